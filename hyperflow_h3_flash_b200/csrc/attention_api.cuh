// Host side of the attention operators (argument checks, tensor maps, launch shapes); included by convrot.cu inside its
// unnamed namespace, after the device state and tensor-map helpers.  Contracts: include/convrot.h.

// Launches a kernel that calls grid_wait() before it touches memory: its start overlaps the end of the one before.
template <class... Params, class... Args>
int launch_overlapped(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                      const Args&... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return e == cudaSuccess ? CONVROT_OK : cuda_fail(e);
}

// ------------------------------------------------------------------------------------------------ rotary table

int rotary_table(const void* pos, int pos_type, int64_t ld_pos, int64_t rows, int axes, const int* dims,
                 const double* theta, float* out, cudaStream_t stream) {
  if (axes < 1 || axes > kRopeMaxAxes) return CONVROT_ERR_SHAPE;
  if (!dims || !theta || pos_type < 0 || pos_type > 3) return CONVROT_ERR_ARG;
  RotaryTableParams p;
  memset(&p, 0, sizeof(p));
  for (int a = 0; a < axes; ++a) {
    if (dims[a] <= 0 || dims[a] % 2 || p.pairs + dims[a] / 2 > kRopeMaxPairs) return CONVROT_ERR_SHAPE;
    if (!(theta[a] > 0.0) || !isfinite(theta[a])) return CONVROT_ERR_ARG;
    for (int i = 0; i < dims[a] / 2; ++i, ++p.pairs) {
      p.freq_over_pi[p.pairs] = pow(theta[a], -2.0 * i / dims[a]) / 3.14159265358979323846;
      p.axis[p.pairs] = static_cast<uint8_t>(a);
    }
  }
  if (rows < 0 || rows > INT32_MAX || ld_pos < axes) return CONVROT_ERR_SHAPE;
  if (rows == 0) return CONVROT_OK;
  if (!pos || !out) return CONVROT_ERR_ARG;
  const int size = pos_type == 1 || pos_type == 3 ? 8 : 4;
  if (reinterpret_cast<uintptr_t>(pos) % size || !aligned16(out)) return CONVROT_ERR_ALIGN;
  DeviceState* st = nullptr;
  int rc = device_state(&st);
  if (rc) return rc;
  p.pos = pos;
  p.ld_pos = ld_pos;
  p.rows = rows;
  p.out = reinterpret_cast<float2*>(out);
  const int64_t need = (rows * p.pairs + 255) / 256, most = 16 * static_cast<int64_t>(st->sms);
  const unsigned grid = static_cast<unsigned>(need < most ? need : most);
  switch (pos_type) {
    case 0: return launch_overlapped(rotary_table_kernel<int32_t>, dim3(grid), 256, 0, stream, p);
    case 1: return launch_overlapped(rotary_table_kernel<int64_t>, dim3(grid), 256, 0, stream, p);
    case 2: return launch_overlapped(rotary_table_kernel<float>, dim3(grid), 256, 0, stream, p);
    default: return launch_overlapped(rotary_table_kernel<double>, dim3(grid), 256, 0, stream, p);
  }
}

// ------------------------------------------------------------------------------------------------ norm and rotation

// Whether rows of D elements, a x b of them, may share an element (the stride of a single one does not count): the rows
// of the smaller stride have to lie side by side within the larger one, (n - 1) stride + D <= larger.
bool rows_overlap(int64_t a, int64_t stride_a, int64_t b, int64_t stride_b, int D) {
  if (a <= 1) return b > 1 && stride_b < D;
  if (b <= 1) return stride_a < D;
  if (stride_a > stride_b) return rows_overlap(b, stride_b, a, stride_a, D);
  return stride_a < D || (stride_b - D) / (a - 1) < stride_a;
}

int qk_norm_rope(const void* q, int64_t q_t, int64_t q_h, void* q_out, int64_t qo_t, int64_t qo_h, int heads_q,
                 const void* k, int64_t k_t, int64_t k_h, void* k_out, int64_t ko_t, int64_t ko_h, int heads_k,
                 int64_t rows, int D, int dtype, int norm, const void* q_weight, const void* k_weight, int weight_f32,
                 float eps, const float* table, int64_t ld_table, int R, int interleaved, cudaStream_t stream) {
  if (dtype < 0 || dtype > 1) return CONVROT_ERR_ARG;
  if (D < 8 || D > 256 || D % 8 || heads_q < 1 || heads_k < 0 || heads_q > (1 << 20) || heads_k > (1 << 20) ||
      rows < 0 || rows > INT32_MAX)
    return CONVROT_ERR_SHAPE;
  if (!norm && !table) return CONVROT_ERR_ARG;
  if (!norm && (q_weight || k_weight)) return CONVROT_ERR_ARG;
  if (norm && !(eps >= 0.0f && eps < 3e38f)) return CONVROT_ERR_ARG;
  if (table) {
    if (R < 8 || R > D || R % (interleaved ? 8 : 16) || ld_table < R / 2) return CONVROT_ERR_SHAPE;
    if (ld_table % 2 || !aligned16(table)) return CONVROT_ERR_ALIGN;
  }
  if (rows == 0) return CONVROT_OK;
  if (!q || !q_out || (heads_k > 0 && (!k || !k_out))) return CONVROT_ERR_ARG;
  // a stride of a dimension of one element does not matter
  if (rows == 1) q_t = qo_t = k_t = ko_t = 0;
  if (heads_q == 1) q_h = qo_h = 0;
  if (heads_k == 1) k_h = ko_h = 0;
  const int64_t strides[] = {q_t, q_h, qo_t, qo_h, k_t, k_h, ko_t, ko_h};
  for (int i = 0; i < (heads_k ? 8 : 4); ++i) {
    if (strides[i] < 0) return CONVROT_ERR_SHAPE;
    if (strides[i] % 8) return CONVROT_ERR_ALIGN;
  }
  if (rows_overlap(rows, qo_t, heads_q, qo_h, D) || (heads_k && rows_overlap(rows, ko_t, heads_k, ko_h, D)))
    return CONVROT_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(q_out) || !aligned16(k) || !aligned16(k_out) || !aligned16(q_weight) ||
      !aligned16(k_weight))
    return CONVROT_ERR_ALIGN;
  DeviceState* st = nullptr;
  int rc = device_state(&st);
  if (rc) return rc;
  QkRopeParams p;
  memset(&p, 0, sizeof(p));
  p.in[0] = q, p.in[1] = k;
  p.out[0] = q_out, p.out[1] = k_out;
  p.in_t[0] = q_t, p.in_h[0] = q_h, p.out_t[0] = qo_t, p.out_h[0] = qo_h;
  p.in_t[1] = k_t, p.in_h[1] = k_h, p.out_t[1] = ko_t, p.out_h[1] = ko_h;
  p.weight[0] = q_weight, p.weight[1] = k_weight;
  p.heads[0] = heads_q, p.heads[1] = heads_k;
  p.table = reinterpret_cast<const float2*>(table);
  p.ld_table = ld_table;
  p.rows = rows;
  p.D = D;
  p.R = table ? R : 0;
  // a lane holds 8 channels (pairs of neighbours), or 8 and their partners, or 16 behind the rotated part
  const bool single = !table || interleaved;
  const int lanes = single ? D / 8 : p.R / 16 + (D - p.R + 15) / 16;
  while ((1 << p.lanes_log2) < lanes) ++p.lanes_log2;
  const int per = (single ? kRopeRows : kRopeRows / 2) * (32 >> p.lanes_log2);
  p.items_q = (heads_q + per - 1) / per;
  p.items = p.items_q + (heads_k + per - 1) / per;
  p.norm = norm;
  p.weight_f32 = weight_f32;
  p.eps = eps;
  p.inv_D = 1.0f / static_cast<float>(D);
  const int64_t blocks = (rows * p.items + kRopeWarps - 1) / kRopeWarps;
  if (blocks > INT32_MAX) return CONVROT_ERR_SHAPE;
  auto bf16 = single ? qk_norm_rope_kernel<__nv_bfloat16, true> : qk_norm_rope_kernel<__nv_bfloat16, false>;
  auto fp16 = single ? qk_norm_rope_kernel<__half, true> : qk_norm_rope_kernel<__half, false>;
  auto kernel = dtype == 0 ? bf16 : fp16;
  return launch_overlapped(kernel, dim3(static_cast<unsigned>(blocks)), kRopeWarps * 32, 0, stream, p);
}

// ------------------------------------------------------------------------------------------------ attention

int attn_check(int64_t Tq, int64_t Tk, int64_t batch, int heads_q, int heads_kv, int D) {
  if (Tq < 0 || Tk < 0 || Tq > INT32_MAX / 2 || Tk > INT32_MAX / 2 || batch < 0 || batch > (1 << 20))
    return CONVROT_ERR_SHAPE;
  if (heads_kv < 1 || heads_q < 1 || heads_q % heads_kv || heads_q / heads_kv > kAtTile || heads_q > (1 << 16))
    return CONVROT_ERR_SHAPE;
  if (D < 8 || D > 128 || D % 8) return CONVROT_ERR_SHAPE;
  return CONVROT_OK;
}

// Query tiles that a call has at most, from host-known sizes.
int64_t attn_items(int64_t Tq, int64_t batch, int heads_q, int heads_kv) {
  const int64_t span = 2 * (kAtTile / (heads_q / heads_kv));
  const int64_t q_tiles = batch == 1 ? (Tq + span - 1) / span : Tq / span + (batch < Tq ? batch : Tq);
  return q_tiles * heads_kv;
}

// CTAs that share the items of the last wave evenly; 0: every item is one CTA's.
//
// Dividing saves the time that CTAs without a last item would idle, an item's work times their share, and costs a second
// launch, a later start of the next kernel and the partial rows' way through memory.  In half steps (one 128 x 128 tile,
// about 0.8 us of a CTA) the fixed part measured 14 and each megabyte of partial rows 0.8:
//   1 token, 8 heads, 1536 / 2048 / 4096 keys (saves 11 / 15 / 30, costs 14): 20.7 / 17.6 / 18.4 us divided, 15.8 / 19.0 /
//     31.8 not;
//   256 tokens, 40 heads, 2048 / 3000 / 8192 keys (23 / 35 / 93, 34): 33.7 / 39.4 / 61.1 divided, 31.6 / 45.4 / 107.0 not;
//   4.3 waves of 40 heads, 2048 / 4096 / 32760 keys (22 / 43 / 346, 35): 173.9 / 310.9 / 2236 divided, 165.7 / 320.2 / 2453
//     not; beyond 24 waves the difference is within 1 % either way.
// Where less than a fifth of the CTAs would idle, the others slow down by as much (power, L2): 120 items for 148 CTAs over
// 8192 / 32760 keys 151 / 487 us divided, 133 / 462 not.
//
// Of several sequences only the sums of the lengths are known here.  One is reckoned with that has a fourth of all keys or
// eight times the mean, and eight times the mean queries too unless the keys are twice the queries (chunks and tokens behind
// caches): its items have the GPU to themselves at last.  If they fill it, half a wave of items of the mean is reckoned
// with.  Single tokens, 8 key heads, divided / not: 100 requests of 40 keys 19.7 / 10.3 us (not divided), 16 of 2000 keys
// 38.9 / 28.6 and 63 of 100 keys before one of 8000 40.3 / 74.7 (divided).  4 prompts of 1000 tokens, 8 heads 51.8 / 21.8
// (not divided).  Chunks of 256 queries, 40 heads, 15 over 200 keys before one over 16000 137 / 247, 40 over 2000 keys 526 /
// 479 (divided).
int attn_shares(int64_t Tq, int64_t Tk, int64_t batch, int heads_q, int heads_kv, int D, int sms) {
  // (the sum of at most kMaxShares items' work has to fit an int)
  if (batch < 1 || Tq < 1 || Tk < 8 * kAtTile || Tk > (1 << 28)) return 0;
  const int shares = sms < kMaxShares ? sms : kMaxShares, group = heads_q / heads_kv;
  const int64_t items = attn_items(Tq, batch, heads_q, heads_kv);
  if (items >= 24 * static_cast<int64_t>(shares)) return 0;
  auto at_most = [](int64_t a, int64_t b) { return a < b ? a : b; };
  const int64_t tile = kAtTile / group;  // query positions
  int64_t queries = (Tq + batch - 1) / batch, keys = (Tk + batch - 1) / batch, last = items % shares, idle = shares - last;
  const int64_t long_queries = Tk / 2 >= Tq ? queries : at_most(Tq, 8 * queries);
  const int64_t long_items = (long_queries + 2 * tile - 1) / (2 * tile) * heads_kv;
  if (batch > 1 && long_items < shares) {
    queries = long_queries;
    keys = at_most(Tk, 8 * keys > Tk / 4 ? 8 * keys : Tk / 4);
    last = at_most(items, shares - 1);
    idle = shares - long_items;
  } else if (batch > 1) {
    last = idle = shares / 2;
  }
  // (one sequence whose items fill whole waves: nothing is left to divide and nothing is launched for it, unless offsets
  // make it shorter)
  if (batch == 1 && last == 0) return shares;
  const int64_t units = (keys + kAtTile - 1) / kAtTile * (queries > tile ? 2 : 1);
  const int64_t parts = at_most(units * last / 8, shares) + last;
  const int64_t part_bytes = parts * at_most(queries, 2 * tile) * group * D * 4;
  return 5 * idle >= shares && units * idle > (14 + part_bytes / 1250000) * shares ? shares : 0;
}

size_t attn_workspace(int shares, int D) {
  return shares ? (kMaxShares + 4 + static_cast<size_t>(shares) * 2 * 256 * (D + 1)) * 4 : 0;
}

int attn_map(CUtensorMap* map, const void* base, int dtype, int D, int64_t heads, int64_t rows, int64_t ld_h,
             int64_t ld_t, int box_heads, int box_rows) {
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld_h * 2), static_cast<cuuint64_t>(ld_t * 2)};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = g_encode(map, dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    t_last_cuda_error = static_cast<int>(r);
    return CONVROT_ERR_CUDA;
  }
  return CONVROT_OK;
}

template <class T, int NP, bool CAUSAL>
int launch_attention(const DeviceState& st, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                     const AttnParams& p, int64_t items, int joined, cudaStream_t stream) {
  auto kernel = attention_kernel<T, NP, CAUSAL>;
  int ready = -1;
  int rc = cached_resident(reinterpret_cast<const void*>(kernel), &ready);
  if (rc) return rc;
  cudaError_t e;
  if (ready < 0) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, AttnCfg<NP>::kSmemBytes);
    if (e != cudaSuccess) return cuda_fail(e);
    store_resident(reinterpret_cast<const void*>(kernel), 1);
  }
  rc = launch_overlapped(kernel, dim3(static_cast<unsigned>(items)), kAtThreads, AttnCfg<NP>::kSmemBytes, stream, tq, tk,
                         tv, p);
  if (rc || joined == 0) return rc;
  // a warp for each row that an item has at most (few tokens have few)
  const int positions = p.Tq < 2 * p.positions ? p.Tq : 2 * p.positions;
  return launch_overlapped(attention_combine_kernel<T>, dim3(joined, (positions * p.group + 7) / 8), 256, 0, stream, p);
}

int attention(const void* q, int64_t q_t, int64_t q_h, const void* k, int64_t k_t, int64_t k_h, const void* v,
              int64_t v_t, int64_t v_h, const int32_t* cu_q, const int32_t* cu_k, int64_t batch, int64_t Tq, int64_t Tk,
              int heads_q, int heads_kv, int D, int dtype, float scale, int causal, void* out, int64_t out_t,
              int64_t out_h, float* lse, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  int rc = attn_check(Tq, Tk, batch, heads_q, heads_kv, D);
  if (rc) return rc;
  const float scale_log2 = scale * 1.4426950408889634f;  // what the kernel multiplies with
  if (dtype < 0 || dtype > 1 || !(scale > 0.0f) || !isfinite(scale_log2)) return CONVROT_ERR_ARG;
  if ((cu_q == nullptr) != (cu_k == nullptr) || (!cu_q && batch != 1)) return CONVROT_ERR_ARG;
  if (Tq == 0 || batch == 0) return CONVROT_OK;
  if (!q || !out || (Tk > 0 && (!k || !v))) return CONVROT_ERR_ARG;
  // a stride of a dimension of one element does not matter
  const int64_t any = 128;
  if (heads_q == 1) q_h = out_h = any;
  if (heads_kv == 1) k_h = v_h = any;
  if (Tq <= 1) q_t = out_t = any;
  if (Tk <= 1) k_t = v_t = any;
  const struct {
    const void* base;
    int64_t t, h, heads, rows;
  } ops[4] = {{q, q_t, q_h, heads_q, Tq}, {out, out_t, out_h, heads_q, Tq}, {k, k_t, k_h, heads_kv, Tk},
              {v, v_t, v_h, heads_kv, Tk}};
  for (int i = 0; i < 4; ++i) {
    if (!aligned16(ops[i].base) || ops[i].t % 8 || ops[i].h % 8) return CONVROT_ERR_ALIGN;
    if (ops[i].t <= 0 || ops[i].h <= 0 || ops[i].t >= (int64_t{1} << 38) || ops[i].h >= (int64_t{1} << 38))
      return CONVROT_ERR_SHAPE;
  }
  if (rows_overlap(Tq, out_t, heads_q, out_h, D)) return CONVROT_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(cu_q) | reinterpret_cast<uintptr_t>(cu_k) | reinterpret_cast<uintptr_t>(lse)) & 3u)
    return CONVROT_ERR_ALIGN;
  DeviceState* st = nullptr;
  if ((rc = device_state(&st))) return rc;
  AttnParams p;
  memset(&p, 0, sizeof(p));
  p.shares = attn_shares(Tq, Tk, batch, heads_q, heads_kv, D, st->sms);
  if (p.shares > 0) {
    if (!workspace || workspace_bytes < attn_workspace(p.shares, D)) return CONVROT_ERR_ARG;
    if (!aligned16(workspace)) return CONVROT_ERR_ALIGN;
    p.meta = static_cast<int*>(workspace);
    p.part_o = static_cast<float*>(workspace) + kMaxShares + 4;
    p.part_lse = p.part_o + static_cast<size_t>(p.shares) * 2 * 256 * D;
  }
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.batch = static_cast<int>(batch);
  p.Tq = static_cast<int>(Tq);
  p.Tk = static_cast<int>(Tk);
  p.heads_kv = heads_kv;
  p.group = heads_q / heads_kv;
  p.D = D;
  p.positions = kAtTile / p.group;
  p.group_inverse = (65536 + p.group - 1) / p.group;
  p.scale_log2 = scale_log2;
  p.causal = causal ? 1 : 0;
  // Causal items go out longest first; over as many heads at once as keep their keys and values in L2, so that the
  // last ones are short.
  const int64_t head_bytes = (Tk + batch - 1) / batch * D * 4 + 1;
  const int64_t block = (int64_t{96} << 20) / head_bytes;
  p.head_block = !causal || block < 1 ? 1 : block < heads_kv ? static_cast<int>(block) : heads_kv;
  p.v = v;
  p.v_t = v_t;
  p.v_h = v_h;
  p.out = out;
  p.out_t = out_t;
  p.out_h = out_h;
  p.lse = lse;
  p.wait_limit_ns = g_wait_limit_ns;
  p.error_word = st->error_word;
  CUtensorMap tq, tk, tv;
  if ((rc = attn_map(&tq, q, dtype, D, heads_q, Tq, q_h, q_t, p.group, p.positions))) return rc;
  // Without a key the maps of k and v are never read; the query's stands in (an empty extent cannot be encoded).
  if ((rc = attn_map(&tk, Tk ? k : q, dtype, D, Tk ? heads_kv : heads_q, Tk ? Tk : Tq, Tk ? k_h : q_h, Tk ? k_t : q_t, 1,
                     kAtTile)))
    return rc;
  if ((rc = attn_map(&tv, Tk ? v : q, dtype, D, Tk ? heads_kv : heads_q, Tk ? Tk : Tq, Tk ? v_h : q_h, Tk ? v_t : q_t, 1,
                     kAtTile)))
    return rc;
  // An upper bound of the work items (the kernel finds their number; what is beyond it finds nothing).
  const int64_t whole = attn_items(Tq, batch, heads_q, heads_kv), items = whole + p.shares;
  if (items > INT32_MAX / 2) return CONVROT_ERR_SHAPE;
  // Items of the divided last wave: known, or at most one short of a wave.
  const int64_t last = !p.shares ? 0 : !cu_q ? whole % p.shares : whole < p.shares ? whole : p.shares - 1;
  const int joined = static_cast<int>(last);
  auto launch = [&](auto type) {
    using T = decltype(type);
    if (D <= 64)
      return causal ? launch_attention<T, 1, true>(*st, tq, tk, tv, p, items, joined, stream)
                    : launch_attention<T, 1, false>(*st, tq, tk, tv, p, items, joined, stream);
    return causal ? launch_attention<T, 2, true>(*st, tq, tk, tv, p, items, joined, stream)
                  : launch_attention<T, 2, false>(*st, tq, tk, tv, p, items, joined, stream);
  };
  return dtype == 0 ? launch(__nv_bfloat16()) : launch(__half());
}
