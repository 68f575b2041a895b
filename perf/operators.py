"""The attention operators between an attention block's q/k/v and out projections: the rotary table of several
position axes, the per-head norm of q and k with its rotation, and attention over packed sequences.

Sizes are this repository's: 40 heads of 128 channels, 32760 video tokens (21 x 30 x 52 latents), 256 or 333 text
tokens, 5 heads per GPU when 40 are split over 8; grouped heads and single-token calls use generic sizes.
"""

import math

import torch

own = False

THETA = 10000.0
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST_SCORES = 5 * 32760 * 32760  # padded scores of one pass of the plain form (fp32): about 21 GB


# ------------------------------------------------------------------------------------------------ cases


def listed():
    video = "21x30x52"
    return [
        # the positions of one clip's latents, computed once per clip and used by every block
        {"name": "table-video-32760", "op": "table", "grid": video, "axes": "44,42,42", "positions": "int32"},
        # text tokens with one axis and fractional positions: a call whose latency counts
        {"name": "table-text-333", "op": "table", "grid": "333", "axes": "128", "positions": "float64"},
        # self-attention of the video tokens on one GPU
        {"name": "norm-video-32760x40", "op": "norm", "T": 32760, "hq": 40, "hkv": 40, "D": 128, "R": 128,
         "dtype": "bf16", "interleaved": True, "fused": False},
        # grouped heads read out of one fused projection, half-split pairs, part of each head rotated, odd length
        {"name": "norm-fused-4099x24", "op": "norm", "T": 4099, "hq": 24, "hkv": 8, "D": 64, "R": 48,
         "dtype": "fp16", "interleaved": False, "fused": True},
        # a few tokens: latency
        {"name": "norm-17x40", "op": "norm", "T": 17, "hq": 40, "hkv": 40, "D": 128, "R": 128, "dtype": "bf16",
         "interleaved": True, "fused": False},
        # one rank's heads of a clip, all tokens, after the 8-GPU exchange
        {"name": "self-32760x5", "op": "attn", "lq": "32760", "lk": "32760", "hq": 5, "hkv": 5, "D": 128,
         "dtype": "bf16", "causal": False, "lse": False},
        # four requests of different lengths packed behind each other
        {"name": "self-packed-4x40", "op": "attn", "lq": "4096,1560,2731,333", "lk": "4096,1560,2731,333",
         "hq": 40, "hkv": 40, "D": 128, "dtype": "bf16", "causal": False, "lse": False},
        # video tokens reading the text
        {"name": "cross-32760x333", "op": "attn", "lq": "32760", "lk": "333", "hq": 40, "hkv": 40, "D": 128,
         "dtype": "bf16", "causal": False, "lse": False},
        # whole prompts, causal, grouped heads, lengths down to one token
        {"name": "causal-packed-6x40", "op": "attn", "lq": "4001,1,129,2500,17,512", "lk": "4001,1,129,2500,17,512",
         "hq": 40, "hkv": 8, "D": 128, "dtype": "fp16", "causal": True, "lse": True},
        # one new token for each of 16 requests over long caches
        {"name": "token-16x32768", "op": "attn", "lq": "1," * 15 + "1",
         "lk": "32768,1,16384,8191,12000,4097,24001,31999,512,20000,9999,15000,30001,7777,2049,28672",
         "hq": 40, "hkv": 8, "D": 128, "dtype": "bf16", "causal": True, "lse": False},
        # the newest latent frame of a stream over everything before it: few rows, long keys
        {"name": "frame-1560x32760", "op": "attn", "lq": "1560", "lk": "32760", "hq": 5, "hkv": 5, "D": 128,
         "dtype": "bf16", "causal": True, "lse": True},
        # a handful of tokens: latency
        {"name": "small-17x333", "op": "attn", "lq": "17", "lk": "333", "hq": 8, "hkv": 8, "D": 64, "dtype": "bf16",
         "causal": False, "lse": False},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["table", "norm", "norm", "attn", "attn", "attn"])
    if op == "table":
        if rng.random() < 0.5:
            t, h, w = _spread(rng, 1, 21), _spread(rng, 1, 40), _spread(rng, 1, 39)
            axes = rng.choice(["44,42,42", "16,56,56", "16,24,24", "32,16,16"])
            return {"op": op, "grid": "%dx%dx%d" % (t, h, w), "axes": axes, "positions": rng.choice(["int32", "int64", "float32"])}
        return {"op": op, "grid": str(_spread(rng, 1, 32761)), "axes": rng.choice(["128", "64", "48"]),
                "positions": rng.choice(["int32", "float32", "float64"])}
    D = rng.choice([64, 64, 72, 80, 96, 128, 128, 128])
    group, hkv = rng.choice([1, 1, 2, 3, 5, 8]), rng.choice([1, 2, 5, 8, 10])
    if group == 1:
        hkv = rng.choice([5, 8, 24, 40])
    hq = hkv * group
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "norm":
        interleaved = rng.random() < 0.5
        R = D if D % 16 == 0 and rng.random() < 0.7 else D // 32 * 16
        T = _spread(rng, 1, max(1, min(32761, 32760 * 80 * 128 // ((hq + hkv) * D))))
        return {"op": op, "T": T, "hq": hq, "hkv": hkv, "D": D, "R": R, "dtype": dtype, "interleaved": interleaved,
                "fused": rng.random() < 0.5}
    kind = rng.choice(["self", "packed", "cross", "token", "frame"])
    most = MOST_SCORES // 2
    if kind == "self":
        n = _spread(rng, 1, min(16384, int(math.sqrt(most / hq))))
        lq = lk = [n]
    elif kind == "packed":
        B = _spread(rng, 2, 24)
        top = int(min(8192, math.sqrt(most / (hq * B))))
        lq = lk = [_spread(rng, 1, top) for _ in range(B)]
    elif kind == "cross":
        B = _spread(rng, 1, 4)
        lk = [_spread(rng, 1, 777) for _ in range(B)]
        lq = [_spread(rng, 1, min(16384, most // (hq * 777 * B))) for _ in range(B)]
    elif kind == "token":
        B = _spread(rng, 1, 64)
        new = rng.choice([1, 1, 1, 2, 4])
        top = max(64, min(32768, 800_000 // (B * hkv)))
        lk = [_spread(rng, new, top) for _ in range(B)]
        lq = [new] * B
    else:
        n = _spread(rng, 2, 2048)
        lk = [max(n, _spread(rng, 64, min(32760, max(n, most // (hq * n)))))]
        lq = [n]
    return {"op": "attn", "lq": ",".join(map(str, lq)), "lk": ",".join(map(str, lk)), "hq": hq, "hkv": hkv, "D": D,
            "dtype": dtype, "causal": kind in ("token", "frame") or (kind in ("self", "packed") and rng.random() < 0.5),
            "lse": rng.random() < 0.3}


def _ints(text, sep=","):
    return [int(v) for v in text.split(sep)]


# ------------------------------------------------------------------------------------------------ inputs


def _grid(case, device):
    """[T, axes] positions: the latent grid, row-major, or a run of text positions with fractional steps."""
    n = _ints(case["grid"], "x")
    dtype = getattr(torch, case["positions"])
    if len(n) == 1:
        pos = torch.arange(n[0], device=device, dtype=torch.float64)[:, None]
        return (pos * (0.75 if dtype.is_floating_point else 1.0)).to(dtype)
    ax = [torch.arange(m, device=device, dtype=torch.float64) for m in n]
    return torch.stack(torch.meshgrid(*ax, indexing="ij"), dim=-1).reshape(-1, len(n)).to(dtype)


def _angles(pos, axes):
    """fp64 angles [T, R / 2] of positions [T, A] over axes of the given widths."""
    parts = []
    for a, d in enumerate(axes):
        inv = THETA ** (-torch.arange(0, d, 2, device=pos.device, dtype=torch.float64) / d)
        parts.append(pos[:, a : a + 1].double() * inv)
    return torch.cat(parts, dim=1)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(1000 + int(seed))
    if case["op"] == "table":
        pos = _grid(case, dev)
        # a clip that starts somewhere in a longer stream: each seed has its own offset
        start = torch.randint(0, 1000, (1, pos.shape[1]), generator=g, device=dev)
        return {"case": case, "pos": pos + start.to(pos.dtype), "axes": tuple(_ints(case["axes"]))}
    dt = DTYPES[case["dtype"]]
    hq, hkv, D = case["hq"], case["hkv"], case["D"]

    def rand(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev) * scale

    if case["op"] == "norm":
        T, R = case["T"], case["R"]
        x = rand(T, (hq + 2 * hkv) * D)
        x *= torch.exp(0.7 * rand(1, x.shape[1]))  # projections whose channels differ in size
        x = x.to(dt)
        q = x[:, : hq * D].unflatten(1, (hq, D))
        k = x[:, hq * D : (hq + hkv) * D].unflatten(1, (hkv, D))
        if not case["fused"]:
            q, k = q.contiguous(), k.contiguous()
        start = torch.randint(0, 1000, (1,), generator=g, device=dev)
        ang = _angles((torch.arange(T, device=dev) + start)[:, None], (R,))
        table = torch.stack([ang.cos(), ang.sin()], dim=-1).float()
        return {"case": case, "q": q, "k": k, "table": table, "wq": (1 + rand(D, scale=0.2)).to(dt),
                "wk": (1 + rand(D, scale=0.2)).to(dt)}
    lq, lk = _ints(case["lq"]), _ints(case["lk"])
    # q and k as the norm leaves them, with a part that all keys of a head share; values with a mean per channel
    q = rand(sum(lq), hq, D, scale=1.3).to(dt)
    k = (rand(sum(lk), hkv, D) + rand(1, hkv, D, scale=0.5)).to(dt)
    v = (rand(sum(lk), hkv, D) + rand(1, hkv, D, scale=0.5)).to(dt)
    cu = [torch.tensor([sum(l[:i]) for i in range(len(l) + 1)], dtype=torch.int32, device=dev) for l in (lq, lk)]
    return {"case": case, "q": q, "k": k, "v": v, "cu_q": cu[0], "cu_k": cu[1], "packed": len(lq) > 1,
            "max_q": max(lq), "max_k": max(lk)}


# ------------------------------------------------------------------------------------------------ one pass


def _rotate(x, table, interleaved):
    """fp32 [T, H, D] with the first R channels of each head rotated by table [T, R / 2, 2]."""
    R = 2 * table.shape[1]
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., : R // 2], x[..., R // 2 : R]
        y[..., : R // 2], y[..., R // 2 : R] = a * c - b * s, b * c + a * s
    return y


def _norm_rope(x, w, table, interleaved):
    f = x.float()
    f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * w.float()
    return _rotate(f, table, interleaved).to(x.dtype)


def _padded(x, cu, longest):
    """[B, longest, H, D] fp32 of packed rows, and which of its rows exist."""
    at = torch.arange(longest, device=x.device)
    here = at < (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + at).clamp(max=max(x.shape[0] - 1, 0))
    return x[rows.reshape(-1)].reshape(*rows.shape, *x.shape[1:]).float(), here, rows


def _attend(s):
    q, k, v, case = s["q"], s["k"], s["v"], s["case"]
    hkv, D, group = case["hkv"], case["D"], case["hq"] // case["hkv"]
    qp, q_here, q_rows = _padded(q, s["cu_q"], s["max_q"])
    kp, k_here, _ = _padded(k, s["cu_k"], s["max_k"])
    vp, _, _ = _padded(v, s["cu_k"], s["max_k"])
    B, Lq = q_here.shape
    qp = qp.reshape(B, Lq, hkv, group, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, group * Lq, D) * D**-0.5
    scores = torch.matmul(qp, kp.permute(0, 2, 3, 1)).view(B, hkv, group, Lq, -1)
    hidden = ~k_here[:, None, :].expand(B, Lq, -1)
    if case["causal"]:
        lq, lk = (s["cu_q"][1:] - s["cu_q"][:-1]), (s["cu_k"][1:] - s["cu_k"][:-1])
        last = torch.arange(Lq, device=q.device)[None, :] + (lk - lq)[:, None]
        hidden = hidden | (torch.arange(s["max_k"], device=q.device) > last[:, :, None])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, hkv, group * Lq, -1), vp.permute(0, 2, 1, 3)).view(B, hkv, group, Lq, D)
    out = out / torch.where(total == 0, 1.0, total)
    place = torch.zeros(q.shape[0], dtype=torch.int64, device=q.device)
    flat = torch.arange(B * Lq, device=q.device).view(B, Lq)
    place.index_put_((torch.where(q_here, q_rows, q_rows.new_zeros(())).long(),),
                     torch.where(q_here, flat, flat.new_zeros(())), accumulate=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(B * Lq, hkv * group, D)[place].to(q.dtype)
    if not case["lse"]:
        return out
    return out, (top + total.log()).permute(0, 3, 1, 2, 4).reshape(B * Lq, hkv * group)[place]


def run(state):
    case = state["case"]
    if own:
        from hyperflow_h3_flash_b200 import attention as A

        if case["op"] == "table":
            return A.rotary_table(state["pos"], state["axes"], theta=THETA)
        if case["op"] == "norm":
            return A.qk_norm_rope(state["q"], state["k"], q_weight=state["wq"], k_weight=state["wk"], eps=EPS,
                                  table=state["table"], interleaved=case["interleaved"])
        cu = {"cu_q": state["cu_q"], "cu_k": state["cu_k"]} if state["packed"] else {}
        return A.attention(state["q"], state["k"], state["v"], causal=case["causal"], return_lse=case["lse"], **cu)
    if case["op"] == "table":
        ang = _angles(state["pos"], state["axes"])
        return torch.stack([ang.cos(), ang.sin()], dim=-1).float()
    if case["op"] == "norm":
        return (_norm_rope(state["q"], state["wq"], state["table"], case["interleaved"]),
                _norm_rope(state["k"], state["wk"], state["table"], case["interleaved"]))
    return _attend(state)


# ------------------------------------------------------------------------------------------------ work and oracle


def work(case):
    if case["op"] == "table":
        T = math.prod(_ints(case["grid"], "x"))
        axes = _ints(case["axes"])
        size = {"int32": 4, "float32": 4, "int64": 8, "float64": 8}[case["positions"]]
        return {"bytes": T * (len(axes) * size + sum(axes) // 2 * 8), "flops": T * sum(axes) // 2 * 3}
    hq, hkv, D = case["hq"], case["hkv"], case["D"]
    if case["op"] == "norm":
        n = case["T"] * (hq + hkv) * D
        return {"bytes": n * 4 + case["T"] * case["R"] * 4 + 4 * D, "flops": n * 8}
    lq, lk = _ints(case["lq"]), _ints(case["lk"])
    pairs = 0
    for a, b in zip(lq, lk):
        if case["causal"]:  # query i sees the first b - a + i + 1 keys
            first = max(0, a - b)
            pairs += sum(range(b - a + first + 1, b + 1)) if a > first else 0
        else:
            pairs += a * b
    moved = 2 * (2 * sum(lq) * hq + 2 * sum(lk) * hkv) * D + (4 * sum(lq) * hq if case["lse"] else 0)
    return {"bytes": moved, "flops": 4 * D * pairs * hq}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "table":
        pos, parts = s["pos"].double(), []
        for a, d in enumerate(s["axes"]):
            for i in range(d // 2):
                ang = pos[:, a] * math.pow(THETA, -2.0 * i / d)
                parts.append(torch.stack([torch.cos(ang), torch.sin(ang)], dim=-1))
        return torch.stack(parts, dim=1)
    if case["op"] == "norm":
        outs, R = [], case["R"]
        z = torch.view_as_complex(s["table"].double().contiguous())  # [T, R / 2]
        for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
            d = x.double()
            d = d / torch.sqrt(torch.linalg.vector_norm(d, dim=-1, keepdim=True) ** 2 / case["D"] + EPS) * w.double()
            part = d[..., :R]
            if case["interleaved"]:
                pair = part.unflatten(-1, (R // 2, 2)).contiguous()
            else:
                pair = part.unflatten(-1, (2, R // 2)).transpose(-1, -2).contiguous()
            turned = torch.view_as_real(torch.view_as_complex(pair) * z[:, None])
            turned = turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2)
            outs.append(torch.cat([turned, d[..., R:]], dim=-1))
        return tuple(outs)
    lq, lk, group = _ints(case["lq"]), _ints(case["lk"]), case["hq"] // case["hkv"]
    out = torch.zeros(sum(lq), case["hq"], case["D"], dtype=torch.float64, device="cuda")
    lse = torch.full((sum(lq), case["hq"]), -math.inf, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for a, b in zip(lq, lk):
        for h in range(case["hq"]):
            K = s["k"][k0 : k0 + b, h // group].double()
            V = s["v"][k0 : k0 + b, h // group].double()
            for r in range(0, a, 8192):
                n = min(8192, a - r)
                x = s["q"][q0 + r : q0 + r + n, h].double() @ K.t() / math.sqrt(case["D"])
                if case["causal"]:
                    i = torch.arange(r, r + n, device="cuda")[:, None]
                    x = torch.where(torch.arange(b, device="cuda")[None, :] - i <= b - a, x, -math.inf)
                z = torch.logsumexp(x, dim=1)
                lse[q0 + r : q0 + r + n, h] = z
                w = torch.where(z[:, None] == -math.inf, 0.0, torch.exp(x - torch.nan_to_num(z, neginf=0.0)[:, None]))
                out[q0 + r : q0 + r + n, h] = w @ V
        q0, k0 = q0 + a, k0 + b
    return (out, lse) if case["lse"] else out
