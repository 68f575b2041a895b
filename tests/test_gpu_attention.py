"""The attention operators on the GPU against plain 64-bit formulas.

Tolerances count roundings.  u = half a step of the 16-bit type, relative (bf16 2^-8, fp16 2^-11).

* rotary table: fp32 cos / sin of an angle known to fp64: one rounding of the reduced angle's head (its remainder is
  carried), sincospif's 2 units in the last place and the correction's two roundings: below 4 * 2^-23 absolute.
* norm and rotation: fp32 steps of 2^-24 each (sum of D squares, rsqrt's 2 ulp, three products, the rotation), together
  below (D + 16) 2^-24 of |a| + |b|, and one rounding u of the result.
* attention: each weight p is rounded once (u) before its product with v, the result once: u (A + |o|) with
  A = sum_k w_k |v_k|; the scores' fp32 sums are off by at most (D + 4) 2^-23 sum_d |q_d k_d| scale = e, which moves a
  weight by a factor exp(2 e); exp2, sums, rescaling and joining in fp32 stay below 2^-17 A for the lengths used here.
  fp16 weights below 2^-14 (of a largest of at least 1) are off by at most 2^-25 each.
"""

from __future__ import annotations

import math

import pytest
import torch

from hyperflow_h3_flash_b200 import _lib
from hyperflow_h3_flash_b200 import attention as A

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.lib().convrot_poll_error(None) == 0


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=_gen(seed), device=DEV) * scale).to(dtype)


def _cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ attention


def reference(q, k, v, lq, lk, causal, scale):
    """(o, lse, bound of |o|'s error, seen rows) in fp64, by the definition, sequence by sequence and head by head."""
    u, D = U[q.dtype], q.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(o)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    lse_bound = torch.zeros_like(lse)
    group = q.shape[1] // k.shape[1]
    q0 = k0 = 0
    for a, b in zip(lq, lk):
        for h in range(q.shape[1]):
            if a and b:
                Q = q[q0 : q0 + a, h].double()
                K, V = (t[k0 : k0 + b, h // group].double() for t in (k, v))
                s = Q @ K.t() * scale
                if causal:
                    i = torch.arange(a, device=DEV)[:, None]
                    s = s.masked_fill(torch.arange(b, device=DEV)[None] > i + b - a, -math.inf)
                top = s.amax(1, keepdim=True)
                e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
                total = e.sum(1, keepdim=True)
                w = e / torch.where(total == 0, 1.0, total)
                o[q0 : q0 + a, h] = w @ V
                lse[q0 : q0 + a, h] = (top + total.log())[:, 0]
                size = w @ V.abs()
                slip = (D + 4) * 2.0**-23 * (Q.abs() @ K.abs().t() * scale).amax(1, keepdim=True)
                tiny = 2.0**-25 * V.abs().sum(0) if q.dtype == torch.float16 else 0.0
                bound[q0 : q0 + a, h] = u * (1 + u) * (size + o[q0 : q0 + a, h].abs()) + size * (
                    torch.expm1(2 * slip) + 2.0**-17) + tiny + 1e-30
                lse_bound[q0 : q0 + a, h] = slip[:, 0] + 2.0**-17
        q0, k0 = q0 + a, k0 + b
    return o, lse, bound, lse_bound


def check(q, k, v, lq, lk, causal=False, scale=None, cu=True, **kw):
    scale_ = q.shape[2] ** -0.5 if scale is None else scale
    args = {"cu_q": _cu(lq), "cu_k": _cu(lk)} if cu else {}
    got, lse = A.attention(q, k, v, causal=causal, scale=scale, return_lse=True, **args, **kw)
    want, want_lse, bound, lse_bound = reference(q, k, v, lq, lk, causal, scale_)
    n = sum(lq)
    assert got.dtype == q.dtype and got.shape == q.shape and lse.shape == q.shape[:2]
    off = (got[:n].double() - want[:n]).abs() - bound[:n]
    assert not torch.isnan(off).any()
    assert (off <= 0).all(), f"{int((off > 0).sum())} of {off.numel()} outside, worst by {off.max().item():.3e}"
    empty = want_lse[:n] == -math.inf
    assert torch.equal(lse[:n] == -math.inf, empty)
    assert (got[:n][empty] == 0).all()
    d = torch.where(empty, 0.0, (lse[:n].double() - want_lse[:n]).abs())
    assert (d <= lse_bound[:n]).all(), f"lse off by {d.max().item():.3e}"
    return got


def qkv(Tq, Tk, Hq, Hkv, D, dtype=torch.bfloat16, seed=0, spread=1.5):
    return (_randn(Tq, Hq, D, seed=seed, dtype=dtype, scale=spread), _randn(Tk, Hkv, D, seed=seed + 1, dtype=dtype),
            _randn(Tk, Hkv, D, seed=seed + 2, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [8, 16, 40, 64, 72, 80, 96, 120, 128])
def test_head_dims_and_types(D, dtype):
    q, k, v = qkv(300, 333, 2, 2, D, dtype, seed=D)
    check(q, k, v, [300], [333], cu=False)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 128), (1, 129), (127, 127), (128, 128), (129, 255), (255, 129), (256, 256),
                                   (257, 640), (17, 1025), (500, 7), (640, 1)])
def test_lengths(lq, lk, causal):
    q, k, v = qkv(lq, lk, 3, 3, 64, seed=lq + lk)
    check(q, k, v, [lq], [lk], causal, cu=False)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 40, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_grouped_heads(group, causal):
    q, k, v = qkv(70, 200, 2 * group, 2, 64, seed=group)
    check(q, k, v, [70], [200], causal, cu=False)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_sequences(causal, dtype):
    lq = [130, 0, 1, 257, 64, 5, 0]
    lk = [131, 9, 0, 300, 63, 700, 0]
    q, k, v = qkv(sum(lq), sum(lk), 4, 2, 128, dtype, seed=3)
    check(q, k, v, lq, lk, causal)


def test_many_sequences():
    """More sequences than one warp looks at in a step, empty ones among them."""
    lq = [(7 * i) % 5 for i in range(101)]
    lk = [(13 * i) % 150 for i in range(101)]
    q, k, v = qkv(sum(lq), sum(lk), 4, 2, 64, seed=4)
    check(q, k, v, lq, lk, True)


@pytest.mark.parametrize("lk", [[2000], [1, 5000, 300, 0, 129]])
@pytest.mark.parametrize("new", [1, 3])
def test_single_tokens_over_long_keys(lk, new):
    lq = [new] * len(lk)
    q, k, v = qkv(sum(lq), sum(lk), 10, 2, 128, seed=5)
    assert _lib.lib().convrot_attention_workspace_size(sum(lq), sum(lk), len(lk), 10, 2, 128) > 0  # keys are split
    check(q, k, v, lq, lk, True)


@pytest.mark.parametrize("D,heads,group,lk", [(64, 2, 64, [2582]), (104, 3, 4, [2560, 0]), (128, 12, 1, [1200] * 9),
                                              (40, 5, 8, [300, 4000, 1, 700]), (128, 1, 127, [260] * 40)])
def test_one_tile_items_behind_each_other(D, heads, group, lk):
    """Items of a single query tile, several to a CTA: what one leaves on the chip is not touched by the next."""
    for seed in range(8):
        q, k, v = qkv(len(lk), sum(lk), heads * group, heads, D, torch.float16 if seed & 1 else torch.bfloat16, seed=seed)
        check(q, k, v, [1] * len(lk), lk, causal=seed & 2 != 0)


def test_scores_that_grow_and_shrink_along_the_keys():
    """Maxima that jump by far more than the lazy rescaling's step, up and down, and rows of equal scores."""
    q, k, v = qkv(200, 1500, 2, 2, 64, seed=6, spread=1.0)
    ramp = torch.linspace(-6, 6, 1500, device=DEV).reshape(-1, 1, 1)
    k = (k + ramp * q.float().mean(0) * 20).to(k.dtype)
    check(q, k, v, [200], [1500], cu=False)
    check(q, k.flip(0).contiguous(), v, [200], [1500], cu=False)
    check(torch.zeros_like(q), k, v, [200], [1500], cu=False)
    check(q, k, v, [200], [1500], cu=False, scale=3.0)


def test_strided_views_of_a_fused_projection():
    T, Hq, Hkv, D = 311, 6, 2, 64
    x = _randn(T, (Hq + 2 * Hkv) * D + 8, seed=7, dtype=torch.bfloat16)
    q = x[:, : Hq * D].unflatten(1, (Hq, D))
    k = x[:, Hq * D : (Hq + Hkv) * D].unflatten(1, (Hkv, D))
    v = x[:, (Hq + Hkv) * D : (Hq + 2 * Hkv) * D].unflatten(1, (Hkv, D))
    check(q, k, v, [T], [T], True, cu=False)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    out = torch.empty(Hq, T, D, dtype=q.dtype, device=DEV).transpose(0, 1)
    check(*heads_first, [T], [T], True, cu=False, out=out)


def test_rows_of_no_sequence_stay_as_they_were():
    lq, lk = [100, 50], [60, 90]
    q, k, v = qkv(200, 300, 2, 2, 64, seed=8)
    out = torch.full_like(q, 7.0)
    A.attention(q, k, v, cu_q=_cu(lq), cu_k=_cu(lk), out=out)
    assert (out[150:] == 7).all() and not (out[:150] == 7).all()
    few = torch.full_like(q[:9], 7.0)
    A.attention(q[:9], k, v, cu_q=_cu([1, 1, 2]), cu_k=_cu([60, 90, 100]), out=few)
    assert (few[4:] == 7).all() and not (few[:4] == 7).any()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_no_query_sees_does_not_reach_it(bad):
    """Rows behind a sequence (another request's, or padding) hold NaN or infinities."""
    lq, lk = [130, 40], [130, 70]
    q, k, v = qkv(sum(lq) + 60, sum(lk) + 60, 2, 2, 128, seed=9)
    clean = check(q, k, v, lq, lk)
    for t, n in ((q, sum(lq)), (k, sum(lk)), (v, sum(lk))):
        t[n:] = bad
    got = A.attention(q, k, v, cu_q=_cu(lq), cu_k=_cu(lk))
    assert torch.equal(got[: sum(lq)], clean[: sum(lq)])
    # another request's rows: sequence 1 is spoilt, sequence 0 is not
    for t, n in ((q, lq[0]), (k, lk[0]), (v, lk[0])):
        t[n:] = bad
    got = A.attention(q, k, v, cu_q=_cu(lq), cu_k=_cu(lk))
    assert torch.equal(got[: lq[0]], clean[: lq[0]])


def test_offsets_that_make_no_sense_stay_inside():
    q, k, v = qkv(64, 64, 2, 2, 64, seed=10)
    for cu in ([0, 1000, 64], [-5, 30, 64], [50, 20, 64]):
        cu = torch.tensor(cu, dtype=torch.int32, device=DEV)
        A.attention(q, k, v, cu_q=cu, cu_k=cu)
    torch.cuda.synchronize()


def test_results_repeat_bitwise():
    lk = [3000, 17, 900]
    q, k, v = qkv(3, sum(lk), 8, 2, 128, seed=11)
    args = {"cu_q": _cu([1, 1, 1]), "cu_k": _cu(lk)}
    first = A.attention(q, k, v, **args)
    for _ in range(5):
        assert torch.equal(A.attention(q, k, v, **args), first)


def test_empty_calls():
    q, k, v = qkv(0, 10, 2, 2, 64)
    assert A.attention(q, k, v).shape == (0, 2, 64)
    q, k, v = qkv(5, 0, 2, 2, 64)
    o, lse = A.attention(q, k, v, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    o = A.attention(q, k, v, cu_q=torch.zeros(1, dtype=torch.int32, device=DEV),
                    cu_k=torch.zeros(1, dtype=torch.int32, device=DEV), out=torch.ones_like(q))
    assert (o == 1).all()


# ------------------------------------------------------------------------------------------------ rotary table


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32, torch.float64])
@pytest.mark.parametrize("axes,theta", [((2,), 10000.0), ((128,), 10000.0), ((44, 42, 42), 10000.0), ((16, 24, 24), (100.0, 1e4, 5e5)),
                                        ((64, 32, 32, 64, 64), 256.0)])
def test_rotary_table(axes, theta, dtype):
    T = 777
    pos = torch.randint(0, 2_000_000, (T, len(axes)), generator=_gen(1), device=DEV).double()
    pos[:40] = torch.arange(40, device=DEV, dtype=torch.float64)[:, None]
    if dtype.is_floating_point:
        pos = pos * 0.37 - 1000
    pos = pos.to(dtype)
    table = A.rotary_table(pos, axes, theta=theta)
    thetas = theta if isinstance(theta, tuple) else (theta,) * len(axes)
    ang = torch.cat([pos[:, a, None].double() * (thetas[a] ** (-torch.arange(0, d, 2, device=DEV).double() / d))
                     for a, d in enumerate(axes)], dim=1)
    want = torch.stack([ang.cos(), ang.sin()], dim=-1)
    assert table.shape == (T, sum(axes) // 2, 2) and table.dtype == torch.float32
    # fp64 angles of 2e6 are themselves known to 2e6 * 2^-52
    assert (table.double() - want).abs().max() <= 4 * 2.0**-23 + 2e6 * 2.0**-51


def test_rotary_table_of_strided_and_few_positions():
    pos = torch.randint(0, 50, (30, 5), generator=_gen(2), device=DEV, dtype=torch.int32)
    assert torch.equal(A.rotary_table(pos[:, 1:4], (16, 24, 24)), A.rotary_table(pos[:, 1:4].contiguous(), (16, 24, 24)))
    assert torch.equal(A.rotary_table(pos[:, 2], (64,)), A.rotary_table(pos[:, 2:3].contiguous(), (64,)))
    assert torch.equal(A.rotary_table(pos[:1, 1:4].expand(30, 3), (16, 24, 24))[29],
                       A.rotary_table(pos[:1, 1:4].contiguous(), (16, 24, 24))[0])
    assert A.rotary_table(pos[:0, :3], (16, 24, 24)).shape == (0, 32, 2)
    assert torch.isnan(A.rotary_table(torch.tensor([math.inf, math.nan], device=DEV), (8,))).all()


# ------------------------------------------------------------------------------------------------ norm and rotation


def norm_rope_reference(x, weight, eps, norm, table, interleaved):
    """(y, bound) in fp64."""
    y = x.double()
    D = x.shape[2]
    if norm:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
    size = y.abs()
    if table is not None:
        R = 2 * table.shape[1]
        c, s = table.double()[:, None, :, 0], table.double()[:, None, :, 1]
        sel = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
        a, b = y[..., sel[0]].clone(), y[..., sel[1]].clone()
        y[..., sel[0]], y[..., sel[1]] = a * c - b * s, b * c + a * s
        size[..., sel[0]] = size[..., sel[1]] = a.abs() + b.abs()
    step = (D + 16) * 2.0**-24 * size
    return y, U[x.dtype] * (y.abs() + step) + step + 2.0**-25 * (x.dtype == torch.float16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,R", [(8, 8), (16, 16), (40, 32), (64, 64), (72, 48), (80, 80), (128, 128), (128, 64), (200, 160),
                                 (256, 256)])
def test_norm_and_rotation(D, R, interleaved, dtype):
    if R % 16 and not interleaved:
        R = None
    T, Hq, Hk = 37, 5, 3
    q = _randn(T, Hq, D, seed=D, dtype=dtype, scale=3.0)
    k = _randn(T, Hk, D, seed=D + 1, dtype=dtype, scale=0.1)
    q[0, 0] = 0
    table = None if R is None else A.rotary_table(torch.arange(T, device=DEV) * 97, (R,))
    for norm, weights in ((True, dtype), (True, torch.float32), (True, None), (False, None)):
        if not norm and table is None:
            continue
        wq, wk = (None, None) if weights is None else (1 + _randn(D, seed=1, scale=0.3), 1 + _randn(D, seed=2, scale=0.3))
        if weights is not None:
            wq, wk = wq.to(weights), wk.to(weights)
        got = A.qk_norm_rope(q, k, q_weight=wq, k_weight=wk, eps=1e-5, norm=norm, table=table, interleaved=interleaved)
        for g, x, w in zip(got, (q, k), (wq, wk)):
            want, bound = norm_rope_reference(x, w, 1e-5, norm, table, interleaved)
            assert g.dtype == dtype and ((g.double() - want).abs() <= bound).all()
        alone = A.qk_norm_rope(q, q_weight=wq, eps=1e-5, norm=norm, table=table, interleaved=interleaved)
        assert torch.equal(alone, got[0])


@pytest.mark.parametrize("T", [0, 1, 2, 1000])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (7, 1), (40, 40), (3, 40)])
def test_norm_and_rotation_of_any_rows_in_place_and_strided(T, Hq, Hk):
    D = 64
    x = _randn(T, (Hq + 2 * Hk) * D, seed=5, dtype=torch.bfloat16)
    q, k = x[:, : Hq * D].unflatten(1, (Hq, D)), x[:, Hq * D : (Hq + Hk) * D].unflatten(1, (Hk, D))
    w = 1 + _randn(D, seed=6, dtype=torch.bfloat16, scale=0.3)
    table = A.rotary_table(torch.arange(T, device=DEV), (48,))
    rest = x[:, (Hq + Hk) * D :].clone()
    args = {"q_weight": w, "k_weight": w, "table": table}
    fresh = A.qk_norm_rope(q.contiguous(), k.contiguous(), **args)
    outs = A.qk_norm_rope(q, k, **args)
    assert torch.equal(outs[0], fresh[0]) and torch.equal(outs[1], fresh[1])
    for g, t in zip(fresh, (q, k)):
        want, bound = norm_rope_reference(t, w, 1e-6, True, table, True)
        assert ((g.double() - want).abs() <= bound).all()
    back = A.qk_norm_rope(q, k, q_out=q, k_out=k, **args)
    assert back[0] is q and torch.equal(q, fresh[0]) and torch.equal(k, fresh[1])
    assert torch.equal(x[:, (Hq + Hk) * D :], rest)


def test_rows_of_nan_stay_in_their_head():
    q = _randn(4, 4, 128, seed=7, dtype=torch.bfloat16)
    clean = A.qk_norm_rope(q)
    q[1, 2, 5] = math.nan
    got = A.qk_norm_rope(q)
    assert torch.isnan(got[1, 2]).all()
    got[1, 2] = clean[1, 2]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("lk", [70, 300])
def test_scores_that_are_not_finite(lk):
    """NaN and +infinity among a row's scores make the row NaN, -infinity a weight of zero; other rows do not change."""
    q, k, v = qkv(140, lk, 2, 2, 64, seed=12)
    q = q.abs() + 0.1
    clean = A.attention(q, k, v)
    for key in range(0, lk, 11):
        bad = k.clone()
        bad[key, 0, 3] = -math.inf
        want, *_ = reference(q, bad, v, [140], [lk], False, 0.125)
        got = A.attention(q, bad, v)
        assert not torch.isnan(got).any() and torch.equal(got[:, 1], clean[:, 1])
        assert (got.double() - want).abs().max() <= 0.03
        bad[key, 0, 3] = math.inf if key % 2 else math.nan
        got = A.attention(q, bad, v)
        assert torch.isnan(got[:, 0]).all() and torch.equal(got[:, 1], clean[:, 1])
    row = q.clone()
    row[77, 1] = math.nan
    got = A.attention(row, k, v)
    assert torch.isnan(got[77, 1]).all()
    got[77, 1] = clean[77, 1]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq,lk,D,group", [(300, 300, 128, 1), (130, 517, 64, 1), (3, 700, 128, 4), (260, 260, 72, 5), (1, 4000, 128, 2)])
def test_values_that_causal_rows_do_not_see(lq, lk, D, group, dtype):
    """A value row that is not finite reaches the rows that see its key, in its columns, and no other."""
    q, k, v = qkv(lq, lk, 2 * group, 2, D, dtype, seed=13, spread=0.5)
    clean = A.attention(q, k, v, causal=True)
    keys = sorted({0, 5, lk // 2, max(lk - lq, 0), lk - lq // 2 - 1, lk - 2, lk - 1} & set(range(lk)))
    for key in keys:
        for bad in (math.nan, math.inf):
            spoilt = v.clone()
            spoilt[key, 1, 3] = bad
            spoilt[key, 1, D - 1] = -bad
            got = A.attention(q, k, spoilt, causal=True)
            hit = torch.zeros(got.shape, dtype=torch.bool, device=DEV)
            sees = torch.arange(lq, device=DEV) + lk - lq >= key
            hit[:, group:, 3] = hit[:, group:, D - 1] = sees[:, None]
            assert torch.equal(~torch.isfinite(got), hit), (key, bad)
            assert torch.equal(got[~hit], clean[~hit])
            if bad == math.inf:
                assert (got[:, group:, 3][sees] == math.inf).all() and (got[:, group:, D - 1][sees] == -math.inf).all()


def test_many_values_that_are_not_finite():
    q, k, v = qkv(200, 200, 1, 1, 64, seed=14, spread=0.5)
    clean = A.attention(q, k, v, causal=True)
    v[90:] = math.nan
    got = A.attention(q, k, v, causal=True)
    assert torch.equal(got[:90], clean[:90]) and torch.isnan(got[90:]).all()


def test_small_weights_of_a_long_row_count():
    """One score far above 30000 others, whose weights together still matter: 16-bit weights must not lose them."""
    for dtype in (torch.float16, torch.bfloat16):
        n = 30000
        q = torch.zeros(1, 1, 64, dtype=dtype, device=DEV)
        q[0, 0, 0] = 8
        k = torch.zeros(n, 1, 64, dtype=dtype, device=DEV)
        k[777, 0, 0] = 14.0  # exp(14) = 1.2e6, the others 1 each
        v = torch.ones(n, 1, 64, dtype=dtype, device=DEV)
        v[777] = 0
        check(q, k, v, [1], [n], cu=False)


def test_strides_of_single_elements_do_not_matter():
    q, k, v = qkv(1, 9, 4, 1, 64, seed=15)
    want = A.attention(q, k, v)
    odd = torch.as_strided(q, q.shape, (3, 64, 1))
    assert torch.equal(A.attention(odd, torch.as_strided(k, k.shape, (64, 5, 1)), torch.as_strided(v, v.shape, (64, 1, 1))), want)
    assert torch.equal(A.qk_norm_rope(odd), A.qk_norm_rope(q))


# ------------------------------------------------------------------------------------------------ as they are used


def test_joined_module_in_an_attention_block():
    """Packed sequences through convrot projections, norms, rotation, attention and the out projection: the block's
    module against the single calls, and those against the formulas on the projections' own outputs."""
    from hyperflow_h3_flash_b200 import int8 as I
    from hyperflow_h3_flash_b200 import synthetic, ulysses

    T, width, heads, D = 410, 1024, 8, 128
    layers = []
    for i in range(4):
        layer = I.Int8RotLinear(width, width, 256, bias=True)
        synthetic.load_into(layer, synthetic.linear_weights(width, width, seed_offset=40 + i))
        layers.append(layer.to(DEV))
    core = A.QKNormAttention(D).to(DEV)
    core.norm_q.weight.copy_(1 + _randn(D, seed=20, scale=0.2))
    core.norm_k.weight.copy_(1 + _randn(D, seed=21, scale=0.2))
    lens = [200, 0, 33, 177]
    grid = torch.stack([torch.arange(T, device=DEV) // 60, torch.arange(T, device=DEV) // 10 % 6, torch.arange(T, device=DEV) % 10], 1)
    table = A.rotary_table(grid, (44, 42, 42))
    core.set_sequences(table, _cu(lens))
    x = synthetic.activations(T, width, seed=22).to(DEV)
    got = ulysses.attention_block_linears(x, *layers, heads, attention=core)
    q, k, v = (layer(x).view(T, heads, D) for layer in layers[:3])
    qn, kn = A.qk_norm_rope(q, k, q_weight=core.norm_q.weight, k_weight=core.norm_k.weight, table=table)
    for g, t, w in ((qn, q, core.norm_q.weight), (kn, k, core.norm_k.weight)):
        want, bound = norm_rope_reference(t, w, 1e-6, True, table, True)
        assert ((g.double() - want).abs() <= bound).all()
    o = check(qn, kn, v, lens, lens)
    assert torch.equal(got, layers[3](o.reshape(T, width)))


def test_captured_and_replayed():
    from hyperflow_h3_flash_b200.graphs import CapturedCall

    q, k, v = qkv(70, 2500, 4, 2, 128, seed=23)
    table = A.rotary_table(torch.arange(70, device=DEV), (128,))

    def call(q, k, v):
        return A.attention(A.qk_norm_rope(q, table=table), k, v, causal=True)

    assert _lib.lib().convrot_attention_workspace_size(70, 2500, 1, 4, 2, 128) > 0
    first, second = CapturedCall(call, q, k, v), CapturedCall(call, q, k, v)  # two graphs, each with its own workspace
    for seed in (24, 25, 26):
        a, b = qkv(70, 2500, 4, 2, 128, seed=seed), qkv(70, 2500, 4, 2, 128, seed=seed + 10)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            two = second(*b)
        one = first(*a)
        torch.cuda.synchronize()
        assert torch.equal(one, call(*a)) and torch.equal(two, call(*b))


def test_calls_on_two_streams_at_once():
    cases = [qkv(300, 3000, 4, 4, 64, seed=30 + i) for i in range(4)]
    want = [A.attention(*c, causal=True) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(A.attention(*c, causal=True))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_more_items_than_the_grid_has_sms():
    """Whole waves of items, and a last one that is divided among the SMs."""
    q, k, v = qkv(4500, 2100, 12, 12, 64, seed=40)
    check(q, k, v, [4500], [2100], cu=False)
    lens = [1000, 1, 2048, 130, 1321]
    check(q, torch.cat([k, k, k])[:4500], torch.cat([v, v, v])[:4500], lens, lens, True)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("packed", [False, True])
def test_items_that_fill_whole_waves(D, packed):
    """Nothing is left over to be divided among the SMs."""
    heads = torch.cuda.get_device_properties(0).multi_processor_count
    q, k, v = qkv(40, 1100, heads, heads, D, seed=41)
    check(q, k, v, [40], [1100], cu=packed)
    assert _lib.lib().convrot_attention_workspace_size(40, 1100, 1, heads, heads, D) > 0


def test_workspace_of_very_long_keys():
    """Keys whose work, summed over the divided items, would pass 32 bits are not divided."""
    size = _lib.lib().convrot_attention_workspace_size
    assert size(1, 1 << 28, 1, 8, 1, 64) > 0 and size(1, (1 << 28) + 1, 1, 8, 1, 64) == 0


def test_offsets_beyond_32_bits():
    """Queries, keys, values and outputs as columns of one wide buffer whose rows reach past 2^31 elements."""
    T, width = 34000, 65536
    buf = torch.empty(T, width, dtype=torch.bfloat16, device=DEV)
    parts = [buf[:, i * 128 : (i + 1) * 128].unflatten(1, (1, 128)) for i in range(4)]
    for i, t in enumerate(parts[:3]):
        t.copy_(_randn(T, 1, 128, seed=50 + i, dtype=torch.bfloat16))
    q, k, v, out = parts
    dense = [t.contiguous() for t in (q, k, v)]
    for causal in (False, True):
        A.attention(q, k, v, causal=causal, out=out)
        assert torch.equal(out, A.attention(*dense, causal=causal))
    few = A.attention(q[-3:], k, v, causal=True)  # single tokens: the keys are divided
    assert torch.equal(few, A.attention(dense[0][-3:], *dense[1:], causal=True))
    table = A.rotary_table(torch.arange(T, device=DEV), (128,))
    A.qk_norm_rope(q, k, table=table, q_out=out, k_out=k)
    assert torch.equal(out, A.qk_norm_rope(dense[0], table=table)) and torch.equal(k, A.qk_norm_rope(dense[1], table=table))
    A.qk_norm_rope(q, table=table, interleaved=False, q_out=q)
    assert torch.equal(q, A.qk_norm_rope(dense[0], table=table, interleaved=False))


def test_compiled_and_interpreted_calls_agree():
    """The compiled form of a call gives what the checked one gives, and hands over what it does not take."""
    fast = A._fast_calls()
    assert fast is not None
    q, k, v = qkv(40, 40, 4, 2, 64, seed=60)
    table = A.rotary_table(torch.arange(40, device=DEV), (64,))
    w = torch.ones(64, device=DEV)
    quick = fast.qk_norm_rope(q, k, w, None, 1e-6, True, table, True)
    slow = A.qk_norm_rope(q, k, q_weight=w, table=table, q_out=torch.empty_like(q), k_out=torch.empty_like(k))
    assert all(torch.equal(a, b) for a, b in zip(quick, slow))
    quick, lse = fast.attention(q, k, v, None, None, True, None, True)
    slow, slow_lse = A.attention(q, k, v, causal=True, out=torch.empty_like(q), return_lse=True)
    assert torch.equal(quick, slow) and torch.equal(lse, slow_lse)
    cu = _cu([40])
    for args in ((q.cpu(), k, v, None, None, True, None, False), (q, k.half(), v, None, None, True, None, False),
                 (q, k, v[:3], None, None, True, None, False), (q, k, v, cu, None, True, None, False),
                 (q, k, v, cu.long(), cu, True, None, False), (q, k, v, None, None, True, -1.0, False),
                 (q.clone().requires_grad_(), k, v, None, None, True, None, False),
                 (q, k[:, :0], v[:, :0], None, None, True, None, False), (q, k, v, None, None, 1, None, False),
                 (q, k, v, None, None, True, "x", False), (q, k, v)):
        assert fast.attention(*args) is None
    for args in ((q, k[:5], None, None, 1e-6, True, table, True), (q, k, w[:3], None, 1e-6, True, table, True),
                 (q, k, w, w.bfloat16(), 1e-6, True, table, True), (q, None, None, w, 1e-6, True, table, True),
                 (q, k, w, None, 1e-6, False, table, True), (q, k, None, None, math.nan, True, table, True),
                 (q, k, None, None, 1e-6, False, None, True), (q, k, None, None, 1e-6, True, table.double(), True),
                 (q, k, None, None, 1e-6, True, table[:, :3], True)):
        assert fast.qk_norm_rope(*args) is None
    for args in ((table, (64,), 1e4), (torch.arange(4, device=DEV)[:, None], (63,), 1e4),
                 (torch.arange(4, device=DEV)[:, None], (64,), 0.0), (torch.arange(4, device=DEV)[:, None], (64, 64), 1e4)):
        assert fast.rotary_table(*args) is None


def test_refusals_on_the_gpu_leave_the_device_usable():
    q, k, v = qkv(8, 8, 2, 2, 64, seed=61)
    wide = torch.empty(8, 2, 65, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: A.attention(q.float(), k.float(), v.float()), lambda: A.attention(wide[..., 1:], k, v),
                lambda: A.attention(q, k.expand(8, 2, 64)[:, :1].expand(8, 2, 64), v), lambda: A.qk_norm_rope(q.float()),
                lambda: A.attention(q, k, v, out=q), lambda: A.qk_norm_rope(wide[..., 1:]), lambda: A.qk_norm_rope(q, k, q_out=k),
                lambda: A.attention(q, k, v, cu_q=torch.zeros(2, dtype=torch.int32), cu_k=torch.zeros(2, dtype=torch.int32)),
                lambda: A.rotary_table(torch.zeros(3, 2, dtype=torch.int16, device=DEV), (8, 8))):
        with pytest.raises(ValueError):
            bad()
    check(q, k, v, [8], [8], cu=False)


# ------------------------------------------------------------------------------------------------ given outputs


def _layer_that_keeps_its_input(width, group):
    from hyperflow_h3_flash_b200 import int8 as I
    from hyperflow_h3_flash_b200 import synthetic

    layer = I.Int8RotLinear(width, 256, group)
    synthetic.load_into(layer, synthetic.linear_weights(width, 256, bias=False, group=group))
    layer.keep_input = True
    return layer.to(DEV)


@pytest.mark.parametrize("inference", [False, True])
@pytest.mark.parametrize("view", [False, True])
def test_a_buffer_that_is_written_again_is_quantised_again(view, inference):
    """A layer with keep_input recognises its last input by the tensor and its version: writing into a given output
    counts as torch's own in-place operations do, for the buffer and for a view of it that was kept."""
    T, H, D = 96, 1 if not view else 2, 128
    layer = _layer_that_keeps_its_input(H * D, 64)
    with torch.inference_mode(inference):
        q, k, v = qkv(T, T, H, H, D, seed=70)
        buf = torch.zeros_like(q)
        x = buf.view(T, H * D) if view else buf
        for write in (lambda: A.attention(q, k, v, out=buf), lambda: A.qk_norm_rope(q, q_out=buf),
                      lambda: A.qk_norm_rope(q, k, q_out=torch.empty_like(q), k_out=buf)):
            before = layer(x)
            write()
            got = layer(x)
            assert torch.equal(got, layer(x.clone())) and not torch.equal(got, before)


# ------------------------------------------------------------------------------------------------ bounds


def _guarded(rows, *rest, dtype, pad=512):
    """A tensor in the middle of a buffer of sevens, and a check that the rows around it are as they were."""
    buf = torch.full((rows + 2 * pad, *rest), 7.0, dtype=dtype, device=DEV)

    def untouched():
        return bool((buf[:pad] == 7).all() and (buf[pad + rows :] == 7).all())

    return buf[pad : pad + rows], untouched


def _attention_entry(q, k, v, cu_q, cu_k, causal, out, lse, space):
    """convrot_attention itself, on a workspace of the caller's."""
    P = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    (Tq, Hq, D), (Tk, Hkv, _) = q.shape, k.shape
    return _lib.lib().convrot_attention(
        P(q), *q.stride()[:2], P(k), *k.stride()[:2], P(v), *v.stride()[:2], P(cu_q), P(cu_k),
        1 if cu_q is None else cu_q.numel() - 1, Tq, Tk, Hq, Hkv, D, 0, D**-0.5, causal, P(out), *out.stride()[:2], P(lse),
        P(space), space.numel() * space.element_size(), torch.cuda.current_stream().cuda_stream)


NO_PLAN = [  # shares, items, first item, all work, then the work before each item in equal steps of the last number
    (0, 0, 0, 0, 0), (5, 100, -37, 4000, 40), (5, 100, -148, 4000, 40), (148, 147, 3, 4000, 20), (148, 147, 1 << 30, 9000, 60),
    (148, 147, 148, 9000, 60), (148, 147, 2**31 - 2, 9000, 60), (1, 191, 0, 2**31 - 1, 10_000_000), (148, 147, 0, 9000, -60)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("plan", NO_PLAN)
def test_a_plan_that_was_never_written_leads_nowhere(plan, causal):
    """Offsets of sequences that overlap, which the arrays must not hold, make more items than the grid has CTAs, and
    the plan for the joining kernel is not written: whatever the workspace held, nothing outside the outputs is."""
    T, heads = 8192, 2
    q, k, v = qkv(T, T, heads, heads, 64, seed=80)
    cu = torch.tensor([0, T] * 10, dtype=torch.int32, device=DEV)
    size = _lib.lib().convrot_attention_workspace_size(T, T, 19, heads, heads, 64)
    assert size > 0
    space = torch.zeros(size // 4, dtype=torch.int32, device=DEV)
    space[:4] = torch.tensor(plan[:4])
    space[4:196] = torch.tensor([max(-(2**31), min(2**31 - 1, i * plan[4])) for i in range(192)])
    out, out_kept = _guarded(T, heads, 64, dtype=torch.bfloat16)
    lse, lse_kept = _guarded(T, heads, dtype=torch.float32)
    assert _attention_entry(q, k, v, cu, cu, causal, out, lse, space) == 0
    torch.cuda.synchronize()
    assert out_kept() and lse_kept()


@pytest.mark.parametrize("cu", [[0, 5000, 2048], [-5, 1100, 2048], [1500, 20, 2048], [2**31 - 1, -(2**31), 2**31 - 1],
                                [0, 2048, 0, 2048], [7, 7, 7]])
def test_offsets_that_make_no_sense_write_nothing_outside(cu):
    T = 2048
    q, k, v = qkv(T, T, 4, 2, 64, seed=81)
    cu = torch.tensor(cu, dtype=torch.int32, device=DEV)
    assert _lib.lib().convrot_attention_workspace_size(T, T, cu.numel() - 1, 4, 2, 64) > 0
    for causal in (False, True):
        for cu_q, cu_k in ((cu, cu), (cu, torch.full_like(cu, T)), (torch.linspace(0, T, cu.numel(), device=DEV).int(), cu)):
            out, kept = _guarded(T, 4, 64, dtype=torch.bfloat16)
            A.attention(q, k, v, cu_q=cu_q, cu_k=cu_k, causal=causal, out=out)
            torch.cuda.synchronize()
            assert kept()


# ------------------------------------------------------------------------------------------------ derivatives


def test_every_input_and_given_output_that_requires_grad_is_refused():
    q, k, v = qkv(5, 5, 2, 2, 64, seed=82)
    table, w = A.rotary_table(torch.arange(5, device=DEV), (64,)), torch.ones(64, device=DEV)
    wants = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda: A.attention(wants(q), k, v), lambda: A.attention(q, wants(k), v), lambda: A.attention(q, k, wants(v)),
             lambda: A.attention(q, k, v, out=wants(q)), lambda: A.qk_norm_rope(wants(q)), lambda: A.qk_norm_rope(q, wants(k)),
             lambda: A.qk_norm_rope(q, q_weight=wants(w)), lambda: A.qk_norm_rope(q, k, table=wants(table)),
             lambda: A.qk_norm_rope(q, k, q_out=wants(q)), lambda: A.qk_norm_rope(q, k, k_out=wants(k)),
             lambda: A.rotary_table(wants(torch.arange(5.0, device=DEV)), (16,)),
             lambda: A.rotary_table(wants(torch.ones(5, 2, device=DEV)), (8, 8))]
    for call in calls:
        with pytest.raises(ValueError, match="inference only"):
            call()
        with torch.no_grad():
            call()


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad

    q, k, v = qkv(5, 5, 2, 2, 64, seed=83)
    table = A.rotary_table(torch.arange(5, device=DEV), (64,))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: A.attention(dual(q), k, v), lambda: A.attention(q, dual(k), v), lambda: A.attention(q, k, dual(v)),
                     lambda: A.qk_norm_rope(dual(q)), lambda: A.qk_norm_rope(q, dual(k)),
                     lambda: A.qk_norm_rope(q, q_weight=dual(torch.ones(64, device=DEV))),
                     lambda: A.qk_norm_rope(q, table=dual(table)), lambda: A.rotary_table(dual(torch.arange(5.0, device=DEV)), (16,)),
                     lambda: A.rotary_table(dual(torch.ones(5, 2, device=DEV)), (8, 8))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="tangent"):
                    call()
        assert torch.equal(A.attention(forward_ad.unpack_dual(dual(q)).primal, k, v), A.attention(q, k, v))


# ------------------------------------------------------------------------------------------------ the wait limit


@pytest.mark.parametrize("causal", [False, True])
def test_an_item_may_take_longer_than_the_wait_limit(causal):
    """The limit of the device-side waits bounds a stall, not the work of an item: here every CTA has one item of 256 key
    tiles (about 350 us), under a limit of 100 us."""
    L = _lib.lib()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    q, k, v = qkv(sms * 256, 32768, 1, 1, 64, seed=84)
    want = A.attention(q, k, v, causal=causal)
    torch.cuda.synchronize()
    L.convrot_set_wait_limit_ns(100_000)
    try:
        got = A.attention(q, k, v, causal=causal)
        torch.cuda.synchronize()
        assert L.convrot_poll_error(None) == 0
    finally:
        L.convrot_set_wait_limit_ns(0)
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ shares


@pytest.mark.parametrize("D,causal", [(64, False), (128, True)])
def test_short_items_of_many_requests(D, causal):
    """Last items that are too short to be cut: each is a share of its own, beside requests of other lengths and with
    one among them that is cut."""
    for lk in ([40] * 100, [128] * 147, [300] * 120, [1 + 7 * i % 300 for i in range(140)], [5000] + [17] * 90,
               [17] * 90 + [5000], [513] * 30 + [2000, 0, 3]):
        lq = [1 + i % 3 for i in range(len(lk))]
        q, k, v = qkv(sum(lq), sum(lk), 4, 1, D, seed=85 + len(lk))
        check(q, k, v, lq, lk, causal)
        check(*qkv(len(lk), sum(lk), 5, 5, D, seed=86 + len(lk)), [1] * len(lk), lk, causal)


@pytest.mark.parametrize("D", [64, 128])
def test_a_last_wave_that_is_divided_behind_whole_ones(D):
    size = _lib.lib().convrot_attention_workspace_size
    q, k, v = qkv(2560, 8192, 20, 20, D, seed=87)
    assert size(2560, 8192, 1, 20, 20, D) > 0
    check(q, k, v, [2560], [8192], cu=False)
    check(q, k, v, [2560], [8192], True, cu=False)
    lq, lk = [1200, 1, 1359], [6000, 8013, 2371]
    assert size(2560, 16384, 3, 20, 20, D) > 0
    check(q, torch.cat([k, k]), torch.cat([v, v]), lq, lk, True)


def test_which_calls_are_divided():
    """Where dividing the last items measured faster, and where it did not (sizes on both sides of the rule)."""
    size = _lib.lib().convrot_attention_workspace_size
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the sizes are for 148 SMs")
    for Tq, Tk, batch, hq, hkv, divided in (
            (1, 1536, 1, 8, 8, False), (1, 2048, 1, 8, 8, True), (256, 2048, 1, 40, 40, False), (256, 3000, 1, 40, 40, True),
            (700, 1024, 1, 40, 40, False), (700, 32760, 1, 40, 40, False), (4096, 2048, 1, 40, 40, False),
            (4096, 4096, 1, 40, 40, True), (32760, 32760, 1, 5, 5, True), (32760, 333, 1, 40, 40, False),
            (33093, 33093, 2, 5, 5, True), (100, 4000, 100, 8, 1, False), (64, 63 * 100 + 8000, 64, 40, 8, True),
            (4000, 4000, 4, 8, 8, False), (8720, 8720, 4, 40, 40, False), (1024, 8300, 4, 8, 8, True),
            (40 * 256, 39 * 200 + 32768, 40, 40, 40, True), (40 * 256, 40 * 500, 40, 40, 40, False), (17, 333, 1, 8, 8, False)):
        assert (size(Tq, Tk, batch, hq, hkv, 128) > 0) == divided, (Tq, Tk, batch, hq, hkv)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_caches_with_room_to_grow(dtype):
    """Rows of a cache that are not filled yet, given as sequences without a query: whatever they hold reaches nobody."""
    room, filled = 640, [1, 640, 300, 129, 511]
    k, v = (_randn(room * len(filled), 2, 128, seed=s, dtype=dtype) for s in (88, 89))
    lq, lk = [], []
    for i, n in enumerate(filled):
        lq += [1, 0]
        lk += [n, room - n]
        for t in (k, v):
            t[i * room + n : (i + 1) * room] = math.nan if i % 2 else math.inf
    q = _randn(len(filled), 10, 128, seed=90, dtype=dtype)
    for causal in (False, True):
        got = A.attention(q, k, v, cu_q=_cu(lq), cu_k=_cu(lk), causal=causal)
        keep = torch.cat([torch.arange(i * room, i * room + n, device=DEV) for i, n in enumerate(filled)])
        want, _, bound, _ = reference(q, k[keep], v[keep], [1] * len(filled), filled, causal, 128**-0.5)
        assert ((got.double() - want).abs() <= bound).all()
    # the next token of each: the offsets move, the cache stays
    for i, n in enumerate(filled):
        if n < room:
            k[i * room + n], v[i * room + n] = 0.5, 2.0
    lk = [x for n in filled for x in (min(n + 1, room), room - min(n + 1, room))]
    assert torch.isfinite(A.attention(q, k, v, cu_q=_cu(lq), cu_k=_cu(lk), causal=True)).all()


# ------------------------------------------------------------------------------------------------ more ways of use


def test_captured_with_a_fork_a_copy_and_changing_offsets():
    """One graph with a copied input, a branch on a second stream that joins again, and offsets that move between replays."""
    T, Tk, H, D = 96, 4096, 4, 128
    q, k, v = qkv(T, Tk, H, H, D, seed=91)
    table = A.rotary_table(torch.arange(T, device=DEV), (D,))
    cu_q, cu_k = _cu([40, 56]), _cu([4000, 96])
    staged = torch.empty_like(q)

    def call():
        main, side = torch.cuda.current_stream(), streams[0]
        staged.copy_(q)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            other = A.attention(staged, k, v, causal=True)
        turned = A.qk_norm_rope(staged, table=table)
        packed = A.attention(turned, k, v, cu_q=cu_q, cu_k=cu_k)
        main.wait_stream(side)
        return other, A.attention(A.qk_norm_rope(other, table=table), k, v), packed

    streams = [torch.cuda.Stream()]
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed, lens in ((92, [(40, 56), (4000, 96)]), (93, [(1, 95), (1, 4095)]), (94, [(96, 0), (4096, 0)])):
        q.copy_(_randn(T, H, D, seed=seed, dtype=q.dtype))
        for cu, length in zip((cu_q, cu_k), lens):
            cu.copy_(_cu(list(length)))
        graph.replay()
        torch.cuda.synchronize()
        first = [t.clone() for t in got]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, got))
        assert all(torch.equal(a, b) for a, b in zip(first, call()))


def test_calls_from_several_threads_at_once():
    import threading

    cases = [(qkv(1 + 64 * i, 3000 + i, 4, 2, 64 + 64 * (i % 2), seed=95 + i), i % 2 == 0) for i in range(4)]
    want = [A.attention(*c, causal=causal) for c, causal in cases]
    tables = [A.rotary_table(torch.arange(c[0].shape[0], device=DEV), (64,)) for c, _ in cases]
    turned = [A.qk_norm_rope(c[0], table=t) for (c, _), t in zip(cases, tables)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        (c, causal), stream = cases[i], torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for n in range(50):
                out = torch.empty_like(c[0]) if n % 2 else None
                got, rot = A.attention(*c, causal=causal, out=out), A.qk_norm_rope(c[0], table=tables[i])
                stream.synchronize()
                if not (torch.equal(got, want[i]) and torch.equal(rot, turned[i])):
                    wrong.append((i, n))
            stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_one_module_for_all_blocks_of_a_pass():
    """The module's table and offsets serve every block, q and k of each are turned in place, and a replay of the captured
    pass on new inputs gives what the calls give."""
    T, H, D = 200, 4, 128
    core = A.QKNormAttention(D, causal=True).to(DEV)
    core.set_sequences(A.rotary_table(torch.arange(T, device=DEV), (D,)), _cu([150, 0, 50]))

    def blocks(q, k, v):
        for _ in range(3):
            o = core(q.clone(), k.clone(), v)
            q, k, v = o, q + o, v + o
        return o

    from hyperflow_h3_flash_b200.graphs import CapturedCall

    call = CapturedCall(blocks, *qkv(T, T, H, H, D, seed=99))
    for seed in (100, 101):
        args = qkv(T, T, H, H, D, seed=seed)
        kept = [t.clone() for t in args]
        assert torch.equal(call(*args), blocks(*args))
        assert all(torch.equal(a, b) for a, b in zip(args, kept))


def test_numbers_of_numpy_are_numbers():
    """In the compiled form, in the interpreted one and for outputs that are given alike."""
    import numpy as np

    q, k, v = qkv(5, 9, 2, 2, 64, seed=102)
    table = A.rotary_table(torch.arange(5, device=DEV), (64,), theta=np.float32(500.0))
    assert torch.equal(table, A.rotary_table(torch.arange(5, device=DEV), (64,), theta=500.0))
    want = A.attention(q, k, v, causal=True, scale=0.25)
    for kw in ({}, {"out": torch.empty_like(q)}):
        assert torch.equal(A.attention(q, k, v, causal=np.True_, scale=np.float32(0.25), **kw), want)
    want = A.qk_norm_rope(q, table=table, eps=0.5, interleaved=False)
    for kw in ({}, {"q_out": torch.empty_like(q)}):
        got = A.qk_norm_rope(q, table=table, eps=np.float32(0.5), norm=np.True_, interleaved=np.False_, **kw)
        assert torch.equal(got, want)


def test_compiled_and_interpreted_calls_agree_on_given_outputs():
    fast = A._fast_calls()
    q, k, _ = qkv(40, 40, 4, 2, 64, seed=103)
    table = A.rotary_table(torch.arange(40, device=DEV), (64,))
    want = A.qk_norm_rope(q, k, table=table)
    qo, ko = torch.empty(4, 40, 64, dtype=q.dtype, device=DEV).transpose(0, 1), torch.empty_like(k)
    versions = qo._version, ko._version
    base = (None, None, 1e-6, True, table, True)
    for outs in ((qo, ko), (None, ko), (qo, None)):
        got = fast.qk_norm_rope(q, k, *base, *outs)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(b is None or a is b for a, b in zip(got, outs))
    assert (qo._version, ko._version) == (versions[0] + 2, versions[1] + 2)
    assert fast.qk_norm_rope(q, None, *base, qo, None) is qo and torch.equal(qo, want[0])
    with torch.inference_mode():
        kept = torch.empty_like(q)
    for args in ((q, k, *base, k, None), (q, k, *base, None, q), (q, k, *base, qo, qo), (q, q, *base, q, q), (q, None, *base, None, ko),
                 (q, k, *base, qo[:3], ko), (q, k, *base, qo.half(), ko), (q, k, *base, qo.cpu(), ko), (q, k, *base, kept, ko),
                 (q, k, *base, qo.clone().requires_grad_(), ko), (q, k, *base, qo)):
        assert fast.qk_norm_rope(*args) is None
    inplace = q.clone(), k.clone()
    back = A.qk_norm_rope(*inplace, table=table, q_out=inplace[0], k_out=inplace[1])
    assert back[0] is inplace[0] and back[1] is inplace[1] and all(torch.equal(a, b) for a, b in zip(back, want))
    # (a truth value that is no bool takes the interpreted way)
    assert fast.qk_norm_rope(q, k, None, None, 1e-6, True, table, 1, None, None) is None
    for outs in ({}, {"q_out": qo, "k_out": ko}):
        assert all(torch.equal(a, b) for a, b in zip(A.qk_norm_rope(q, k, table=table, interleaved=1, **outs), want))


def test_compiled_and_interpreted_attention_agree_on_a_given_output():
    fast = A._fast_calls()
    q, k, v = qkv(40, 70, 4, 2, 64, seed=104)
    want, want_lse = A.attention(q, k, v, causal=1, return_lse=True)  # (no bool: the interpreted way)
    out = torch.empty(4, 40, 64, dtype=q.dtype, device=DEV).transpose(0, 1)
    version, base = out._version, (None, None, True, None)
    assert fast.attention(q, k, v, *base, False, out) is out and torch.equal(out, want) and out._version == version + 1
    out.zero_()
    got, lse = fast.attention(q, k, v, *base, True, out)
    assert got is out and torch.equal(out, want) and torch.equal(lse, want_lse)
    assert A.attention(q, k, v, causal=1, out=out.zero_()) is out and torch.equal(out, want)
    with torch.inference_mode():
        kept = torch.empty_like(q)
    same = q[:, :2].clone()
    for args in ((q, k, v, *base, False, q), (q, k, v, *base, False, out[:3]), (q, k, v, *base, False, out.half()),
                 (q, k, v, *base, False, out.cpu()), (q, k, v, *base, False, kept), (same, same, v[:40], *base, False, same),
                 (q[:, :2], k[:40], v[:40], *base, False, v[:40]), (q, k, v, *base, False, out.clone().requires_grad_())):
        assert fast.attention(*args) is None
    # the workspace of a divided call, and rows of no sequence
    q, k, v = qkv(9, 5000, 4, 2, 64, seed=105)
    out = torch.full_like(q, 7.0)
    assert A.attention(q, k, v, cu_q=_cu([1, 3]), cu_k=_cu([4000, 1000]), out=out) is out
    assert (out[4:] == 7).all() and torch.equal(out[:4], A.attention(q, k, v, cu_q=_cu([1, 3]), cu_k=_cu([4000, 1000]))[:4])
