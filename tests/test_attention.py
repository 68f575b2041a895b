"""The attention operators without a GPU: the CPU path against the formulas, and what the Python and C entries refuse
before any device call."""

from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

from hyperflow_h3_flash_b200 import attention as A
from hyperflow_h3_flash_b200 import ulysses
from tests.test_abi import lib  # noqa: F401  (builds the library)


def _qkv(Tq=6, Tk=9, Hq=4, Hkv=2, D=16, dtype=torch.float32):
    g = torch.Generator().manual_seed(0)
    return tuple(torch.randn(t, h, D, generator=g).to(dtype) for t, h in ((Tq, Hq), (Tk, Hkv), (Tk, Hkv)))


# ------------------------------------------------------------------------------------------------ CPU path


def test_attention_on_cpu_follows_the_definition():
    q, k, v = _qkv(7, 9)
    lq, lk = [3, 0, 4], [5, 2, 2]
    cu = [torch.tensor([0, 3, 3, 7], dtype=torch.int32), torch.tensor([0, 5, 7, 9], dtype=torch.int32)]
    out, lse = A.attention(q, k, v, cu_q=cu[0], cu_k=cu[1], causal=True, return_lse=True)
    q0 = k0 = 0
    for a, b in zip(lq, lk):
        for i in range(a):
            for h in range(4):
                n = i + b - a + 1  # keys that this query sees
                if n <= 0:
                    assert (out[q0 + i, h] == 0).all() and lse[q0 + i, h] == -math.inf
                    continue
                s = k[k0 : k0 + n, h // 2].double() @ q[q0 + i, h].double() / 4
                w = torch.softmax(s, 0)
                assert torch.allclose(out[q0 + i, h].double(), w @ v[k0 : k0 + n, h // 2].double(), atol=1e-5)
                assert abs(lse[q0 + i, h].item() - torch.logsumexp(s, 0).item()) < 1e-5
        q0, k0 = q0 + a, k0 + b


@pytest.mark.parametrize("interleaved", [True, False])
def test_norm_and_rotation_on_cpu(interleaved):
    q, k, _ = _qkv(5, 5)
    w = torch.linspace(0.5, 1.5, 16)
    table = A.rotary_table(torch.tensor([[0, 0], [1, 5], [2, 7], [1000, 3], [7, 7]]), (8, 8), theta=(100.0, 1e4))
    out = A.qk_norm_rope(q, k, q_weight=w, table=table[:, :8], interleaved=interleaved)
    for x, y, weight in ((q, out[0], w), (k, out[1], torch.ones(16))):
        n = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6) * weight.double()
        for j in range(8):
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + 8)
            c, s = table[:, j, 0].double()[:, None], table[:, j, 1].double()[:, None]
            assert torch.allclose(y[..., a].double(), n[..., a] * c - n[..., b] * s, atol=1e-5)
            assert torch.allclose(y[..., b].double(), n[..., b] * c + n[..., a] * s, atol=1e-5)
    # a rotation keeps the length of each pair, and position 0 does not turn
    assert torch.allclose(out[1].square().sum(-1), torch.full((5, 2), 16.0), atol=1e-3)
    assert torch.equal(A.qk_norm_rope(q, norm=False, table=table, interleaved=interleaved)[0], q[0])


def test_rotary_table_on_cpu_splits_the_axes():
    pos = torch.tensor([[3, 50, 7]])
    table = A.rotary_table(pos, (4, 6, 2))
    want = [3.0, 3.0 / 100, 50.0, 50 * 10000 ** (-1 / 3), 50 * 10000 ** (-2 / 3), 7.0]
    assert torch.allclose(table[0, :, 0], torch.tensor([math.cos(a) for a in want]))
    assert torch.allclose(table[0, :, 1], torch.tensor([math.sin(a) for a in want]))


def test_the_joined_module_is_the_callable_of_an_attention_block():
    core = A.QKNormAttention(16, dtype=torch.float32)
    core.norm_q.weight.copy_(torch.linspace(0.5, 2, 16))
    x = torch.randn(12, 64, generator=torch.Generator().manual_seed(1))
    table = A.rotary_table(torch.arange(12), (16,))
    cu = torch.tensor([0, 7, 12], dtype=torch.int32)
    core.set_sequences(table, cu)
    eye = lambda t: t.clone()  # noqa: E731
    got = ulysses.attention_block_linears(x, eye, eye, eye, eye, 4, attention=core)
    q = k = v = x.view(12, 4, 16)
    qn, kn = A.qk_norm_rope(q, k, q_weight=core.norm_q.weight, k_weight=core.norm_k.weight, table=table)
    want = A.attention(qn, kn, v, cu_q=cu, cu_k=cu).reshape(12, 64)
    assert torch.equal(got, want)
    assert sorted(core.state_dict()) == ["norm_k.weight", "norm_q.weight"]
    assert not any(p.requires_grad for p in core.parameters())


def test_what_a_causal_row_does_not_see_does_not_reach_it_on_cpu():
    q, k, v = _qkv(6, 9, 4, 2)
    want = A.attention(q, k, v, causal=True)
    v[7, 1, 3], v[8, 0, 0] = math.nan, math.inf
    got = A.attention(q, k, v, causal=True)
    assert got[4:, 2:, 3].isnan().all() and (got[5:, :2, 0] == math.inf).all()
    got[4:, 2:, 3] = want[4:, 2:, 3]
    got[5:, :2, 0] = want[5:, :2, 0]
    torch.testing.assert_close(got, want, rtol=0, atol=1e-6)


# ------------------------------------------------------------------------------------------------ refusals


def test_attention_refuses_what_it_does_not_compute():
    q, k, v = _qkv()
    cu = torch.tensor([0, 6], dtype=torch.int32)

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            A.attention(*(args or (q, k, v)), **kw)

    refused("tokens, heads", q[0], k, v)
    refused("must be \\[Tk", q, k, v[:5])
    refused("must be \\[Tk", q, k[..., :8], v[..., :8])
    refused("torch.float32 on cpu", q, k.half(), v)
    refused("cannot share", q[:, :3], k, v)
    refused("cannot share", q[:, :0], k, v)
    refused("head_dim", *_qkv(D=12))
    refused("head_dim", *_qkv(D=136))
    refused("contiguous in its last", q.transpose(1, 2).contiguous().transpose(1, 2), k, v)
    refused("scale", scale=0.0)
    refused("scale", scale=-1.0)
    refused("scale", scale=math.nan)
    refused("come together", cu_q=cu)
    refused("cu_q must be", cu_q=cu.long(), cu_k=cu)
    refused("cu_k must be", cu_q=cu, cu_k=cu[None])
    refused("one length", cu_q=cu, cu_k=torch.tensor([0, 4, 9], dtype=torch.int32))
    refused("out must have", out=q[:3])
    refused("one of the inputs", out=q)
    same = _qkv(Tk=6, Hkv=4)
    refused("one of the inputs", *same, out=same[2])
    refused("inference only", q.requires_grad_(), k, v)
    with torch.no_grad():
        assert not A.attention(q, k, v).requires_grad


def test_norm_and_rotation_refuse_what_they_do_not_compute():
    q, k, _ = _qkv(5, 5)
    table = A.rotary_table(torch.arange(5), (16,))

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            A.qk_norm_rope(*(args or (q, k)), **kw)

    refused("q's tokens", q, k[:4])
    refused("nothing to do", norm=False)
    refused("need norm", norm=False, table=table, q_weight=torch.ones(16))
    refused("need k", q, k_weight=torch.ones(16))
    refused("norm weights must", q_weight=torch.ones(8))
    refused("norm weights must", q_weight=torch.ones(16, dtype=torch.float64))
    refused("one type", *(t.to(torch.bfloat16) for t in (q, k)), q_weight=torch.ones(16), k_weight=torch.ones(16).bfloat16())
    refused("eps", eps=-1.0)
    refused("eps", eps=math.nan)
    refused("table must be", table=table[:4])
    refused("table must be", table=table.double())
    refused("rotates", table=table[:, :2])
    refused("rotates", table=table[:, :4], interleaved=False)
    refused("rotates", q[..., :8], k[..., :8], table=table)
    refused("q_out must have", q_out=q[:2])
    refused("inference only", q, k, q_weight=torch.ones(16, requires_grad=True))


def test_rotary_table_refuses_what_it_does_not_compute():
    pos = torch.zeros(4, 2, dtype=torch.int32)
    for axes, kw in (((16,), {}), ((15, 16), {}), ((0, 16), {}), ((256, 16), {}), ((16, 16), {"theta": 0.0}),
                     ((16, 16), {"theta": math.inf}), ((16, 16), {"theta": (1.0,)})):
        with pytest.raises(ValueError):
            A.rotary_table(pos, axes, **kw)
    with pytest.raises(ValueError, match="positions must be int32"):
        A.rotary_table(pos.to(torch.int16), (16, 16))


def test_c_entries_refuse_bad_arguments_before_any_device_call(lib):  # noqa: F811
    L = lib.lib()
    p = ctypes.c_void_p(4096)
    base = dict(q=p, q_t=256, q_h=64, k=p, k_t=128, k_h=64, v=p, v_t=128, v_h=64, cu_q=None, cu_k=None, batch=1, Tq=8,
                Tk=8, Hq=4, Hkv=2, D=64, dtype=0, scale=0.125, causal=0, out=p, o_t=256, o_h=64, lse=None, ws=None,
                nbytes=0, stream=None)

    def attention(**kw):
        return L.convrot_attention(*{**base, **kw}.values())

    assert attention(Tq=-1) == attention(Hq=3) == attention(D=60) == attention(D=136) == attention(D=0) == lib.ERR_SHAPE
    assert attention(Hq=258) == attention(Hkv=0) == attention(batch=-1) == attention(q_t=0) == lib.ERR_SHAPE
    assert attention(dtype=2) == attention(scale=0.0) == attention(scale=math.inf) == lib.ERR_ARG
    assert attention(scale=math.nan) == attention(cu_q=p) == attention(batch=2) == lib.ERR_ARG
    assert attention(q=None) == attention(v=None) == attention(out=None) == lib.ERR_ARG
    assert attention(k_t=129) == attention(v_h=60) == attention(out=ctypes.c_void_p(4104)) == lib.ERR_ALIGN
    assert attention(lse=ctypes.c_void_p(4097)) == lib.ERR_ALIGN
    assert attention(o_h=32) == attention(o_t=128) == attention(o_t=8, o_h=8) == lib.ERR_SHAPE  # rows that overlap
    assert attention(Tq=0) == attention(batch=0, cu_q=p, cu_k=p) == lib.OK
    assert L.convrot_attention_workspace_size(8, 8, 1, 3, 2, 64) == -1
    assert L.convrot_attention_workspace_size(0, 8, 1, 4, 2, 64) == 0

    base2 = dict(q=p, q_t=256, q_h=64, qo=p, qo_t=256, qo_h=64, Hq=4, k=p, k_t=256, k_h=64, ko=p, ko_t=256, ko_h=64, Hk=4,
                 rows=8, D=64, dtype=0, norm=1, wq=None, wk=None, f32=0, eps=1e-6, table=p, ld=32, R=64, inter=1,
                 stream=None)

    def rope(**kw):
        return L.convrot_qk_norm_rope(*{**base2, **kw}.values())

    assert rope(D=60) == rope(D=264) == rope(Hq=0) == rope(Hk=-1) == rope(rows=-1) == lib.ERR_SHAPE
    assert rope(R=60) == rope(R=72) == rope(R=24, inter=0) == rope(ld=16) == lib.ERR_SHAPE
    assert rope(dtype=3) == rope(norm=0, table=None) == rope(norm=0, wq=p) == rope(eps=-1.0) == lib.ERR_ARG
    assert rope(q=None) == rope(ko=None) == rope(eps=math.nan) == lib.ERR_ARG
    assert rope(q_t=257) == rope(ko_h=4) == rope(ld=33) == rope(wq=ctypes.c_void_p(4100)) == lib.ERR_ALIGN
    assert rope(qo_h=0) == rope(ko_t=0) == rope(qo_t=128) == rope(ko_h=56) == lib.ERR_SHAPE  # rows that overlap
    assert rope(rows=0) == lib.OK

    def table(pos=p, kind=0, ld=2, rows=4, dims=(16, 16), theta=(1e4, 1e4), out=p):
        return L.convrot_rotary_table(pos, kind, ld, rows, len(dims), (ctypes.c_int * len(dims))(*dims),
                                      (ctypes.c_double * len(theta))(*theta), out, None)

    assert table(dims=(15, 16)) == table(dims=(256, 16)) == table(ld=1) == table(rows=-1) == lib.ERR_SHAPE
    assert table(kind=4) == table(theta=(1.0, 0.0)) == table(pos=None) == table(out=None) == lib.ERR_ARG
    assert table(dims=(2,) * 9, theta=(1.0,) * 9) == lib.ERR_SHAPE
    assert table(pos=ctypes.c_void_p(4098)) == table(kind=3, pos=ctypes.c_void_p(4100)) == lib.ERR_ALIGN
    assert table(rows=0) == lib.OK


def test_every_input_and_given_output_that_requires_grad_is_refused():
    q, k, v = _qkv(5, 5)
    table = A.rotary_table(torch.arange(5), (16,))
    wants = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda: A.attention(q, wants(k), v), lambda: A.attention(q, k, wants(v)), lambda: A.attention(q, k, v, out=wants(q)),
             lambda: A.qk_norm_rope(q, wants(k)), lambda: A.qk_norm_rope(q, k, table=wants(table)),
             lambda: A.qk_norm_rope(q, k, q_out=wants(q)), lambda: A.qk_norm_rope(q, k, k_out=wants(k)),
             lambda: A.rotary_table(wants(torch.arange(5.0)), (16,)), lambda: A.rotary_table(wants(torch.ones(5, 2)), (8, 8))]
    for call in calls:
        with pytest.raises(ValueError, match="inference only"):
            call()
        with torch.no_grad():
            call()


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad

    q, k, v = _qkv(5, 5)
    table = A.rotary_table(torch.arange(5), (16,))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: A.attention(dual(q), k, v), lambda: A.attention(q, k, dual(v)),
                     lambda: A.qk_norm_rope(q, dual(k)), lambda: A.qk_norm_rope(q, q_weight=dual(torch.ones(16))),
                     lambda: A.qk_norm_rope(q, table=dual(table)), lambda: A.rotary_table(dual(torch.arange(5.0)), (16,))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="tangent"):
                    call()
        A.attention(forward_ad.unpack_dual(dual(q)).primal, k, v)
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda t: A.attention(t, k, v), (q,), (torch.ones_like(q),))


# ------------------------------------------------------------------------------------------------ the compiled calls


def test_the_library_is_built_where_the_compiled_calls_cannot_be(tmp_path, monkeypatch):
    """The module of the compiled calls needs Python.h and torch's headers; the library does not, and comes first."""
    import subprocess

    from hyperflow_h3_flash_b200 import build

    made = []

    def run(cmd, check):
        made.append(os.path.basename(cmd[0]))
        if "-gencode" not in cmd:
            raise subprocess.CalledProcessError(1, cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass

    monkeypatch.setattr(build, "LIB", str(tmp_path / "libconvrot.so"))
    monkeypatch.setattr(build, "nvcc", lambda: "nvcc")
    monkeypatch.setattr(build.subprocess, "run", run)
    with pytest.warns(RuntimeWarning, match="compiled calls"):
        assert build.build(force=True) == build.LIB
    assert os.path.exists(build.LIB) and made == ["nvcc", os.path.basename(os.environ.get("CXX", "g++"))]


def test_compiled_calls_of_another_torch_or_python_are_not_taken(monkeypatch):
    """The module's file carries the versions that it was compiled for; without one of these the way through ctypes is
    taken, and a warning says so."""
    from hyperflow_h3_flash_b200 import build

    mine = build.fast_path()
    assert torch.__version__ in mine and os.path.dirname(mine) == build.HERE
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    assert build.fast_path() != mine and build.stale(build.fast_path(), [build.FAST_SOURCE])
    with pytest.warns(RuntimeWarning, match="compiled calls"):
        assert A._fast_calls.__wrapped__() is None


def test_a_compiled_module_that_cannot_be_loaded_is_not_taken(monkeypatch, tmp_path):
    from hyperflow_h3_flash_b200 import build

    broken = tmp_path / "_fast.so"
    broken.write_bytes(b"not a module")
    monkeypatch.setattr(build, "fast_path", lambda: str(broken))
    with pytest.warns(RuntimeWarning, match="compiled calls"):
        assert A._fast_calls.__wrapped__() is None


def test_rows_of_an_output_may_end_where_the_buffer_does(lib):  # noqa: F811
    """Outputs whose last row has no padding behind it do not overlap; one element less and they do.  (A misaligned
    pointer ends each call behind that check.)"""
    L = lib.lib()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4104 - 6)

    def attention(Tq, Hq, o_t, o_h):
        return L.convrot_attention(p, 256, 64, p, 128, 64, p, 128, 64, None, None, 1, Tq, 8, Hq, 2, 64, 0, 0.125, 0, p, o_t,
                                   o_h, odd, None, 0, None)

    def rope(T, H, qo_t, qo_h, ko_t, ko_h):
        return L.convrot_qk_norm_rope(p, 256, 64, p, qo_t, qo_h, H, p, 256, 64, p, ko_t, ko_h, H, T, 64, 0, 1, odd, None, 0,
                                      1e-6, None, 0, 0, 1, None)

    for a, b in ((3, 4), (2, 2), (7, 4), (8, 2)):
        for tight in (72, 640, 1 << 20):
            wide = (a - 1) * tight + 64
            assert attention(a, b, tight, wide) == lib.ERR_ALIGN  # heads first
            assert attention(a, b, tight, wide - 8) == lib.ERR_SHAPE
            assert rope(a, b, tight, wide, tight, wide + 8) == lib.ERR_ALIGN
            assert rope(a, b, tight, wide, tight, wide - 8) == rope(a, b, tight, wide - 8, tight, wide) == lib.ERR_SHAPE
            wide = (b - 1) * tight + 64
            assert attention(a, b, wide, tight) == lib.ERR_ALIGN  # tokens first
            assert attention(a, b, wide - 8, tight) == lib.ERR_SHAPE
    assert attention(1 << 29, 2, 1 << 37, 64) == lib.ERR_ALIGN and attention(1 << 29, 2, 1 << 37, 1 << 37) == lib.ERR_SHAPE


def test_a_scale_that_overflows_in_units_of_log2_is_refused(lib):  # noqa: F811
    """The kernel takes scores times scale * log2(e), which has to be finite in fp32.  (A misaligned pointer ends the calls
    with a good scale.)"""
    L = lib.lib()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)

    def attention(scale):
        return L.convrot_attention(p, 256, 64, p, 128, 64, p, 128, 64, None, None, 1, 8, 8, 4, 2, 64, 0, scale, 0, p, 256, 64,
                                   odd, None, 0, None)

    assert attention(2.3e38) == attention(1e-40) == attention(1.0) == lib.ERR_ALIGN
    assert attention(2.4e38) == attention(2.9e38) == attention(3.4e38) == lib.ERR_ARG


def test_outputs_of_the_norm_must_not_be_the_other_ones_memory_on_cpu_either():
    """As on the GPU: q's output over k's input (or both outputs in one place) would change what the other half reads."""
    q, k, _ = _qkv(5, 5, 4, 4)
    kept = k.clone()
    for kw in ({"q_out": k}, {"k_out": q}, {"q_out": q, "k_out": q}):
        with pytest.raises(ValueError, match="each other"):
            A.qk_norm_rope(q, k, **kw)
    with pytest.raises(ValueError, match="each other"):
        A.qk_norm_rope(q, q, q_out=q, k_out=q)
    assert torch.equal(k, kept)
    want = A.qk_norm_rope(q, k)
    got = A.qk_norm_rope(q, k, q_out=q, k_out=k)
    assert got[0] is q and got[1] is k and all(torch.equal(a, b) for a, b in zip(got, want))
