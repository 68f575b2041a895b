"""What an attention block computes between its q / k / v and out projections, on B200 (sm_100a).

The reference leaves these steps to diffusers (called from chunk_block, src/hyperflow_h3_flash/transformer.py:350-358);
``ulysses.attention_block_linears`` takes them as its ``attention`` callable.  Here:

* ``rotary_table``: (cos, sin) of a rotation with several position axes (time, height, width of a latent video);
* ``qk_norm_rope``: the per-head RMS norm of q and k and their rotation, one pass over both;
* ``attention``: softmax attention over sequences packed behind each other, grouped heads, causal or not;
* ``QKNormAttention``: the three joined, with the norms' weights: the callable for ``attention_block_linears``.

The layout is ``[tokens, heads, head_dim]``, bf16 or fp16, with any token and head strides that are positive multiples of
8 elements (slices of a fused projection go in as they are; heads that ``expand`` repeats do not: give them once, as
grouped heads).  Sequences of a batch are packed along the tokens with int32 offsets on the device (``cu_q``, ``cu_k``:
``[batch + 1]``), which are read on the GPU only: no call synchronises.

CUDA tensors run the kernels of ``libconvrot.so``; there is no other path on CUDA.  CPU tensors take plain torch
operations in fp32, as the package's layers do.  Inference only, like the layers around them: an input or a given output
that requires grad is refused while grad mode is on, and one with a forward-mode tangent always.
"""

from __future__ import annotations

import ctypes
import functools
import importlib.util
import math
import numbers
import warnings
from collections.abc import Sequence

import torch
from torch import Tensor, nn
from torch.autograd import forward_ad

from . import _lib, build
from .int8 import _written

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}
MAX_HEAD_DIM = 128  # of attention; qk_norm_rope takes heads up to 256


@functools.cache
def _fast_calls():
    """The compiled form of the common calls (csrc/fast_call.cpp), or None if it was not built for this Python and torch:
    it calls the same C entries, and answers None to every call that is not plainly in order, which then takes the way
    below."""
    path = build.fast_path()
    try:
        spec = importlib.util.spec_from_file_location(f"{__package__}._fast", path)
        fast = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(fast)
    except ImportError as e:
        warnings.warn(f"attention operators without their compiled calls ({e}): short calls take about 10 us longer; build "
                      f"with `python -m {__package__}.build`", RuntimeWarning, stacklevel=3)
        return None
    handle = _lib.lib()
    names = ("rotary_table", "qk_norm_rope", "attention", "attention_workspace_size")
    fast.init(*(ctypes.cast(getattr(handle, f"convrot_{name}"), ctypes.c_void_p).value for name in names))
    return fast


def _no_grad(*tensors: Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("attention operators are inference only: use torch.no_grad() or detach the inputs")
    if forward_ad._current_level >= 0:  # within a dual_level (no_grad() leaves forward mode on)
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("attention operators are inference only: a forward-mode tangent would be lost")


def _call(entry, device: torch.device, *args):
    """One library call on the tensors' device and its current stream."""
    # (the raw stream: a torch.cuda.Stream object takes as long to make as the launch)
    index = device.index
    if index == torch._C._cuda_getDevice():
        return entry(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(device):
        return entry(*args, torch._C._cuda_getCurrentRawStream(index))


def _heads(t: Tensor, name: str, like: Tensor | None = None) -> tuple[torch.Size, tuple[int, ...]]:
    """Shape and strides of a [tokens, heads, head_dim] tensor, of the type and device of ``like``."""
    shape, strides = t.shape, t.stride()
    if len(shape) != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got shape {tuple(shape)}")
    if like is None:
        if t.dtype not in _DTYPES and t.is_cuda:
            raise ValueError(f"{name} must be bfloat16 or float16, got {t.dtype}")
    elif t.dtype is not like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    if strides[2] != 1 and shape[2] != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return shape, strides


def _output(out: Tensor | None, x: Tensor, name: str) -> Tensor:
    if out is None:
        if x.is_contiguous():
            return torch.empty_like(x)
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    if _heads(out, name, x)[0] != x.shape:
        raise ValueError(f"{name} must have shape {tuple(x.shape)}, got {tuple(out.shape)}")
    return out


# ------------------------------------------------------------------------------------------------ positions


@functools.lru_cache(maxsize=64)
def _host_arrays(axes: tuple[int, ...], thetas: tuple[float, ...]):
    return (ctypes.c_int * len(axes))(*axes), (ctypes.c_double * len(thetas))(*thetas)


def rotary_table(positions: Tensor, axes: Sequence[int], *, theta: float | Sequence[float] = 10000.0) -> Tensor:
    """(cos, sin) of a rotation over several position axes, fp32 ``[T, R / 2, 2]`` with ``R = sum(axes)``.

    ``positions`` is ``[T, len(axes)]`` (``[T]`` for one axis) of int32, int64, float32 or float64, fractional ones
    included; axis ``a`` turns ``axes[a] / 2`` pairs of channels, pair ``i`` by ``pos * theta[a] ** (-2 i / axes[a])``.
    Angles are formed and reduced in fp64, so far positions lose nothing.  Made once per clip and shared by every block:
    ``qk_norm_rope(table=...)`` reads it."""
    if positions.is_cuda and (fast := _fast_calls()) is not None:
        table = fast.rotary_table(positions, axes, theta)
        if table is not None:
            return table
    _no_grad(positions)
    axes = tuple(int(d) for d in axes)
    if not 1 <= len(axes) <= 8 or any(d <= 0 or d % 2 for d in axes) or sum(axes) > 256:
        raise ValueError(f"axes must be 1 to 8 even positive widths of at most 256 channels in all, got {axes}")
    thetas = [float(theta)] * len(axes) if isinstance(theta, numbers.Real) else [float(v) for v in theta]
    if len(thetas) != len(axes) or any(not (v > 0 and math.isfinite(v)) for v in thetas):
        raise ValueError(f"theta must be positive, one value or one per axis, got {theta!r}")
    if positions.dim() == 1:
        positions = positions[:, None]
    if positions.dim() != 2 or positions.shape[1] != len(axes):
        raise ValueError(f"positions must be [T, {len(axes)}], got shape {tuple(positions.shape)}")
    if positions.dtype not in _POSITIONS:
        raise ValueError(f"positions must be int32, int64, float32 or float64, got {positions.dtype}")
    T, R = positions.shape[0], sum(axes)
    if not positions.is_cuda:
        parts = []
        for a, (d, base) in enumerate(zip(axes, thetas)):
            freq = base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
            parts.append(positions[:, a : a + 1].double() * freq)
        angle = torch.cat(parts, dim=1)
        return torch.stack([angle.cos(), angle.sin()], dim=-1).float()
    if positions.stride(1) != 1 and len(axes) > 1 or positions.stride(0) < len(axes):
        positions = positions.contiguous()
    out = torch.empty(T, R // 2, 2, dtype=torch.float32, device=positions.device)
    rc = _call(_lib.lib().convrot_rotary_table, positions.device, positions.data_ptr(), _POSITIONS[positions.dtype],
               max(positions.stride(0), len(axes)), T, len(axes), *_host_arrays(axes, tuple(thetas)), out.data_ptr())
    if rc:
        _lib.check(rc, "convrot_rotary_table")
    return out


# ------------------------------------------------------------------------------------------------ norm and rotation


def _norm_rope_torch(x: Tensor, weight: Tensor | None, eps: float, norm: bool, table: Tensor | None,
                     interleaved: bool) -> Tensor:
    y = x.float()
    if norm:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.float()
    if table is not None:
        half = table.shape[1]
        c, s = table[:, None, :, 0], table[:, None, :, 1]
        part = y[..., : 2 * half]
        if interleaved:
            a, b = part[..., 0::2], part[..., 1::2]
            turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
        else:
            a, b = part[..., :half], part[..., half:]
            turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
        y = torch.cat([turned, y[..., 2 * half :]], dim=-1)
    return y.to(x.dtype)


def _weight(w: Tensor, D: int, q: Tensor) -> bool:
    """Whether a norm weight is fp32 (else it is of q's type)."""
    f32 = w.dtype is torch.float32
    if w.shape != (D,) or not (f32 or w.dtype is q.dtype) or w.device != q.device or not w.is_contiguous():
        raise ValueError(f"norm weights must be contiguous [{D}] of {q.dtype} or float32 on {q.device}")
    return f32


def qk_norm_rope(q: Tensor, k: Tensor | None = None, *, q_weight: Tensor | None = None, k_weight: Tensor | None = None,
                 eps: float = 1e-6, norm: bool = True, table: Tensor | None = None, interleaved: bool = True,
                 q_out: Tensor | None = None, k_out: Tensor | None = None) -> Tensor | tuple[Tensor, Tensor]:
    """The per-head RMS norm of q ``[T, Hq, D]`` and k ``[T, Hk, D]`` and their rotation, in one pass over both.

    ``y = x * rsqrt(mean(x^2) + eps) * weight`` over each head's D channels (``norm=False`` leaves it out; weights ``[D]``
    in the inputs' type or fp32, or None), then the first ``R = 2 * table.shape[1]`` channels are rotated by ``table``
    (``rotary_table``'s, fp32 ``[T, R / 2, 2]``; None: no rotation): pairs of neighbours if ``interleaved``, else
    ``(j, j + R / 2)``.  fp32 arithmetic, one rounding.  Returns the new q (and k when given).  ``q_out`` / ``k_out`` may
    be the inputs themselves; an output that overlaps an input in any other way is not supported."""
    if q.is_cuda and (fast := _fast_calls()) is not None:
        made = fast.qk_norm_rope(q, k, q_weight, k_weight, eps, norm, table, interleaved, q_out, k_out)
        if made is not None:
            return made
    _no_grad(q, k, q_weight, k_weight, table, q_out, k_out)
    (T, Hq, D), qs = _heads(q, "q")
    if k is not None:
        k_shape, ks = _heads(k, "k", q)
        if k_shape[0] != T or k_shape[2] != D:
            raise ValueError(f"k must have q's tokens and head_dim, got {tuple(k_shape)} beside {tuple(q.shape)}")
    elif k_weight is not None or k_out is not None:
        raise ValueError("k_weight and k_out need k")
    f32 = None
    if q_weight is not None:
        f32 = _weight(q_weight, D, q)
    if k_weight is not None:
        k_f32 = _weight(k_weight, D, q)
        if f32 is not None and f32 != k_f32:
            raise ValueError("q_weight and k_weight must have one type")
        f32 = k_f32
    if not norm:
        if table is None:
            raise ValueError("nothing to do: norm=False and no table")
        if f32 is not None:
            raise ValueError("norm weights need norm=True")
    eps, norm, interleaved = float(eps), bool(norm), bool(interleaved)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    R = 0
    if table is not None:
        shape = table.shape
        if len(shape) != 3 or shape[0] != T or shape[2] != 2 or table.dtype is not torch.float32 or \
                table.device != q.device:
            raise ValueError(f"table must be float32 [{T}, R / 2, 2] on {q.device}, got {table.dtype} {tuple(shape)} on "
                             f"{table.device}")
        R = 2 * shape[1]
        if R > D or R % (8 if interleaved else 16) or R == 0:
            raise ValueError(f"the table rotates {R} channels: must be a multiple of {8 if interleaved else 16} up to "
                             f"head_dim {D}")
        if not table.is_contiguous():
            table = table.contiguous()
    if q.is_cuda and (D % 8 or not 8 <= D <= 256):
        raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {D}")
    if q.is_cuda and (Hq == 0 or (k is not None and k_shape[1] == 0)):
        raise ValueError("q and k need at least one head")
    qo, ko = _output(q_out, q, "q_out"), None if k is None else _output(k_out, k, "k_out")
    if q.is_cuda or q_out is not None or k_out is not None:
        qos, q_ptr, qo_ptr = qo.stride(), q.data_ptr(), qo.data_ptr()
        kk = (None, 0, 0, None, 0, 0, 0)
        if k is not None:
            kos, k_ptr, ko_ptr = ko.stride(), k.data_ptr(), ko.data_ptr()
            if (qo_ptr == k_ptr or qo_ptr == ko_ptr or ko_ptr == q_ptr) and qo.numel() and ko.numel():
                raise ValueError("q_out and k_out must not be the other's input or each other")
            kk = (k_ptr, ks[0], ks[1], ko_ptr, kos[0], kos[1], k_shape[1])
    if not q.is_cuda:
        qo.copy_(_norm_rope_torch(q, q_weight, eps, norm, table, interleaved))
        if k is None:
            return qo
        return qo, ko.copy_(_norm_rope_torch(k, k_weight, eps, norm, table, interleaved))
    rc = _call(_lib.lib().convrot_qk_norm_rope, q.device, q_ptr, qs[0], qs[1], qo_ptr, qos[0], qos[1], Hq, *kk, T, D,
               _DTYPES[q.dtype], norm, None if q_weight is None else q_weight.data_ptr(),
               None if k_weight is None else k_weight.data_ptr(), f32 is True, eps,
               None if table is None else table.data_ptr(), R // 2, R, interleaved)
    if rc:
        _lib.check(rc, "convrot_qk_norm_rope")
    _written(q_out, k_out)
    return qo if k is None else (qo, ko)


# ------------------------------------------------------------------------------------------------ attention


def _attention_torch(q: Tensor, k: Tensor, v: Tensor, cu_q: Tensor | None, cu_k: Tensor | None, causal: bool,
                     scale: float, out: Tensor, lse: Tensor | None) -> None:
    bq = [0, q.shape[0]] if cu_q is None else cu_q.tolist()
    bk = [0, k.shape[0]] if cu_k is None else cu_k.tolist()
    group = q.shape[1] // k.shape[1]
    for (q0, q1), (k0, k1) in zip(zip(bq, bq[1:]), zip(bk, bk[1:])):
        kf = k[k0:k1].float().repeat_interleave(group, dim=1).transpose(0, 1)
        vf = v[k0:k1].float().repeat_interleave(group, dim=1).transpose(0, 1)
        s = q[q0:q1].float().transpose(0, 1) @ kf.transpose(1, 2) * scale
        if causal:
            seen = torch.arange(k1 - k0) <= torch.arange(q1 - q0)[:, None] + (k1 - k0) - (q1 - q0)
            s = s.masked_fill(~seen, -math.inf)
        z = torch.logsumexp(s, dim=-1) if k1 > k0 else s.new_full(s.shape[:2], -math.inf)
        w = torch.exp(s - torch.where(z == -math.inf, 0.0, z)[..., None])
        o = w @ vf
        if causal and not vf.isfinite().all():  # a weight of zero does not keep a NaN or an infinity out of a product
            o = w @ vf.nan_to_num(0.0, 0.0, 0.0)
            for key in (~vf.isfinite()).any(2).any(0).nonzero().flatten().tolist():
                value = torch.where(vf[:, key].isfinite(), 0.0, vf[:, key])
                o += torch.where(seen[:, key, None], value[:, None], 0.0)
        out[q0:q1] = o.transpose(0, 1).to(q.dtype)
        if lse is not None:
            lse[q0:q1] = z.transpose(0, 1)


def attention(q: Tensor, k: Tensor, v: Tensor, *, cu_q: Tensor | None = None, cu_k: Tensor | None = None,
              causal: bool = False, scale: float | None = None, out: Tensor | None = None,
              return_lse: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """``softmax(scale q k^T + mask) v`` for q ``[Tq, Hq, D]``, k and v ``[Tk, Hkv, D]``; returns ``[Tq, Hq, D]``.

    * Query head ``h`` reads key head ``h // (Hq // Hkv)``.  D is a multiple of 8 up to 128; ``scale`` is ``D ** -0.5`` by
      default.
    * ``cu_q`` / ``cu_k`` (int32 ``[batch + 1]``, non-decreasing, on the device): sequence b is rows ``cu_q[b]:cu_q[b + 1]``
      of q and ``cu_k[b]:cu_k[b + 1]`` of k and v; None: one sequence.  Rows of no sequence (padding behind the last one)
      are not written: they keep what ``out`` held.
    * A cache with room to grow: its rows that are not filled yet are a sequence without a query (``cu_q`` repeats its
      offset, ``cu_k`` spans them); what they hold reaches no row.  With m caches of ``room`` rows and n[i] filled,
      ``cu_k`` is ``[0, n[0], room, room + n[1], 2 * room, ...]`` and ``cu_q`` ``[0, 1, 1, 2, 2, ...]`` for a token each.
    * ``causal``: query i of lq sees the keys up to ``i + lk - lq`` (the last query sees all of them), so a prompt, a
      chunk behind a cache and a single new token are the same call.
    * A query that sees no key gives zeros (and ``-inf`` in the log-sum-exp).
    * ``return_lse`` adds the natural log-sum-exp of each row's scores, fp32 ``[Tq, Hq]``.

    ``out`` must not overlap the inputs, nor its rows each other.  Scores, statistics and sums are fp32; the weights are
    rounded to the inputs' type for their product with v.  Few queries over long keys are split over the GPU and joined
    in a fixed order: results do not vary from run to run."""
    if q.is_cuda and (fast := _fast_calls()) is not None:
        made = fast.attention(q, k, v, cu_q, cu_k, causal, scale, return_lse, out)
        if made is not None:
            return made
    _no_grad(q, k, v, out)
    (Tq, Hq, D), qs = _heads(q, "q")
    (Tk, Hkv, Dk), ks = _heads(k, "k", q)
    v_shape, vs = _heads(v, "v", q)
    if Dk != D or v_shape != k.shape:
        raise ValueError(f"k and v must be [Tk, Hkv, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if Hkv == 0 or Hq == 0 or Hq % Hkv or Hq // Hkv > 128:
        raise ValueError(f"{Hq} query heads cannot share {Hkv} key heads (at most 128 each)")
    if D % 8 or not 8 <= D <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}, got {D}")
    causal, scale = bool(causal), D**-0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    batch = 1
    if (cu_q is None) != (cu_k is None):
        raise ValueError("cu_q and cu_k come together")
    if cu_q is not None:
        for name, cu in (("cu_q", cu_q), ("cu_k", cu_k)):
            if cu.dtype != torch.int32 or cu.dim() != 1 or cu.shape[0] < 1 or cu.device != q.device or \
                    not cu.is_contiguous():
                raise ValueError(f"{name} must be contiguous int32 [batch + 1] on {q.device}")
        if cu_q.shape != cu_k.shape:
            raise ValueError(f"cu_q and cu_k must have one length, got {cu_q.shape[0]} and {cu_k.shape[0]}")
        batch = cu_q.shape[0] - 1
    given, out = out, _output(out, q, "out")
    if Tq and out.data_ptr() in (q.data_ptr(), k.data_ptr(), v.data_ptr()):
        raise ValueError("out must not be one of the inputs")
    lse = torch.empty(Tq, Hq, dtype=torch.float32, device=q.device) if return_lse else None
    if not q.is_cuda:
        _attention_torch(q, k, v, cu_q, cu_k, causal, scale, out, lse)
        return out if lse is None else (out, lse)
    handle, device = _lib.lib(), q.device
    if device.index == torch._C._cuda_getDevice():
        size = handle.convrot_attention_workspace_size(Tq, Tk, batch, Hq, Hkv, D)
    else:
        with torch.cuda.device(device):
            size = handle.convrot_attention_workspace_size(Tq, Tk, batch, Hq, Hkv, D)
    if size < 0:
        raise ValueError(f"attention does not take {Tq} queries and {Tk} keys in {batch} sequences of {Hq} heads")
    # from torch's stream-ordered allocator: freed at return, reused only by later work of this stream (or graph)
    space = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    os = out.stride()
    rc = _call(handle.convrot_attention, device, q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(),
               vs[0], vs[1], None if cu_q is None else cu_q.data_ptr(), None if cu_k is None else cu_k.data_ptr(), batch,
               Tq, Tk, Hq, Hkv, D, _DTYPES[q.dtype], scale, causal, out.data_ptr(), os[0], os[1],
               None if lse is None else lse.data_ptr(), None if space is None else space.data_ptr(), size)
    if rc:
        _lib.check(rc, "convrot_attention")
    _written(given)
    return out if lse is None else (out, lse)


# ------------------------------------------------------------------------------------------------ joined


class QKNormAttention(nn.Module):
    """Per-head q / k norms, rotation and attention: the ``attention`` callable of ``ulysses.attention_block_linears``.

    ``norm_q.weight`` / ``norm_k.weight`` (``[head_dim]``, frozen) as a checkpoint's per-head norms name them.  The
    positions of the next calls are set with ``set_sequences(table, cu)``: the rotary table of every token (after the
    exchange a rank holds all tokens of its heads) and the packed sequences' offsets, both kept for all blocks of a
    forward pass.  q and k are normalised and rotated in place."""

    def __init__(self, head_dim: int, *, eps: float = 1e-6, interleaved: bool = True, causal: bool = False,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.head_dim, self.eps, self.interleaved, self.causal = head_dim, eps, interleaved, causal
        self.norm_q, self.norm_k = nn.Module(), nn.Module()
        for norm in (self.norm_q, self.norm_k):
            norm.weight = nn.Parameter(torch.ones(head_dim, dtype=dtype), requires_grad=False)
        self.table: Tensor | None = None
        self.cu: Tensor | None = None

    def set_sequences(self, table: Tensor | None, cu: Tensor | None = None) -> None:
        self.table, self.cu = table, cu

    def forward(self, q: Tensor, k: Tensor, v: Tensor) -> Tensor:
        q, k = qk_norm_rope(q, k, q_weight=self.norm_q.weight, k_weight=self.norm_k.weight, eps=self.eps,
                            table=self.table, interleaved=self.interleaved, q_out=q, k_out=k)
        return attention(q, k, v, cu_q=self.cu, cu_k=self.cu, causal=self.causal)


__all__ = ["MAX_HEAD_DIM", "QKNormAttention", "attention", "qk_norm_rope", "rotary_table"]
