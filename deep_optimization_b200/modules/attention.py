"""The q/k/v split of a fused qkv projection with a one-pass backward.

`split_heads(qkv, heads)` returns what the reference's attention builds with view, permute and
index (Model/ViT/ViT.py:39-42): three [B, heads, T, head_dim] tensors, here strided views of the
projection's output (no copy).  Its backward hands the three gradients of the attention kernel to
`act_merge_heads`, which writes the gradient of the projection's output directly; autograd's own
route is a stack of the three followed by a strided copy of the result.

`RotaryAxes` is the split with rotary positions in it: q and k are turned by angles that grow with a
token's coordinates on one or several axes (height and width of an image, time of a video), in the pass
that lays the three tensors out, and their gradients are turned back in the pass that merges them.
`rotary_split` / `rotary_merge` are its two directions without autograd."""
from __future__ import annotations

import ctypes
import functools
import math

import torch
import torch.fx
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib
from ..codec import _DTYPES


def _merge_heads(grads, B, H, T, Dh, dtype, device):
    out = torch.empty((B, T, len(grads) * H * Dh), dtype=dtype, device=device)
    ptrs = (ctypes.c_void_p * len(grads))(*[g.data_ptr() for g in grads])
    strides = (ctypes.c_int64 * (3 * len(grads)))(*[s for g in grads for s in (g.stride(0), g.stride(1), g.stride(2))])
    with _lib.device_of(out):
        rc = _lib.load().act_merge_heads(ptrs, strides, len(grads), B, H, T, Dh, out.element_size(), out.data_ptr(),
                                         _lib.stream_ptr(out))
    _lib.check(rc, "act_merge_heads")
    return out


def _mergeable(g, Dh):
    es = g.element_size()
    return (g.stride(3) == 1 and g.data_ptr() % 16 == 0 and (Dh * es) % 16 == 0
            and all((g.stride(i) * es) % 16 == 0 for i in range(3)))


class _SplitHeads(Function):
    @staticmethod
    def forward(ctx, qkv, heads):
        B, T, D3 = qkv.shape
        Dh = D3 // (3 * heads)
        ctx.dims = (B, heads, T, Dh)
        return qkv.view(B, T, 3, heads, Dh).permute(2, 0, 3, 1, 4).unbind(0)

    @staticmethod
    def backward(ctx, dq, dk, dv):
        B, H, T, Dh = ctx.dims
        ref = next(g for g in (dq, dk, dv) if g is not None)
        grads = [g if g is not None else torch.zeros((B, H, T, Dh), dtype=ref.dtype, device=ref.device)
                 for g in (dq, dk, dv)]
        if all(g.dtype == ref.dtype for g in grads) and ref.element_size() in (2, 4) \
                and all(_mergeable(g, Dh) for g in grads):
            return _merge_heads(grads, B, H, T, Dh, ref.dtype, ref.device), None
        return torch.stack(grads, 0).permute(1, 3, 0, 2, 4).reshape(B, T, 3 * H * Dh), None


def split_heads(qkv: torch.Tensor, heads: int):
    """q, k, v of shape [B, heads, T, head_dim] from the [B, T, 3 * heads * head_dim] output of a fused
    projection, as views.  On a CUDA tensor that needs a gradient the backward is one gather pass.
    A model that is traced with torch.fx registers the name it imports this under with
    `torch.fx.wrap("split_heads")`, so that the trace keeps the call instead of its branches."""
    B, T, D3 = qkv.shape
    if qkv.is_cuda and qkv.requires_grad and qkv.is_contiguous():
        return _SplitHeads.apply(qkv, heads)
    return qkv.view(B, T, 3, heads, D3 // (3 * heads)).permute(2, 0, 3, 1, 4).unbind(0)


# ---------------------------------------------------------------- rotary positions

def rotary_turns(sections, base: float = 10000.0, device=None) -> torch.Tensor:
    """int64 [sum(sections)]: the frequencies base ** (-i / n), i < n, of an axis with n pairs, axis after
    axis, as 64-bit binary fractions of a turn per position.  Their products with integer positions keep
    the fraction of the turn however far the position."""
    if base < 1.0:
        raise ValueError(f"rotary_turns: base must be at least 1, got {base}")
    out = []
    for n in sections:
        out += [int(round(base ** (-i / n) / (2.0 * math.pi) * 2.0 ** 64)) for i in range(n)]
    return torch.tensor(out, dtype=torch.int64, device=device)


_I64x3, _I64x9 = ctypes.c_int64 * 3, ctypes.c_int64 * 9


@functools.lru_cache(maxsize=64)
def _sections_array(sections):
    """The C array of a tuple of pair counts, and their sum."""
    if not 1 <= len(sections) <= 4 or min(sections) < 0:
        raise ValueError(f"rotary: one to four sections of zero or more pairs, got {sections}")
    return (ctypes.c_int * len(sections))(*sections), sum(sections)


def _rotary_args(ref, B, T, Dh, positions, turns, sections):
    """Checks, and (pos pointer, bytes, three strides, turns pointer, sections, axes) for the library."""
    array, pairs = _sections_array(tuple(sections))
    axes = len(array)
    if 2 * pairs > Dh:
        raise ValueError(f"rotary: the sections' pairs {tuple(sections)} do not fit into a head of {Dh}")
    dev = ref.device
    if turns.dtype != torch.int64 or turns.numel() != pairs or turns.device != dev or not turns.is_contiguous():
        raise ValueError("rotary: turns must be a contiguous int64 tensor on the tensors' device with one entry per pair")
    es = 8 if positions.dtype == torch.int64 else 4
    if (es == 4 and positions.dtype != torch.int32) or positions.device != dev:
        raise TypeError("rotary: positions must be int32 or int64 on the tensors' device")
    shape = positions.shape
    if shape == (T, axes):
        st, sa = positions.stride()
        sb = 0
    elif shape == (B, T, axes):
        sb, st, sa = positions.stride()
    else:
        raise ValueError(f"rotary: positions must be [T, axes] or [B, T, axes] = [{B}, {T}, {axes}], got {tuple(shape)}")
    return positions.data_ptr(), es, sb, st, sa, turns.data_ptr(), array, axes


def _split_views(qkv, heads, kv_heads, Dh):
    x = qkv.view(qkv.shape[0], qkv.shape[1], heads + 2 * kv_heads, Dh).transpose(1, 2)
    return x.split((heads, kv_heads, kv_heads), 1)


def _dtype_code(t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"unsupported activation dtype {t.dtype}")
    return code


def rotary_split(qkv: torch.Tensor, heads: int, positions: torch.Tensor, turns: torch.Tensor, sections,
                 kv_heads=None, interleaved: bool = False):
    """q [B, heads, T, Dh] and k, v [B, kv_heads, T, Dh] from a fused projection's output
    [B, T, (heads + 2 kv_heads) Dh], q and k turned; the three are views of one new buffer of qkv's
    layout, so that qkv itself is not kept alive by them.  positions: int32 or int64 [T, axes] or
    [B, T, axes], any values; turns: `rotary_turns(sections)`; sections: pairs per axis.  Pairs are
    (j, P + j) in a head, or (2 j, 2 j + 1) if `interleaved`; elements behind the pairs are copied."""
    if not qkv.is_cuda:
        raise RuntimeError("rotary_split needs a CUDA tensor: there is no CPU path")
    kv_heads = heads if kv_heads is None else kv_heads
    if heads < 1 or kv_heads < 1 or qkv.dim() != 3 or qkv.shape[2] % (heads + 2 * kv_heads) or qkv.shape[2] == 0:
        raise ValueError("rotary_split: qkv must be [B, T, (heads + 2 * kv_heads) * Dh]")
    qkv = qkv.contiguous()
    B, T, W = qkv.shape
    Dh = W // (heads + 2 * kv_heads)
    pos, es, sb, st, sa, tp, array, axes = _rotary_args(qkv, B, T, Dh, positions, turns, sections)
    out = torch.empty_like(qkv)
    with _lib.device_of(qkv):
        rc = _lib.load().act_rotary_split(qkv.data_ptr(), out.data_ptr(), heads, kv_heads, _dtype_code(qkv), B, T, Dh, pos, es,
                                          sb, st, sa, tp, array, axes, int(interleaved), _lib.stream_ptr(qkv))
    _lib.check(rc, "act_rotary_split")
    return tuple(_split_views(out, heads, kv_heads, Dh))


def rotary_merge(dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, positions: torch.Tensor, turns: torch.Tensor,
                 sections, interleaved: bool = False) -> torch.Tensor:
    """The gradient of `rotary_split`'s qkv from the gradients of its q, k and v (any strides): dq and dk
    turned back, the three merged, one pass."""
    if not dq.is_cuda:
        raise RuntimeError("rotary_merge needs CUDA tensors: there is no CPU path")
    B, H, T, Dh = dq.shape
    K = dk.shape[1]
    if dk.shape != (B, K, T, Dh) or dv.shape != dk.shape or dk.dtype != dq.dtype or dv.dtype != dq.dtype \
            or dk.device != dq.device or dv.device != dq.device:
        raise ValueError("rotary_merge: dq [B, heads, T, Dh] and dk, dv [B, kv_heads, T, Dh] of one type and device")
    pos, es, sb, st, sa, tp, array, axes = _rotary_args(dq, B, T, Dh, positions, turns, sections)
    (q0, q1, q2, q3), (k0, k1, k2, k3), (v0, v1, v2, v3) = dq.stride(), dk.stride(), dv.stride()
    if not q3 == k3 == v3 == 1:
        dq, dk, dv = dq.contiguous(), dk.contiguous(), dv.contiguous()
        (q0, q1, q2, _), (k0, k1, k2, _), (v0, v1, v2, _) = dq.stride(), dk.stride(), dv.stride()
    out = torch.empty((B, T, (H + 2 * K) * Dh), dtype=dq.dtype, device=dq.device)
    with _lib.device_of(dq):
        rc = _lib.load().act_rotary_merge(dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                          _I64x9(q0, q1, q2, k0, k1, k2, v0, v1, v2), out.data_ptr(), H, K, _dtype_code(dq),
                                          B, T, Dh, pos, es, sb, st, sa, tp, array, axes, int(interleaved),
                                          _lib.stream_ptr(dq))
    _lib.check(rc, "act_rotary_merge")
    return out


def rotary_heads(x: torch.Tensor, positions: torch.Tensor, turns: torch.Tensor, sections, interleaved: bool = False,
                 inverse: bool = False) -> torch.Tensor:
    """One [B, heads, T, Dh] tensor (any strides) turned, or turned back; the result is contiguous."""
    if not x.is_cuda:
        raise RuntimeError("rotary_heads needs a CUDA tensor: there is no CPU path")
    if x.dim() != 4:
        raise ValueError("rotary_heads: x must be [B, heads, T, Dh]")
    if x.stride(3) != 1:
        x = x.contiguous()
    B, H, T, Dh = x.shape
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return out
    pos, es, sb, st, sa, tp, array, axes = _rotary_args(x, B, T, Dh, positions, turns, sections)
    one = ctypes.c_int * 1
    with _lib.device_of(x):
        rc = _lib.load().act_rotary_heads(
            (ctypes.c_void_p * 1)(x.data_ptr()), _I64x3(*x.stride()[:3]), (ctypes.c_void_p * 1)(out.data_ptr()),
            _I64x3(*out.stride()[:3]), one(H), one(1), 1, _dtype_code(x), B, T, Dh, pos, es, _I64x3(sb, st, sa), tp, array,
            axes, int(interleaved), int(inverse), _lib.stream_ptr(x))
    _lib.check(rc, "act_rotary_heads")
    return out


class _RotarySplit(Function):
    @staticmethod
    def forward(ctx, qkv, heads, positions, turns, sections, kv_heads, interleaved):
        ctx.save_for_backward(positions, turns)
        ctx.how = (sections, interleaved)
        ctx.set_materialize_grads(False)
        q, k, v = rotary_split(qkv, heads, positions, turns, sections, kv_heads, interleaved)
        ctx.like = (q.shape, k.shape)
        return q, k, v

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk, dv):
        positions, turns = ctx.saved_tensors
        sections, interleaved = ctx.how
        ref = next((g for g in (dq, dk, dv) if g is not None), None)
        if ref is None:
            return (None,) * 7
        grads = [torch.zeros(s, dtype=ref.dtype, device=ref.device) if g is None else g.to(ref.dtype)
                 for g, s in ((dq, ctx.like[0]), (dk, ctx.like[1]), (dv, ctx.like[1]))]
        return rotary_merge(*grads, positions, turns, sections, interleaved), None, None, None, None, None, None


class _RotaryHeads(Function):
    @staticmethod
    def forward(ctx, x, positions, turns, sections, interleaved):
        ctx.save_for_backward(positions, turns)
        ctx.how = (sections, interleaved)
        return rotary_heads(x, positions, turns, sections, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        positions, turns = ctx.saved_tensors
        sections, interleaved = ctx.how
        return rotary_heads(dy, positions, turns, sections, interleaved, inverse=True), None, None, None, None


def rotary_split_heads(qkv, heads, positions, turns, sections, kv_heads=None, interleaved=False):
    """`rotary_split` that differentiates (once) with respect to qkv.  Tensors on the meta device get the
    results' shapes, which is what shape propagation asks for."""
    if qkv.is_meta:
        K = heads if kv_heads is None else kv_heads
        return tuple(_split_views(qkv, heads, K, qkv.shape[2] // (heads + 2 * K)))
    return _RotarySplit.apply(qkv, heads, positions, turns, sections, kv_heads, interleaved)


def rotary_turn_heads(x, positions, turns, sections, interleaved=False):
    """`rotary_heads` that differentiates (once) with respect to x."""
    if x.is_meta:
        return torch.empty_like(x)
    return _RotaryHeads.apply(x, positions, turns, sections, interleaved)


# leaves for torch.fx: a trace keeps the calls that RotaryAxes makes, not their branches
torch.fx.wrap("rotary_split_heads")
torch.fx.wrap("rotary_turn_heads")


class RotaryAxes(nn.Module):
    """Rotary positions with one to four axes.  `sections` are the pairs of a head that each axis turns
    (their sum at most half the head); `base` sets the frequencies base ** (-i / n).

    `forward(qkv, heads, positions, kv_heads=None)` splits a fused projection's output as `split_heads`
    does, q and k turned; `turn(x, positions)` turns one [B, heads, T, Dh] tensor.  Both differentiate
    (once) with respect to their tensor.  positions: integers, [T, axes] or [B, T, axes]; a token at the
    origin, such as a class token, is not turned."""

    def __init__(self, sections, base: float = 10000.0, interleaved: bool = False):
        super().__init__()
        self.sections, self.base, self.interleaved = tuple(int(n) for n in sections), float(base), bool(interleaved)
        self.register_buffer("turns", rotary_turns(self.sections, self.base))

    def forward(self, qkv, heads, positions, kv_heads=None):
        return rotary_split_heads(qkv, heads, positions, self.turns, self.sections, kv_heads, self.interleaved)

    def turn(self, x, positions):
        return rotary_turn_heads(x, positions, self.turns, self.sections, self.interleaved)


def image_positions(height: int, width: int, leading: int = 1, device=None) -> torch.Tensor:
    """int64 [leading + height * width, 2]: the row and column, counted from 1, of the patches of an image
    in row-major order, behind `leading` tokens at the origin (a class token)."""
    y, x = torch.meshgrid(torch.arange(1, height + 1), torch.arange(1, width + 1), indexing="ij")
    grid = torch.stack([y.reshape(-1), x.reshape(-1)], -1)
    return torch.cat([torch.zeros(leading, 2, dtype=torch.int64), grid]).to(device)
