"""FP8 e4m3 GEMM with per-row / per-column scales (tcgen05 kernel behind the C ABI).

`fp8_gemm(A8, B8, sa, sb)` computes bf16((A8 @ B8) * sa[:,None] * sb[None,:]) for
A8 [M,K] and B8 [K,N] (the operand layout of the reference's Triton_Linear,
Activation_Compression/triton_kernel/linear.py:43-95) or, with `b_is_nk=True`,
B8 given as [N,K] like an nn.Linear weight.  `quantize_e4m3` produces the
operands and scales the way the evaluation configuration describes (amax / 448).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

E4M3_MAX = 448.0


def quantize_e4m3(x: torch.Tensor, dim: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Scale each slice along `dim` to the e4m3 range; returns (fp8 tensor, fp32 scales)."""
    amax = x.abs().amax(dim=dim, keepdim=True).float().clamp_min(1e-12)
    scale = amax / E4M3_MAX
    q = (x.float() / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q, scale.squeeze(dim).contiguous()


def workspace_bytes(M: int, N: int, K: int, b_is_nk: bool) -> int:
    return int(_lib.load().act_fp8_gemm_workspace(M, N, K, _lib.ACT_GEMM_B_IS_NK if b_is_nk else 0))


def fp8_gemm(A8: torch.Tensor, B8: torch.Tensor, sa: torch.Tensor, sb: torch.Tensor,
             b_is_nk: bool = False, out: Optional[torch.Tensor] = None,
             workspace: Optional[torch.Tensor] = None, single_cta: bool = False) -> torch.Tensor:
    if not A8.is_cuda:
        raise RuntimeError("fp8_gemm needs CUDA tensors: there is no CPU path")
    if A8.dtype != torch.float8_e4m3fn or B8.dtype != torch.float8_e4m3fn:
        raise TypeError("operands must be torch.float8_e4m3fn")
    A8, B8 = A8.contiguous(), B8.contiguous()
    M, K = A8.shape
    N = B8.shape[0] if b_is_nk else B8.shape[1]
    if (B8.shape[1] if b_is_nk else B8.shape[0]) != K:
        raise ValueError("inner dimensions differ")
    sa = sa.to(torch.float32).contiguous()
    sb = sb.to(torch.float32).contiguous()
    if sa.numel() != M or sb.numel() != N:
        raise ValueError("sa must have M entries and sb N entries")
    C = out if out is not None else torch.empty((M, N), dtype=torch.bfloat16, device=A8.device)
    flags = (_lib.ACT_GEMM_B_IS_NK if b_is_nk else 0) | (_lib.ACT_GEMM_SINGLE_CTA if single_cta else 0)
    need = workspace_bytes(M, N, K, b_is_nk)
    ws_ptr, ws_len = None, 0
    if need:
        if workspace is None or workspace.numel() * workspace.element_size() < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=A8.device)
        ws_ptr, ws_len = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    with _lib.device_of(A8):
        rc = _lib.load().act_fp8_gemm(A8.data_ptr(), B8.data_ptr(), sa.data_ptr(), sb.data_ptr(), C.data_ptr(),
                                      M, N, K, A8.stride(0), B8.stride(0), C.stride(0), flags, ws_ptr, ws_len,
                                      _lib.stream_ptr(A8))
    _lib.check(rc, "act_fp8_gemm")
    return C


def gemm_status(clear: bool = True) -> int:
    """Abort reason of the last GEMM (0 = none).  Synchronises the device."""
    import ctypes
    v = ctypes.c_uint(0)
    _lib.check(_lib.load().act_fp8_gemm_status(ctypes.byref(v), 1 if clear else 0), "act_fp8_gemm_status")
    return int(v.value)


def dw_from_packed(dy: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, mn: torch.Tensor, bits: int,
                   group_size: int, K: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dW [N, K] (fp32) = dy[M, N]^T @ X~[M, K] with X~ decoded from `packed / scale / mn` (the
    output of codec.quant_pack on the row-major [M, K] layer input, flat groups) inside the
    GEMM: the step `dequant_unpack` + `dy.T.mm(x)` of a linear layer's backward
    (Activation_Compression/modules/ops.py:496-526) without the dequantised copy."""
    if not dy.is_cuda:
        raise RuntimeError("dw_from_packed needs CUDA tensors: there is no CPU path")
    if dy.dtype != torch.bfloat16:
        raise TypeError("dy must be bfloat16")
    dy = dy.reshape(-1, dy.shape[-1])
    if dy.stride(1) != 1:
        dy = dy.contiguous()
    M, N = dy.shape
    packed = packed.contiguous()
    scale = scale.reshape(-1).to(torch.float32).contiguous()
    mn = mn.reshape(-1).to(torch.float32).contiguous()
    if scale.numel() * group_size != M * K:
        raise ValueError("scale does not have one entry per group of the [M, K] input")
    dw = out if out is not None else torch.empty((N, K), dtype=torch.float32, device=dy.device)
    if dw.dtype != torch.float32 or dw.shape != (N, K) or dw.stride(1) != 1:
        raise ValueError("out must be a float32 [N, K] tensor with unit column stride")
    with _lib.device_of(dy):
        rc = _lib.load().act_dw_from_packed(dy.data_ptr(), packed.data_ptr(), scale.data_ptr(), mn.data_ptr(), bits,
                                            group_size, M, N, K, dy.stride(0), dw.data_ptr(), dw.stride(0),
                                            _lib.stream_ptr(dy))
    _lib.check(rc, "act_dw_from_packed")
    return dw


def dw_status(clear: bool = True) -> int:
    """Abort reason of the last dw_from_packed (0 = none).  Synchronises the device."""
    import ctypes
    v = ctypes.c_uint(0)
    _lib.check(_lib.load().act_dw_from_packed_status(ctypes.byref(v), 1 if clear else 0), "act_dw_from_packed_status")
    return int(v.value)


# ---------------------------------------------------------------- linear with its epilogue

_ACTIVATIONS = {"none": _lib.ACT_KIND_NONE, "relu": _lib.ACT_KIND_RELU, "gelu": _lib.ACT_KIND_GELU,
                "gelu_erf": _lib.ACT_KIND_GELU_ERF, "silu": _lib.ACT_KIND_SILU}
_DTYPE16 = {torch.bfloat16: _lib.ACT_DTYPE_BF16, torch.float16: _lib.ACT_DTYPE_F16}
_DTYPES = {torch.float32: _lib.ACT_DTYPE_F32, **_DTYPE16}


def _rows(t: torch.Tensor):
    """(t as a matrix of its last dimension whose rows are contiguous and do not overlap, its pitch)."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    rows, cols = t.shape
    pitch, step = t.stride()
    if (step != 1 and cols > 1) or (pitch < cols and rows > 1):
        return t.contiguous(), cols
    return t, pitch if rows > 1 else cols


def _check_sizes(what: str, *sizes: int) -> None:
    if max(sizes) > 0x7FFFFC00:
        raise ValueError(f"{what}: at most {0x7FFFFC00} rows, features or columns, got {sizes}")


def linear_act_applies(x: torch.Tensor, weight: torch.Tensor, cast_weight: bool = False) -> bool:
    """linear_act takes bf16 or fp16 CUDA tensors of one type (`cast_weight`: the weight will be cast to x's)
    and device, at least one input feature."""
    return (x.is_cuda and x.dtype in _DTYPE16 and (cast_weight or weight.dtype == x.dtype) and weight.device == x.device
            and weight.dim() == 2 and x.dim() >= 1 and x.shape[-1] == weight.shape[1] > 0)


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
               residual: Optional[torch.Tensor] = None, derivative: bool = False, variant: int = 0):
    """y = f(x @ weight.T + bias) + residual in one kernel (the sum in fp32, rounded once), for bf16 or fp16
    x [..., K] and weight [N, K] of the same type; bias [N] bf16, fp16 or fp32; residual [..., N] of x's type.
    `activation`: "none", "relu", "gelu" (tanh form), "gelu_erf" or "silu".  With `derivative` (GELU and SiLU)
    the result is (y, f'(...)): what a layer that saves the derivative, not its input, keeps for backward.
    Without autograd; `layers.DOLinearAct` is the module.  `variant` names a kernel (ACT_LINEAR_*) instead of
    the library's own choice."""
    if not x.is_cuda:
        raise RuntimeError("linear_act needs CUDA tensors: there is no CPU path")
    dtype, dev = x.dtype, x.device
    dt = _DTYPE16.get(dtype)
    if dt is None or weight.dtype != dtype:
        raise TypeError(f"linear_act: x and weight must both be bfloat16 or both float16, got {dtype} and {weight.dtype}")
    kind = _ACTIVATIONS.get(activation)
    if kind is None:
        raise ValueError(f"linear_act: activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if derivative and kind in (_lib.ACT_KIND_NONE, _lib.ACT_KIND_RELU):
        raise ValueError("linear_act: the derivative is an output of the GELU and SiLU forms only")
    xs, ws = x.shape, weight.shape
    if len(ws) != 2 or len(xs) < 1 or xs[-1] != ws[1] or ws[1] == 0:
        raise ValueError(f"linear_act: x [..., K] and weight [N, K] with K > 0, got {tuple(xs)} and {tuple(ws)}")
    N, K = ws
    shape = (xs[0], N) if len(xs) == 2 else xs[:-1] + (N,)
    bias_ptr, bias_dt = None, 0
    if bias is not None:
        bias_dt = _DTYPES.get(bias.dtype)
        if bias_dt is None or bias.dim() != 1 or bias.shape[0] != N or bias.device != dev:
            raise ValueError("linear_act: bias must be [N], of a floating type of 16 or 32 bits, on x's device")
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    if weight.device != dev:
        raise ValueError("linear_act: weight must be on x's device")
    x2, ldx = _rows(x)
    w2, ldw = _rows(weight)
    M = x2.numel() // K
    _check_sizes("linear_act", M, N, K)
    res_ptr, ldr = None, 0
    if residual is not None:
        if residual.shape != shape or residual.dtype != dtype or residual.device != dev:
            raise ValueError(f"linear_act: residual must have the result's shape {tuple(shape)}, type and device")
        residual, ldr = _rows(residual)
        res_ptr = residual.data_ptr()
    y = x.new_empty(shape)
    d = x.new_empty(shape) if derivative else None
    lib = _lib.load()
    xp, wp = x2.data_ptr(), w2.data_ptr()
    ws_ptr, need = None, 0
    if (xp | wp) & 15 or (ldx | ldw) & 7:                  # rows that may have to be copied first
        need = lib.act_linear_fwd_workspace(xp, ldx, wp, ldw, M, N, K, variant)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
            ws_ptr = workspace.data_ptr()
    with _lib.device_of(x):
        rc = lib.act_linear_fwd(xp, ldx, wp, ldw, bias_ptr, bias_dt, res_ptr, ldr, dt, M, N, K, kind, y.data_ptr(), N,
                                None if d is None else d.data_ptr(), N, variant, ws_ptr, need, _lib.stream_ptr(x))
    if rc:
        _lib.check(rc, "act_linear_fwd")
    return (y, d) if derivative else y


def act_backward(dy: torch.Tensor, derivative: torch.Tensor, bias_grad: bool = True):
    """(dz, db) of z -> f(z) with f'(z) = `derivative`: dz = dy * derivative in their type and, with
    `bias_grad`, db = its sum over everything but the last dimension, fp32, of the products before that
    rounding; None otherwise.  bf16 or fp16, one pass; the sum's order is fixed."""
    if not dy.is_cuda:
        raise RuntimeError("act_backward needs CUDA tensors: there is no CPU path")
    if dy.dtype not in _DTYPE16 or derivative.dtype != dy.dtype:
        raise TypeError("act_backward: dy and derivative must both be bfloat16 or both float16")
    if derivative.shape != dy.shape or dy.dim() < 1 or derivative.device != dy.device:
        raise ValueError("act_backward: dy and derivative must have one shape and device")
    dy, derivative = dy.contiguous(), derivative.contiguous()
    N = dy.shape[-1]
    M = dy.numel() // N if N else 0
    _check_sizes("act_backward", N)
    dz = torch.empty_like(dy)
    lib = _lib.load()
    db = db_ptr = ws_ptr = None
    need = 0
    with _lib.device_of(dy):
        if bias_grad:
            db = torch.empty(N, dtype=torch.float32, device=dy.device)
            db_ptr = db.data_ptr()
            need = lib.act_mul_col_sum_workspace(M, N)
            if need:
                workspace = torch.empty(need, dtype=torch.uint8, device=dy.device)
                ws_ptr = workspace.data_ptr()
        rc = lib.act_mul_col_sum(dy.data_ptr(), derivative.data_ptr(), _DTYPE16[dy.dtype], M, N, dz.data_ptr(), db_ptr, ws_ptr,
                                 need, _lib.stream_ptr(dy))
    _lib.check(rc, "act_mul_col_sum")
    return dz, db


def linear_backward(dz: torch.Tensor, x: Optional[torch.Tensor], weight: Optional[torch.Tensor], need_dx: bool = True,
                    need_dw: bool = True, dw_dtype: Optional[torch.dtype] = None, variant: int = 0):
    """(dx, dw) of z = x @ weight.T from dz [..., N]: dx = dz @ weight and dw = dz.T @ x over all rows, in dz's
    type (dw in float32 if `dw_dtype` says so), None where not needed (x or weight may then be None).
    bf16 or fp16, sums in fp32; dw's long reduction is split over the GPU and joined in a fixed order."""
    if not dz.is_cuda:
        raise RuntimeError("linear_backward needs CUDA tensors: there is no CPU path")
    dt = _DTYPE16.get(dz.dtype)
    x = x if need_dw else None
    weight = weight if need_dx else None
    if dt is None or any(t is not None and t.dtype != dz.dtype for t in (x, weight)):
        raise TypeError("linear_backward: dz, x and weight must all be bfloat16 or all float16")
    dw_dtype = dz.dtype if dw_dtype is None else dw_dtype
    if dw_dtype not in (dz.dtype, torch.float32):
        raise TypeError("linear_backward: dw comes in dz's type or in float32")
    if dz.dim() < 1 or (need_dw and (x is None or x.shape[:-1] != dz.shape[:-1])) \
            or (need_dx and (weight is None or weight.dim() != 2 or weight.shape[0] != dz.shape[-1])) \
            or any(t is not None and t.device != dz.device for t in (x, weight)) \
            or (need_dx and need_dw and x.shape[-1] != weight.shape[1]):
        raise ValueError("linear_backward: dz [..., N], x [..., K] and weight [N, K] on one device")
    if not need_dx and not need_dw:
        return None, None
    N = dz.shape[-1]
    K = weight.shape[1] if need_dx else x.shape[-1]
    M = dz.numel() // N if N else 0
    dx = dz.new_empty(dz.shape[:-1] + (K,)) if need_dx else None
    dw = torch.empty((N, K), dtype=dw_dtype, device=dz.device) if need_dw else None
    _check_sizes("linear_backward", M, N, K)
    if M == 0 or N == 0 or K == 0:                          # empty sums
        return (None if dx is None else dx.zero_()), (None if dw is None else dw.zero_())
    g, ldg = _rows(dz)
    xp = wp = None
    ldx = ldw = 0
    if need_dw:
        x, ldx = _rows(x)
        xp = x.data_ptr()
    if need_dx:
        weight, ldw = _rows(weight)
        wp = weight.data_ptr()
    lib = _lib.load()
    args = (g.data_ptr(), ldg, xp, ldx, wp, ldw)
    with _lib.device_of(dz):
        need = lib.act_linear_bwd_workspace(*args, M, N, K, _DTYPES[dw_dtype], need_dx, need_dw, variant)
        ws = torch.empty(need, dtype=torch.uint8, device=dz.device) if need else None
        rc = lib.act_linear_bwd(*args, dt, M, N, K, None if dx is None else dx.data_ptr(), K,
                                None if dw is None else dw.data_ptr(), K, _DTYPES[dw_dtype], variant,
                                None if ws is None else ws.data_ptr(), need, _lib.stream_ptr(dz))
    _lib.check(rc, "act_linear_bwd")
    return dx, dw


def linear_status(clear: bool = True) -> int:
    """Abort reason of the last linear_act / linear_backward kernel (0 = none).  Synchronises the device."""
    import ctypes
    v = ctypes.c_uint(0)
    _lib.check(_lib.load().act_linear_status(ctypes.byref(v), 1 if clear else 0), "act_linear_status")
    return int(v.value)
