"""Refusals and host logic of the linear, dropout and rotary operators, without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

from .philox import keep_mask, philox


@pytest.fixture(scope="module")
def lib():
    from deep_optimization_b200 import _lib, build
    build.build()
    return _lib.load()


P = ctypes.c_void_p(4096)          # never dereferenced: the checks come first
ODD = ctypes.c_void_p(4097)
DTYPE, ALIGN, SIZE, NULL, WORKSPACE, UNSUPPORTED = 1, 4, 5, 6, 8, 11


def test_generator_known_answers():
    """The three published known answers of Philox-4x32-10."""
    ones = 2 ** 64 - 1
    for ctr, key, want in (((0, 0), 0, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
                           ((ones, ones), ones, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
                           ((0x85a308d3243f6a88, 0x0370734413198a2e), 0x299f31d0a4093822,
                            "d16cfe09 94fdcceb 5001e420 24126ea1")):
        got = philox(np.array([ctr], dtype=np.uint64), key)[0]
        assert " ".join(f"{int(v):08x}" for v in got) == want
    m = keep_mask(0, 1 << 16, 0.25, 3, 5)
    assert abs(m.mean() - 0.75) < 5 * (0.25 * 0.75 / (1 << 16)) ** 0.5
    assert (keep_mask(13, 100, 0.25, 3, 5) == m[13:113]).all()


def _fwd(lib, x=P, ldx=64, w=P, ldw=64, bias=None, bias_dt=0, res=None, ldr=0, dt=1, M=32, N=64, K=64, kind=0, y=P, ldy=64,
         d=None, ldd=0, variant=0, ws=None, ws_bytes=0):
    return lib.act_linear_fwd(x, ldx, w, ldw, bias, bias_dt, res, ldr, dt, M, N, K, kind, y, ldy, d, ldd, variant, ws, ws_bytes, None)


def test_linear_forward_refusals(lib):
    assert _fwd(lib, dt=0) == DTYPE and _fwd(lib, dt=9) == DTYPE
    assert _fwd(lib, bias=P, bias_dt=7) == DTYPE
    assert _fwd(lib, M=-1) == SIZE and _fwd(lib, N=-1) == SIZE and _fwd(lib, K=0) == SIZE
    assert _fwd(lib, ldx=63) == SIZE and _fwd(lib, ldw=63) == SIZE and _fwd(lib, ldy=63) == SIZE
    assert _fwd(lib, res=P, ldr=63) == SIZE and _fwd(lib, kind=1, d=P, ldd=63) == SIZE
    assert _fwd(lib, kind=5) == UNSUPPORTED and _fwd(lib, kind=-1) == UNSUPPORTED
    assert _fwd(lib, variant=5) == UNSUPPORTED and _fwd(lib, variant=4, M=9) == UNSUPPORTED
    assert _fwd(lib, kind=0, d=P, ldd=64) == UNSUPPORTED and _fwd(lib, kind=4, d=P, ldd=64) == UNSUPPORTED
    assert _fwd(lib, x=None) == NULL and _fwd(lib, w=None) == NULL and _fwd(lib, y=None) == NULL
    assert _fwd(lib, x=ODD) == ALIGN and _fwd(lib, bias=ctypes.c_void_p(4098), bias_dt=0) == ALIGN
    assert _fwd(lib, M=0x7FFFFC01) == SIZE and _fwd(lib, N=0x7FFFFFFF, ldy=1 << 31) == SIZE
    assert _fwd(lib, M=0) == 0 and _fwd(lib, N=0, ldy=0) == 0
    # rows that a bulk copy cannot read need the workspace
    need = lib.act_linear_fwd_workspace(P, 65, P, 64, 32, 64, 64, 0)
    assert need == 32 * 64 * 2
    assert _fwd(lib, ldx=65) == WORKSPACE and _fwd(lib, ldx=65, ws=P, ws_bytes=need - 1) == WORKSPACE
    assert _fwd(lib, ldx=65, ws=ctypes.c_void_p(4104), ws_bytes=need) == ALIGN
    assert lib.act_linear_fwd_workspace(P, 64, P, 64, 32, 64, 64, 0) == 0
    assert lib.act_linear_fwd_workspace(P, 65, P, 64, 4, 64, 64, 0) == 0        # few rows read in place


def _bwd(lib, dz=P, lddz=64, x=P, ldx=64, w=P, ldw=64, dt=1, M=32, N=64, K=64, dx=P, lddx=64, dw=P, lddw=64, dwt=1, variant=0,
         ws=None, n=0):
    return lib.act_linear_bwd(dz, lddz, x, ldx, w, ldw, dt, M, N, K, dx, lddx, dw, lddw, dwt, variant, ws, n, None)


def test_linear_backward_refusals(lib):
    assert _bwd(lib, dt=0) == DTYPE and _bwd(lib, dwt=2) == DTYPE
    assert _bwd(lib, M=0) == SIZE and _bwd(lib, N=0) == SIZE and _bwd(lib, K=0) == SIZE
    assert _bwd(lib, lddz=63) == SIZE and _bwd(lib, ldx=63) == SIZE and _bwd(lib, ldw=63) == SIZE
    assert _bwd(lib, lddx=63) == SIZE and _bwd(lib, lddw=63) == SIZE
    assert _bwd(lib, M=0x7FFFFC01) == SIZE
    assert _bwd(lib, variant=4) == UNSUPPORTED
    assert _bwd(lib, dx=None, dw=None) == 0
    assert _bwd(lib, dz=None) == NULL and _bwd(lib, w=None) == NULL and _bwd(lib, x=None) == NULL
    assert _bwd(lib, dz=ODD) == ALIGN and _bwd(lib, dw=ctypes.c_void_p(4098), dwt=0) == ALIGN
    assert _bwd(lib, lddz=65) == WORKSPACE and _bwd(lib, dwt=0) == WORKSPACE     # fp32 dw goes through a partial plane
    assert lib.act_linear_bwd_workspace(P, 64, P, 64, P, 64, 32, 64, 64, 0, 0, 1, 0) == 64 * 64 * 4


def test_mul_col_sum_refusals(lib):
    f = lib.act_mul_col_sum
    assert f(P, P, 0, 4, 8, P, P, P, 1 << 20, None) == DTYPE
    assert f(P, P, 1, -1, 8, P, P, P, 1 << 20, None) == SIZE
    assert f(None, P, 1, 4, 8, P, P, P, 1 << 20, None) == NULL
    assert f(ODD, P, 1, 4, 8, P, P, P, 1 << 20, None) == ALIGN
    assert f(P, P, 1, 4, 8, P, ctypes.c_void_p(4098), P, 1 << 20, None) == ALIGN
    assert f(P, P, 1, 40000, 8, P, P, None, 0, None) == WORKSPACE
    assert lib.act_mul_col_sum_workspace(4, 8) == 0 and lib.act_mul_col_sum_workspace(0, 8) == 0
    assert f(P, P, 1, 4, 0, P, P, None, 0, None) == 0


def test_dropout_refusals(lib):
    f = lib.act_dropout
    assert f(P, None, 7, 8, 10, 0, 0, None, P, None) == DTYPE
    assert f(P, None, 1, -1, 10, 0, 0, None, P, None) == SIZE
    assert f(P, None, 1, 8, 65537, 0, 0, None, P, None) == SIZE
    assert f(None, None, 1, 8, 10, 0, 0, None, P, None) == NULL
    assert f(ODD, None, 1, 8, 10, 0, 0, None, P, None) == ALIGN
    assert f(ctypes.c_void_p(4098), None, 0, 8, 10, 0, 0, None, P, None) == ALIGN
    assert f(P, None, 1, 8, 10, 0, 0, ctypes.c_void_p(4100), P, None) == ALIGN
    assert f(P, None, 1, 0, 10, 0, 0, None, P, None) == 0
    assert lib.act_rng_ticket(None, P, None) == NULL and lib.act_rng_ticket(P, ctypes.c_void_p(4100), None) == ALIGN
    from deep_optimization_b200 import codec
    assert codec.dropout_threshold(0.1) == 6554 and codec.dropout_threshold(1.0) == 65536 and codec.dropout_threshold(0.0) == 0
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            codec.dropout_threshold(p)
    with pytest.raises(RuntimeError):
        codec.dropout(torch.zeros(8), 0.1, (1, 1))


def _rotary(lib, src=4096, dst=4096, heads=2, parts=1, dt=1, B=1, T=4, Dh=64, pos=P, pos_bytes=8, turns=P, sections=(16, 16), axes=None):
    n = max(parts, 1)
    strides = (ctypes.c_int64 * (3 * n))(*([512, 64, 128] * n))
    return lib.act_rotary_heads((ctypes.c_void_p * n)(*([src] * n)), strides, (ctypes.c_void_p * n)(*([dst] * n)), strides,
                                (ctypes.c_int * n)(*([heads] * n)), (ctypes.c_int * n)(*([1] * n)), parts, dt, B, T, Dh, pos,
                                pos_bytes, (ctypes.c_int64 * 3)(0, 2, 1), turns, (ctypes.c_int * len(sections))(*sections),
                                len(sections) if axes is None else axes, 0, 0, None)


def test_rotary_refusals(lib):
    assert _rotary(lib, dt=5) == DTYPE and _rotary(lib, pos_bytes=2) == DTYPE
    assert _rotary(lib, parts=0) == SIZE and _rotary(lib, parts=4) == SIZE
    assert _rotary(lib, axes=0) == SIZE and _rotary(lib, sections=(1, 1, 1, 1, 1)) == SIZE
    assert _rotary(lib, B=-1) == SIZE and _rotary(lib, T=-1) == SIZE and _rotary(lib, Dh=0) == SIZE and _rotary(lib, Dh=1025) == SIZE
    assert _rotary(lib, sections=(16, 17)) == SIZE and _rotary(lib, sections=(-1, 2)) == SIZE and _rotary(lib, heads=-1) == SIZE
    assert _rotary(lib, src=None) == NULL and _rotary(lib, dst=None) == NULL and _rotary(lib, pos=None) == NULL and _rotary(lib, turns=None) == NULL
    assert _rotary(lib, src=4097) == ALIGN and _rotary(lib, pos=ctypes.c_void_p(4100)) == ALIGN and _rotary(lib, turns=ctypes.c_void_p(4100)) == ALIGN
    assert _rotary(lib, B=0) == 0 and _rotary(lib, T=0) == 0 and _rotary(lib, heads=0) == 0


def test_rotary_split_and_merge_refusals(lib):
    sec = (ctypes.c_int * 1)(16)
    split = lambda q=P, o=P, h=2, k=1, dt=1, T=4, Dh=64: lib.act_rotary_split(q, o, h, k, dt, 1, T, Dh, P, 8, 0, 1, 1, P, sec, 1, 0, None)
    assert split(dt=4) == DTYPE and split(h=-1) == SIZE and split(T=-1) == SIZE and split(Dh=0) == SIZE and split(Dh=31) == SIZE
    assert split(q=None) == NULL and split(o=None) == NULL and split(q=ODD) == ALIGN and split(T=0) == 0
    st = (ctypes.c_int64 * 9)(*([256, 64, 64] * 3))
    merge = lambda q=P, k=P, v=P, o=P, dt=1, T=4, Dh=64: lib.act_rotary_merge(q, k, v, st, o, 2, 1, dt, 1, T, Dh, P, 8, 0, 1, 1, P, sec, 1, 0, None)
    assert merge(dt=4) == DTYPE and merge(T=-1) == SIZE and merge(Dh=31) == SIZE
    assert merge(q=None) == NULL and merge(k=None) == NULL and merge(v=None) == NULL and merge(o=None) == NULL
    assert merge(v=ODD) == ALIGN and merge(T=0) == 0


def test_cpu_tensors_are_refused():
    from deep_optimization_b200 import gemm
    from deep_optimization_b200.modules import attention
    x, w = torch.zeros(4, 8).bfloat16(), torch.zeros(8, 8).bfloat16()
    with pytest.raises(RuntimeError):
        gemm.linear_act(x, w)
    with pytest.raises(RuntimeError):
        gemm.act_backward(x, x)
    with pytest.raises(RuntimeError):
        gemm.linear_backward(x, x, w)
    turns = attention.rotary_turns((2,))
    with pytest.raises(RuntimeError):
        attention.rotary_split(torch.zeros(1, 4, 24), 1, torch.zeros(4, 1, dtype=torch.int64), turns, (2,))
    with pytest.raises(RuntimeError):
        attention.rotary_heads(torch.zeros(1, 1, 4, 8), torch.zeros(4, 1, dtype=torch.int64), turns, (2,))
    with pytest.raises(ValueError):
        attention.rotary_turns((2,), base=0.5)


def test_image_positions():
    from deep_optimization_b200.modules import attention
    p = attention.image_positions(2, 3)
    assert p.tolist() == [[0, 0], [1, 1], [1, 2], [1, 3], [2, 1], [2, 2], [2, 3]]


def test_turns_are_the_frequencies():
    from fractions import Fraction
    import math
    from deep_optimization_b200.modules import attention
    t = attention.rotary_turns((3, 2), base=100.0).tolist()
    for got, f in zip(t, (1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3), 1.0, 0.1)):
        # three roundings of 2^-53 relative, then half a unit
        assert abs(Fraction(got) - Fraction(f / (2 * math.pi)) * 2 ** 64) <= Fraction(f) * 2 ** 12


def test_dropout_in_a_capture_needs_a_step_outside_first(monkeypatch):
    from deep_optimization_b200 import codec
    monkeypatch.setattr(codec, "_graph_rng", {})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="outside the capture"):
        codec.dropout_rng(torch.device("cuda", 0))
