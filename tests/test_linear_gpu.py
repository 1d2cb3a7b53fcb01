"""Linear with bias, activation and residual in its epilogue, and its backward, against 64 bits.

Tolerances.  The sum of K products of 16-bit numbers (each exact in 24 bits or less) in fp32 is off by
at most K steps of 2^-23 of the sum of the products' sizes S, in any order and with truncation; f and
f' have slopes of at most 1.2 and 1.0, are themselves within 2^-20 of max(|z|, 1), and the result is
rounded once, by half a step of its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = (torch.bfloat16, torch.float16)
ACTS = ("none", "relu", "gelu", "gelu_erf", "silu")
VARIANTS = (0, 1, 2, 3)


def _gemm():
    from deep_optimization_b200 import gemm
    return gemm


def _f(z, act):
    if act == "none":
        return z, None
    if act == "relu":
        return z.clamp_min(0), None
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if act == "gelu":
        k = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * k * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * (1 - s) * 2 * k * (1 + 3 * 0.044715 * z * z)
    cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _check(got, want, noise):
    eps = torch.finfo(got.dtype).eps / 2
    floor = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -134     # half the smallest subnormal
    tol = (want.abs() + noise) * eps + noise + floor
    off = (got.double() - want).abs()
    assert (off <= tol).all(), f"worst {(off / tol).max().item():.2f} of the tolerance"


def _linear_case(M, N, K, dtype, act, residual, bias, derivative, variant, dev, seed=0, layout=None):
    gemm = _gemm()
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=dev).to(dtype)
    w = (torch.randn(N, K, generator=g, device=dev) / math.sqrt(K)).to(dtype)
    b = torch.randn(N, generator=g, device=dev).to({"16": dtype, "32": torch.float32}[bias]) if bias else None
    r = torch.randn(M, N, generator=g, device=dev).to(dtype) if residual else None
    if layout:
        x, w, r = layout(x), layout(w), None if r is None else layout(r)
    out = gemm.linear_act(x, w, b, act, residual=r, derivative=derivative, variant=variant)
    assert gemm.linear_status() == 0
    X, W = x.double(), w.double()
    z = X @ W.t()
    S = X.abs() @ W.abs().t()
    if b is not None:
        z, S = z + b.double(), S + b.double().abs()
    y, d = _f(z, act)
    noise = 1.2 * (K + 4) * 2.0 ** -23 * S + 2.0 ** -20 * z.abs().clamp_min(1)
    if r is not None:
        y = y + r.double()
        noise = noise + 2.0 ** -23 * (r.double().abs() + y.abs())
    _check(out[0] if derivative else out, y, noise)
    if derivative:
        _check(out[1], d, noise)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("shape", [(300, 264, 136), (129, 72, 64), (257, 321, 203), (9, 1, 1)])
def test_forward(cuda_device, dtype, act, variant, shape):
    M, N, K = shape
    smooth = act not in ("none", "relu")
    for residual, bias, derivative in ((False, "", False), (True, "16", False), (False, "32", smooth), (True, "16", smooth)):
        _linear_case(M, N, K, dtype, act, residual, bias, derivative, variant, cuda_device, seed=M)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("shape", [(768, 768), (1, 1), (33, 7), (100, 264), (2304, 776), (5, 4096), (130, 4099), (3, 1025)])
def test_few_rows(cuda_device, dtype, M, shape):
    for i, act in enumerate(ACTS):
        for variant in (0, 4):
            _linear_case(M, *shape, dtype, act, i % 2 == 0, ("", "16", "32")[i % 3], act not in ("none", "relu"), variant,
                         cuda_device, seed=M + i)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("shape", [(2560, 2304, 768), (5000, 1000, 520), (20000, 768, 256), (1024, 4096, 1024)])
def test_more_tiles_than_ctas(cuda_device, variant, shape):
    _linear_case(*shape, torch.bfloat16, "gelu", False, "16", True, variant, cuda_device)
    _linear_case(*shape, torch.bfloat16, "none", True, "16", False, variant, cuda_device)
    _linear_case(*shape, torch.bfloat16, "silu", True, "16", True, variant, cuda_device)


@pytest.mark.parametrize("variant", VARIANTS)
def test_strides_and_bases(cuda_device, variant):
    def offset(t):                                        # rows pitched by 3 more elements, base off by one
        big = torch.zeros(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device=t.device)
        big[:, 1:1 + t.shape[1]] = t
        return big[:, 1:1 + t.shape[1]]

    def pitched(t):                                       # aligned rows with a gap
        big = torch.zeros(t.shape[0], t.shape[1] + 40, dtype=t.dtype, device=t.device)
        big[:, :t.shape[1]] = t
        return big[:, :t.shape[1]]

    for layout in (offset, pitched, lambda t: t.t().contiguous().t()):
        for shape in ((200, 136, 72), (4, 40, 64)):
            if variant in (0, 3) or shape[0] > 8:
                _linear_case(*shape, torch.bfloat16, "gelu", True, "16", True, variant, cuda_device, layout=layout)


def test_leading_dimensions_and_empty(cuda_device):
    gemm = _gemm()
    x = torch.randn(2, 3, 5, 64, device=cuda_device).bfloat16()
    w = torch.randn(24, 64, device=cuda_device).bfloat16()
    r = torch.randn(2, 3, 5, 24, device=cuda_device).bfloat16()
    y = gemm.linear_act(x, w, residual=r)
    assert torch.equal(y.view(30, 24), gemm.linear_act(x.view(30, 64), w, residual=r.view(30, 24)))
    assert gemm.linear_act(x[0, 0, 0], w).shape == (24,)
    assert gemm.linear_act(x[:0], w).shape == (0, 3, 5, 24)
    assert gemm.linear_act(x, w[:0]).shape == (2, 3, 5, 0)
    # one row broadcast over the batch has a zero stride
    e = x[0, 0, :1].expand(20, 64)
    assert torch.equal(gemm.linear_act(e, w, variant=3)[7], gemm.linear_act(e.contiguous(), w, variant=3)[0])


@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("rows", [1, 40])
def test_extreme_pre_activations(cuda_device, act, rows):
    """z far from zero, infinite and NaN: through a product with one nonzero column."""
    gemm = _gemm()
    vals = torch.tensor([0.0, -0.0, 1e-30, 30.0, -30.0, 1000.0, -1000.0, 1e20, -1e20, float("inf"), float("nan"), 3e38],
                        device=cuda_device).bfloat16()
    w = vals.view(-1, 1)
    x = torch.ones(rows, 1, dtype=torch.bfloat16, device=cuda_device)
    deriv = act != "relu"
    out = gemm.linear_act(x, w, activation=act, derivative=deriv)
    y = (out[0] if deriv else out)[0].double()
    z = vals.double()
    finite = torch.isfinite(z)
    want, d = _f(z.clamp(-1e6, 1e6), act)
    big = z.abs() > 1e5
    want = torch.where(big, torch.where(z > 0, z, torch.zeros_like(z)), want)
    assert torch.allclose(y[finite], want[finite].bfloat16().double(), rtol=2.0 ** -8, atol=1e-30 if act == "relu" else 1e-12)
    assert torch.isnan(y[10]) and y[9] == float("inf")
    if deriv:
        got = out[1][0].double()
        want_d = torch.where(z > 25, torch.ones_like(z), torch.where(z < -25, torch.zeros_like(z), d))
        assert ((got - want_d).abs()[finite] <= 2.0 ** -9 * want_d.abs()[finite] + 2.0 ** -20).all()
        assert torch.isnan(got[10])


# ---------------------------------------------------------------- backward

def _mul_case(M, N, dtype, dev, seed=0):
    gemm = _gemm()
    g = torch.Generator(device=dev).manual_seed(seed)
    dy, d = torch.randn(M, N, generator=g, device=dev).to(dtype), torch.rand(M, N, generator=g, device=dev).to(dtype)
    dz, db = gemm.act_backward(dy, d)
    p = dy.double() * d.double()
    # a product of two 16-bit numbers fits 24 bits (fp16: 22): one rounding
    _check(dz, p, p.abs() * 2.0 ** -24)
    S = p.abs().sum(0)
    assert ((db.double() - p.sum(0)).abs() <= (M + 1) * 2.0 ** -24 * S).all()
    dz2, none = gemm.act_backward(dy, d, bias_grad=False)
    assert none is None and torch.equal(dz, dz2)
    again = gemm.act_backward(dy, d)[1]
    assert torch.equal(db, again)                          # the same order every time


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 8), (3, 7), (1003, 997), (5000, 768), (40, 4096), (9, 2056), (20000, 64), (333, 3001), (16, 2048), (17, 2048), (16, 2049), (17, 301)])
def test_act_backward(cuda_device, dtype, shape):
    _mul_case(*shape, dtype, cuda_device)


def test_act_backward_empty_and_unaligned(cuda_device):
    gemm = _gemm()
    e = torch.empty(0, 24, dtype=torch.bfloat16, device=cuda_device)
    dz, db = gemm.act_backward(e, e)
    assert dz.shape == (0, 24) and torch.equal(db, torch.zeros(24, device=cuda_device))
    flat = torch.randn(1 + 64 * 40, device=cuda_device).bfloat16()
    dy = flat[1:].view(64, 40)
    d = flat[:-1].view(64, 40)
    dz, db = gemm.act_backward(dy, d)
    _check(dz, dy.double() * d.double(), (dy.double() * d.double()).abs() * 2.0 ** -24)
    assert (db.double() - (dy.double() * d.double()).sum(0)).abs().max() < 1e-4


def _backward_case(M, N, K, dtype, variant, dev, dw_dtype=None, layout=None):
    gemm = _gemm()
    g = torch.Generator(device=dev).manual_seed(M + N)
    dz = torch.randn(M, N, generator=g, device=dev).to(dtype)
    x = torch.randn(M, K, generator=g, device=dev).to(dtype)
    w = (torch.randn(N, K, generator=g, device=dev) / math.sqrt(N)).to(dtype)
    if layout:
        dz, x, w = layout(dz), layout(x), layout(w)
    dx, dw = gemm.linear_backward(dz, x, w, dw_dtype=dw_dtype, variant=variant)
    assert gemm.linear_status() == 0
    assert dw.dtype == (dw_dtype or dtype)
    Z, X, W = dz.double(), x.double(), w.double()
    _check(dx, Z @ W, (N + 2) * 2.0 ** -23 * (Z.abs() @ W.abs()))
    _check(dw, Z.t() @ X, (M + 150) * 2.0 ** -23 * (Z.abs().t() @ X.abs()))
    again = gemm.linear_backward(dz, x, w, dw_dtype=dw_dtype, variant=variant)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("shape", [(1, 64, 64), (300, 136, 264), (203, 321, 257), (1003, 997, 771), (4096, 64, 64), (7, 1, 1), (2000, 520, 8)])
def test_backward(cuda_device, dtype, variant, shape):
    _backward_case(*shape, dtype, variant, cuda_device)
    _backward_case(*shape, dtype, variant, cuda_device, dw_dtype=torch.float32)


def test_backward_long_and_strided(cuda_device):
    _backward_case(50432, 768, 256, torch.bfloat16, 0, cuda_device)
    _backward_case(400, 72, 40, torch.bfloat16, 0, cuda_device, layout=lambda t: t.t().contiguous().t())

    def offset(t):
        big = torch.zeros(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device=t.device)
        big[:, 1:1 + t.shape[1]] = t
        return big[:, 1:1 + t.shape[1]]
    _backward_case(400, 72, 40, torch.float16, 0, cuda_device, layout=offset)


def test_backward_parts_and_empty(cuda_device):
    gemm = _gemm()
    dz = torch.randn(64, 40, device=cuda_device).bfloat16()
    x, w = torch.randn(64, 24, device=cuda_device).bfloat16(), torch.randn(40, 24, device=cuda_device).bfloat16()
    dx, dw = gemm.linear_backward(dz, x, w)
    assert torch.equal(gemm.linear_backward(dz, None, w, need_dw=False)[0], dx)
    assert torch.equal(gemm.linear_backward(dz, x, None, need_dx=False)[1], dw)
    dx, dw = gemm.linear_backward(dz[:0], x[:0], w)
    assert dx.shape == (0, 24) and torch.equal(dw, torch.zeros_like(w))


def test_captured_and_on_another_stream(cuda_device):
    gemm = _gemm()
    x = torch.randn(1003, 771, device=cuda_device).bfloat16()
    w = torch.randn(997, 771, device=cuda_device).bfloat16()
    y, d = gemm.linear_act(x, w, activation="silu", derivative=True)
    dx, dw = gemm.linear_backward(y, x, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y2, d2 = gemm.linear_act(x, w, activation="silu", derivative=True)
        dx2, dw2 = gemm.linear_backward(y2, x, w)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and torch.equal(d, d2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y3 = gemm.linear_act(x, w, activation="silu")
    side.synchronize()
    assert torch.equal(y, y3)
