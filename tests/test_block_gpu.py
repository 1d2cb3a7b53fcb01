"""The operators of a transformer block together: DOLinearAct, RotaryAxes and DODropout as modules, in a
block and in a Controller's model."""
import math

import pytest
import torch
import torch.nn.functional as F
from torch import nn

pytestmark = pytest.mark.gpu
ACTS = ("none", "relu", "gelu", "gelu_erf", "silu")


def _f64(z, act):
    if act == "gelu":
        return F.gelu(z, approximate="tanh")
    return {"none": lambda v: v, "relu": F.relu, "gelu_erf": F.gelu, "silu": F.silu}[act](z)


def _norm_close(got, want, steps, dtype):
    """2-norm of the difference against `steps` roundings of the type, each off by at most half a step."""
    eps = torch.finfo(dtype).eps / 2
    off, size = (got.double() - want).norm(), want.norm()
    assert off <= steps * eps * size, f"{(off / size / eps).item():.2f} roundings, {steps} allowed"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [((3, 50, 96), 136), ((77, 33), 51), ((5, 64), 128)])
def test_linear_act_module_gradients(cuda_device, dtype, act, residual, shape):
    """y rounds once; dz = dy * f' holds the roundings of f' and of dz, and each gradient its own."""
    from deep_optimization_b200.layers import DOLinearAct
    torch.manual_seed(1)
    (xs, N) = shape
    m = DOLinearAct(xs[-1], N, act).to(cuda_device, dtype).train()
    x = torch.randn(xs, device=cuda_device).to(dtype).requires_grad_()
    r = torch.randn(xs[:-1] + (N,), device=cuda_device).to(dtype).requires_grad_() if residual else None
    dy = torch.randn(xs[:-1] + (N,), device=cuda_device).to(dtype)
    y = m(x, r)
    wrt = [x, m.weight, m.bias] + ([r] if residual else [])
    got = torch.autograd.grad(y, wrt, dy)
    X, W, B = (t.detach().double().requires_grad_() for t in (x, m.weight, m.bias))
    Y = _f64(X @ W.t() + B, act)
    want = torch.autograd.grad(Y, (X, W, B), dy.double())
    if residual:
        Y = Y + r.detach().double()
        assert torch.equal(got[3], dy)
    # a ReLU with a residual rounds before and after the sum
    _norm_close(y, Y.detach(), 2 if act == "relu" and residual else 1, dtype)
    for g, w in zip(got, want):
        _norm_close(g, w, 3, dtype)
    m.eval()
    with torch.no_grad():
        _norm_close(m(x, r), Y.detach(), 1, dtype)


def test_linear_act_gradient_against_differences(cuda_device):
    """d/dt of sum(f(x(t) W^T + b) * g) along a direction, in 64 bits by a central difference, against
    the gradient the module gives: three roundings of bf16 in the gradient, and the difference's own
    step squared."""
    from deep_optimization_b200.layers import DOLinearAct
    torch.manual_seed(2)
    m = DOLinearAct(64, 96, "gelu").to(cuda_device, torch.bfloat16)
    x = torch.randn(40, 64, device=cuda_device).bfloat16().requires_grad_()
    g = torch.randn(40, 96, device=cuda_device).bfloat16()
    (grad,) = torch.autograd.grad(m(x), x, g)
    v = torch.randn(40, 64, device=cuda_device, dtype=torch.float64)

    def value(t):
        z = (x.detach().double() + t * v) @ m.weight.double().t() + m.bias.double()
        return (F.gelu(z, approximate="tanh") * g.double()).sum()

    h = 1e-4
    diff = (value(h) - value(-h)) / (2 * h)
    # 64 * 40 independent roundings add up as a norm; five times that
    tol = 5 * 3 * 2.0 ** -9 * (grad.double() * v).norm() + 1e-6
    assert (diff - (grad.double() * v).sum()).abs() <= tol


def test_linear_act_other_tensors_take_the_stock_operators(cuda_device):
    from deep_optimization_b200.layers import DOLinearAct
    m = DOLinearAct(8, 6, "silu").to(cuda_device)
    x = torch.randn(4, 8, device=cuda_device)
    assert torch.equal(m(x), F.silu(F.linear(x, m.weight, m.bias)))
    r32 = torch.randn(4, 6, device=cuda_device)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x)
        assert y.dtype == torch.bfloat16
        # a residual of another type is added outside, with its promotion
        assert torch.equal(m(x, r32), y + r32)
    x.requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x)
    y.float().sum().backward()
    assert x.grad.dtype == torch.float32 and m.weight.grad.dtype == torch.float32 and m.bias.grad.dtype == torch.float32
    c = m.cpu()
    assert c(torch.randn(2, 8)).shape == (2, 6)
    with pytest.raises(ValueError):
        DOLinearAct(4, 4, "tanh")


@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True)])
@pytest.mark.parametrize("act", ("none", "relu", "gelu"))
def test_linear_act_gradients_one_at_a_time(cuda_device, needs, act):
    from deep_optimization_b200.layers import DOLinearAct
    torch.manual_seed(3)
    m = DOLinearAct(40, 24, act).to(cuda_device, torch.bfloat16)
    x = torch.randn(30, 40, device=cuda_device).bfloat16()
    full = [x.clone().requires_grad_(), m.weight, m.bias]
    dy = torch.randn(30, 24, device=cuda_device).bfloat16()
    want = torch.autograd.grad(m(full[0]), full, dy)
    for p, n in zip((m.weight, m.bias), needs[1:]):
        p.requires_grad_(n)
    x.requires_grad_(needs[0])
    i = needs.index(True)
    (got,) = torch.autograd.grad(m(x), (x, m.weight, m.bias)[i], dy)
    assert torch.equal(got, want[i])


class _Block(nn.Module):
    """x + drop(proj(attention(rotary(qkv(norm x))))), then + drop(fc2(f(fc1(norm x))))."""

    def __init__(self, dim, heads, kv, hidden, p):
        super().__init__()
        from deep_optimization_b200.layers import DOLinearAct
        from deep_optimization_b200.modules.activations.act_layers import DODropout
        from deep_optimization_b200.modules.attention import RotaryAxes
        self.heads, self.kv = heads, kv
        d = dim // heads
        self.norm1, self.norm2 = nn.LayerNorm(dim), nn.LayerNorm(dim)
        self.qkv = DOLinearAct(dim, (heads + 2 * kv) * d)
        self.rotary = RotaryAxes((d // 8, d // 8, d // 4))
        self.proj, self.fc1, self.fc2 = DOLinearAct(dim, dim), DOLinearAct(dim, hidden, "gelu"), DOLinearAct(hidden, dim)
        self.drop1, self.drop2 = DODropout(p), DODropout(p)

    def forward(self, x, pos):
        q, k, v = self.rotary(self.qkv(self.norm1(x)), self.heads, pos, self.kv)
        a = F.scaled_dot_product_attention(q, k, v, enable_gqa=self.kv != self.heads)
        x = self.drop1(self.proj(a.transpose(1, 2).reshape(x.shape)), x)
        return self.drop2(self.fc2(self.fc1(self.norm2(x))), x)


def _plain_block(m, x, pos, masks):
    """The same in 64 bits with the masks given (kept elements hold their factor)."""
    P = {n: p.detach().double().requires_grad_() for n, p in m.named_parameters()}
    B, T, D = x.shape
    d = D // m.heads
    lin = lambda n, v: v @ P[n + ".weight"].t() + P[n + ".bias"]
    h = F.layer_norm(x, (D,), P["norm1.weight"], P["norm1.bias"])
    q, k, v = lin("qkv", h).view(B, T, m.heads + 2 * m.kv, d).transpose(1, 2).split((m.heads, m.kv, m.kv), 1)
    f = torch.cat([torch.tensor([10000.0 ** (-i / n) for i in range(n)], dtype=torch.float64) for n in m.rotary.sections]).to(x.device)
    axis = torch.repeat_interleave(torch.arange(3), torch.tensor(m.rotary.sections)).to(x.device)
    ang = pos.double()[:, axis] * f
    c, s, n = torch.cos(ang), torch.sin(ang), f.numel()
    rot = lambda t: torch.cat([t[..., :n] * c - t[..., n:2 * n] * s, t[..., n:2 * n] * c + t[..., :n] * s, t[..., 2 * n:]], -1)
    rep = m.heads // m.kv
    q, k, v = rot(q), rot(k).repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    a = torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(d), -1) @ v
    x = x + masks[0] * lin("proj", a.transpose(1, 2).reshape(x.shape))
    h = F.gelu(lin("fc1", F.layer_norm(x, (D,), P["norm2.weight"], P["norm2.bias"])), approximate="tanh")
    return x + masks[1] * lin("fc2", h), P


def test_block_together(cuda_device):
    from deep_optimization_b200 import codec
    torch.manual_seed(4)
    B, T, D = 3, 49, 128
    m = _Block(D, 4, 2, 320, 0.25).to(cuda_device, torch.bfloat16).train()
    pos = torch.randint(0, 30, (T, 3), device=cuda_device)
    x = torch.randn(B, T, D, device=cuda_device).bfloat16().requires_grad_()
    g = torch.randn(B, T, D, device=cuda_device).bfloat16()
    torch.manual_seed(11)
    rngs = [codec.dropout_rng(cuda_device), codec.dropout_rng(cuda_device)]
    masks = [codec.dropout(torch.ones(B, T, D, device=cuda_device), 0.25, r).double() for r in rngs]
    torch.manual_seed(11)
    y = m(x, pos)
    grads = torch.autograd.grad(y, [x] + list(m.parameters()), g)
    X = x.detach().double().requires_grad_()
    Y, P = _plain_block(m, X, pos, masks)
    want = torch.autograd.grad(Y, [X] + list(P.values()), g.double())
    # Roundings of bf16 along the longest path, one per tensor that is written: forward norm1, qkv, q, k, the
    # attention's probabilities and output, proj, the sum, norm2, fc1, fc2, the sum = 12; backward as many
    # again and the saved derivative.  A LayerNorm's and a softmax's gradients subtract two parts and can
    # double what comes in; 50 covers the paths, whose errors are independent and mostly add as squares.
    _norm_close(y, Y.detach(), 12, torch.bfloat16)
    for a, b in zip(grads, want):
        _norm_close(a, b, 50, torch.bfloat16)


def test_block_captured_against_eager(cuda_device):
    """A training step in a graph: new masks at each replay, each replay's gradients those of its masks."""
    torch.manual_seed(5)
    B, T, D = 2, 17, 64
    m = _Block(D, 2, 2, 96, 0.5).to(cuda_device, torch.bfloat16).train()
    pos = torch.randint(0, 9, (T, 3), device=cuda_device)
    x = torch.randn(B, T, D, device=cuda_device).bfloat16().requires_grad_()
    params = list(m.parameters())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(m(x, pos).float().square().sum(), [x] + params)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x, pos)
        grads = torch.autograd.grad(y.float().square().sum(), [x] + params)
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.isfinite(t).all() for t in grads)
        seen.append((y.detach().clone(), [t.clone() for t in grads]))
    assert not torch.equal(seen[0][0], seen[1][0]) and not torch.equal(seen[1][0], seen[2][0])
    m.eval()
    with torch.no_grad():
        a = m(x, pos)
        assert torch.equal(a, m(x, pos))


def _vit(**kw):
    from deep_optimization_b200.payload.vit import VisionTransformer
    return VisionTransformer(image=48, patch=8, dim=128, depth=2, heads=4, mlp_dim=256, num_classes=10, **kw)


def _controlled(model, dev, **extra):
    from deep_optimization_b200.controller import Controller
    cfg = {"default_bits": 8, "group_size": 256, "batch_size": 16, "min_activation_mib": -1, **extra}
    return Controller(model, cfg, input_shape=(3, 48, 48), test=False, device=dev)


def _grads(model, x, target):
    model.zero_grad()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = F.cross_entropy(model(x).float(), target)
    loss.backward()
    return torch.cat([p.grad.flatten().double() for p in model.parameters()])


@pytest.mark.parametrize("rotary", [False, True])
def test_controller_fuses_the_mlp(cuda_device, rotary):
    """fc1 and its GELU become one module; its gradients are as near to the stock model's as those of the
    unfused compressed model are, whose only difference is that z is rounded before the GELU."""
    import copy
    torch.manual_seed(6)
    base = _vit(rotary=rotary).to(cuda_device)
    x = torch.randn(16, 3, 48, 48, device=cuda_device)
    target = torch.randint(0, 10, (16,), device=cuda_device)
    want = _grads(base, x, target)
    c = _controlled(copy.deepcopy(base), cuda_device, fuse_linear_act=True)
    assert c.fused_linear_act == ["blocks.0.fc1", "blocks.1.fc1"]
    assert set(c.traced_model.state_dict()) == set(base.state_dict())
    fused = _grads(c.traced_model, x, target)
    plain = _grads(_controlled(copy.deepcopy(base), cuda_device).traced_model, x, target)
    off = lambda g: ((g - want).norm() / want.norm()).item()
    # 8-bit storage is random rounding: two draws of one distance
    assert off(fused) <= 1.3 * off(plain) + 2.0 ** -9
    c.traced_model.eval()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.isfinite(c.traced_model(x)).all()


@pytest.mark.parametrize("features", [256, 200])
@pytest.mark.parametrize("offset", [0, 1])
def test_linear_act_compressed_gradients(cuda_device, features, offset):
    """DOLinearAct with a meta: 8-bit x and f', whole groups (256 features) or padded ones (200), against the
    gradients of the same layer without: a stored value is off by less than a step of its group, range / 255,
    at most 12 / 255 of x and 1.3 / 255 of f', as independent errors; bf16 roundings as above."""
    from deep_optimization_b200.controller import find_group_size
    from deep_optimization_b200.layers import DOLinearAct
    torch.manual_seed(9)
    meta = {}
    for name, f in (("lin", 128), ("act", features)):
        gs, pad = find_group_size(40 * f, 8)
        meta[name] = {"pack_only": False, "bits": 8, "group_size": gs, "act_padding": pad, "N": 48, "AVG_ALAM": False,
                      "ALAM_BITS": 0, "DIVISION": None}
    m = DOLinearAct(128, features, "gelu").to(cuda_device, torch.bfloat16).train()
    x = torch.randn(48, 40, 128, device=cuda_device).bfloat16().requires_grad_()
    flat = torch.randn(48 * 40 * features + 8, device=cuda_device).bfloat16()
    dy = flat[offset:offset + 48 * 40 * features].view(48, 40, features)      # one element off: not 16-byte aligned
    wrt = [x, m.weight, m.bias]
    want = torch.autograd.grad(m(x), wrt, dy)
    m.meta, m.target_name, m.act_name = meta, "lin", "act"
    got = torch.autograd.grad(m(x), wrt, dy)
    eps = 2.0 ** -9
    # f' has a root mean square of at least 0.5, x of 1: relative errors of a stored value, then the roundings
    err_d, err_x = 1.3 / 255 / 0.5, 12.0 / 255
    for a, b, e in zip(got, want, (err_d, err_d + err_x, err_d)):
        assert (a.double() - b.double()).norm() <= (e + 6 * eps) * b.double().norm()


def test_controller_with_everything(cuda_device):
    torch.manual_seed(7)
    c = _controlled(_vit(rotary=True, dropout=0.1), cuda_device, fuse_linear_act=True, compress_dropout=True)
    x = torch.randn(16, 3, 48, 48, device=cuda_device)
    g = _grads(c.traced_model, x, torch.randint(0, 10, (16,), device=cuda_device))
    assert torch.isfinite(g).all() and g.abs().sum() > 0


def test_payload_defaults_are_unchanged(cuda_device):
    keys = set(_vit().state_dict())
    assert "pos_embed" in keys and not any("positions" in k or "turns" in k for k in keys)
    assert "pos_embed" not in set(_vit(rotary=True).state_dict())


def test_refusals(cuda_device):
    """Arguments that the host turns down before anything is launched."""
    from deep_optimization_b200 import codec, gemm
    from deep_optimization_b200.modules import attention
    t = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device=cuda_device)
    x, w = t(4, 16), t(8, 16)
    for bad in (dict(x=t(4, 16, dt=torch.float32)), dict(w=t(8, 16, dt=torch.float16)), dict(w=t(8, 16, dt=torch.float32))):
        with pytest.raises(TypeError):
            gemm.linear_act(bad.get("x", x), bad.get("w", w))
    for kw in (dict(activation="tanh"), dict(derivative=True), dict(activation="relu", derivative=True), dict(bias=t(9)),
               dict(bias=t(8, dt=torch.int32)), dict(bias=torch.zeros(8)), dict(residual=t(4, 9)),
               dict(residual=t(4, 8, dt=torch.float32)), dict(residual=t(8))):
        with pytest.raises(ValueError):
            gemm.linear_act(x, w, **kw)
    for a, b in ((t(4, 15), w), (t(4, 0), t(8, 0)), (x, t(16)), (x, w.cpu())):
        with pytest.raises(ValueError):
            gemm.linear_act(a, b)
    with pytest.raises(TypeError):
        gemm.act_backward(x, t(4, 16, dt=torch.float16))
    with pytest.raises(ValueError):
        gemm.act_backward(x, t(4, 8))
    with pytest.raises(TypeError):
        gemm.linear_backward(t(4, 8, dt=torch.float32), x, w)
    with pytest.raises(TypeError):
        gemm.linear_backward(t(4, 8), x, w, dw_dtype=torch.float16)
    for args in ((t(4, 9), x, w), (t(5, 8), x, w), (t(4, 8), t(4, 15), w), (t(4, 8), None, w), (t(4, 8), x, None)):
        with pytest.raises(ValueError):
            gemm.linear_backward(*args)
    with pytest.raises(TypeError):
        codec.dropout(t(4, dt=torch.int32), 0.5, (1, 1))
    for kw in (dict(p=1.5), dict(residual=t(5)), dict(residual=t(4, dt=torch.float32)), dict(rng=t(2)), dict(rng=torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            codec.dropout(t(4), kw.get("p", 0.5), kw.get("rng", (1, 1)), kw.get("residual"))
    turns = attention.rotary_turns((4, 4), device=cuda_device)
    pos = t(5, 2, dt=torch.int64)
    qkv = t(2, 5, 3 * 2 * 16)
    ok = dict(qkv=qkv, heads=2, positions=pos, turns=turns, sections=(4, 4))
    for kw in (dict(heads=5), dict(heads=0), dict(qkv=t(2, 96)), dict(positions=t(4, 2, dt=torch.int64)),
               dict(positions=t(5, 1, dt=torch.int64)), dict(positions=t(3, 5, 2, dt=torch.int64)), dict(turns=turns[:7]),
               dict(turns=turns.int()), dict(turns=turns.cpu()), dict(sections=(4, 5)), dict(sections=(4, 4, 0, 0, 0)),
               dict(sections=(-1, 9)), dict(sections=())):
        with pytest.raises(ValueError):
            attention.rotary_split(**{**ok, **kw})
    for kw in (dict(positions=pos.float()), dict(positions=pos.cpu()), dict(qkv=qkv.double())):
        with pytest.raises(TypeError):
            attention.rotary_split(**{**ok, **kw})
    g = t(2, 2, 5, 16)
    for dk, dv in ((t(2, 2, 4, 16), g), (g, t(2, 1, 5, 16)), (g, t(2, 2, 5, 16, dt=torch.float16))):
        with pytest.raises(ValueError):
            attention.rotary_merge(g, dk, dv, pos, turns, (4, 4))
    with pytest.raises(ValueError):
        attention.rotary_heads(t(5, 16), pos, turns, (4, 4))


def test_two_streams_at_once(cuda_device):
    """Calls in flight on two streams share nothing: each result is that of its own call."""
    from deep_optimization_b200 import gemm
    torch.manual_seed(8)
    pairs = [(torch.randn(1003, 771, device=cuda_device).bfloat16(), torch.randn(997, 771, device=cuda_device).bfloat16()) for _ in range(2)]
    want = []
    for x, w in pairs:
        y, d = gemm.linear_act(x, w, activation="gelu", derivative=True)
        dz, db = gemm.act_backward(y, d)
        want.append((y, d, dz, db, *gemm.linear_backward(dz, x, w)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, (x, w) in enumerate(pairs):
            with torch.cuda.stream(streams[i]):
                y, d = gemm.linear_act(x, w, activation="gelu", derivative=True)
                dz, db = gemm.act_backward(y, d)
                got[i] = (y, d, dz, db, *gemm.linear_backward(dz, x, w))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
