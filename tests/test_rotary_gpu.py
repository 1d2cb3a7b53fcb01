"""Rotary positions with several axes against the rotation in 64 bits.

Tolerance: cos and sin are within 2^-23 (a rounding each of the angle's fraction and of the result),
two products and a sum of 24 bits, then the rounding to the type, half a step.  The frequencies and the
reference's angle are float64: five roundings of 2^-53 of the angle, at most |pos| radians, between them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _attn():
    from deep_optimization_b200.modules import attention
    return attention


def _want(x, pos, sections, base=10000.0, interleaved=False, sign=1.0):
    """x [B, H, T, D] (CPU), pos [T, A] or [B, T, A]; the result and the size of what is summed, float64."""
    x = x.double()
    pos = pos.double()
    if pos.dim() == 2:
        pos = pos.expand(x.shape[0], *pos.shape)
    f = torch.cat([torch.tensor([base ** (-i / n) for i in range(n)], dtype=torch.float64) for n in sections if n] or [torch.zeros(0, dtype=torch.float64)])
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angle = sign * torch.remainder(pos[..., axis] * f, 2.0 * math.pi).unsqueeze(1)
    c, s = torch.cos(angle), torch.sin(angle)
    P = f.numel()
    i = torch.arange(P)
    i1, i2 = (2 * i, 2 * i + 1) if interleaved else (i, i + P)
    y, size = x.clone(), x.abs()
    y[..., i1] = x[..., i1] * c - x[..., i2] * s
    y[..., i2] = x[..., i2] * c + x[..., i1] * s
    size[..., i1] = size[..., i2] = x[..., i1].abs() + x[..., i2].abs()
    return y, size


def _close(got, want, size, far=1000):
    tol = want.abs() * torch.finfo(got.dtype).eps / 2 + size * (2.0 ** -21 + 5 * 2.0 ** -53 * (far + 1000)) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert ((got.double().cpu() - want).abs() <= tol).all()


def _inputs(B, T, H, K, D, dtype, dev, axes, far=0, batch_pos=False, pos_dtype=torch.int64, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, T, (H + 2 * K) * D, generator=g).to(dtype)
    pos = torch.randint(-40, 1000, ((B, T, axes) if batch_pos else (T, axes)), generator=g) + far
    return qkv, pos.to(pos_dtype)


CASES = [
    # B, T, H, K, D, sections, interleaved
    (2, 197, 12, 12, 64, (16, 16), False),
    (1, 1, 4, 1, 128, (64,), False),
    (3, 17, 6, 2, 80, (8, 12, 12), True),
    (2, 33, 4, 4, 72, (5, 4, 9), False),              # pair count no multiple of a vector
    (2, 5, 2, 1, 36, (3, 3, 3, 3), True),
    (1, 9, 3, 3, 7, (1, 2), False),                   # an odd head
    (2, 6, 2, 2, 64, (0, 0, 8), False),               # axes without pairs
    (1, 300, 40, 8, 96, (24, 24), True),              # more work items than threads
    (2, 4, 2, 2, 32, (0,), False),                    # nothing to turn
    (1, 3, 1, 1, 1024, (256, 256), False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("far", [0, 10 ** 9])
def test_split_and_merge(cuda_device, dtype, case, far):
    a = _attn()
    B, T, H, K, D, sections, inter = case
    qkv, pos = _inputs(B, T, H, K, D, dtype, cuda_device, len(sections), far)
    turns = a.rotary_turns(sections, device=cuda_device)
    q, k, v = a.rotary_split(qkv.to(cuda_device), H, pos.to(cuda_device), turns, sections, K, inter)
    x = qkv.view(B, T, H + 2 * K, D).transpose(1, 2)
    _close(q, *_want(x[:, :H], pos, sections, interleaved=inter), far)
    _close(k, *_want(x[:, H:H + K], pos, sections, interleaved=inter), far)
    assert torch.equal(v.cpu(), x[:, H + K:])
    g = torch.Generator().manual_seed(1)
    dq, dk, dv = (torch.randn(B, n, T, D, generator=g).to(dtype) for n in (H, K, K))
    back = a.rotary_merge(dq.to(cuda_device), dk.to(cuda_device), dv.to(cuda_device), pos.to(cuda_device), turns, sections, inter)
    b = back.view(B, T, H + 2 * K, D).transpose(1, 2)
    _close(b[:, :H], *_want(dq, pos, sections, interleaved=inter, sign=-1.0), far)
    _close(b[:, H:H + K], *_want(dk, pos, sections, interleaved=inter, sign=-1.0), far)
    assert torch.equal(b[:, H + K:].cpu(), dv)


@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_positions_per_batch_and_strided(cuda_device, pos_dtype):
    a = _attn()
    sections = (8, 8)
    qkv, pos = _inputs(3, 21, 2, 2, 32, torch.float32, cuda_device, 2, batch_pos=True, pos_dtype=pos_dtype)
    turns = a.rotary_turns(sections, device=cuda_device)
    q, _, _ = a.rotary_split(qkv.to(cuda_device), 2, pos.to(cuda_device), turns, sections)
    x = qkv.view(3, 21, 6, 32).transpose(1, 2)
    _close(q, *_want(x[:, :2], pos, sections))
    # the same numbers in another memory order
    turned = pos.to(cuda_device).permute(2, 1, 0).contiguous().permute(2, 1, 0)
    assert not turned.is_contiguous()
    q2, _, _ = a.rotary_split(qkv.to(cuda_device), 2, turned, turns, sections)
    assert torch.equal(q, q2)


@pytest.mark.parametrize("dtype", TYPES)
def test_any_strides_and_bases(cuda_device, dtype):
    a = _attn()
    sections = (8, 8)
    turns = a.rotary_turns(sections, device=cuda_device)
    pos = torch.randint(0, 50, (19, 2), generator=torch.Generator().manual_seed(2))
    big = torch.randn(2, 3, 40, 67, generator=torch.Generator().manual_seed(3)).to(dtype)
    for x in (big[:, :, ::2, :64][:, :, :19], big[:, :, :19, 3:67], big.transpose(1, 2)[:, :3, :, :64][:, :, :3],
              big.permute(0, 1, 3, 2)[:, :, :19, :40], big[:1, :, :19, :64].expand(4, 3, 19, 64)):
        t = x.shape[2]
        got = a.rotary_heads(x.to(cuda_device) if x.is_contiguous() else _same_strides(x, cuda_device), pos[:t].to(cuda_device), turns, sections)
        assert got.is_contiguous()
        _close(got, *_want(x, pos[:t], sections))


def _same_strides(x, dev):
    span = sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1
    flat = torch.as_strided(x, (x.storage_offset() + span,), (1,), 0).to(dev)
    return torch.as_strided(flat, x.shape, x.stride(), x.storage_offset())


def test_turning_back_and_empty(cuda_device):
    a = _attn()
    sections = (8, 4)
    turns = a.rotary_turns(sections, device=cuda_device)
    x = torch.randn(2, 3, 11, 32, device=cuda_device)
    pos = torch.randint(0, 2 ** 40, (11, 2), device=cuda_device)
    y = a.rotary_heads(a.rotary_heads(x, pos, turns, sections), pos, turns, sections, inverse=True)
    # two turns, each within the tolerance above, of pairs of norm at most |x1| + |x2|
    assert ((y - x).abs() <= 2.0 ** -19 * x.abs().amax()).all()
    assert torch.equal(a.rotary_heads(x, torch.zeros_like(pos), turns, sections), x)
    for shape in ((0, 3, 5, 32), (2, 3, 0, 32)):
        z = torch.empty(shape, device=cuda_device)
        assert a.rotary_heads(z, pos[:shape[2]], turns, sections).shape == shape


def test_module_gradients(cuda_device):
    """Against autograd through the 64-bit rotation, and against differences."""
    a = _attn()
    B, T, H, K, D = 2, 10, 4, 2, 40
    rope = a.RotaryAxes((6, 10), interleaved=True).to(cuda_device)
    pos = a.image_positions(3, 3, 1, cuda_device)
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(B, T, (H + 2 * K) * D, generator=g).to(cuda_device).requires_grad_()
    wq, wk, wv = (torch.randn(B, n, T, D, generator=g).to(cuda_device) for n in (H, K, K))
    q, k, v = rope(qkv, H, pos, K)
    loss = (q * wq).sum() + (k * wk).sum() + (v * wv).sum()
    (grad,) = torch.autograd.grad(loss, qkv, retain_graph=True)
    ref = qkv.detach().double().cpu().requires_grad_()
    x = ref.view(B, T, H + 2 * K, D).transpose(1, 2)
    turned = [_turn64(x[:, :H], pos.cpu(), (6, 10)), _turn64(x[:, H:H + K], pos.cpu(), (6, 10)), x[:, H + K:]]
    (want,) = torch.autograd.grad(sum((t * w.double().cpu()).sum() for t, w in zip(turned, (wq, wk, wv))), ref)
    assert (grad.double().cpu() - want).abs().max() <= 2.0 ** -19 * want.abs().max()
    # a difference along one direction: the map is linear, so the quotient has no error of its own
    step = torch.randn(qkv.shape, generator=g).to(cuda_device)
    with torch.no_grad():
        q2, k2, v2 = rope(qkv + step, H, pos, K)
        diff = ((q2 - q) * wq).double().sum() + ((k2 - k) * wk).double().sum() + ((v2 - v) * wv).double().sum()
    along = (grad.double() * step.double()).sum()
    size = (grad.double().abs() * step.double().abs()).sum()
    assert (diff - along).abs() <= 2.0 ** -18 * size + 2.0 ** -20 * qkv.numel() ** 0.5 * 10
    # only one of the three used downstream
    (gv,) = torch.autograd.grad((rope(qkv, H, pos, K)[2] * wv).sum(), qkv)
    assert torch.equal(gv.view(B, T, -1, D)[:, :, H + K:].transpose(1, 2), wv) and (gv.view(B, T, -1, D)[:, :, :H + K] == 0).all()


def _turn64(x, pos, sections):
    f = torch.cat([torch.tensor([10000.0 ** (-i / n) for i in range(n)], dtype=torch.float64) for n in sections])
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angle = pos.double()[:, axis] * f
    P = f.numel()
    a, b = x[..., 0:2 * P:2], x[..., 1:2 * P:2]
    c, s = torch.cos(angle), torch.sin(angle)
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., 2 * P:]], -1)


def test_single_tensor_module_gradient(cuda_device):
    a = _attn()
    rope = a.RotaryAxes((16,)).to(cuda_device)
    pos = torch.arange(6, device=cuda_device).view(6, 1)
    x = torch.randn(1, 2, 6, 32, device=cuda_device, requires_grad=True)
    w = torch.randn(1, 2, 6, 32, device=cuda_device)
    (g,) = torch.autograd.grad((rope.turn(x, pos) * w).sum(), x)
    _close(g, *_want(w.cpu(), pos.cpu(), (16,), sign=-1.0))


def test_captured_and_on_another_stream(cuda_device):
    a = _attn()
    rope = a.RotaryAxes((16, 16)).to(cuda_device)
    pos = a.image_positions(7, 7, 1, cuda_device)
    qkv = torch.randn(2, 50, 3 * 2 * 64, device=cuda_device, dtype=torch.bfloat16)
    eager = rope(qkv, 2, pos)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = rope(qkv, 2, pos)
    qkv.neg_()
    g.replay()
    torch.cuda.synchronize()
    for x, y in zip(held, eager):
        assert torch.equal(x, -y)
