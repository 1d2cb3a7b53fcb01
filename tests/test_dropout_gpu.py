"""Dropout without a stored mask against the same counter generator in numpy.

Tolerance: the product with the survivors' factor and the sum with the residual are rounded to 24
bits each, the result to its type, every rounding off by at most half a step."""
import numpy as np
import pytest
import torch

from .philox import keep_mask

pytestmark = pytest.mark.gpu
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _codec():
    from deep_optimization_b200 import codec
    return codec


def _want(x, p, seed, offset, r=None, first=0):
    t = int(p * 65536.0 + 0.5)
    keep = torch.from_numpy(keep_mask(first, x.numel(), p, seed, offset)).view(x.shape)
    factor = 65536.0 / (65536 - t) if t < 65536 else 0.0
    y = torch.where(keep, x.double().cpu() * factor, torch.zeros((), dtype=torch.float64))
    size = y.abs()
    if r is not None:
        y = y + r.double().cpu()
        size = size + r.double().abs().cpu()
    return y, size


def _close(got, want, size):
    tol = want.abs() * torch.finfo(got.dtype).eps / 2 + size * 3 * 2.0 ** -24 + 2.0 ** -25
    if got.dtype == torch.float32:
        tol = want.abs() * 2.0 ** -24 + size * 3 * 2.0 ** -24
    assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 15, 16, 17, 31, 8191, 8192, 8193, 100003])
@pytest.mark.parametrize("residual", [False, True])
def test_against_numpy(cuda_device, dtype, n, residual):
    codec = _codec()
    g = torch.Generator().manual_seed(n)
    x, r = torch.randn(n, generator=g).to(dtype), torch.randn(n, generator=g).to(dtype)
    for p, seed, offset in ((0.1, 7, 0), (0.5, (1 << 64) - 3, (5 << 32) + 9), (0.973, 1 << 40, 12)):
        got = codec.dropout(x.to(cuda_device), p, (seed, offset), r.to(cuda_device) if residual else None)
        _close(got, *_want(x, p, seed, offset, r if residual else None))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [1, 3, 8])
def test_unaligned_base(cuda_device, dtype, shift):
    codec = _codec()
    base = torch.randn(5000, generator=torch.Generator().manual_seed(3)).to(dtype).to(cuda_device)
    x = base[shift:shift + 4001]
    r = base[:4001]
    _close(codec.dropout(x, 0.25, (11, 2), r), *_want(x.cpu(), 0.25, 11, 2, r.cpu()))


def test_probabilities_zero_and_one(cuda_device):
    codec = _codec()
    x = torch.randn(1003, device=cuda_device, dtype=torch.bfloat16)
    assert torch.equal(codec.dropout(x, 0.0, (1, 1)), x)
    assert torch.equal(codec.dropout(x, 1.0, (1, 1)), torch.zeros_like(x))
    assert torch.equal(codec.dropout(x, 1.0, (1, 1), x), x)
    assert codec.dropout(x[:0], 0.5, (1, 1)).shape == (0,)


@pytest.mark.parametrize("dtype", TYPES)
def test_dropped_elements_are_zero_whatever_they_hold(cuda_device, dtype):
    codec = _codec()
    n = 4099
    keep = torch.from_numpy(keep_mask(0, n, 0.5, 21, 4))
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.where(keep, 1.0, bad).to(dtype).to(cuda_device)
        y = codec.dropout(x, 0.5, (21, 4)).cpu()
        assert torch.equal(y, torch.where(keep, 2.0, 0.0).to(dtype))


def test_elements_past_32_bits(cuda_device):
    """The element number is 64 bits wide: the end of a tensor of 2^32 + 4099 elements."""
    codec = _codec()
    n = (1 << 32) + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device=cuda_device)
    y = codec.dropout(x, 0.5, (3, 1))
    tail = 8200
    keep = torch.from_numpy(keep_mask(n - tail, tail, 0.5, 3, 1))
    assert torch.equal(y[-tail:].cpu(), torch.where(keep, 2.0, 0.0).to(torch.bfloat16))


def test_numbers_from_the_device(cuda_device):
    codec = _codec()
    x = torch.randn(777, device=cuda_device)
    seed, offset = (1 << 63) + 5, (1 << 62) + 1
    rng = torch.tensor([seed - (1 << 64), offset], dtype=torch.int64, device=cuda_device)
    assert torch.equal(codec.dropout(x, 0.3, rng), codec.dropout(x, 0.3, (seed, offset)))


def test_in_another_layout_and_on_another_stream(cuda_device):
    codec = _codec()
    x = torch.randn(3, 40, 6, 5, device=cuda_device).to(memory_format=torch.channels_last)
    y = codec.dropout(x, 0.4, (5, 6))
    assert y.is_contiguous(memory_format=torch.channels_last)
    flat = x.permute(0, 2, 3, 1).reshape(-1)
    want, size = _want(flat.cpu(), 0.4, 5, 6)
    _close(y.permute(0, 2, 3, 1).reshape(-1), want, size)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = codec.dropout(x, 0.4, (5, 6))
    side.synchronize()
    assert torch.equal(y, z)


# ---------------------------------------------------------------- module

def _module(p):
    from deep_optimization_b200.modules.activations.act_layers import DODropout
    return DODropout(p).train()


@pytest.mark.parametrize("dtype", TYPES)
def test_module_gradient_is_the_forward_mask(cuda_device, dtype):
    drop = _module(0.3)
    x = torch.randn(37, 129, device=cuda_device, dtype=dtype, requires_grad=True)
    r = torch.randn(37, 129, device=cuda_device, dtype=dtype, requires_grad=True)
    y = drop(x, r)
    with torch.no_grad():
        kept = (y - r) != 0
    dy = torch.ones_like(y)
    dx, dr = torch.autograd.grad(y, (x, r), dy)
    factor = torch.tensor(65536.0 / (65536 - round(0.3 * 65536)), dtype=dtype)
    # where y - r rounds to nothing the element was tiny, not dropped
    sure = x.detach().abs() > 0.1
    assert torch.equal(dx[sure], torch.where(kept, factor.to(cuda_device), torch.zeros((), dtype=dtype, device=cuda_device))[sure])
    assert torch.equal(dr, dy)
    share = (dx == 0).float().mean().item()
    # 4773 draws: five standard deviations of the share
    assert abs(share - 0.3) < 5 * (0.3 * 0.7 / 4773) ** 0.5


def test_module_saves_no_tensor_and_follows_the_seed(cuda_device):
    drop = _module(0.5)
    x = torch.randn(64, 64, device=cuda_device, requires_grad=True)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        drop(x)
    assert not saved
    torch.manual_seed(5)
    a, b = drop(x), drop(x)
    torch.manual_seed(5)
    c = drop(x)
    assert torch.equal(a, c) and not torch.equal(a, b)


@pytest.mark.parametrize("reentrant", [False, True])
def test_module_under_checkpoint(cuda_device, reentrant):
    from torch.utils.checkpoint import checkpoint
    drop = _module(0.5)
    x = torch.randn(300, 33, device=cuda_device, requires_grad=True)
    w = torch.randn(300, 33, device=cuda_device)

    def block(v):
        return drop(v * w).square()

    torch.manual_seed(9)
    plain = torch.autograd.grad(block(x).sum(), x)[0]
    torch.manual_seed(9)
    y = checkpoint(block, x, use_reentrant=reentrant)
    again = x.detach().clone().requires_grad_()
    torch.manual_seed(9)
    checkpoint(block, again, use_reentrant=reentrant).sum().backward()
    assert torch.equal(plain, again.grad)
    del y


def test_module_shapes_types_and_eval(cuda_device):
    drop = _module(0.5)
    x = torch.randn(4, 6, device=cuda_device, dtype=torch.bfloat16)
    # a residual of another type or shape is added the ordinary way, with its promotion
    assert drop(x, torch.zeros(4, 6, device=cuda_device)).dtype == torch.float32
    assert drop(x, torch.zeros(6, device=cuda_device, dtype=torch.bfloat16)).shape == (4, 6)
    drop.eval()
    assert torch.equal(drop(x), x) and torch.equal(drop(x, x), x + x)


def test_captured_step_draws_new_masks_and_keeps_its_gradient(cuda_device):
    drop = _module(0.5)
    x = torch.randn(64, 256, device=cuda_device, requires_grad=True)
    drop(x)                                              # outside the capture: the stream of numbers
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            y = drop(x)
            (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        graphs.append(g)
        outs.append((y, dx))
    seen = []
    for g, (y, dx) in list(zip(graphs, outs)) * 2:
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, (y != 0).float() * 2.0)
        seen.append(y.detach().clone() != 0)
    for i in range(4):
        for j in range(i):
            assert not torch.equal(seen[i], seen[j])


def test_controller_swaps_dropout_on_request(cuda_device):
    from torch import nn
    from deep_optimization_b200.controller import Controller
    from deep_optimization_b200.modules.activations.act_layers import DODropout
    cfg = {"default_bits": 2, "group_size": 256, "batch_size": 8, "compress_dropout": True}
    make = lambda: nn.Sequential(nn.Linear(64, 64), nn.Dropout(0.2), nn.Linear(64, 8))
    c = Controller(make(), cfg, input_shape=(64,), test=False, device=cuda_device)
    assert type(c.traced_model.get_submodule("1")) is DODropout and c.traced_model.get_submodule("1").p == 0.2
    out = c.traced_model(torch.randn(8, 64, device=cuda_device))
    out.sum().backward()
    cfg.pop("compress_dropout")
    c = Controller(make(), cfg, input_shape=(64,), test=False, device=cuda_device)
    assert type(c.traced_model.get_submodule("1")) is nn.Dropout
