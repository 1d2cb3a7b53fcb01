"""Cases of the operators of a transformer block between its norms: the matrix product with bias,
activation and residual in its epilogue, its backward, dropout whose mask is never stored, and
rotary positions with several axes on the q/k/v split.

`run` computes a case in its plain form (elementary torch operations in 32 bits) or, with `own`
set, through the calls a user of this package makes.  `exact` computes it once more from the
definition in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_DEV = "cuda"


# ------------------------------------------------------------------------------------- cases

def _linear(name, m, k, n, act, dtype="bf16", residual=False, derivative=False):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "act": act, "dtype": dtype, "residual": residual,
            "derivative": derivative}


def _backward(name, m, k, n, dtype="bf16"):
    return {"name": name, "op": "backward", "m": m, "k": k, "n": n, "dtype": dtype}


def _dropout(name, rows, cols, p, dtype="bf16", residual=False, train=True):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "p": p, "dtype": dtype, "residual": residual,
            "train": train}


def _rotary(name, b, frames, height, width, heads, kv_heads, dim, s0, s1, s2, dtype="bf16", interleaved=False, far=0,
            train=False):
    return {"name": name, "op": "rotary", "b": b, "frames": frames, "height": height, "width": width, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "s0": s0, "s1": s1, "s2": s2, "dtype": dtype,
            "interleaved": interleaved, "far": far, "train": train}


def listed():
    return [
        # one token through the fused q/k/v projection of ViT-B/16: latency
        _linear("linear one token", 1, 768, 2304, "none"),
        # one 224 x 224 image (197 tokens) through an attention's output projection and its skip
        _linear("linear one image + skip", 197, 768, 768, "none", dtype="fp16", residual=True),
        # a ragged classifier-like product: no size a multiple of eight
        _linear("linear ragged silu", 1003, 771, 997, "silu", residual=True, derivative=True),
        # the widening half of an MLP in training: the derivative is what the compressed layer saves
        _linear("linear mlp gelu train", 32768, 1024, 4096, "gelu", derivative=True),
        # backward of the ragged product
        _backward("backward ragged", 1003, 771, 997, dtype="fp16"),
        # backward of a 768 -> 2304 layer of ViT-B/16 at batch 256 (197 tokens each)
        _backward("backward batch 256", 50432, 768, 2304),
        # one token's hidden state: latency
        _dropout("dropout one token", 1, 768, 0.1, train=False),
        # hidden states of batch 256 in front of the skip, forward and backward
        _dropout("dropout batch 256 + skip", 50432, 768, 0.1, residual=True),
        # an odd fp32 tensor
        _dropout("dropout odd fp32", 2331, 1001, 0.3, dtype="fp32"),
        # q, k, v of one image, class token first: two axes, forward only
        _rotary("rotary one image", 1, 1, 14, 14, 12, 12, 64, 0, 16, 16),
        # a training batch of images, forward and backward
        _rotary("rotary batch 256 train", 256, 1, 14, 14, 12, 12, 64, 0, 16, 16, train=True),
        # video, three axes, shared key/value heads, part of the head rotated, far into a stream
        _rotary("rotary video", 2, 8, 23, 25, 16, 4, 80, 8, 12, 12, dtype="fp32", interleaved=True, far=1000003),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd_or_not(rng, v, step):
    """As it is (mostly odd sizes) or rounded up to a multiple of `step`, evenly."""
    return v if rng.random() < 0.5 else -(-v // step) * step


def draw(rng):
    op = rng.choice(("linear", "backward", "dropout", "rotary"))
    half = rng.choice(("bf16", "fp16"))
    if op in ("linear", "backward"):
        k, n = (_odd_or_not(rng, _log(rng, 64, 4064), 32) for _ in range(2))
        most = 2.7e11 / (2.0 * k * n * (2 if op == "backward" else 1))
        m = max(1, min(_log(rng, 1, 50432), int(most)))
        if op == "backward":
            return _backward("drawn", m, k, n, half)
        act = rng.choice(("none", "relu", "gelu", "gelu_erf", "silu"))
        # the smooth activations have a derivative to save; a ReLU's is the sign of its result
        return _linear("drawn", m, k, n, act, half, rng.random() < 0.5,
                       act not in ("none", "relu") and rng.random() < 0.7)
    if op == "dropout":
        cols = _odd_or_not(rng, _log(rng, 1, 8192), 8)
        rows = max(1, min(_log(rng, 1, 50432), 38000000 // cols))
        return _dropout("drawn", rows, cols, round(rng.uniform(0.01, 0.9), 3), rng.choice(("bf16", "fp16", "fp32")),
                        rng.random() < 0.5, rng.random() < 0.7)
    dim = rng.choice((32, 48, 64, 72, 80, 96, 128))
    pairs = rng.randint(3, dim // 2)
    s0, s1 = pairs // rng.randint(3, 6), pairs // 3
    kv = rng.choice((1, 2, 4, 6))
    heads = kv * rng.randint(1, 4)
    frames, height, width = rng.choice((1, 1, 3, 8)), _log(rng, 1, 40), _log(rng, 1, 40)
    most = 38000000 * 3 // ((frames * height * width + 1) * (heads + 2 * kv) * dim)
    return _rotary("drawn", max(1, min(_log(rng, 1, 256), most)), frames, height, width, heads, kv, dim, s0, s1,
                   pairs - s0 - s1, rng.choice(("bf16", "fp16", "fp32")), rng.random() < 0.4,
                   rng.choice((0, 0, 4099, 1000003)), rng.random() < 0.5)


# ------------------------------------------------------------------------------------ inputs

def _randn(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=_DEV) * scale).to(_TYPES[dtype])


def _turns(case, base=10000.0):
    """The frequency ladder of each axis, base ** (-i / n) radians per position, as 64-bit binary
    fractions of a turn: a product with an integer position that drops the carry out of bit 64 is
    the angle modulo a whole turn, however far the position."""
    out = []
    for n in (case["s0"], case["s1"], case["s2"]):
        out += [int(round(base ** (-i / n) / (2.0 * math.pi) * 2.0 ** 64)) for i in range(n)]
    return torch.tensor(out, dtype=torch.int64, device=_DEV)


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(int(seed) * 7919 + 11)
    dt = case.get("dtype")
    state = {"case": case}
    if case["op"] in ("linear", "backward"):
        m, k, n = case["m"], case["k"], case["n"]
        state["x"] = _randn((m, k), gen, dt)
        state["w"] = _randn((n, k), gen, dt, 1.0 / math.sqrt(k))
        if case["op"] == "linear":
            state["b"] = _randn((n,), gen, dt, 0.1)
            state["r"] = _randn((m, n), gen, dt) if case["residual"] else None
        else:
            state["dy"] = _randn((m, n), gen, dt)
            # derivatives of an activation: between a little below 0 and a little above 1
            state["d"] = (torch.rand((m, n), generator=gen, device=_DEV) * 1.2 - 0.1).to(_TYPES[dt])
    elif case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        state["x"] = _randn(shape, gen, dt)
        state["r"] = _randn(shape, gen, dt) if case["residual"] else None
        state["dy"] = _randn(shape, gen, dt) if case["train"] else None
        # the generator's key and the number of this call in its stream
        state["rng"] = (0x9E3779B97F4A7C15 ^ (int(seed) * 0x1000193), 5 + int(seed) % 97)
    else:
        b, h, kv, d = case["b"], case["heads"], case["kv_heads"], case["dim"]
        t = case["frames"] * case["height"] * case["width"] + 1
        state["qkv"] = _randn((b, t, (h + 2 * kv) * d), gen, dt)
        grid = torch.stack(torch.meshgrid(torch.arange(case["frames"]), torch.arange(case["height"]),
                                          torch.arange(case["width"]), indexing="ij"), -1).reshape(-1, 3)
        # the class token sits at the origin and is not turned
        state["pos"] = torch.cat([torch.zeros(1, 3, dtype=torch.int64), grid + case["far"] + 1]).to(_DEV)
        state["turns"] = _turns(case)
        state["sections"] = (case["s0"], case["s1"], case["s2"])
        if case["train"]:
            state["grads"] = [_randn((b, heads, t, d), gen, dt) for heads in (h, kv, kv)]
    return state


# -------------------------------------------------------------------------------- plain forms

_K = math.sqrt(2.0 / math.pi)


def _activation(z, act):
    """f(z) and, for the smooth activations, f'(z)."""
    if act == "none":
        return z, None
    if act == "relu":
        return z.clamp_min(0.0), None
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s + z * s * (1.0 - s)
    if act == "gelu":
        th = torch.tanh(_K * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * _K * (1.0 + 3 * 0.044715 * z * z)
    cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)


def _plain_linear(s):
    c = s["case"]
    z = s["x"].float() @ s["w"].float().t() + s["b"].float()
    y, d = _activation(z, c["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    y = y.to(s["x"].dtype)
    return (y, d.to(s["x"].dtype)) if c["derivative"] else y


def _plain_backward(s):
    dz = s["dy"].float() * s["d"].float()
    db = dz.sum(0)
    # the gradient of the pre-activation is handed on in the tensors' own type (it is returned, and
    # it is the operand that both products read)
    dz = dz.to(s["x"].dtype)
    dx = dz.float() @ s["w"].float()
    dw = dz.float().t() @ s["x"].float()
    return dz, db, dx.to(s["x"].dtype), dw.to(s["w"].dtype)


def _philox_words(blocks, key, offset):
    """Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
    2011) of the counters (block, offset) under a 64-bit key: four 32-bit words per block.  64-bit
    integers wrap, so the product of two 32-bit words keeps all its bits."""
    low = 0xFFFFFFFF
    c0, c1 = blocks & low, (blocks >> 32) & low
    c2, c3 = torch.full_like(c0, offset & low), torch.full_like(c0, (offset >> 32) & low)
    k0, k1 = key & low, (key >> 32) & low
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((q >> 32) & low) ^ c1 ^ k0, q & low, ((p >> 32) & low) ^ c3 ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], -1)


def _plain_dropout(x, p, rng, r):
    t = int(math.floor(p * 65536.0 + 0.5))          # the probability in 2**-16
    n = x.numel()
    words = _philox_words(torch.arange((n + 7) // 8, device=x.device), rng[0], rng[1])
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:n].view(x.shape)
    y = torch.where(halves >= t, x.float() * (65536.0 / (65536 - t)), 0.0)
    if r is not None:
        y = y + r.float()
    return y.to(x.dtype)


def _turn(x, cos, sin, pairs, interleaved):
    """x [B, H, T, D] with its first 2 * pairs elements turned by the angles [T, pairs]."""
    x = x.float()
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * pairs:]], -1)


def _angles(s):
    pairs = s["turns"].numel()
    axis = torch.repeat_interleave(torch.arange(3, device=_DEV), torch.tensor(s["sections"], device=_DEV), output_size=pairs)
    angle = (s["pos"][:, axis] * s["turns"]).double() * (2.0 * math.pi / 2.0 ** 64)
    return torch.cos(angle).float(), torch.sin(angle).float(), pairs


def _plain_rotary(s):
    c = s["case"]
    b, t, _ = s["qkv"].shape
    h, kv, d, inter = c["heads"], c["kv_heads"], c["dim"], c["interleaved"]
    cos, sin, pairs = _angles(s)
    x = s["qkv"].view(b, t, h + 2 * kv, d).transpose(1, 2)
    dt = s["qkv"].dtype
    out = [_turn(x[:, :h], cos, sin, pairs, inter).to(dt), _turn(x[:, h:h + kv], cos, sin, pairs, inter).to(dt),
           x[:, h + kv:]]
    if c["train"]:
        dq, dk, dv = s["grads"]
        back = torch.cat([_turn(dq, cos, -sin, pairs, inter).to(dt), _turn(dk, cos, -sin, pairs, inter).to(dt), dv], 1)
        out.append(back.transpose(1, 2).reshape(b, t, -1))
    return out


# -------------------------------------------------------------------------------------- calls

def run(state):
    c = state["case"]
    op = c["op"]
    if own:
        from deep_optimization_b200 import codec, gemm
        from deep_optimization_b200.modules import attention
        if op == "linear":
            return gemm.linear_act(state["x"], state["w"], state["b"], c["act"], residual=state["r"],
                                   derivative=c["derivative"])
        if op == "backward":
            dz, db = gemm.act_backward(state["dy"], state["d"])
            dx, dw = gemm.linear_backward(dz, state["x"], state["w"])
            return dz, db, dx, dw
        if op == "dropout":
            y = codec.dropout(state["x"], c["p"], state["rng"], residual=state["r"])
            return (y, codec.dropout(state["dy"], c["p"], state["rng"])) if c["train"] else y
        q, k, v = attention.rotary_split(state["qkv"], c["heads"], state["pos"], state["turns"], state["sections"],
                                         kv_heads=c["kv_heads"], interleaved=c["interleaved"])
        if not c["train"]:
            return [q, k, v]
        dq, dk, dv = state["grads"]
        return [q, k, v, attention.rotary_merge(dq, dk, dv, state["pos"], state["turns"], state["sections"],
                                                interleaved=c["interleaved"])]
    if op == "linear":
        return _plain_linear(state)
    if op == "backward":
        return _plain_backward(state)
    if op == "dropout":
        y = _plain_dropout(state["x"], c["p"], state["rng"], state["r"])
        return (y, _plain_dropout(state["dy"], c["p"], state["rng"], None)) if c["train"] else y
    return _plain_rotary(state)


# --------------------------------------------------------------------------------------- work

def work(case):
    """Every input read once, every output written once; the products' operations."""
    es = _BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": es * (m * k + n * k + n + m * n * (1 + case["residual"] + case["derivative"])),
                "flops": 2 * m * n * k}
    if case["op"] == "backward":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": es * (2 * m * n + m * k + n * k) + es * (m * n + m * k + n * k) + 4 * n, "flops": 4 * m * n * k}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": es * n * (2 + case["residual"] + 2 * case["train"]), "flops": 0}
    t = case["frames"] * case["height"] * case["width"] + 1
    n = case["b"] * t * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    return {"bytes": es * n * 2 * (1 + case["train"]), "flops": 0}


# ----------------------------------------------------------------------- the definition, 64 bits

def _exact_linear(s, c):
    z = torch.addmm(s["b"].double(), s["x"].double(), s["w"].double().mT)
    act = c["act"]
    if act == "none":
        y, d = z, None
    elif act == "relu":
        y, d = torch.maximum(z, torch.zeros_like(z)), None
    else:
        if act == "silu":
            g, dg = torch.sigmoid(z), lambda g: g * torch.sigmoid(-z)
        elif act == "gelu":                          # (1 + tanh u) / 2 is the logistic function of 2 u
            u = 2.0 * _K * z * (1.0 + 0.044715 * z.square())
            g, dg = torch.sigmoid(u), lambda g: g * torch.sigmoid(-u) * 2.0 * _K * (1.0 + 0.134145 * z.square())
        else:
            g, dg = 0.5 * torch.special.erfc(-z / math.sqrt(2.0)), lambda g: torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
        y, d = z * g, g + z * dg(g)
    if s["r"] is not None:
        y = y + s["r"].double()
    return (y, d) if c["derivative"] else y


def _exact_backward(s):
    product = torch.mul(s["dy"].double(), s["d"].double())
    handed_on = product.to(s["x"].dtype).double()
    return (product, torch.ones(1, product.shape[0], dtype=torch.float64, device=product.device).mm(product)[0],
            torch.mm(handed_on, s["w"].double()), torch.mm(handed_on.mT, s["x"].double()))


def _exact_mask(n, key, offset):
    """Philox-4x32-10 once more, in numpy's unsigned integers; the sixteen bits of each element."""
    mask32 = np.uint64(0xFFFFFFFF)
    x = np.zeros((4, (n + 7) // 8), dtype=np.uint64)
    x[0] = np.arange(x.shape[1], dtype=np.uint64)
    x[2], x[3] = offset % 2 ** 32, offset >> 32
    key = [key % 2 ** 32, key >> 32]
    for r in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        k = [np.uint64((key[0] + r * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + r * 0xBB67AE85) % 2 ** 32)]
        x = np.stack([(b >> np.uint64(32)) ^ x[1] ^ k[0], b & mask32, (a >> np.uint64(32)) ^ x[3] ^ k[1], a & mask32])
    return np.ascontiguousarray(x.T).astype("<u4").view("<u2").reshape(-1)[:n]


def _exact_dropout(s, c):
    t = int(math.floor(c["p"] * 65536 + 0.5))
    kept = torch.from_numpy((_exact_mask(s["x"].numel(), *s["rng"]) >= t)).to(_DEV).view(s["x"].shape)
    factor = kept.double() * 65536.0 / (65536.0 - t)
    y = s["x"].double() * factor
    if s["r"] is not None:
        y += s["r"].double()
    return (y, s["dy"].double() * factor) if c["train"] else y


def _exact_rotary(s, c, base=10000.0):
    b, t, _ = s["qkv"].shape
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    pos = s["pos"].cpu().numpy().astype(np.float64)
    z = np.concatenate([np.exp(1j * pos[:, a, None] * base ** (-np.arange(n) / max(n, 1)))
                        for a, n in enumerate((c["s0"], c["s1"], c["s2"]))], axis=1)
    z = torch.from_numpy(z).to(_DEV)
    pairs = z.shape[1]
    at = torch.arange(pairs, device=_DEV)
    first, second = (2 * at, 2 * at + 1) if c["interleaved"] else (at, at + pairs)

    def turned(x, w):                                # pairs as complex numbers, times e^(i angle)
        x = x.double().clone()
        v = torch.complex(x[..., first], x[..., second]) * w
        x[..., first], x[..., second] = v.real, v.imag
        return x

    q, k, v = s["qkv"].view(b, t, h + 2 * kv, d).permute(0, 2, 1, 3).split((h, kv, kv), 1)
    out = [turned(q, z), turned(k, z), v.double()]
    if c["train"]:
        dq, dk, dv = s["grads"]
        out.append(torch.cat([turned(dq, z.conj()), turned(dk, z.conj()), dv.double()], 1).permute(0, 2, 1, 3).reshape(b, t, -1))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(s, case)
    if case["op"] == "backward":
        return _exact_backward(s)
    if case["op"] == "dropout":
        return _exact_dropout(s, case)
    return _exact_rotary(s, case)
