"""The fully connected layer and the 8-bit activation checkpoints, as cases that can be timed and compared.

Kinds of case:

* ``linear`` -- y = act(x W^T + b) + r without gradients, as a serving program calls it;
* ``train``  -- the same layer forward and backward: y and the gradients of x, W, b and r.  What the backward pass needs of the
  pre-activation z is kept from the forward pass in the layer's own 16-bit type (``bits`` = 16), or x and z are kept in 8 bits
  (``bits`` = 8);
* ``pack``   -- a tensor packed into 8 bits and unpacked again.

Eight bits: 32 neighbours of the last dimension share a power of two, the smallest that brings the largest of them within
e4m3's 448, and are rounded to e4m3 (half to even).

Where ``own`` is true, ``run`` calls the framework; else it computes the same in elementary operations.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32


def _linear(name, rows, k, n, dtype, act, bias=True, residual=False, kind="linear", bits=16):
    case = {"kind": kind, "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "residual": residual, "bits": bits}
    return case if name is None else dict(case, name=name)


def _pack(name, rows, k, dtype):
    case = {"kind": "pack", "rows": rows, "k": k, "dtype": dtype}
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # one token through an output projection with the skip connection: latency, one pass over the weights
        _linear("linear_1x4096x4096_bf16", 1, 4096, 4096, "bf16", "none", residual=True),
        # a batch of users, one token each, into a wide feed-forward layer
        _linear("linear_24x4096x16384_f16", 24, 4096, 16384, "f16", "gelu_tanh"),
        # a short ragged prompt, an odd number of outputs
        _linear("linear_509x1000x1531_f16", 509, 1000, 1531, "f16", "silu", residual=True),
        # the features of 256 images into a classifier's hidden layer
        _linear("linear_256x25088x4096_f16", 256, 25088, 4096, "f16", "relu"),
        # a long prompt into a wide feed-forward layer: the largest case
        _linear("linear_8192x4096x16384_bf16", 8192, 4096, 16384, "bf16", "gelu"),
        # a training step of a feed-forward layer
        _linear("train_4096x2048x8192_bf16", 4096, 2048, 8192, "bf16", "gelu_tanh", kind="train"),
        # a small ragged step whose rows do not start on 16 bytes
        _linear("train_333x500x750_f16", 333, 500, 750, "f16", "silu", residual=True, kind="train"),
        # the same step as above with both activations kept in 8 bits
        _linear("train8_4096x2048x8192_bf16", 4096, 2048, 8192, "bf16", "gelu_tanh", kind="train", bits=8),
        # the way back to the model's width, with the skip connection, ragged
        _linear("train8_1111x1000x776_f16", 1111, 1000, 776, "f16", "relu", residual=True, kind="train", bits=8),
        # one layer's activations of a long batch
        _pack("pack_8192x4096_bf16", 8192, 4096, "bf16"),
        # odd rows whose last block is short
        _pack("pack_1001x777_f16", 1001, 777, "f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of 8, as networks have them; one in four as it comes."""
    c = _log_int(rng, lo, hi)
    return c if rng.random() < 0.25 else (c + 7) // 8 * 8


def draw(rng):
    """Rows from one to 8192, widths from 64 to 16384, at most the largest listed case's multiplications."""
    dtype = rng.choice(("f16", "bf16"))
    kind = rng.choice(("linear", "linear", "train", "train8", "pack"))
    if kind == "pack":
        return _pack(None, _log_int(rng, 1, 8192), _width(rng, 20, 8192), dtype)
    act = rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu"))
    rows, k, n = _log_int(rng, 1, 8192), _width(rng, 64, 16384), _width(rng, 64, 16384)
    most = 8192 * 4096 * 16384 // (1 if kind == "linear" else 3)
    rows = max(1, min(rows, most // (k * n)))
    if kind == "linear":
        return _linear(None, rows, k, n, dtype, act, rng.random() < 0.8, rng.random() < 0.5)
    return _linear(None, rows, k, n, dtype, act, rng.random() < 0.8, rng.random() < 0.5, "train", 8 if kind == "train8" else 16)


def prepare(case, seed):
    """Activations of unit size with a few channels that stand out, weights of a trained layer's size, small gradients."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale)

    rows, k = case["rows"], case["k"]
    loud = torch.where(torch.rand(k, generator=gen, device="cuda") < 0.01, 8.0, 1.0)
    state = {"case": dict(case), "x": (normal(rows, k) * loud).to(dtype)}
    if case["kind"] == "pack":
        return state
    n = case["n"]
    state["w"] = normal(n, k, scale=k ** -0.5).to(dtype)
    state["b"] = normal(n, scale=0.1).to(dtype) if case["bias"] else None
    state["r"] = normal(rows, n).to(dtype) if case["residual"] else None
    if case["kind"] == "train":
        state["gy"] = normal(rows, n, scale=0.01).to(dtype)
        for name in ("x", "w", "b", "r"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


def work(case):
    rows, k = case["rows"], case["k"]
    if case["kind"] == "pack":
        return {"bytes": rows * k * (2 + 2) + 2 * rows * k + 2 * rows * -(-k // BLOCK), "flops": 4 * rows * k}
    n = case["n"]
    forward = 2 * (rows * k + n * k + rows * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0))
    if case["kind"] == "linear":
        return {"bytes": forward, "flops": 2 * rows * k * n}
    # x, W, r, gy in; y, dx, dW, db out; what is kept of x and z is written and read again
    kept = 0 if case["act"] == "none" else rows * n * 2
    if case["bits"] == 8:
        kept = rows * k + (0 if case["act"] == "none" else rows * n)
    backward = 2 * (rows * n + rows * k + n * k + (n if case["bias"] else 0))
    return {"bytes": forward + backward + 2 * kept, "flops": 6 * rows * k * n}


# ---- plain form --------------------------------------------------------------------------------------------------------
def _act(z, name):
    if name == "relu":
        return z * (z > 0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _eight(x, dtype):
    """x (f32) as eight bits hold it, and the blocks' powers of two."""
    rows, k = x.shape
    blocks = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(rows, -1, BLOCK)
    m, e = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    e = torch.where(m > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -127)).clamp_min(-127)
    q = torch.ldexp(blocks, -e).to(torch.float8_e4m3fn).float()
    most = torch.finfo(dtype).max
    values = torch.ldexp(q, e).clamp(-most, most).reshape(rows, -1)[:, :k]
    return values, torch.ldexp(torch.ones_like(m), e).squeeze(-1)


def _plain(state):
    case = state["case"]
    dtype, act = DTYPES[case["dtype"]], case.get("act")
    with torch.no_grad():
        x = state["x"].float()
        if case["kind"] == "pack":
            values, scale = _eight(x, dtype)
            return {"values": values.to(dtype), "scale": scale}
        w = state["w"].float()
        z = x @ w.t()
        if case["bias"]:
            z = z + state["b"].float()
        y = _act(z, act)
        if case["residual"]:
            y = y + state["r"].float()
        y = y.to(dtype)
        if case["kind"] == "linear":
            return {"y": y}
        gy = state["gy"].float()
        if case["bits"] == 8:
            x, z = _eight(x, dtype)[0], _eight(z, dtype)[0]
        else:
            z = z.to(dtype).float()
        dz = gy * _slope(z, act)
        out = {"y": y, "dx": (dz @ w).to(dtype), "dw": (dz.t() @ x).to(dtype)}
        if case["bias"]:
            out["db"] = dz.sum(0).to(dtype)
        if case["residual"]:
            out["dr"] = gy.to(dtype)
        return out


def run(state):
    if not own:
        return _plain(state)
    from pytorch_winoconv_b200 import checkpoint, linear

    case = state["case"]
    if case["kind"] == "pack":
        q, scale = checkpoint.pack(state["x"])
        return {"values": checkpoint.unpack(q, scale, state["x"].dtype), "scale": scale.float()}
    act = None if case["act"] == "none" else case["act"]
    if case["kind"] == "linear":
        return {"y": linear.linear(state["x"], state["w"], state["b"], state["r"], activation=act)}
    y = linear.linear(state["x"], state["w"], state["b"], state["r"], activation=act, checkpoint="e4m3" if case["bits"] == 8 else None)
    wanted = {"d" + name: state[name] for name in ("x", "w", "b", "r") if state[name] is not None}
    return {"y": y.detach(), **dict(zip(wanted, torch.autograd.grad(y, list(wanted.values()), state["gy"])))}


# ---- in 64 bits --------------------------------------------------------------------------------------------------------
def _eight64(x, dtype):
    """The same from the definition: the exponent from a logarithm, the rounding as a division by the step at each value."""
    rows, k = x.shape
    values, scale = torch.zeros_like(x), torch.zeros(rows, -(-k // BLOCK), dtype=torch.float64, device=x.device)
    for c in range(0, k, BLOCK):
        part = x[:, c:c + BLOCK]
        top = part.abs().amax(1, keepdim=True)
        log = torch.log2(top.clamp_min(1e-300))
        low = torch.floor(log)
        low = torch.where(torch.exp2(low + 1) <= top, low + 1, torch.where(torch.exp2(low) > top, low - 1, low))
        e = (low - 8 + (top > 1.75 * torch.exp2(low)).double()).clamp_min(-127)
        v = part * torch.exp2(-e)
        at = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
        at = torch.where(torch.exp2(at) > v.abs().clamp_min(2.0 ** -6), at - 1, at)
        step = torch.exp2(at - 3)
        values[:, c:c + BLOCK] = torch.round(v / step) * step * torch.exp2(e)
        scale[:, c // BLOCK] = torch.exp2(e).squeeze(1)
    most = torch.finfo(dtype).max
    return values.clamp(-most, most), scale


def exact(case, seed):
    state = prepare(case, seed)
    dtype = DTYPES[case["dtype"]]
    x = state["x"].detach().double()
    if case["kind"] == "pack":
        values, scale = _eight64(x, dtype)
        return {"values": values, "scale": scale}
    f = torch.nn.functional
    act = {"none": lambda t: t, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh"), "silu": f.silu}[case["act"]]
    w = state["w"].detach().double()
    z = torch.einsum("mk,nk->mn", x, w)
    if case["bias"]:
        z += state["b"].detach().double()
    y = act(z)
    if case["residual"]:
        y = y + state["r"].detach().double()
    if case["kind"] == "linear":
        return {"y": y}
    if case["bits"] == 8:
        x, z = _eight64(x, dtype)[0], _eight64(z, dtype)[0]
    else:
        z = z.to(dtype).double()
    gy = state["gy"].double()
    z.requires_grad_()
    dz, = torch.autograd.grad(act(z), z, gy)
    out = {"y": y, "dx": torch.einsum("mn,nk->mk", dz, w), "dw": torch.einsum("mn,mk->nk", dz, x)}
    if case["bias"]:
        out["db"] = dz.sum(0)
    if case["residual"]:
        out["dr"] = gy
    return out
