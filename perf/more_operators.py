"""What is measured of the feed-forward sub-layer's operators: layer norm, dropout from a counter-based generator with a
residual added, and the gated feed-forward block.

``run`` computes one pass of a case: with ``own`` false in plain form (elementary torch operations in 32 bits, rounded
once at the end), with ``own`` true through the package's fronts, as a training or serving program calls them. A case
with ``train`` true is forward and backward; the others are the forward of inference.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NORM_EPS = 1e-5
GOLDEN, MIX_1, MIX_2 = 0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB  # SplitMix64


def listed():
    return [
        # the norm of one decode step: 256 streams of a d = 2048 model
        dict(name="norm-step", op="norm", rows=256, width=2048, dtype="bf16", weights="same", bias=True, train=False),
        # a training batch of 8 x 4096 tokens, its scale and shift kept in fp32
        dict(name="norm-train", op="norm", rows=32768, width=2048, dtype="bf16", weights="f32", bias=True, train=True),
        # a ragged batch of an odd width: rows that no vector load fits
        dict(name="norm-odd", op="norm", rows=10007, width=1021, dtype="f16", weights="same", bias=False, train=True),
        # wide rows in fp32, few of them
        dict(name="norm-wide", op="norm", rows=2048, width=16384, dtype="f32", weights="same", bias=True, train=True),
        # a training batch of the byte-vocabulary model (d = 128)
        dict(name="dropout-small", op="dropout", rows=4096, width=128, dtype="f32", p=0.1, residual=True, train=True),
        # 8 x 4096 tokens of a d = 2048 block, the sub-layer's output dropped out and added to the residual stream
        dict(name="dropout-train", op="dropout", rows=32768, width=2048, dtype="bf16", p=0.1, residual=True, train=True),
        # an odd number of values, no residual, half of them dropped
        dict(name="dropout-odd", op="dropout", rows=10007, width=1021, dtype="f16", p=0.5, residual=False, train=True),
        # one token of one stream: latency, and every weight once
        dict(name="block-single", op="block", rows=1, width=2048, hidden=4096, dtype="bf16", bias=True, train=False),
        # one decode step of 256 streams
        dict(name="block-step", op="block", rows=256, width=2048, hidden=4096, dtype="bf16", bias=True, train=False),
        # a training batch of 8 x 4096 tokens
        dict(name="block-train", op="block", rows=32768, width=2048, hidden=4096, dtype="bf16", bias=False, train=True),
        # the byte-vocabulary model (d = 128) in fp32
        dict(name="block-small", op="block", rows=4096, width=128, hidden=256, dtype="f32", bias=True, train=True),
        # a ragged batch of an odd model in half precision
        dict(name="block-odd", op="block", rows=1777, width=515, hidden=1030, dtype="f16", bias=True, train=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "block", "block"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "block":
        width, hidden = _spread(rng, 32, 4096), _spread(rng, 32, 8192)
        if rng.random() < 0.6:
            width, hidden = max(32, width // 32 * 32), max(32, hidden // 32 * 32)
        most = 32768 * 2048 * 4096 // (8 if dtype == "f32" else 1)
        rows = max(1, min(_spread(rng, 1, 32768), most // (width * hidden)))
        return dict(op=op, rows=rows, width=width, hidden=hidden, dtype=dtype, bias=rng.random() < 0.5, train=rng.random() < 0.6)
    width = _spread(rng, 16, 16384)
    if rng.random() < 0.6:
        width = max(16, width // 32 * 32)
    rows = max(1, min(_spread(rng, 1, 262144), (1 << 26) // width))
    if op == "norm":
        return dict(op=op, rows=rows, width=width, dtype=dtype, weights=rng.choice(["same", "f32"]), bias=rng.random() < 0.7,
                    train=rng.random() < 0.7)
    return dict(op=op, rows=rows, width=width, dtype=dtype, p=rng.choice([0.02, 0.1, 0.25, 0.5]), residual=rng.random() < 0.6,
                train=rng.random() < 0.8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, width, train = case["op"], case["rows"], case["width"], case["train"]
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, kind=dtype):
        return (shift + scale * torch.randn(*shape, generator=g, device="cuda")).to(kind)

    state = {"case": case, "x": normal(rows, width)}
    if op == "norm":  # a residual stream: rows of different sizes, off centre
        state["x"] = (torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda")) * (0.2 + state["x"].float())).to(dtype)
        kind = torch.float32 if case["weights"] == "f32" else dtype
        state["weight"] = normal(width, scale=0.1, shift=1.0, kind=kind)
        state["bias"] = normal(width, scale=0.1, kind=kind) if case["bias"] else None
        leaves = ["x", "weight", "bias"]
    elif op == "dropout":
        state["residual"] = normal(rows, width) if case["residual"] else None
        # a seed, a place in the model and a step of the program
        state["numbers"] = (0x5DEECE66D * (seed + 1) % (1 << 62), seed % 48, seed % 1009)
        leaves = ["x", "residual"]
    else:
        hidden = case["hidden"]
        state["gate_weight"] = normal(hidden, width, scale=width ** -0.5)
        state["value_weight"] = normal(hidden, width, scale=width ** -0.5)
        state["output_weight"] = normal(width, hidden, scale=hidden ** -0.5)
        leaves = ["x", "gate_weight", "value_weight", "output_weight"]
        for name, size in (("gate_bias", hidden), ("value_bias", hidden), ("output_bias", width)):
            state[name] = normal(size, scale=0.1) if case["bias"] else None
            leaves.append(name)
    state["leaves"] = [n for n in leaves if state[n] is not None]
    if train:
        for name in state["leaves"]:
            state[name].requires_grad_(True)
        state["grad"] = normal(rows, width)
    return state


def run(state):
    call = {"norm": _norm, "dropout": _dropout, "block": _block}[state["case"]["op"]]
    if not own:
        with torch.no_grad():
            return call(state)
    train = state["case"]["train"]
    with torch.set_grad_enabled(train):
        y = call(state)
    if not train:
        return y
    return y.detach(), *torch.autograd.grad(y, [state[n] for n in state["leaves"]], state["grad"])


# ------------------------------------------------------------------ layer norm

def _norm(state):
    x, weight, bias = state["x"], state["weight"], state["bias"]
    if own:
        from koemi_5hom_b200.cuda_kernels.core import layer_norm

        return layer_norm(x, weight, bias, eps=NORM_EPS)
    dtype, kind = x.dtype, weight.dtype
    x, weight = x.float(), weight.float()
    centred = x - x.mean(-1, keepdim=True)
    inverse = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + NORM_EPS)
    unit = centred * inverse
    y = unit * weight
    if bias is not None:
        y = y + bias.float()
    if not state["case"]["train"]:
        return y.to(dtype)
    grad = state["grad"].float()
    inner = grad * weight
    dx = inverse * (inner - inner.mean(-1, keepdim=True) - unit * (inner * unit).mean(-1, keepdim=True))
    grads = [dx.to(dtype), (grad * unit).sum(0).to(kind)]
    if bias is not None:
        grads.append(grad.sum(0).to(kind))
    return y.to(dtype), *grads


def _norm_exact(state, x, weight, bias=None):
    deviation = x - x.sum(-1, keepdim=True) / x.shape[-1]
    y = deviation / torch.sqrt(deviation.square().sum(-1, keepdim=True) / x.shape[-1] + NORM_EPS) * weight
    return y if bias is None else y + bias


# ------------------------------------------------------------------ dropout

def _mix(z):
    """SplitMix64's finaliser; torch's int64 products wrap, its shifts carry the sign."""
    def signed(c):
        return c - (1 << 64) if c >> 63 else c

    z = z + signed(GOLDEN)
    z = (z ^ ((z >> 30) & ((1 << 34) - 1))) * signed(MIX_1)
    z = (z ^ ((z >> 27) & ((1 << 37) - 1))) * signed(MIX_2)
    return z ^ ((z >> 31) & ((1 << 33) - 1))


def _kept(count, numbers, dropped):
    """Which of ``count`` values stay: 16 bits each, four from every number of the generator."""
    seed, site, step = (torch.full((), v, dtype=torch.int64, device="cuda") for v in numbers)
    key = _mix(seed ^ _mix(site ^ _mix(step)))
    words = _mix(key + torch.arange((count + 3) // 4, device="cuda") * (GOLDEN - (1 << 64)))
    lanes = torch.stack([(words >> s) & 0xFFFF for s in (0, 16, 32, 48)], -1).reshape(-1)[:count]
    return lanes >= dropped


def _dropout(state):
    case, x, residual = state["case"], state["x"], state["residual"]
    if own:
        from koemi_5hom_b200.cuda_kernels.core import dropout

        seed, site, step = state["numbers"]
        return dropout(x, case["p"], seed=seed, site=site, step=step, residual=residual)
    dropped = int(math.floor(case["p"] * 65536 + 0.5))
    kept = _kept(x.numel(), state["numbers"], dropped).view(x.shape)
    scale = 65536 / (65536 - dropped)
    y = torch.where(kept, x.float() * scale, 0.0)
    if residual is not None:
        y = y + residual.float()
    if not case["train"]:
        return y.to(x.dtype)
    grads = [torch.where(kept, state["grad"].float() * scale, 0.0).to(x.dtype)]
    if residual is not None:
        grads.append(state["grad"].clone())
    return y.to(x.dtype), *grads


def _dropout_exact(state, x, residual=None):
    """The mask in unsigned numbers on the host."""
    def mix(z):
        z = z + np.uint64(GOLDEN)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(MIX_1)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(MIX_2)
        return z ^ (z >> np.uint64(31))

    dropped = round(state["case"]["p"] * 65536)
    with np.errstate(over="ignore"):
        seed, site, step = (np.array([v], dtype=np.uint64) for v in state["numbers"])
        key = mix(seed ^ mix(site ^ mix(step)))
        words = mix(key + np.arange((x.numel() + 3) // 4, dtype=np.uint64) * np.uint64(GOLDEN))
    factor = torch.from_numpy(words.view("<u2")[:x.numel()] >= dropped).to(x.device).view(x.shape).double() / (1 - dropped / 65536)
    return x * factor if residual is None else x * factor + residual


# ------------------------------------------------------------------ the gated feed-forward block

def _block(state):
    x, dtype = state["x"], state["x"].dtype
    if own:
        from koemi_5hom_b200.cuda_kernels.dense import gated_feed_forward

        return gated_feed_forward(x, state["gate_weight"], state["value_weight"], state["output_weight"],
                                  gate_bias=state["gate_bias"], value_bias=state["value_bias"], output_bias=state["output_bias"])
    x, wg, wv, wo = (state[n].float() for n in ("x", "gate_weight", "value_weight", "output_weight"))
    bias = state["gate_bias"] is not None
    gate, value = x @ wg.T, x @ wv.T
    if bias:
        gate, value = gate + state["gate_bias"].float(), value + state["value_bias"].float()
    sigmoid = torch.sigmoid(gate)
    active = gate * sigmoid
    hidden = active * value
    y = hidden @ wo.T
    if bias:
        y = y + state["output_bias"].float()
    if not state["case"]["train"]:
        return y.to(dtype)
    grad = state["grad"].float()
    inner = grad @ wo
    dgate, dvalue = inner * value * (sigmoid * (1 + gate * (1 - sigmoid))), inner * active
    grads = [dgate @ wg + dvalue @ wv, dgate.T @ x, dvalue.T @ x, grad.T @ hidden]
    if bias:
        grads += [dgate.sum(0), dvalue.sum(0), grad.sum(0)]
    return y.to(dtype), *[t.to(dtype) for t in grads]


def _block_exact(state, x, gate_weight, value_weight, output_weight, gate_bias=0.0, value_bias=0.0, output_bias=0.0):
    p = torch.einsum("rw,hw->rh", x, gate_weight) + gate_bias
    q = torch.einsum("rw,hw->rh", x, value_weight) + value_bias
    return torch.einsum("rh,wh->rw", p / (1 + torch.exp(-p)) * q, output_weight) + output_bias


# ------------------------------------------------------------------ what a pass needs

def exact(case, seed):
    """The definition in 64 bits, its gradients by automatic differentiation."""
    state = prepare(case, seed)
    leaves = [state[n].detach().double().requires_grad_(case["train"]) for n in state["leaves"]]
    definition = {"norm": _norm_exact, "dropout": _dropout_exact, "block": _block_exact}[case["op"]]
    with torch.set_grad_enabled(case["train"]):
        y = definition(state, **dict(zip(state["leaves"], leaves)))
    return (y.detach(), *torch.autograd.grad(y, leaves, state["grad"].double())) if case["train"] else y


def work(case):
    rows, width, train = case["rows"], case["width"], case["train"]
    size = DTYPES[case["dtype"]].itemsize
    values = rows * width
    if case["op"] == "norm":  # x in, y out; backward: y's gradient in, x's out; the weights and their gradients
        weights = width * (4 if case["weights"] == "f32" else size) * (1 + case["bias"])
        return {"bytes": values * size * (2 + 2 * train) + weights * (1 + train), "flops": values * (8 + 14 * train)}
    if case["op"] == "dropout":  # x and the residual in, y out; backward: y's gradient in, x's out (the residual's is y's)
        return {"bytes": values * size * (2 + case["residual"] + 2 * train), "flops": values * (2 + 2 * train)}
    hidden = case["hidden"]
    weights = 3 * width * hidden + case["bias"] * (2 * hidden + width)
    return {"bytes": ((2 + 2 * train) * values + (1 + train) * weights) * size, "flops": 6 * values * hidden * (1 + 2 * train)}
