"""What is measured of the training operators: the gated recurrence, the learned route with its balance loss, the
clipped policy loss and the clipping of gradients by their global norm.

``run`` computes one pass of a case: with ``own`` false in plain form (elementary torch operations in 32 bits, rounded
once at the end), with ``own`` true through the package's fronts, as a training program calls them. A case with
``train`` true is forward and backward; the others are the forward of inference or evaluation.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LOW, HIGH = 2.0 ** -8, 1.0 - 2.0 ** -8          # the recurrence's retention bounds
CLIP_LOW, CLIP_HIGH, KL_WEIGHT = 0.2, 0.28, 0.04


def listed():
    return [
        # one decode step of the recurrence: 256 streams of a d = 2048 model, no history beyond the carried state
        dict(name="recurrence-step", op="recurrence", batch=256, length=1, features=2048, dtype="bf16", masks=False, train=False),
        # a prefill window of 64 streams, 128 positions each, padded at the right; fp32 projections as the GEMM emits them
        dict(name="recurrence-window", op="recurrence", batch=64, length=128, features=2048, dtype="f32", masks=True, train=False),
        # a training batch of packed documents (restarts inside the rows)
        dict(name="recurrence-train", op="recurrence", batch=8, length=4096, features=1024, dtype="bf16", masks=True, train=True),
        # one long document: few rows, so the work has to be split over the length
        dict(name="recurrence-long", op="recurrence", batch=1, length=32768, features=2048, dtype="bf16", masks=False, train=True),
        # a ragged small model: odd width, odd length, half precision
        dict(name="recurrence-odd", op="recurrence", batch=3, length=1777, features=515, dtype="f16", masks=True, train=True),
        # the route of one decode step: 256 tokens, 64 experts
        dict(name="route-step", op="route", tokens=256, experts=64, top_k=2, dtype="f32", renormalize=False, masks=False, train=False),
        # the route of a training batch of 8 x 4096 tokens
        dict(name="route-train", op="route", tokens=32768, experts=64, top_k=2, dtype="f32", renormalize=False, masks=True, train=True),
        # many small experts, 16-bit logits (so ties are common), renormalised weights, a ragged token count
        dict(name="route-odd", op="route", tokens=10007, experts=122, top_k=5, dtype="bf16", renormalize=True, masks=True, train=True),
        # policy tuning of the byte-vocabulary model: rows of 257 logits, which no vector load fits
        dict(name="policy-bytes", op="policy", batch=16, length=256, vocabulary=257, dtype="f32", train=True),
        # policy tuning of the hybrid-vocabulary model: the bf16 logits of 8 answers of 1024 tokens
        dict(name="policy-vocabulary", op="policy", batch=8, length=1024, vocabulary=32768, dtype="bf16", train=True),
        # the gradients of a 12-block d = 128 model without experts in one flat fp32 buffer: 144 small tensors
        dict(name="clip-small", op="clip", layers=12, width=128, experts=0, dtype="f32", flat=True),
        # the gradients of one d = 2048 block with 16 experts, each tensor by itself, bf16
        dict(name="clip-block", op="clip", layers=1, width=2048, experts=16, dtype="bf16", flat=False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "route", "policy", "clip"])
    if op == "recurrence":
        features = _spread(rng, 48, 4096)
        if rng.random() < 0.6:
            features = max(64, features // 64 * 64)
        dtype = rng.choice(["bf16", "f16", "f32"])
        most = (1 << 27) // DTYPES[dtype].itemsize  # elements
        length = min(_spread(rng, 1, 32768), most // features)
        batch = max(1, min(_spread(rng, 1, 256), most // (length * features)))
        return dict(op=op, batch=batch, length=length, features=features, dtype=dtype,
                    masks=rng.random() < 0.5, train=rng.random() < 0.7)
    if op == "route":
        experts = _spread(rng, 4, 256)
        return dict(op=op, tokens=_spread(rng, 1, 65536), experts=experts, top_k=min(experts, rng.randint(1, 8)),
                    dtype=rng.choice(["f32", "bf16", "f16"]), renormalize=rng.random() < 0.5, masks=rng.random() < 0.5,
                    train=rng.random() < 0.7)
    if op == "policy":
        vocabulary = _spread(rng, 257, 131072)
        if rng.random() < 0.6:
            vocabulary = max(320, vocabulary // 64 * 64)
        batch = rng.randint(1, 16)
        length = max(1, min(_spread(rng, 1, 2048), (1 << 27) // (batch * vocabulary)))
        return dict(op=op, batch=batch, length=length, vocabulary=vocabulary, dtype=rng.choice(["bf16", "f16", "f32"]),
                    train=rng.random() < 0.7)
    flat = rng.random() < 0.5
    case = dict(op="clip", layers=1, width=_spread(rng, 40, 1024), experts=rng.randint(0, 8), dtype=rng.choice(["bf16", "f32"]), flat=flat)
    most = max(1, (1 << 27) // sum(math.prod(s) for s in _shapes(case)))
    return dict(case, layers=min(most, rng.randint(1, 16) if flat else rng.randint(1, 3)))


def _shapes(case):
    """The parameter shapes of ``layers`` HERM blocks of ``width`` with ``experts`` experts (16 memory features)."""
    d, e = case["width"], case["experts"]
    block = [(d,), (2 * d, d), (2 * d,), (3 * d + 2, d), (3 * d + 2,), (16, d), (16,), (2 * d, d), (2 * d,), (d, 4 * d), (d,), (d,)]
    if e:
        block += [(e, 2 * d, d), (e, 2 * d), (e, 2 * d, d), (e, 2 * d), (e, d, 2 * d), (e, d), (d,), (e, d)]
    return block * case["layers"]


def _padding(batch, length, generator):
    """Right padding: sequences between half and all of ``length`` long."""
    lengths = torch.randint((length + 1) // 2, length + 1, (batch, 1), generator=generator, device="cuda")
    return torch.arange(length, device="cuda") < lengths


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if op == "recurrence":
        batch, length, features = case["batch"], case["length"], case["features"]
        state = {"case": case, "projections": (1.5 * normal(batch, length, 2 * features)).to(dtype),
                 "initial": normal(batch, features).tanh(), "valid": None, "restart": None}
        if case["masks"]:
            state["valid"] = _padding(batch, length, g)
            if case["train"]:  # packed documents of about 500 tokens
                state["restart"] = torch.rand(batch, length, generator=g, device="cuda") < 1 / 500
        if case["train"]:
            state["projections"].requires_grad_(True)
            state["initial"].requires_grad_(True)
            state["grad_states"] = normal(batch, length, features).to(dtype)
            state["grad_final"] = normal(batch, features)
        return state
    if op == "route":
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        state = {"case": case, "logits": (normal(tokens, experts) + 0.5 * normal(experts)).to(dtype), "valid": None}
        if case["masks"]:
            state["valid"] = torch.rand(tokens, generator=g, device="cuda") < 0.9
        if case["train"]:
            state["logits"].requires_grad_(True)
            state["grad_weights"] = normal(tokens, top_k)
            state["grad_balance"] = torch.full((), 0.01, device="cuda")
        return state
    if op == "policy":
        batch, length, vocabulary = case["batch"], case["length"], case["vocabulary"]
        logits = torch.empty(batch, length, vocabulary, dtype=dtype, device="cuda")
        targets = torch.empty(batch, length, dtype=torch.int64, device="cuda")
        log_probs = torch.empty(batch, length, device="cuda")
        for row in range(batch):  # the answers were sampled from (nearly) this policy
            values = (2.5 * normal(length, vocabulary)).to(dtype)
            noise = torch.rand(length, vocabulary, generator=g, device="cuda").clamp_(1e-20, 1 - 1e-7)
            logits[row] = values
            targets[row] = (values.float() - torch.log(-torch.log(noise))).argmax(-1)
            log_probs[row] = torch.log_softmax(values.float(), -1).gather(-1, targets[row].unsqueeze(-1)).squeeze(-1)
        drift = 0.2 * normal(batch, length)
        for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):  # a ratio is hardly ever on the edge itself
            drift = torch.where((drift - edge).abs() < 1e-3, edge + 2e-3, drift)
        state = {"case": case, "logits": logits.requires_grad_(case["train"]), "targets": targets, "old": log_probs - drift,
                 "reference": log_probs + 0.1 * normal(batch, length), "advantages": 0.25 + normal(batch, length),
                 "valid": _padding(batch, length, g)}
        # half precision is trained with a scaled loss: its gradients would underflow otherwise
        state["scale"] = torch.full((), 32.0 * batch * length if dtype == torch.float16 else 1.0, device="cuda")
        return state
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    if case["flat"]:
        flat, out = (0.02 * normal(sum(sizes))).to(dtype), torch.zeros(sum(sizes), dtype=dtype, device="cuda")
        return {"case": case, "gradients": [t.view(s) for t, s in zip(flat.split(sizes), shapes)], "flat": out,
                "out": [t.view(s) for t, s in zip(out.split(sizes), shapes)]}
    gradients = [(0.02 * normal(*s)).to(dtype) for s in shapes]
    return {"case": case, "gradients": gradients, "out": [torch.zeros_like(t) for t in gradients]}


def run(state):
    return {"recurrence": _recurrence, "route": _route, "policy": _policy, "clip": _clip}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the gated recurrence

def _affine_scan(a, b):
    """h_t = a_t h_{t-1} + b_t by doubling: after the round of step s every pair covers 2 s positions. Its rounds are
    log2(length) whole-array operations; one operation for the whole scan does not exist among the elementary ones."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat((b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]), 1)
        a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return b


def _recurrence(state):
    case = state["case"]
    train = case["train"]
    if own:
        from koemi_5hom_b200.cuda_kernels.dense import gated_recurrence

        with torch.set_grad_enabled(train):
            states, final = gated_recurrence(state["projections"], state["initial"], valid=state["valid"],
                                             restart=state["restart"], minimum_retention=LOW, maximum_retention=HIGH)
        if not train:
            return states, final
        grads = torch.autograd.grad((states, final), (state["projections"], state["initial"]),
                                    (state["grad_states"], state["grad_final"]))
        return states.detach(), final.detach(), *grads
    with torch.no_grad():
        dtype = state["projections"].dtype
        p, c = state["projections"].float().chunk(2, -1)
        s, k = torch.sigmoid(p), torch.tanh(c)
        a = LOW + (HIGH - LOW) * s
        increment = (1 - a) * k
        if state["valid"] is not None:
            valid = state["valid"].unsqueeze(-1)
            a, increment = torch.where(valid, a, 1.0), torch.where(valid, increment, 0.0)
        carry = a if state["restart"] is None else torch.where(state["restart"].unsqueeze(-1), 0.0, a)
        b = increment.clone()
        b[:, 0] += carry[:, 0] * state["initial"]
        h = _affine_scan(carry, b)
        if not train:
            return h.to(dtype), h[:, -1].clone()
        # the adjoint is the same scan from the end: adj_t = g_t + carry_{t+1} adj_{t+1}
        g = state["grad_states"].float().clone()
        g[:, -1] += state["grad_final"]
        later = torch.cat((carry[:, 1:], torch.zeros_like(carry[:, :1])), 1)
        adjoint = _affine_scan(later.flip(1), g.flip(1)).flip(1)
        before = torch.cat((state["initial"].unsqueeze(1), h[:, :-1]), 1)
        if state["restart"] is not None:
            before = torch.where(state["restart"].unsqueeze(-1), 0.0, before)
        dp = adjoint * (before - k) * ((HIGH - LOW) * s * (1 - s))
        dc = adjoint * (1 - a) * (1 - k * k)
        if state["valid"] is not None:
            dp, dc = torch.where(valid, dp, 0.0), torch.where(valid, dc, 0.0)
        return h.to(dtype), h[:, -1].clone(), torch.cat((dp, dc), -1).to(dtype), carry[:, 0] * adjoint[:, 0]


def _recurrence_exact(state):
    """Position by position in 64 bits."""
    case = state["case"]
    x = state["projections"].detach().double()
    features, length = case["features"], case["length"]
    s = 1 / (1 + torch.exp(-x[..., :features]))
    k = torch.tanh(x[..., features:])
    a = LOW + (HIGH - LOW) * s
    ones = torch.ones(case["batch"], length, dtype=torch.bool, device="cuda")
    valid = (ones if state["valid"] is None else state["valid"]).unsqueeze(-1)
    restart = (~ones if state["restart"] is None else state["restart"]).unsqueeze(-1)
    retain = torch.where(valid, a, 1.0) * (~restart)
    gain = torch.where(valid, (1 - a) * k, 0.0)
    h = torch.empty_like(a)
    running = state["initial"].detach().double()
    for t in range(length):
        running = retain[:, t] * running + gain[:, t]
        h[:, t] = running
    if not case["train"]:
        return h, running
    grad = state["grad_states"].double()
    dp, dc = torch.empty_like(a), torch.empty_like(a)
    incoming = state["grad_final"].double()
    for t in range(length - 1, -1, -1):
        adjoint = grad[:, t] + incoming
        dp[:, t], dc[:, t] = adjoint, adjoint
        incoming = retain[:, t] * adjoint
    before = torch.cat((state["initial"].detach().double().unsqueeze(1), h[:, :-1]), 1) * (~restart)
    dp *= valid * (before - k) * (HIGH - LOW) * s * (1 - s)
    dc *= valid * (1 - a) * (1 - k * k)
    return h, running, torch.cat((dp, dc), -1), incoming


# ------------------------------------------------------------------ the learned route

def _route(state):
    case = state["case"]
    train, top_k, renormalize = case["train"], case["top_k"], case["renormalize"]
    if own:
        from koemi_5hom_b200.cuda_kernels.moe import route_learned_topk

        with torch.set_grad_enabled(train):
            route = route_learned_topk(state["logits"], state["valid"], top_k=top_k, renormalize=renormalize)
        outputs = (route.expert_ids, route.weights.detach(), route.counts, route.balance_loss.detach())
        if not train:
            return outputs
        return *outputs, *torch.autograd.grad((route.weights, route.balance_loss), (state["logits"],),
                                              (state["grad_weights"], state["grad_balance"]))
    with torch.no_grad():
        logits = state["logits"].float()
        tokens, experts = logits.shape
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top_k]
        chosen = p.gather(-1, ids)
        total = chosen.sum(-1, keepdim=True)
        weights = chosen / total if renormalize else chosen
        if state["valid"] is None:
            count = torch.full((), float(tokens), device="cuda")
            mask = torch.ones(tokens, 1, dtype=torch.bool, device="cuda")
        else:
            mask = state["valid"].unsqueeze(-1)
            count = mask.sum().float()
        ids, weights = torch.where(mask, ids, -1), torch.where(mask, weights, 0.0)
        counts = torch.zeros(experts, dtype=torch.int64, device="cuda")
        counts.scatter_add_(0, ids.clamp_min(0).reshape(-1), mask.expand_as(ids).reshape(-1).long())
        load = counts / counts.sum().clamp_min(1)
        importance = torch.where(mask, p, 0.0).sum(0) / count.clamp_min(1)
        balance = experts * (importance * load).sum()
        if not train:
            return ids, weights, counts, balance
        grad = state["grad_weights"]
        if renormalize:
            grad = (grad - (grad * weights).sum(-1, keepdim=True)) / total
        dp = (state["grad_balance"] * experts / count.clamp_min(1) * load).expand(tokens, experts).clone()
        dp.scatter_add_(1, ids.clamp_min(0), grad)
        dlogits = torch.where(mask, p * (dp - (p * dp).sum(-1, keepdim=True)), 0.0)
        return ids, weights, counts, balance, dlogits.to(state["logits"].dtype)


def _route_exact(state):
    """Row by row definitions in 64 bits; the gradient through the softmax's Jacobian."""
    case = state["case"]
    x = state["logits"].detach().double()
    tokens, experts = x.shape
    p = torch.softmax(x, -1)
    rank = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
    live = torch.ones(tokens, dtype=torch.bool, device="cuda") if state["valid"] is None else state["valid"]
    one_hot = torch.zeros(tokens, experts, dtype=torch.float64, device="cuda").scatter_(1, rank, 1.0) * live.unsqueeze(-1)
    raw = p.gather(1, rank)
    norm = raw.sum(1, keepdim=True) if case["renormalize"] else torch.ones_like(raw[:, :1])
    weights = raw / norm * live.unsqueeze(-1)
    counts = one_hot.sum(0)
    alive = max(1, int(live.sum()))
    share = counts / counts.sum().clamp_min(1)
    balance = experts * ((p * live.unsqueeze(-1)).sum(0) / alive * share).sum()
    ids = torch.where(live.unsqueeze(-1), rank, -1)
    if not case["train"]:
        return ids, weights, counts.long(), balance
    gw = state["grad_weights"].double()
    if case["renormalize"]:
        gw = (gw - (gw * raw / norm).sum(1, keepdim=True)) / norm
    slope = torch.zeros_like(p).scatter_(1, rank, gw) + float(state["grad_balance"]) * experts / alive * share
    grad = (slope - (slope * p).sum(1, keepdim=True)) * p * live.unsqueeze(-1)
    return ids, weights, counts.long(), balance, grad


# ------------------------------------------------------------------ the policy loss

def _policy(state):
    train = state["case"]["train"]
    if own:
        from koemi_5hom_b200.cuda_kernels.think import policy_loss

        with torch.set_grad_enabled(train):
            result = policy_loss(state["logits"], state["targets"], state["old"], state["advantages"],
                                 reference_log_probs=state["reference"], valid_mask=state["valid"], clip_low=CLIP_LOW,
                                 clip_high=CLIP_HIGH, kl_weight=KL_WEIGHT)
        outputs = (result.loss.detach(), result.kl, result.log_probs)
        return (*outputs, *torch.autograd.grad(result.loss, (state["logits"],), (state["scale"],))) if train else outputs
    with torch.no_grad():
        logits = state["logits"].float()
        valid, advantages = state["valid"], state["advantages"]
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        total = e.sum(-1, keepdim=True)
        target = state["targets"].unsqueeze(-1)
        log_probs = (logits.gather(-1, target) - logits.amax(-1, keepdim=True) - torch.log(total)).squeeze(-1)
        ratio = torch.exp(log_probs - state["old"])
        free = ratio * advantages
        clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * advantages
        gap = state["reference"] - log_probs
        kl = torch.exp(gap) - gap - 1
        count = valid.sum().clamp_min(1)
        loss = torch.where(valid, KL_WEIGHT * kl - torch.minimum(free, clipped), 0.0).sum() / count
        outputs = (loss, torch.where(valid, kl, 0.0).sum() / count, torch.where(valid, log_probs, 0.0))
        if not train:
            return outputs
        slope = torch.where(free <= clipped, -free, 0.0) + KL_WEIGHT * (1 - torch.exp(gap))
        slope = torch.where(valid, slope * (state["scale"] / count), 0.0).unsqueeze(-1)
        dlogits = e * (-slope / total)
        dlogits.scatter_add_(-1, target, slope)
        return *outputs, dlogits.to(state["logits"].dtype)


def _policy_exact(state):
    """Sequence by sequence in 64 bits."""
    count = max(1, int(state["valid"].sum()))
    loss = divergence = 0.0
    log_probs, grads = [], []
    for row in range(state["targets"].shape[0]):
        lp = torch.log_softmax(state["logits"][row].detach().double(), -1)
        target, live = state["targets"][row], state["valid"][row]
        chosen = lp.gather(1, target.unsqueeze(1)).squeeze(1)
        advantage, old, reference = (state[n][row].double() for n in ("advantages", "old", "reference"))
        r = torch.exp(chosen - old)
        bounded = torch.clamp(r, 1 - CLIP_LOW, 1 + CLIP_HIGH)
        kl = torch.expm1(reference - chosen) - (reference - chosen)
        loss += float((live * (KL_WEIGHT * kl - torch.minimum(r * advantage, bounded * advantage))).sum())
        divergence += float((live * kl).sum())
        log_probs.append(chosen * live)
        if state["case"]["train"]:
            d = -r * advantage * (r * advantage <= bounded * advantage) - KL_WEIGHT * torch.expm1(reference - chosen)
            d = (d * live * float(state["scale"]) / count).unsqueeze(1)
            grads.append((-d * torch.exp(lp)).scatter_add_(1, target.unsqueeze(1), d))
    outputs = (torch.tensor(loss / count, dtype=torch.float64), torch.tensor(divergence / count, dtype=torch.float64), torch.stack(log_probs))
    return (*outputs, torch.stack(grads)) if grads else outputs


# ------------------------------------------------------------------ the clipping of gradients

MAX_NORM = 1.0


def _clip(state):
    flat = state["case"]["flat"]
    if own:
        from koemi_5hom_b200.cuda_kernels.core import clip_gradients

        norm = clip_gradients(state["gradients"], MAX_NORM, out=state["out"])
        return (norm, state["flat"]) if flat else (norm, *state["out"])
    values = torch.cat([g.reshape(-1) for g in state["gradients"]]).float()
    norm = torch.sqrt((values * values).sum())
    scaled = (values * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)).to(state["gradients"][0].dtype)
    if flat:
        return norm, scaled
    pieces = scaled.split([g.numel() for g in state["gradients"]])
    return norm, *[p.view(g.shape) for p, g in zip(pieces, state["gradients"])]


def _clip_exact(state):
    square = torch.stack([g.double().square().sum() for g in state["gradients"]]).sum()
    norm = torch.sqrt(square)
    factor = min(1.0, MAX_NORM / (float(norm) + 1e-6))
    if state["case"]["flat"]:
        return norm, torch.cat([g.double().reshape(-1) * factor for g in state["gradients"]])
    return norm, *[g.double() * factor for g in state["gradients"]]


# ------------------------------------------------------------------ what a pass needs

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"recurrence": _recurrence_exact, "route": _route_exact, "policy": _policy_exact, "clip": _clip_exact}[case["op"]](state)


def work(case):
    op, train = case["op"], case.get("train", False)
    size = DTYPES[case["dtype"]].itemsize
    if op == "recurrence":
        lanes = case["batch"] * case["features"]
        elements = lanes * case["length"]
        flags = case["batch"] * case["length"] * (case["masks"] * (1 + train))
        # forward: projections in, states out; backward: projections and states' gradient in, projections' gradient out
        return {"bytes": elements * size * (3 + 5 * train) + lanes * 8 * (1 + train) + flags * (1 + train), "flops": elements * (15 + 40 * train)}
    if op == "route":
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        forward = tokens * experts * size + tokens * top_k * 12 + tokens * case["masks"] + experts * 8
        backward = 2 * tokens * experts * size + tokens * top_k * 12
        return {"bytes": forward + train * backward, "flops": tokens * experts * (8 + 8 * train)}
    if op == "policy":
        rows = case["batch"] * case["length"]
        return {"bytes": rows * case["vocabulary"] * size * (1 + train) + rows * 25, "flops": rows * case["vocabulary"] * (5 + 3 * train)}
    elements = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": 2 * elements * size, "flops": 3 * elements}
