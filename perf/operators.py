"""Cases of the operators around the layers of a mixture-of-experts decoder in training and serving: the gated norm that
joins a block to the residual stream, the router's balance loss, the token embedding and its gradient.

`run` computes them from elementary torch operations, or with `own` set through popcorn_b200."""

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decoding step of eight sequences: the norm between two blocks, latency alone
        dict(name="norm decode bf16", op="norm", direction="forward", batch=8, seq=1, hidden=4096, dtype="bf16", post=True, gate="channel",
             activation="identity", scale=1.0, residual_scale=1.0, offset=0.0),
        # a long prompt through a wide model, norms on both sides of the block
        dict(name="norm prefill bf16", op="norm", direction="forward", batch=2, seq=8192, hidden=8192, dtype="bf16", post=True, gate="none",
             activation="identity", scale=0.5, residual_scale=1.0, offset=1.0),
        # a training step with a learned gate per channel
        dict(name="norm train bf16", op="norm", direction="training", batch=4, seq=4096, hidden=4096, dtype="bf16", post=True, gate="channel",
             activation="identity", scale=1.0, residual_scale=0.7, offset=0.0),
        # an adaptive gate per sequence (its gradient sums over the sequence)
        dict(name="norm train adaptive fp16", op="norm", direction="training", batch=8, seq=2047, hidden=5120, dtype="fp16", post=True, gate="sequence",
             activation="tanh", scale=1.0, residual_scale=1.0, offset=0.0),
        # a gate per token, fp32, a width that no wide load divides
        dict(name="norm train odd fp32", op="norm", direction="training", batch=3, seq=1365, hidden=2050, dtype="fp32", post=False, gate="token",
             activation="sigmoid", scale=2.0, residual_scale=1.0, offset=0.0),
        # the router of a training step: the benchmark's own MoE sizes
        dict(name="balance train fp32", op="balance", direction="training", batch=16, seq=4096, experts=64, top_k=8, dtype="fp32", masked=False, per_sequence=False),
        # a padded batch with the loss taken sequence by sequence over many experts
        dict(name="balance sequences fp32", op="balance", direction="training", batch=32, seq=4001, experts=256, top_k=8, dtype="fp32", masked=True, per_sequence=True),
        # a small evaluation batch, few experts
        dict(name="balance eval bf16", op="balance", direction="forward", batch=1, seq=509, experts=8, top_k=2, dtype="bf16", masked=False, per_sequence=False),
        # one decoding step: 64 ids out of a large table
        dict(name="embedding decode bf16", op="embedding", direction="forward", batch=64, seq=1, vocab=131072, hidden=4096, dtype="bf16", scale=1.0, padded=False),
        # a training step over a small vocabulary: most rows of the gradient are hit
        dict(name="embedding train bf16", op="embedding", direction="training", batch=4, seq=4096, vocab=32000, hidden=4096, dtype="bf16", scale=64.0, padded=False),
        # a large one: frequent tokens, and a gradient whose rows are mostly zero
        dict(name="embedding large fp16", op="embedding", direction="training", batch=16, seq=4096, vocab=131072, hidden=4096, dtype="fp16", scale=1.0, padded=True),
        # odd sizes, fp32
        dict(name="embedding odd fp32", op="embedding", direction="training", batch=3, seq=2731, vocab=50257, hidden=1002, dtype="fp32", scale=31.0, padded=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "balance", "embedding"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    direction = rng.choice(("forward", "training", "training"))
    if op == "norm":
        hidden = _log(rng, 256, 8192)
        hidden = hidden if rng.random() < 0.2 else max(256, hidden // 64 * 64)
        rows = _log(rng, 1, min(32768, 16384 * 4096 // hidden))
        batch = rng.randint(1, min(rows, 16))
        return dict(op=op, direction=direction, batch=batch, seq=rows // batch, hidden=hidden, dtype=dtype, post=rng.random() < 0.7,
                    gate=rng.choice(("none", "channel", "sequence", "token")), activation=rng.choice(("identity", "tanh", "sigmoid")),
                    scale=rng.choice((1.0, 0.25)), residual_scale=rng.choice((1.0, 0.8)), offset=rng.choice((0.0, 1.0)))
    if op == "balance":
        experts = rng.choice((8, 16, 32, 64, 128, 256, 512, rng.randint(4, 300)))
        tokens = _log(rng, 1, min(131072, 131072 * 256 // experts))
        batch = rng.randint(1, min(tokens, 32))
        return dict(op=op, direction=direction, batch=batch, seq=tokens // batch, experts=experts, top_k=rng.randint(1, min(8, experts)),
                    dtype=rng.choice(("fp32", "fp32", dtype)), masked=rng.random() < 0.5, per_sequence=rng.random() < 0.5)
    hidden = _log(rng, 256, 8192)
    hidden = hidden if rng.random() < 0.2 else max(256, hidden // 64 * 64)
    vocab = _log(rng, 1000, min(262144, 131072 * 4096 // hidden))
    tokens = _log(rng, 1, min(65536, 65536 * 2048 // hidden))
    batch = rng.randint(1, min(tokens, 16))
    return dict(op=op, direction=direction, batch=batch, seq=tokens // batch, vocab=vocab, hidden=hidden, dtype=dtype,
                scale=rng.choice((1.0, 45.25)), padded=rng.random() < 0.5)


def _lengths(batch, seq, generator):
    """Lengths of the sequences of a padded batch: most are long, some may be empty."""
    share = torch.rand(batch, 1, generator=generator, device="cuda").sqrt()
    return torch.floor(share * (seq + 1)).clamp(max=seq)


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    batch, seq, dtype, training = case["batch"], case["seq"], TYPES[case["dtype"]], case["direction"] == "training"

    def normal(*shape, mean=0.0, std=1.0, dtype=dtype):
        return torch.randn(shape, generator=generator, device="cuda", dtype=dtype).mul_(std).add_(mean)

    if case["op"] == "norm":
        hidden = case["hidden"]
        state = dict(x=normal(batch, seq, hidden, std=2.0), residual=normal(batch, seq, hidden, std=3.0), weight=normal(hidden, mean=1.0 - case["offset"], std=0.1),
                     post_weight=normal(hidden, mean=1.0 - case["offset"], std=0.1) if case["post"] else None)
        shape = {"none": None, "channel": (hidden,), "sequence": (batch, 1, hidden), "token": (batch, seq, hidden)}[case["gate"]]
        state["gate"] = None if shape is None else normal(*shape, mean=0.5, std=0.5)
        leaves = [name for name in ("x", "residual", "weight", "post_weight", "gate") if state[name] is not None]
        if training:
            state["grads"] = (normal(batch, seq, hidden), normal(batch, seq, hidden))
    elif case["op"] == "balance":
        experts = case["experts"]
        # some experts are liked more than others, as in a router that needs the loss
        logits = (torch.randn((batch, seq, experts), generator=generator, device="cuda") + normal(experts, std=0.7, dtype=torch.float32)).to(dtype)
        state = dict(router_logits=logits, indices=logits.float().topk(case["top_k"], -1).indices.to(torch.int32), mask=None)
        if case["masked"]:
            state["mask"] = torch.arange(seq, device="cuda")[None] < _lengths(batch, seq, generator)
        leaves = ["router_logits"]
        if training:
            state["grads"] = (torch.full((), 0.01, device="cuda"), torch.full((), 0.001, device="cuda"))
    else:
        vocab, hidden = case["vocab"], case["hidden"]
        # token frequencies fall like one over their rank; ranks are scattered over the table
        rank = torch.exp(torch.rand((batch, seq), generator=generator, device="cuda", dtype=torch.float64) * math.log(vocab)).long() - 1
        ids = (rank.clamp(0, vocab - 1) * 7919 + 13) % vocab
        if case["padded"]:
            ids = torch.where(torch.arange(seq, device="cuda")[None] < _lengths(batch, seq, generator), ids, 0)
        state = dict(ids=ids, weight=normal(vocab, hidden, std=0.02))
        leaves = ["weight"]
        if training:
            state["grads"] = (normal(batch, seq, hidden),)
    if training:
        for name in leaves:
            state[name].requires_grad_(True)
    state["case"], state["leaves"] = case, leaves
    return state


def _run_own(state):
    from popcorn_b200 import autograd

    case = state["case"]
    if case["op"] == "norm":
        outputs = autograd.gated_add_rms_norm(state["x"], state["residual"], state["weight"], state["post_weight"], state["gate"], activation=case["activation"],
                                              scale=case["scale"], residual_scale=case["residual_scale"], eps=1e-6, offset=case["offset"])
    elif case["op"] == "balance":
        *outputs, counts = autograd.moe_balance_loss(state["router_logits"], state["indices"], state["mask"], per_sequence=case["per_sequence"])
    else:
        outputs = (autograd.embedding(state["ids"], state["weight"], scale=case["scale"], padding_idx=0 if case["padded"] else None),)
    result = {"out%d" % i: t.detach() for i, t in enumerate(outputs)}
    if case["op"] == "balance":
        result["counts"] = counts
    if case["direction"] == "training":
        grads = torch.autograd.grad(outputs, [state[name] for name in state["leaves"]], state["grads"])
        result.update({"grad_" + name: grad for name, grad in zip(state["leaves"], grads)})
    return result


def _gate(gate, activation):
    """The gate's factor and the factor's derivative."""
    if activation == "tanh":
        value = torch.tanh(gate)
        return value, 1 - value * value
    if activation == "sigmoid":
        value = torch.sigmoid(gate)
        return value, value * (1 - value)
    return gate, torch.ones_like(gate)


def _plain_norm(state):
    case, dtype = state["case"], state["x"].dtype
    x, residual, weight, post, gate = (None if state[n] is None else state[n].float() for n in ("x", "residual", "weight", "post_weight", "gate"))
    hidden, eps, offset, scale, residual_scale = x.shape[-1], 1e-6, case["offset"], case["scale"], case["residual_scale"]
    r1 = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    unit = x if post is None else x * r1
    n = unit if post is None else unit * (post + offset)
    act, slope = (1.0, None) if gate is None else _gate(gate, case["activation"])
    branch = scale * act
    s = residual_scale * residual + branch * n
    r2 = torch.rsqrt(s.square().mean(-1, keepdim=True) + eps)
    result = {"out0": (s * r2 * (weight + offset)).to(dtype), "out1": s.to(dtype)}
    if case["direction"] != "training":
        return result
    gy, gs = (g.float() for g in state["grads"])
    gw = gy * (weight + offset)
    ds = gs + r2 * gw - s * (r2 ** 3 * (gw * s).sum(-1, keepdim=True) / hidden)
    dn = branch * ds
    if post is None:
        dx = dn
    else:
        dw = dn * (post + offset)
        dx = r1 * dw - x * (r1 ** 3 * (dw * x).sum(-1, keepdim=True) / hidden)
        result["grad_post_weight"] = (dn * unit).sum((0, 1)).to(dtype)
    result.update(grad_x=dx.to(dtype), grad_residual=(residual_scale * ds).to(dtype), grad_weight=(gy * s * r2).sum((0, 1)).to(dtype))
    if gate is not None:
        dg = scale * slope * n * ds
        if case["gate"] == "channel":
            dg = dg.sum((0, 1))
        elif case["gate"] == "sequence":
            dg = dg.sum(1, keepdim=True)
        result["grad_gate"] = dg.to(dtype)
    return result


def _plain_balance(state):
    case = state["case"]
    logits, indices = state["router_logits"].float(), state["indices"].long()
    batch, seq, experts = logits.shape
    mask = torch.ones((batch, seq), device=logits.device) if state["mask"] is None else state["mask"].float()
    if not case["per_sequence"]:
        logits, indices, mask = logits.reshape(1, -1, experts), indices.reshape(1, batch * seq, -1), mask.reshape(1, -1)
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    p, lse = e / total, (top + torch.log(total))[..., 0]
    n = mask.sum(-1, keepdim=True)
    picks = torch.zeros((logits.shape[0], experts), device=logits.device)
    picks.scatter_add_(1, indices.flatten(1), mask.repeat_interleave(case["top_k"], dim=1))
    used = n.clamp(min=1)
    f = picks * experts / (used * case["top_k"])
    groups = (n > 0).sum().clamp(min=1)
    everything = n.sum().clamp(min=1)
    mean = (p * mask[..., None]).sum(1, dtype=torch.float64).float() / used
    counts = picks if case["per_sequence"] else picks[0]
    result = {"out0": (f * mean).sum() / groups, "out1": (lse.square() * mask).sum(dtype=torch.float64).float() / everything, "counts": counts.to(torch.int32)}
    if case["direction"] == "training":
        gb, gz = state["grads"]
        inner = (p * f[:, None]).sum(-1, keepdim=True)
        slope = gb / (groups * used)[..., None] * (f[:, None] - inner) + (2 * gz / everything * lse)[..., None]
        result["grad_router_logits"] = (p * slope * mask[..., None]).reshape(batch, seq, experts).to(state["router_logits"].dtype)
    return result


def _plain_embedding(state):
    case, ids, weight = state["case"], state["ids"], state["weight"].detach()
    result = {"out0": (case["scale"] * weight[ids].float()).to(weight.dtype)}
    if case["direction"] == "training":
        grad = state["grads"][0].float().reshape(-1, case["hidden"])
        if case["padded"]:
            grad = grad * (ids.reshape(-1, 1) != 0)
        total = torch.zeros(weight.shape, device=weight.device).index_add_(0, ids.reshape(-1), grad)
        result["grad_weight"] = (case["scale"] * total).to(weight.dtype)
    return result


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "balance": _plain_balance, "embedding": _plain_embedding}[state["case"]["op"]](state)


def work(case):
    size, tokens, training = 4 if case["dtype"] == "fp32" else 2, case["batch"] * case["seq"], case["direction"] == "training"
    if case["op"] == "norm":
        elements = tokens * case["hidden"]
        gate = {"none": 0, "channel": case["hidden"], "sequence": case["batch"] * case["hidden"], "token": elements}[case["gate"]]
        small = case["hidden"] * (2 if case["post"] else 1)
        return {"bytes": size * (8 if training else 4) * elements + size * (2 if training else 1) * (gate + small), "flops": (40 if training else 12) * elements}
    if case["op"] == "balance":
        elements = tokens * case["experts"]
        picks = 4 * tokens * case["top_k"] + (tokens if case["masked"] else 0)
        groups = case["batch"] if case["per_sequence"] else 1
        return {"bytes": size * (2 if training else 1) * elements + picks + 4 * groups * case["experts"], "flops": (18 if training else 8) * elements}
    # the table's rows are read once for each distinct id, about: the ids are drawn with a density of one over their rank
    vocab, hidden = case["vocab"], case["hidden"]
    steps = [math.exp(math.log(vocab) * i / 64) for i in range(65)]
    rows = sum((hi - lo) * (1 - (1 - min(1.0, math.log(1 + 1 / lo) / math.log(vocab))) ** tokens) for lo, hi in zip(steps, steps[1:]))
    rows = max(1, min(tokens, vocab, int(rows)))
    forward = 8 * tokens + size * hidden * (rows + tokens)
    return {"bytes": forward + (size * hidden * (tokens + vocab) if training else 0), "flops": (3 if training else 1) * tokens * hidden}


def _exact_norm(state, case):
    wide = {n: None if state[n] is None else state[n].detach().double().requires_grad_(True) for n in ("x", "residual", "weight", "post_weight", "gate")}
    x, gate = wide["x"], wide["gate"]

    def norm(t, weight):
        return t / torch.sqrt(torch.linalg.vector_norm(t, dim=-1, keepdim=True) ** 2 / t.shape[-1] + 1e-6) * (weight + case["offset"])

    branch = x if wide["post_weight"] is None else norm(x, wide["post_weight"])
    if gate is not None:
        branch = {"identity": lambda g: g, "tanh": torch.tanh, "sigmoid": torch.sigmoid}[case["activation"]](gate) * branch
    s = case["residual_scale"] * wide["residual"] + case["scale"] * branch
    return (norm(s, wide["weight"]), s), {}, wide


def _exact_balance(state, case):
    logits = state["router_logits"].detach().double().requires_grad_(True)
    batch, seq, experts = logits.shape
    keep = torch.ones((batch, seq), dtype=torch.bool, device=logits.device) if state["mask"] is None else state["mask"]
    p, lse = torch.softmax(logits, -1), torch.logsumexp(logits, -1)
    parts = [slice(b, b + 1) for b in range(batch)] if case["per_sequence"] else [slice(0, batch)]
    losses, counts = [], []
    for part in parts:
        kept = keep[part]
        picked = torch.bincount(state["indices"][part][kept].reshape(-1).long(), minlength=experts)
        counts.append(picked)
        if kept.any():
            share = picked.double() / picked.sum()
            losses.append(experts * (share * p[part][kept].mean(0)).sum())
    balance = sum(losses) / len(losses) if losses else logits.sum() * 0
    z = (lse[keep] ** 2).mean() if keep.any() else logits.sum() * 0
    counts = torch.stack(counts) if case["per_sequence"] else counts[0]
    return (balance, z), {"counts": counts.to(torch.int32)}, {"router_logits": logits}


def _exact_embedding(state, case):
    ids, weight = state["ids"], state["weight"].detach()
    outputs = {"out0": weight[ids].double() * case["scale"]}
    if case["direction"] == "training":
        grad = state["grads"][0].reshape(-1, case["hidden"])
        order = torch.argsort(ids.reshape(-1), stable=True)
        found, count = torch.unique_consecutive(ids.reshape(-1)[order], return_counts=True)
        ends = torch.cumsum(count, 0)
        total = torch.zeros(weight.shape, dtype=torch.float64, device=weight.device)
        for at in range(0, case["hidden"], 512):  # in columns, to keep the 64-bit sums small
            sums = torch.cumsum(torch.cat((torch.zeros_like(grad[:1, at:at + 512]), grad[order, at:at + 512])).double(), 0)
            total[found, at:at + 512] = case["scale"] * (sums[ends] - sums[ends - count])
        if case["padded"]:
            total[0] = 0
        outputs["grad_weight"] = total
    return outputs


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "embedding":
        return _exact_embedding(state, case)
    outputs, whole, wide = (_exact_norm if case["op"] == "norm" else _exact_balance)(state, case)
    result = {"out%d" % i: t.detach() for i, t in enumerate(outputs)}
    result.update(whole)
    if case["direction"] == "training":
        grads = torch.autograd.grad(outputs, [wide[n] for n in state["leaves"]], [g.double() for g in state["grads"]], allow_unused=True)
        result.update({"grad_" + n: torch.zeros_like(wide[n]) if g is None else g for n, g in zip(state["leaves"], grads)})
    return result
