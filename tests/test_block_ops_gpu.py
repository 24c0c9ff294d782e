"""The operators around the layers (gated norm, balance loss, embedding) against their definitions in 64 bits.

Tolerances: the kernels are fp32 up to one rounding of each output to T, so an output v may be off by half a step of T,
finfo(T).eps / 2 * |v|, plus the fp32 error of its chain, ROUNDINGS * 2^-24 * m, where m is the same expression with every
term replaced by its magnitude (what the rounding errors are relative to, whatever cancels)."""

import pytest
import torch

from popcorn_b200 import _lib, autograd, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# a thread adds at most 16384 / 256 = 64 values of a row one after the other, a row's threads meet in at most 10 steps, and an
# element's own chain has some 20 operations
ROUNDINGS = 96
TINY = {F32: 1e-40, F16: 2.0 ** -24, BF16: 1e-40}  # the step of the smallest numbers


def normal(seed, *shape, dtype=F32, std=1.0, mean=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * std + mean).to(dtype).to(DEV)


def near(got, want, magnitude, roundings=ROUNDINGS, what=""):
    dtype = got.dtype
    bound = torch.finfo(dtype).eps / 2 * want.abs() + roundings * 2.0 ** -24 * magnitude + TINY[dtype]
    off = (got.double() - want).abs()
    assert got.shape == want.shape, what
    assert bool((off <= bound).all()), f"{what}: off by up to {float((off / bound).max()):.2f} of what may be"


# ------------------------------------------------------------------------------------------------------------ gated norm --

ACT = {"identity": (lambda g: g, lambda v: torch.ones_like(v)), "tanh": (torch.tanh, lambda v: 1 - v * v), "sigmoid": (torch.sigmoid, lambda v: v * (1 - v))}


def norm_reference(x, residual, weight, post, gate, activation, scale, residual_scale, eps, offset, gy, gs):
    """Values and magnitudes of the outputs and gradients, by name, in 64 bits."""
    x, residual, weight, post, gate, gy, gs = (None if t is None else t.double() for t in (x, residual, weight, post, gate, gy, gs))
    n, lead = x.shape[-1], tuple(range(x.dim() - 1))
    mean = lambda t: t.sum(-1, keepdim=True) / n  # noqa: E731
    p = 1.0 if post is None else post + offset
    r1 = 1.0 if post is None else 1 / torch.sqrt(mean(x * x) + eps)
    value = 1.0 if gate is None else ACT[activation][0](gate)
    f = scale * value * p * torch.ones_like(x)
    s = residual_scale * residual + f * x * r1
    s_mag = (residual_scale * residual).abs() + (f * x * r1).abs()
    r2 = 1 / torch.sqrt(mean(s * s) + eps)
    w = weight + offset
    # a row whose s cancels carries the error of s into r2: relative to s_mag, like s itself
    amplify = torch.sqrt(mean(s_mag * s_mag) + eps) * r2
    out = {"y": (s * r2 * w, s_mag * r2 * w.abs() * amplify), "s": (s, s_mag)}
    if gy is None and gs is None:
        return out
    gy = torch.zeros_like(x) if gy is None else gy
    gs = torch.zeros_like(x) if gs is None else gs
    gw = gy * w
    c2, c2_mag = r2 ** 3 * mean(gw * s), r2 ** 3 * mean(gw.abs() * s_mag) * amplify
    ds = gs + r2 * gw - c2 * s
    ds_mag = gs.abs() + r2 * gw.abs() * amplify + c2_mag * s_mag
    dn, dn_mag = f * ds, f.abs() * ds_mag
    if post is None:
        c1 = c1_mag = torch.zeros_like(c2)
    else:
        c1, c1_mag = r1 ** 3 * mean(dn * x), r1 ** 3 * mean(dn_mag * x.abs())
    out["x"] = (r1 * dn - c1 * x, r1 * dn_mag + c1_mag * x.abs())
    out["residual"] = (residual_scale * ds, abs(residual_scale) * ds_mag)
    out["weight"] = ((gy * s * r2).sum(lead), (gy.abs() * s_mag * r2 * amplify).sum(lead))
    k, k_mag = ds * x * r1, ds_mag * x.abs() * r1
    if post is not None:
        out["post"] = ((scale * value * k).sum(lead), ((scale * value * torch.ones_like(k)).abs() * k_mag).sum(lead))
    if gate is not None:
        slope = scale * ACT[activation][1](value) * p
        dims = [d for d in lead if d < x.dim() - gate.dim() or gate.shape[d - (x.dim() - gate.dim())] == 1]
        # 1 - v^2 and v (1 - v) round relative to 1, not to what is left of it
        dg, dg_mag = slope * k, scale * abs(p) * k_mag
        for d in dims:
            dg, dg_mag = dg.sum(d, keepdim=True), dg_mag.sum(d, keepdim=True)
        out["gate"] = (dg.reshape(gate.shape), dg_mag.reshape(gate.shape))
    return out


def check_norm(x, residual, weight, post, gate, activation="identity", scale=1.0, residual_scale=1.0, eps=1e-6, offset=0.0, gy=None, gs=None):
    named = {"x": x, "residual": residual, "weight": weight, "post": post, "gate": gate}
    leaves = {n: t.detach().requires_grad_(True) for n, t in named.items() if t is not None}
    y, s = autograd.gated_add_rms_norm(leaves["x"], leaves["residual"], leaves["weight"], leaves.get("post"), leaves.get("gate"), activation, scale, residual_scale, eps, offset)
    want = norm_reference(x, residual, weight, post, gate, activation, scale, residual_scale, eps, offset, gy, gs)
    rows = x.numel() // max(x.shape[-1], 1)
    got = {"y": y.detach(), "s": s.detach()}
    outputs = [(o, g) for o, g in ((y, gy), (s, gs)) if g is not None]
    if outputs:
        grads = torch.autograd.grad([o for o, _ in outputs], list(leaves.values()), [g for _, g in outputs])
        got.update(zip(leaves, grads))
    plain = ops.gated_add_rms_norm(x, residual, weight, post, gate, activation, scale, residual_scale, eps, offset)
    assert torch.equal(plain[0], got["y"]) and torch.equal(plain[1], got["s"])  # with and without a gradient
    for name in got:
        # sums over rows: any order of n terms is off by at most n - 1 roundings of their magnitudes
        near(got[name], *want[name], roundings=ROUNDINGS + (rows if name in ("weight", "post", "gate") else 0), what=name)
    return got


def norm_inputs(seed, lead, hidden, dtype, post=True, gate=None):
    shape = {None: None, "channel": (hidden,), "first": (lead[0], *[1] * (len(lead) - 1), hidden), "row": (*lead, hidden)}[gate]
    return (normal(seed, *lead, hidden, dtype=dtype, std=2.0), normal(seed + 1, *lead, hidden, dtype=dtype, std=3.0), normal(seed + 2, hidden, dtype=dtype, std=0.2, mean=1.0),
            normal(seed + 3, hidden, dtype=dtype, std=0.2, mean=1.0) if post else None, None if shape is None else normal(seed + 4, *shape, dtype=dtype, std=0.7, mean=0.3))


@pytest.mark.parametrize("lead,hidden,dtype,post,gate,activation,scale,residual_scale,offset", [
    ((1,), 4096, BF16, True, "channel", "identity", 1.0, 1.0, 0.0),            # one token
    ((1, 1), 64, F32, False, None, "identity", 0.5, 1.0, 0.0),
    ((3,), 1, F32, True, "channel", "tanh", 1.0, 1.0, 0.0),                    # a row of one channel
    ((5,), 7, BF16, True, "row", "sigmoid", 1.0, 0.5, 1.0),
    ((2, 33), 256, BF16, True, "first", "tanh", 1.0, 1.0, 0.0),
    ((4, 9), 512, F16, False, "first", "sigmoid", 2.0, 0.9, 0.0),
    ((300,), 1000, BF16, True, None, "identity", 0.25, 1.0, 1.0),              # no power of two
    ((65,), 1001, F32, True, "channel", "sigmoid", 1.0, 1.0, 0.0),             # element by element
    ((3, 50), 257, F16, True, "first", "identity", 1.0, 1.0, 0.0),
    ((700, 3), 1024, BF16, True, "first", "tanh", 1.0, 1.0, 0.0),              # many short groups: more than walkers
    ((1, 1, 400), 2048, BF16, True, "row", "tanh", 1.0, 0.7, 0.0),
    ((7, 100), 2050, F32, True, "first", "sigmoid", 1.0, 1.0, 0.0),
    ((1000,), 4096, BF16, True, "channel", "identity", 1.0, 0.7, 0.0),
    ((2, 301), 5120, F16, True, "first", "tanh", 1.0, 1.0, 0.0),
    ((310,), 8192, BF16, False, "row", "identity", 1.0, 1.0, 0.0),
    ((40,), 8192, F32, True, "row", "identity", 1.0, 1.0, 0.0),
    ((20,), 16384, BF16, True, "channel", "tanh", 1.0, 1.0, 0.0),
    ((3, 4), 16400, F32, True, "first", "sigmoid", 1.0, 1.0, 0.0),             # wider than registers
    ((5,), 40000, BF16, True, "row", "tanh", 1.0, 0.5, 0.0),
    ((3000,), 128, BF16, True, "channel", "identity", 1.0, 1.0, 0.0),
])
def test_norm_forward_and_gradients(lead, hidden, dtype, post, gate, activation, scale, residual_scale, offset):
    seed = 100 * hidden + len(lead)
    gy, gs = normal(seed + 5, *lead, hidden, dtype=dtype), normal(seed + 6, *lead, hidden, dtype=dtype)
    check_norm(*norm_inputs(seed, lead, hidden, dtype, post, gate), activation, scale, residual_scale, 1e-6, offset, gy, gs)


@pytest.mark.parametrize("hidden,dtype", [(512, BF16), (4096, BF16), (515, F32)])
def test_norm_gradient_from_one_output_alone(hidden, dtype):
    inputs = norm_inputs(7, (9,), hidden, dtype, True, "channel")
    check_norm(*inputs, gy=normal(8, 9, hidden, dtype=dtype))
    check_norm(*inputs, gs=normal(9, 9, hidden, dtype=dtype))


@pytest.mark.parametrize("hidden,dtype", [(1024, BF16), (4096, F16), (1023, F32)])
def test_norm_strides(hidden, dtype):
    """Column slices of wider buffers, a transposed gradient, rows that start off a 16-byte boundary."""
    wide = normal(20, 6, 5, 3 * hidden + 8, dtype=dtype)
    gates = normal(21, 6, 6 * hidden, dtype=dtype)  # the chunks of one modulation projection
    weight = normal(22, 2 * hidden, dtype=dtype, mean=1.0, std=0.2)[::2]
    gy = normal(23, hidden, 6, 5, dtype=dtype).permute(1, 2, 0)
    for start in (0, 8, 3):
        x, residual = wide[..., start: start + hidden], wide[..., hidden + start: 2 * hidden + start]
        gate = gates[:, None, 2 * hidden + start: 3 * hidden + start]
        check_norm(x, residual, weight, weight.flip(0), gate, "tanh", gy=gy, gs=wide[..., start + 1: start + 1 + hidden])
    check_norm(x[:1, :1].expand_as(x), residual, weight, None, gate, gy=gy[:1, :1].expand_as(x), gs=gy[:, :1].expand_as(x))  # rows that overlap


@pytest.mark.parametrize("hidden,dtype", [(2048, BF16), (100, F32)])
def test_norm_where_the_branch_cancels_the_residual(hidden, dtype):
    x = normal(30, 12, hidden, dtype=dtype)
    residual = -x + normal(31, 12, hidden, dtype=dtype, std=2.0 ** -6)
    weight = torch.ones(hidden, dtype=dtype, device=DEV)
    check_norm(x, residual, weight, None, None, gy=normal(32, 12, hidden, dtype=dtype), gs=normal(33, 12, hidden, dtype=dtype))


def test_norm_rows_of_zeros_and_of_infinities_stay_their_own():
    inputs = list(norm_inputs(40, (16,), 1024, BF16, True, "channel"))
    gy, gs = normal(41, 16, 1024, dtype=BF16), normal(42, 16, 1024, dtype=BF16)
    clean = check_norm(*inputs, gy=gy, gs=gs)
    x, residual = inputs[0].clone(), inputs[1].clone()
    x[3] = 0
    residual[3] = 0
    x[5, 7] = float("inf")
    x[6, 9] = float("nan")
    y, s = ops.gated_add_rms_norm(x, residual, *inputs[2:])
    assert not y[3].any() and not s[3].any()
    assert y[5].isnan().any() and y[6].isnan().all()
    rest = [i for i in range(16) if i not in (3, 5, 6)]
    assert torch.equal(y[rest], clean["y"][rest]) and torch.equal(s[rest], clean["s"][rest])


@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 64), (4, 0)])
def test_norm_of_nothing(shape):
    x = torch.zeros(shape, dtype=BF16, device=DEV, requires_grad=True)
    weight, gate = (torch.ones(shape[-1], dtype=BF16, device=DEV, requires_grad=True) for _ in range(2))
    y, s = autograd.gated_add_rms_norm(x, x.detach(), weight, None, gate)
    grads = torch.autograd.grad((y, s), (x, weight, gate), (torch.ones_like(y), torch.ones_like(s)))
    assert y.shape == s.shape == x.shape
    assert not any(g.any() for g in grads)


@pytest.mark.parametrize("gate", ["channel", "first", "row"])
def test_norm_gradient_against_differences(gate):
    """<gradient, direction> against the difference of the definition in 64 bits along that direction."""
    inputs = norm_inputs(50, (3, 5), 96, F32, True, gate)
    gy, gs = normal(51, 3, 5, 96), normal(52, 3, 5, 96)
    got = check_norm(*inputs, "tanh", 0.7, 0.9, 1e-6, 0.5, gy, gs)
    step = 1e-5
    for name, at in (("x", 0), ("residual", 1), ("weight", 2), ("post", 3), ("gate", 4)):
        direction = normal(53 + at, *inputs[at].shape).double()
        value = []
        for sign in (1, -1):
            moved = [t.double() for t in inputs]
            moved[at] = moved[at] + sign * step * direction
            out = norm_reference(*moved, "tanh", 0.7, 0.9, 1e-6, 0.5, None, None)
            value.append((out["y"][0] * gy.double()).sum() + (out["s"][0] * gs.double()).sum())
        want, mine = float((value[0] - value[1]) / (2 * step)), float((got[name].double() * direction).sum())
        # the difference is off by step^2 times a third derivative of some thousands of order-one terms (1e-6), the gradient by fp32
        assert abs(want - mine) <= 1e-5 + 2e-5 * float((got[name].double() * direction).abs().sum()), name


def test_norm_refuses():
    x, residual, weight, post, gate = norm_inputs(60, (4, 6), 64, BF16, True, "first")
    for kwargs, error in ((dict(weight=weight[:32]), ValueError), (dict(post_weight=post.float()), TypeError), (dict(residual=residual[:, :3]), ValueError),
                          (dict(gate=gate.float()), TypeError), (dict(gate=gate[:3]), ValueError), (dict(activation="relu"), ValueError), (dict(weight=weight.cpu()), RuntimeError)):
        with pytest.raises(error):
            ops.gated_add_rms_norm(**{**dict(x=x, residual=residual, weight=weight, post_weight=post, gate=gate), **kwargs})
    with pytest.raises(RuntimeError, match="forward-only"):
        ops.gated_add_rms_norm(x.requires_grad_(True), residual, weight)
    with pytest.raises(TypeError, match="not supported"):
        ops.gated_add_rms_norm(*(t.detach().double() for t in (x, residual, weight)))


# ---------------------------------------------------------------------------------------------------------- balance loss --


def balance_reference(logits, indices, mask, per_sequence, weights=(1.0, 1.0)):
    """(balance, z, counts, gradient of weights . losses, bounds of their fp32 error) in 64 bits, by autograd."""
    experts, top_k = logits.shape[-1], indices.shape[-1]
    wide = logits.double().reshape(-1 if not per_sequence else logits.shape[0], *logits.shape[-2:]) if per_sequence else logits.double().reshape(1, -1, experts)
    wide = wide.detach().requires_grad_(True)
    keep = torch.ones(logits.shape[:-1], dtype=torch.bool, device=logits.device) if mask is None else mask
    keep, picks = keep.reshape(wide.shape[:2]), indices.reshape(*wide.shape[:2], top_k).long()
    losses, counts, slopes = [], [], torch.zeros_like(wide)
    for g in range(wide.shape[0]):
        kept = picks[g][keep[g]].reshape(-1)
        counts.append(torch.bincount(kept[(kept >= 0) & (kept < experts)], minlength=experts))
        n = int(keep[g].sum())
        if n:
            losses.append((counts[-1].double() * experts / (n * top_k) * torch.softmax(wide[g][keep[g]], -1).sum(0) / n).sum())
    balance = sum(losses) / len(losses) if losses else wide.sum() * 0
    rows = wide[keep]
    z = torch.logsumexp(rows, -1).square().mean() if len(rows) else wide.sum() * 0
    (grad,) = torch.autograd.grad(weights[0] * balance + weights[1] * z, wide)
    grad = torch.where(keep[..., None], grad, 0.0)
    # magnitudes: p and the terms of its factor; exp of a difference of logits is off by 2^-24 of the larger of them
    with torch.no_grad():
        size = 1 + torch.where(wide.isfinite(), wide, 0.0).abs().amax(-1, keepdim=True)
        for g in range(wide.shape[0]):
            n = int(keep[g].sum())
            if n:
                f = counts[g].double() * experts / (n * top_k)
                p = torch.softmax(wide[g], -1)
                lse = torch.logsumexp(wide[g], -1, keepdim=True).abs()
                slopes[g] = p * (abs(weights[0]) / (len(losses) * n) * (f + (p * f).sum(-1, keepdim=True)) + 2 * abs(weights[1]) / len(rows) * (lse + 1)) * size[g]
        slopes = torch.where(keep[..., None], slopes, 0.0)
    counts = torch.stack(counts) if per_sequence else counts[0]
    return balance.detach(), z.detach(), counts.int(), grad.reshape(logits.shape), slopes.reshape(logits.shape), float(size.max())


def picks_of(logits, top_k):
    return torch.nan_to_num(logits.float(), nan=0.0).topk(top_k, -1).indices.int()


def check_balance(logits, indices, mask=None, per_sequence=False, weights=(0.3, 0.02)):
    leaf = logits.detach().requires_grad_(True)
    balance, z, counts = autograd.moe_balance_loss(leaf, indices, mask, per_sequence)
    (grad,) = torch.autograd.grad((balance, z), leaf, tuple(torch.tensor(w, device=DEV) for w in weights))
    want_b, want_z, want_c, want_g, mag_g, size = balance_reference(logits, indices, mask, per_sequence, tuple(float(torch.tensor(w)) for w in weights))
    assert torch.equal(counts, want_c)
    # a CTA adds a few hundred tokens in fp32, the rest is fp64; a probability is off by `size` roundings
    near(balance.detach(), want_b, want_b * size)
    near(z.detach(), want_z, want_z + size)
    near(grad, want_g, mag_g, what="grad")
    plain = ops.moe_balance_loss(logits, indices, mask, per_sequence)
    assert torch.equal(plain[0], balance.detach()) and torch.equal(plain[1], z.detach()) and torch.equal(plain[2], counts)
    return balance.detach(), z.detach(), counts, grad


@pytest.mark.parametrize("lead,experts,top_k,dtype,masked,per_sequence", [
    ((1,), 8, 2, F32, False, False), ((1, 1), 1, 1, F32, False, True), ((3,), 2, 1, BF16, False, False), ((5,), 3, 3, F16, True, False),
    ((7, 33), 8, 2, BF16, True, True), ((2, 509), 60, 4, F32, False, False), ((4, 257), 64, 8, F32, True, True), ((4, 257), 64, 8, BF16, True, False),
    ((1000,), 65, 6, F32, False, False), ((6, 100), 128, 8, F16, False, True), ((3, 500), 256, 8, F32, True, True), ((2, 3, 100), 256, 8, BF16, True, False),
    ((400,), 300, 32, F32, False, False), ((2, 100), 512, 4, F32, True, True), ((2, 100), 520, 4, BF16, True, True), ((300,), 1000, 2, F32, True, False),
    ((150,), 1023, 2, BF16, False, False), ((3, 70), 1024, 8, F32, False, True), ((20000,), 16, 4, F32, True, False), ((70, 5), 32, 4, F32, True, True),
])
def test_balance_and_gradient(lead, experts, top_k, dtype, masked, per_sequence):
    logits = normal(experts, *lead, experts, dtype=dtype, std=2.0)
    mask = normal(experts + 1, *lead) > -0.5 if masked else None
    check_balance(logits, picks_of(logits, top_k), mask, per_sequence)


def test_balance_masks_that_leave_nothing():
    logits = normal(1, 4, 50, 16)
    indices = picks_of(logits, 2)
    mask = torch.zeros(4, 50, dtype=torch.bool, device=DEV)
    for per_sequence in (False, True):
        balance, z, counts, grad = check_balance(logits, indices, mask, per_sequence)
        assert balance == 0 and z == 0 and not counts.any() and not grad.any()
    mask[2, 7] = True  # one token of one sequence
    mask[3] = True
    for per_sequence in (False, True):
        check_balance(logits, indices, mask, per_sequence)


def test_balance_does_not_look_at_masked_tokens():
    logits = normal(2, 3, 70, 64)
    indices = picks_of(logits, 4)
    mask = normal(3, 3, 70) > 0
    for per_sequence in (False, True):
        want = check_balance(logits, indices, mask, per_sequence)
        dirty, wrong = logits.clone(), indices.clone()
        dirty[~mask] = float("nan")
        dirty[0][~mask[0]] = float("inf")
        wrong[~mask] = 1 << 30
        leaf = dirty.requires_grad_(True)
        balance, z, counts = autograd.moe_balance_loss(leaf, wrong, mask, per_sequence)
        (grad,) = torch.autograd.grad((balance, z), leaf, (torch.tensor(0.3, device=DEV), torch.tensor(0.02, device=DEV)))
        for have, wanted in zip((balance, z, counts, grad), want):
            assert torch.equal(have, wanted)


@pytest.mark.parametrize("experts,dtype", [(64, F32), (64, BF16), (61, F32)])
def test_balance_with_experts_switched_off(experts, dtype):
    logits = normal(4, 200, experts, dtype=dtype)
    logits[:, 5] = float("-inf")
    logits[::3, 8:20] = torch.finfo(dtype).min
    logits[7, 1:] = float("-inf")  # one expert is left
    logits[8, :] = 0.0
    check_balance(logits, picks_of(logits, 2))


def test_balance_of_a_row_without_experts_is_nan():
    logits = normal(5, 40, 8)
    logits[3] = float("-inf")
    balance, z, _ = ops.moe_balance_loss(logits, picks_of(normal(5, 40, 8), 2))
    assert balance.isnan() and z.isnan()


def test_balance_picks_outside_the_experts_are_left_out():
    logits = normal(6, 100, 10)
    indices = picks_of(logits, 3)
    indices[::7, 1] = -1
    indices[::5, 0] = 10
    check_balance(logits, indices)


def test_balance_strides():
    wide = normal(7, 6, 40, 100)
    indices = picks_of(wide[..., :32], 4)
    for start in (0, 4, 3):
        logits = wide[..., start: start + 32]
        check_balance(logits, picks_of(logits, 4), normal(8, 40, 6).t() > 0, True)
    check_balance(wide.permute(2, 0, 1)[:96], picks_of(wide.permute(2, 0, 1)[:96], 4).flip(1).flip(1))
    check_balance(wide[..., :32], indices.transpose(0, 1).contiguous().transpose(0, 1))


@pytest.mark.parametrize("shape", [(0, 8), (3, 0, 8), (0, 5, 8)])
def test_balance_of_nothing(shape):
    logits = torch.zeros(shape, device=DEV, requires_grad=True)
    indices = torch.zeros(*shape[:-1], 2, dtype=torch.int32, device=DEV)
    for per_sequence in {False, len(shape) == 3}:
        balance, z, counts = autograd.moe_balance_loss(logits, indices, None, per_sequence)
        (grad,) = torch.autograd.grad(balance + z, logits)
        assert balance == 0 and z == 0 and not counts.any() and grad.shape == logits.shape


def test_balance_gradient_against_differences():
    logits = normal(9, 5, 40, 24)
    indices, mask = picks_of(logits, 3), normal(10, 5, 40) > -0.3
    *_, grad = check_balance(logits, indices, mask, True, weights=(0.3, 0.02))
    direction, step = normal(11, *logits.shape).double(), 1e-5
    value = []
    for sign in (1, -1):
        balance, z, *_ = balance_reference(logits.double() + sign * step * direction, indices, mask, True)
        value.append(float(torch.tensor(0.3)) * balance + float(torch.tensor(0.02)) * z)
    want, terms = float((value[0] - value[1]) / (2 * step)), grad.double() * direction
    # 64-bit losses of order one over 2 step are off by 1e-11, the second order by step^2; the gradient by fp32
    assert abs(want - float(terms.sum())) <= 1e-8 + 1e-5 * float(terms.abs().sum())


def test_balance_loss_alone_and_z_alone():
    logits = normal(12, 90, 64)
    indices = picks_of(logits, 8)
    both = check_balance(logits, indices, weights=(1.0, 0.0))[3], check_balance(logits, indices, weights=(0.0, 1.0))[3]
    for which in (0, 1):
        leaf = logits.detach().requires_grad_(True)
        (grad,) = torch.autograd.grad(autograd.moe_balance_loss(leaf, indices)[which], leaf)
        assert torch.equal(grad, both[which])


def test_balance_refuses():
    logits = normal(13, 4, 6, 8)
    indices = picks_of(logits, 2)
    for args, error in (((logits, indices.long()), ValueError), ((logits, indices[:3]), ValueError), ((logits, indices, torch.ones(4, 6, device=DEV)), ValueError),
                        ((logits, indices, torch.ones(4, 5, dtype=torch.bool, device=DEV)), ValueError), ((logits[0], indices[0], None, True), ValueError),
                        ((logits.double(), indices), TypeError), ((logits, indices.cpu()), RuntimeError)):
        with pytest.raises(error):
            ops.moe_balance_loss(*args)
    with pytest.raises(_lib.B200Error, match="experts"):
        ops.moe_balance_loss(normal(14, 4, 1025), indices[0, :4])


# -------------------------------------------------------------------------------------------------------------- embedding --


def check_embedding(ids, weight, grad, scale=1.0, padding_idx=None):
    leaf = weight.detach().requires_grad_(True)
    out = autograd.embedding(ids, leaf, scale, padding_idx)
    (got,) = torch.autograd.grad(out, leaf, grad)
    vocab, width = weight.shape
    flat = ids.reshape(-1).long()
    there = (flat >= 0) & (flat < vocab)
    table = scale * torch.where(there[:, None], weight.double()[flat.clamp(0, max(vocab - 1, 0))], 0.0) if vocab else torch.zeros(len(flat), width, dtype=torch.float64, device=DEV)
    near(out.detach().reshape(-1, width), table, table.abs(), roundings=1, what="out")
    if padding_idx is not None:
        there &= flat != padding_idx % vocab
    rows = torch.where(there[:, None], grad.reshape(-1, width).double(), 0.0)
    want, magnitude = (torch.zeros(vocab, width, dtype=torch.float64, device=DEV).index_add_(0, torch.where(there, flat, 0), t) for t in (rows, rows.abs()))
    most = int(torch.bincount(flat[there]).max()) if bool(there.any()) else 0
    near(got, scale * want, abs(scale) * magnitude, roundings=most + 2, what="grad")  # any order of n terms: n - 1 roundings
    assert torch.equal(got, ops.embedding_backward(grad, ids, vocab, scale, padding_idx))  # the same bits again
    return out.detach(), got


def ids_of(kind, tokens, vocab, seed):
    gen = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(vocab, (tokens,), generator=gen)
    if kind == "one":
        return torch.full((tokens,), vocab // 2)
    if kind == "few":
        return torch.randint(3, (tokens,), generator=gen) * (vocab // 3)
    rank = torch.exp(torch.rand(tokens, generator=gen, dtype=torch.float64) * torch.tensor(vocab, dtype=torch.float64).log()).long() - 1
    return rank.clamp(0, vocab - 1) * 31 % vocab


@pytest.mark.parametrize("tokens,vocab,hidden,dtype,kind,scale,wide", [
    (1, 1, 1, F32, "one", 1.0, True), (1, 50257, 64, BF16, "uniform", 2.0, False), (7, 5, 3, F16, "uniform", 1.0, True), (8, 100, 256, BF16, "one", 0.5, True),
    (9, 100, 256, BF16, "one", 0.5, True), (31, 1000, 1000, F32, "few", 1.0, False), (33, 1000, 1001, BF16, "zipf", 31.6, True), (1000, 32000, 512, BF16, "zipf", 22.6, False),
    (8191, 1000, 130, F32, "zipf", 1.0, True), (8192, 1000, 128, F32, "zipf", 1.0, False), (8195, 300, 264, F16, "few", 1.0, True), (8200, 7, 520, BF16, "one", 0.1, True),
    (20011, 131072 + 3, 96, BF16, "zipf", 1.0, True), (20011, 131072 + 3, 1032, F32, "uniform", 1.0, False), (40000, 262144, 40, F16, "zipf", 1.0, True), (3000, 2, 2048, BF16, "uniform", 1.0, False),
    (100, 5000, 9000, BF16, "few", 1.0, True),
])
def test_embedding_and_gradient(tokens, vocab, hidden, dtype, kind, scale, wide):
    ids = ids_of(kind, tokens, vocab, tokens).to(DEV).to(torch.int64 if wide else torch.int32)
    check_embedding(ids, normal(tokens, vocab, hidden, dtype=dtype), normal(tokens + 1, tokens, hidden, dtype=dtype), scale)


@pytest.mark.parametrize("padding_idx", [0, 17, -1, None])
def test_embedding_padding_and_ids_outside_the_table(padding_idx):
    weight, ids = normal(1, 50, 72, dtype=BF16), ids_of("uniform", 600, 50, 2).to(DEV).reshape(4, 150)
    ids[:, 100:] = 0 if padding_idx is None else padding_idx % 50
    grad = normal(3, 4, 150, 72, dtype=BF16)
    _, plain = check_embedding(ids, weight, grad, 1.0, padding_idx)
    if padding_idx is not None:
        assert not plain[padding_idx].any()
    ids[1, :40] = -1
    ids[2, 10:20] = 50
    ids[3, 5] = 1 << 40
    ids[0, 0] = -(1 << 62)
    out, _ = check_embedding(ids, weight, grad, 1.0, padding_idx)
    assert not out[1, :40].any() and not out[2, 10:20].any()
    none = torch.full_like(ids, -5)
    out, got = check_embedding(none, weight, grad, 1.0, padding_idx)
    assert not out.any() and not got.any()


def test_embedding_shards_of_a_table_add_up():
    weight, ids = normal(1, 1000, 64, dtype=F32), ids_of("zipf", 500, 1000, 2).to(DEV)
    grad = normal(3, 500, 64)
    out, want = check_embedding(ids, weight, grad)
    parts = [check_embedding(ids - start, weight[start: start + 250], grad) for start in range(0, 1000, 250)]
    assert torch.equal(sum(p[0] for p in parts), out)
    # where the sorted list is cut depends on the tokens before a run, so a shard groups a run's terms in its own way: either sum is
    # within (n - 1) roundings of the terms' magnitudes of the exact one, hence within 2 (n - 1) of the other
    most = int(torch.bincount(ids).max())
    magnitude = torch.zeros(1000, 64, dtype=torch.float64, device=DEV).index_add_(0, ids, grad.abs().double())
    near(torch.cat([p[1] for p in parts]), want.double(), magnitude, roundings=2 * (most + 2))


def test_embedding_strides():
    table, grads = normal(4, 300, 200, dtype=BF16), normal(5, 3, 70, 200, dtype=BF16)
    ids = ids_of("zipf", 210, 300, 6).to(DEV).reshape(70, 3).t()
    for start, width in ((0, 128), (8, 128), (3, 128), (0, 65)):
        check_embedding(ids, table[:, start: start + width], grads[..., start: start + width])
    check_embedding(ids, table.t()[:150].contiguous().t()[:, :150], grads.transpose(0, 1).contiguous().transpose(0, 1)[..., :150])


@pytest.mark.parametrize("tokens,vocab,hidden", [(0, 10, 8), (5, 10, 0), (0, 0, 8)])
def test_embedding_of_nothing(tokens, vocab, hidden):
    weight = torch.ones(vocab, hidden, dtype=BF16, device=DEV, requires_grad=True)
    out = autograd.embedding(torch.zeros(tokens, dtype=torch.int64, device=DEV), weight)
    (grad,) = torch.autograd.grad(out, weight, torch.ones_like(out))
    assert out.shape == (tokens, hidden) and grad.shape == weight.shape and not grad.any()


def test_embedding_offsets_beyond_32_bits():
    vocab, hidden = 270000, 8192  # 2.2e9 elements
    weight = torch.zeros(vocab, hidden, dtype=BF16, device=DEV)
    ids = torch.tensor([0, vocab - 1, 262150, vocab - 1], device=DEV)
    for i, row in enumerate((0, vocab - 1, 262150)):
        weight[row] = normal(i, hidden, dtype=BF16)
    assert torch.equal(ops.embedding(ids, weight), weight[ids])
    grad = normal(9, 4, hidden, dtype=BF16)
    got = ops.embedding_backward(grad, ids, vocab)
    assert torch.equal(got[0], grad[0]) and torch.equal(got[262150], grad[2])
    assert torch.equal(got[vocab - 1], (grad[1].float() + grad[3].float()).to(BF16))
    got[ids] = 0
    assert not got.any()


def test_embedding_refuses():
    weight, ids = normal(1, 10, 8), torch.zeros(3, dtype=torch.int64, device=DEV)
    for args, error in (((ids.float(), weight), TypeError), ((ids, weight[0]), ValueError), ((ids, weight.double()), TypeError), ((ids, weight, 1.0, 10), ValueError),
                        ((ids, weight, 1.0, -11), ValueError), ((ids.cpu(), weight), RuntimeError)):
        with pytest.raises(error):
            ops.embedding(*args)
    with pytest.raises(ValueError):
        ops.embedding_backward(normal(2, 4, 8), ids, 10)


# --------------------------------------------------------------------------------------------------------------- together --


def layer_inputs(tokens=200, hidden=256, vocab=500, experts=8, inter=128):
    d = dict(table=normal(1, vocab, hidden, dtype=BF16, std=0.05), first=normal(2, hidden, dtype=BF16, std=0.1, mean=1.0), post=normal(3, hidden, dtype=BF16, std=0.1, mean=1.0),
             second=normal(4, hidden, dtype=BF16, std=0.1, mean=1.0), gate=normal(5, hidden, dtype=BF16, std=0.3, mean=0.5), router=normal(6, hidden, experts, std=hidden ** -0.5),
             gate_proj=normal(7, experts, hidden, inter, dtype=BF16, std=hidden ** -0.5), up_proj=normal(8, experts, hidden, inter, dtype=BF16, std=hidden ** -0.5),
             down_proj=normal(9, experts, inter, hidden, dtype=BF16, std=inter ** -0.5))
    return d, ids_of("zipf", tokens, vocab, 10).to(DEV).reshape(2, -1)


def layer(p, ids, mask):
    """A mixture-of-experts block between its norms, from the ids to the losses."""
    from popcorn_b200 import kernels

    stream = kernels.embedding(ids, p["table"], 16.0, 0)
    y = kernels.rms_norm(stream, p["first"])
    logits = y.float() @ p["router"]
    indices, _ = kernels.moe_route(logits.detach(), 2)
    balance, z, counts = kernels.moe_balance_loss(logits, indices, mask, True)
    block = kernels.momoe(y, p["gate_proj"], p["up_proj"], p["down_proj"], logits, 2)
    y, stream = kernels.gated_add_rms_norm(block, stream, p["second"], p["post"], p["gate"], "tanh", residual_scale=0.9)
    return y, stream, balance, z, counts


def test_a_layer_of_them_together():
    p, ids = layer_inputs()
    mask = ids != 0
    leaves = {n: t.requires_grad_(True) for n, t in p.items()}
    y, stream, balance, z, counts = layer(leaves, ids, mask)
    gy, gs = normal(11, *y.shape, dtype=BF16), normal(12, *y.shape, dtype=BF16)
    grads = torch.autograd.grad((y, stream, balance, z), list(leaves.values()), (gy, gs, torch.tensor(0.01, device=DEV), torch.tensor(0.001, device=DEV)))
    assert int(counts.sum()) == 2 * int(mask.sum())
    # the same layer from plain 64-bit pieces, with the picks given: bf16 rounds between the pieces by up to 2^-8 each time
    wide = {n: t.detach().double().requires_grad_(True) for n, t in p.items()}
    norm = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    start = 16.0 * torch.where(mask[..., None], wide["table"][ids], wide["table"][ids].detach())
    x = norm(start, wide["first"])
    logits = x @ wide["router"]
    indices = ops.moe_route((autograd.rms_norm(autograd.embedding(ids, p["table"].detach(), 16.0), p["first"].detach()).float() @ p["router"].detach()), 2)[0].long()
    share = torch.softmax(logits.gather(-1, indices), -1)
    every = torch.einsum("btei,eih->bteh", torch.nn.functional.silu(torch.einsum("bth,ehi->btei", x, wide["gate_proj"])) * torch.einsum("bth,ehi->btei", x, wide["up_proj"]), wide["down_proj"])
    block = (every.gather(2, indices[..., None].expand(*indices.shape, every.shape[-1])) * share[..., None]).sum(2)
    out_s = 0.9 * start + torch.tanh(wide["gate"]) * norm(block, wide["post"])
    out_y = norm(out_s, wide["second"])
    f = torch.stack([torch.bincount(indices[b][mask[b]].reshape(-1), minlength=8).double() * 8 / (2 * mask[b].sum()) for b in range(2)])
    want_b = torch.stack([(f[b] * torch.softmax(logits[b][mask[b]], -1).mean(0)).sum() for b in range(2)]).mean()
    want_z = torch.logsumexp(logits[mask], -1).square().mean()
    want = torch.autograd.grad((out_y, out_s, want_b, want_z), list(wide.values()), (gy.double(), gs.double(), *(torch.tensor(v, device=DEV, dtype=torch.float64) for v in (0.01, 0.001))))

    def far(a, b):
        return float((a.double() - b).norm() / b.norm())

    # some ten roundings to bf16 (2^-9 on average each) lie between the ids and an output, some twenty on the way back
    assert far(y, out_y.detach()) < 0.02 and far(stream, out_s.detach()) < 0.02 and far(balance, want_b.detach()) < 0.01 and far(z, want_z.detach()) < 0.01
    for name, g, w in zip(leaves, grads, want):
        assert far(g, w) < 0.04, f"{name}: {far(g, w):.3f}"


def test_captured_and_replayed_forward_and_backward():
    """Both directions of the three operators in a graph (fresh leaves, ops called directly), replayed on other values, beside a second
    graph of the same calls and with eager calls between: every replay gives the eager bits."""
    hidden, vocab, experts = 512, 3000, 32
    weight, post, gate = (normal(i, hidden, dtype=BF16, mean=1.0, std=0.2) for i in range(3))
    table = normal(3, vocab, hidden, dtype=BF16)

    def buffers(seed):
        ids = ids_of("zipf", 300, vocab, seed).to(DEV).reshape(3, 100)
        logits = normal(seed + 2, 3, 100, experts)
        return dict(ids=ids, block=normal(seed, 3, 100, hidden, dtype=BF16), logits=logits, indices=picks_of(logits, 4), mask=normal(seed + 3, 3, 100) > 0,
                    gy=normal(seed + 4, 3, 100, hidden, dtype=BF16), gs=normal(seed + 5, 3, 100, hidden, dtype=BF16), gb=torch.tensor(0.5, device=DEV), gz=torch.tensor(0.1, device=DEV))

    def step(b):
        stream = ops.embedding(b["ids"], table, 2.0)
        y, s, stats = ops.gated_add_rms_norm_forward(b["block"], stream, weight, post, gate, "sigmoid")
        balance, z, counts, row_stats, shares = ops.moe_balance_loss_forward(b["logits"], b["indices"], b["mask"], True)
        grads = ops.gated_add_rms_norm_backward(b["gy"], b["gs"], b["block"], stream, weight, post, gate, stats, "sigmoid")
        dl = ops.moe_balance_loss_backward(b["gb"], b["gz"], b["logits"], b["mask"], row_stats, shares, True)
        return (y, s, balance, z, counts, *grads, dl, ops.embedding_backward(grads[1], b["ids"], vocab, 2.0, 0))

    sets = [buffers(100), buffers(200)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for b in sets:
            step(b)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for b in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(b)
        graphs.append((graph, out))
    for seed in (300, 400):
        for k, (graph, out) in enumerate(graphs):
            for name, value in buffers(seed + 50 * k).items():
                sets[k][name].copy_(value)
            graph.replay()
        replayed = [[t.clone() for t in out] for _, out in graphs]
        for k in range(2):
            for have, want in zip(replayed[k], step(sets[k])):
                assert torch.equal(have, want)


def test_two_streams_at_once():
    x, residual, weight, post, gate = norm_inputs(70, (2000,), 1024, BF16, True, "channel")
    logits = normal(71, 4000, 64)
    indices = picks_of(logits, 8)
    ids = ids_of("zipf", 9000, 5000, 72).to(DEV)
    grad = normal(73, 9000, 256, dtype=BF16)
    calls = (lambda: ops.gated_add_rms_norm_forward(x, residual, weight, post, gate), lambda: ops.moe_balance_loss(logits, indices), lambda: (ops.embedding_backward(grad, ids, 5000),),
             lambda: ops.gated_add_rms_norm_backward(x, residual, x, residual, weight, post, gate, ops.gated_add_rms_norm_forward(x, residual, weight, post, gate)[2]))
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for k, call in enumerate(calls):
            with torch.cuda.stream(streams[k % 2]):
                got.append((k, call()))
    torch.cuda.synchronize()
    for k, out in got:
        for have, wanted in zip(out, want[k]):
            assert torch.equal(have, wanted)


def test_losses_on_shared_leaves_and_a_second_backward():
    """One leaf under several of the operators: its gradients add up; a second pass over fresh graphs gives the same bits."""
    table = normal(80, 400, 128, dtype=F32).requires_grad_(True)
    weight = normal(81, 128, mean=1.0, std=0.1).requires_grad_(True)
    ids = ids_of("zipf", 90, 400, 82).to(DEV)
    picks = picks_of(normal(83, 90, 128), 4)

    def gradients():
        stream = autograd.embedding(ids, table, 2.0)
        y, s = autograd.gated_add_rms_norm(stream, stream, weight, weight, weight)  # x is its own residual, one weight three times
        balance, z, _ = autograd.moe_balance_loss(s, picks)
        return torch.autograd.grad(y.square().sum() + balance + 0.1 * z, (table, weight))

    first, second = gradients(), gradients()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    wide = [t.detach().double().requires_grad_(True) for t in (table, weight)]
    stream = 2.0 * wide[0][ids]
    unit = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    s = stream + wide[1] * unit(stream) * wide[1]
    y = unit(s) * wide[1]
    f = torch.bincount(picks.reshape(-1).long(), minlength=128).double() * 128 / (4 * 90)
    want = torch.autograd.grad(y.square().sum() + (f * torch.softmax(s, -1).mean(0)).sum() + 0.1 * torch.logsumexp(s, -1).square().mean(), wide)
    for have, wanted in zip(first, want):
        # some four hundred fp32 roundings at most lie on any path, each 2^-24 of numbers no larger than the gradients' own norm
        assert float((have.double() - wanted).norm() / wanted.norm()) < 400 * 2.0 ** -24


def test_calls_beside_a_stream_that_is_not_the_current_one():
    """Inputs made on a side stream, used on another after an event; memory handed back while kernels are still to run."""
    x, residual, weight, post, gate = norm_inputs(90, (3000,), 2048, BF16, True, "channel")
    want = ops.gated_add_rms_norm(x, residual, weight, post, gate)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            got = ops.gated_add_rms_norm(x.t().contiguous().t(), residual, weight.flip(0).flip(0), post, gate)  # copies that die with the call
    torch.cuda.current_stream().wait_stream(side)
    for have, wanted in zip(got, want):
        have.record_stream(torch.cuda.current_stream())
        assert torch.equal(have, wanted)
