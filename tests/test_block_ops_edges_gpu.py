"""Calls at the edges of the operators around the layers: gates and logits that are no ordinary numbers, calls from several threads,
derivatives that the kernels do not have."""

import os
import subprocess
import sys
import threading
import time
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from popcorn_b200 import _lib, autograd, ops
from tests.test_block_ops_gpu import BF16, DEV, F16, F32, check_norm, ids_of, near, norm_inputs, norm_reference, normal, picks_of

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
GATE_FORMS = [(hidden, dtype, activation, gate) for hidden, dtype in ((256, BF16), (256, F16), (256, F32), (130, BF16), (129, F16), (130, F32), (4096, BF16), (16390, F16), (16390, F32))
              for activation in ("tanh", "sigmoid") for gate in ("channel", "first", "row")]


@pytest.mark.parametrize("hidden,dtype,activation,gate", GATE_FORMS)
def test_norm_gate_of_infinities_is_open_or_shut(hidden, dtype, activation, gate):
    """tanh is 1 and -1 there, the sigmoid 1 and 0, both slopes 0: everything stays finite."""
    inputs = norm_inputs(hidden, (3, 5), hidden, dtype, True, gate)
    rows = inputs[4].view(-1, hidden)
    rows[-1, 3], rows[-1, 8] = INF, -INF
    gy, gs = normal(1, 3, 5, hidden, dtype=dtype), normal(2, 3, 5, hidden, dtype=dtype)
    got = check_norm(*inputs, activation, gy=gy, gs=gs)
    shut = got["gate"].view(-1, hidden)[-1]
    assert shut[3] == 0 and shut[8] == 0


@pytest.mark.parametrize("hidden,dtype,activation,gate", GATE_FORMS)
def test_norm_gate_that_is_nan_shows(hidden, dtype, activation, gate):
    """Where the definition gives NaN the outputs and gradients do, and nowhere else."""
    inputs = norm_inputs(hidden, (3, 5), hidden, dtype, True, gate)
    inputs[4].view(-1, hidden)[-1, 5] = NAN
    gy, gs = normal(3, 3, 5, hidden, dtype=dtype), normal(4, 3, 5, hidden, dtype=dtype)
    y, s, stats = ops.gated_add_rms_norm_forward(*inputs, activation)
    grads = ops.gated_add_rms_norm_backward(gy, gs, *inputs, stats, activation)
    want = norm_reference(*inputs, activation, 1.0, 1.0, 1e-6, 0.0, gy, gs)
    assert want["s"][0].isnan().any() and not want["s"][0].isnan().all()
    for name, got in zip(("y", "s", "x", "residual", "weight", "post", "gate"), (y, s, *grads)):
        value, magnitude = want[name]
        lost = value.isnan()
        assert torch.equal(got.isnan(), lost), name
        near(torch.where(lost, 0.0, got).to(dtype), torch.where(lost, 0.0, value), torch.where(lost, 0.0, magnitude), roundings=96 + 15, what=name)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rms_norm_gated_by_a_sigmoid_of_nan(dtype):
    """The sigmoid is the one of the gated norm."""
    x, g, weight = normal(1, 4, 64, dtype=dtype), normal(2, 4, 64, dtype=dtype), torch.ones(64, dtype=dtype, device=DEV)
    g[2, 9] = NAN
    for activation in ("sigmoid", "swish"):
        got = ops.rms_norm_gated(x, g, weight, activation=activation).isnan()
        assert got[2, 9] and int(got.sum()) == 1
    for backward in (ops.sigmoid_gate_backward, ops.swiglu_backward):
        da, db = backward(x, g, x)
        assert da[2, 9].isnan() and db[2, 9].isnan() and int(da.isnan().sum()) == int(db.isnan().sum()) == 1


def errors_from_threads(makers, seconds):
    """Each maker's call, over and over, from a thread and on a stream of its own; what they raised."""
    errors, stop = [], threading.Event()

    def calls(make):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            call, is_right = make(stream)
        while not stop.is_set():
            for _ in range(20):
                try:
                    call()
                except _lib.B200Error as error:
                    errors.append(str(error))
            stream.synchronize()
        if not is_right():
            errors.append("wrong values")

    threads = [threading.Thread(target=calls, args=(make,)) for make in makers]
    for thread in threads:
        thread.start()
    time.sleep(seconds)
    stop.set()
    for thread in threads:
        thread.join()
    return errors


def test_embedding_gradients_of_small_and_large_tables_from_several_threads():
    """The listing kernel's shared memory goes with the rows of the table: no call may narrow another's."""
    def table_of(vocab):
        def make(stream):
            ids, grad, out = torch.arange(16, device=DEV), torch.ones(16, 8, device=DEV), torch.empty(vocab, 8, device=DEV)
            scratch = torch.empty(ops._scratch_bytes(0, "b200_embedding_backward_scratch_bytes", 16, vocab, 8), dtype=torch.uint8, device=DEV)
            return (lambda: _lib.call("b200_embedding_backward", grad.data_ptr(), ids.data_ptr(), out.data_ptr(), 16, vocab, 8, 8, -1, 1, _lib.F32, 1.0, scratch.data_ptr(),
                                      scratch.numel(), stream.cuda_stream),
                    lambda: bool((out[:16] == 1).all()) and not out[16:].any())
        return make
    assert not errors_from_threads([table_of(vocab) for vocab in (100, 100, 100, 100, 200000)], 1.5)


def test_rms_norm_gradients_of_several_widths_from_several_threads():
    """The ring of the plain norm's backward takes as many rows as fit: more shared memory at 4160 columns than at 6144."""
    def width_of(hidden):
        def make(stream):
            x, grad, weight = normal(1, 4, hidden, dtype=BF16), normal(2, 4, hidden, dtype=BF16), torch.ones(hidden, dtype=BF16, device=DEV)
            grad_x, grad_w = torch.empty_like(x), torch.empty_like(weight)
            scratch = ops._norm_scratch(4, hidden, False, x.device)
            want = ops.rms_norm_backward(grad, x, weight)
            return (lambda: _lib.call("b200_rms_norm_backward", grad.data_ptr(), x.data_ptr(), weight.data_ptr(), grad_x.data_ptr(), grad_w.data_ptr(), None, 4, hidden,
                                      hidden, hidden, hidden, _lib.BF16, 1e-6, scratch.data_ptr(), scratch.numel(), stream.cuda_stream),
                    lambda: torch.equal(grad_x, want[0]) and torch.equal(grad_w, want[1]))
        return make
    assert not errors_from_threads([width_of(hidden) for hidden in (6144, 6144, 6144, 6144, 4160)], 1.5)


def backwards_whose_waits_run_out():
    """Run in a process of its own: the library counts such waits, and elsewhere there are none."""
    before = 0
    for rows, hidden, dtype, post, gate, with_gs in (
            (12000, 256, BF16, True, "channel", True), (9000, 1000, BF16, True, "row", True), (3001, 4096, BF16, True, "row", True), (3001, 4096, F16, False, None, False),
            (1000, 5120, F16, True, "first", True), (700, 8192, F32, True, "row", True), (700, 8192, F32, True, "channel", True), (700, 8192, BF16, True, "first", False),
            (1, 4096, BF16, True, "channel", True), (2000, 2050, F32, True, "row", True), (2000, 2049, BF16, True, "channel", True), (9000, 515, F32, False, "first", True)):
        lead = (rows // 100, 100) if gate == "first" else (rows,)
        inputs = norm_inputs(hidden, lead, hidden, dtype, post, gate)
        gy, gs = normal(5, *lead, hidden, dtype=dtype), normal(6, *lead, hidden, dtype=dtype) if with_gs else None
        stats = ops.gated_add_rms_norm_forward(*inputs, "tanh")[2]
        want = ops.gated_add_rms_norm_backward(gy, gs, *inputs, stats, "tanh")
        torch.cuda.synchronize()
        assert _lib.wait_timeouts() == before
        for probes in (0, 1, 3):
            os.environ["B200_GATED_WAIT_PROBES"] = str(probes)
            for _ in range(3):
                got = ops.gated_add_rms_norm_backward(gy, gs, *inputs, stats, "tanh")
                for have, wanted in zip(got, want):
                    assert have is wanted is None or torch.equal(have, wanted), (rows, hidden, dtype, gate, probes)
            now = _lib.wait_timeouts()
            assert probes > 0 or now > before
            before = now
        del os.environ["B200_GATED_WAIT_PROBES"]


def test_norm_backward_whose_waits_run_out():
    """Rows that are not there when their wait ends are fetched without the ring: the same bits, and the count of such waits goes up."""
    child = subprocess.run([sys.executable, "-c", "from tests.test_block_ops_edges_gpu import backwards_whose_waits_run_out as run; run()"], cwd=Path(__file__).resolve().parents[1],
                           capture_output=True, text=True, timeout=300)
    assert child.returncode == 0, child.stderr[-2000:]


def test_second_derivatives_are_refused():
    """A gradient penalty would otherwise go without these operators' share; first derivatives of a recorded backward stay as they are."""
    x, residual, weight, post, gate = (t.requires_grad_(True) for t in norm_inputs(1, (6,), 64, F32, True, "channel"))
    logits = normal(2, 20, 8).requires_grad_(True)
    table = normal(3, 30, 16).requires_grad_(True)
    picks, ids = picks_of(logits.detach(), 2), ids_of("zipf", 20, 30, 4).to(DEV)
    for leaf, value in ((x, lambda: autograd.gated_add_rms_norm(x, residual, weight, post, gate)[0].sum()), (gate, lambda: autograd.gated_add_rms_norm(x, residual, weight, post, gate)[1].square().sum()),
                        (logits, lambda: autograd.moe_balance_loss(logits, picks)[0]), (table, lambda: autograd.embedding(ids, table).square().sum())):
        (plain,) = torch.autograd.grad(value(), leaf)
        (recorded,) = torch.autograd.grad(value(), leaf, create_graph=True)
        assert torch.equal(plain, recorded)
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(recorded.square().sum() + leaf.square().sum(), leaf)
    # the gradient of a table does not depend on the table
    (recorded,) = torch.autograd.grad(autograd.embedding(ids, table).sum(), table, create_graph=True)
    (got,) = torch.autograd.grad(recorded.sum() + table.square().sum(), table)
    assert torch.equal(got, 2 * table.detach())


def test_forward_mode_is_refused():
    x, residual, weight, post, gate = norm_inputs(1, (6,), 64, BF16, True, "channel")
    logits, table, ids = normal(2, 20, 8), normal(3, 30, 16), ids_of("zipf", 20, 30, 4).to(DEV)
    picks = picks_of(logits, 2)
    rows, offsets, experts = normal(4, 32, 64, dtype=BF16), torch.tensor([0, 16, 32], dtype=torch.int32, device=DEV), normal(5, 2, 64, 64, dtype=BF16)
    calls = ((x, lambda t: autograd.gated_add_rms_norm(t, residual, weight, post, gate)), (gate, lambda t: autograd.gated_add_rms_norm(x, residual, weight, post, t)),
             (logits, lambda t: autograd.moe_balance_loss(t, picks)), (table, lambda t: autograd.embedding(ids, t)), (experts, lambda t: autograd.moe_grouped_gemm(rows, t, offsets)))
    for enabled in (True, False):
        with torch.set_grad_enabled(enabled), forward_ad.dual_level():
            for tensor, call in calls:
                call(tensor)
                with pytest.raises(RuntimeError):
                    call(forward_ad.make_dual(tensor, torch.ones_like(tensor)))


@pytest.mark.parametrize("per_sequence", [False, True])
@pytest.mark.parametrize("experts,dtype", [(64, F32), (64, BF16), (61, F32), (8, F16), (512, F32)])
def test_balance_values_with_experts_switched_off(experts, dtype, per_sequence):
    """Experts at -inf or at the type's lowest value have no share at all; the losses and the other experts' gradients are held to
    bounds that those logits do not enter."""
    logits = normal(4, 4, 50, experts, dtype=dtype)
    off = torch.zeros(4, 50, experts, dtype=torch.bool, device=DEV)
    off[..., 5] = True
    off[:, ::3, experts // 4: experts // 2] = True
    lowest = torch.zeros_like(off)
    lowest[:, ::3, experts // 4: experts // 2] = True
    off[1, 7, 1:] = True  # one expert is left
    logits[off] = float("-inf")
    logits[lowest & (normal(6, 4, 50, experts) > 0)] = torch.finfo(dtype).min
    indices = picks_of(logits, 2)
    weights = (0.3, 0.02)
    leaf = logits.detach().requires_grad_(True)
    balance, z, counts = autograd.moe_balance_loss(leaf, indices, None, per_sequence)
    (grad,) = torch.autograd.grad((balance, z), leaf, tuple(torch.tensor(w, device=DEV) for w in weights))
    groups = [slice(b, b + 1) for b in range(4)] if per_sequence else [slice(0, 4)]
    wide = logits.double().masked_fill(off, float("-inf"))
    p, lse = torch.softmax(wide, -1), torch.logsumexp(wide, -1, keepdim=True)
    # exp of a difference of logits is off by roundings of the largest difference that counts; the rest as in the plain test
    top = wide.amax(-1, keepdim=True)
    size = 1 + torch.where(off, 0.0, top - wide).amax(-1, keepdim=True)
    gb, gz = (float(torch.tensor(w)) for w in weights)
    want_b, want_grad, bound = 0.0, torch.zeros_like(wide), torch.zeros_like(wide)
    for g in groups:
        picked = torch.bincount(indices[g].reshape(-1).long(), minlength=experts)
        n = logits[g].shape[0] * 50
        f = picked.double() * experts / (2 * n)
        want_b = want_b + (f * p[g].reshape(-1, experts).mean(0)).sum() / len(groups)
        inner = (p[g] * f).sum(-1, keepdim=True)
        want_grad[g] = p[g] * (gb / (len(groups) * n) * (f - inner) + 2 * gz / 200 * lse[g])
        bound[g] = p[g] * (gb / (len(groups) * n) * (f + inner) + 2 * gz / 200 * (lse[g].abs() + top[g].abs() + 1)) * size[g]
        assert torch.equal((counts[g.start] if per_sequence else counts).long(), picked)
    near(balance.detach(), want_b, want_b * float(size.max()), what="balance")
    near(z.detach(), lse.square().mean(), (lse.abs() + top.abs() + 1).square().mean(), what="z")
    near(grad, want_grad, bound, what="grad")
    assert not grad[off].any()
    # and each tolerance is far below the value that it is for
    assert float(size.max()) < 50 and float((lse.abs() + top.abs() + 1).square().mean()) < 50 * float(lse.square().mean())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_expanded_rows_go_through_the_plain_ops(dtype):
    """Rows that overlap in memory (stride 0) are copied first: the values of the contiguous call."""
    row, other, weight = normal(1, 64, dtype=dtype), normal(2, 5, 64, dtype=dtype), normal(3, 64, dtype=dtype)
    x = row.expand(5, 64)
    for call in (lambda t: (ops.rms_norm(t, weight),), lambda t: ops.add_rms_norm(t, other, weight), lambda t: (ops.swiglu(t, other),), lambda t: (ops.layer_norm(t, weight),),
                 lambda t: ops.rms_norm_backward(other, t, weight)[:2], lambda t: ops.swiglu_backward(t, other, other), lambda t: ops.moe_route(t, 4)):
        for have, want in zip(call(x), call(x.contiguous())):
            assert torch.equal(have, want)
    assert torch.equal(x, row.expand(5, 64)) and x.stride(0) == 0
