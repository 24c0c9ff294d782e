"""Refusals of the operators around the layers (gated norm, balance loss, embedding): nothing here touches a GPU."""

import ctypes

import pytest
import torch

from popcorn_b200 import _lib, autograd, kernels, ops

FAKE, NULL = ctypes.c_void_p(4096), ctypes.c_void_p(0)  # FAKE is never dereferenced: validation fails first


def refused(name, *args):
    with pytest.raises(_lib.B200Error) as err:
        _lib.call(name, *args)
    return err.value.status_name


def test_python_entry_points_refuse_cpu_tensors():
    x, w = torch.randn(4, 8), torch.ones(8)
    for call in (lambda: ops.gated_add_rms_norm(x, x, w), lambda: autograd.gated_add_rms_norm(x, x, w), lambda: kernels.gated_add_rms_norm(x, x, w),
                 lambda: ops.moe_balance_loss(x, torch.zeros(4, 2, dtype=torch.int32)), lambda: kernels.moe_balance_loss(x, torch.zeros(4, 2, dtype=torch.int32)),
                 lambda: ops.embedding(torch.zeros(3, dtype=torch.int64), x), lambda: kernels.embedding(torch.zeros(3, dtype=torch.int64), x)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_the_ops_are_on_the_registry_in_their_differentiable_form():
    for name in ("gated_add_rms_norm", "moe_balance_loss", "embedding"):
        op = getattr(kernels, name)
        assert op.available_backends() == ("b200",) and not op["b200"].forward_only


@pytest.mark.parametrize("gate,rows", [((8,), 1), ((1, 1, 8), 1), ((2, 1, 8), 2), ((2, 5, 8), 10), ((5, 8), None), ((1, 8), 1), ((1, 5, 8), None), ((3, 1, 8), None),
                                       ((2, 5, 4), None), ((1, 2, 5, 8), None), ((2, 1, 1), None), ((), None)])
def test_gate_shapes(gate, rows):
    x = torch.zeros(2, 5, 8)
    if rows is None:
        with pytest.raises(ValueError, match="gate must be"):
            ops._gate_rows(x, torch.zeros(gate))
    else:
        assert ops._gate_rows(x, torch.zeros(gate)) == rows


def norm(rows=4, cols=8, gate_rows=0, x=FAKE, gate=NULL, ld=8, ldgate=8, dtype=_lib.BF16, act=0, stats=NULL, y=FAKE):
    return ("b200_gated_add_rms_norm", x, FAKE, FAKE, NULL, gate, y, FAKE, stats, rows, cols, gate_rows, ld, 8, ldgate, 8, 8, dtype, act, 1.0, 1.0, 1e-6, 0.0, NULL)


@pytest.mark.parametrize("change,status", [(dict(rows=-1), "SHAPE"), (dict(rows=1 << 31), "SHAPE"), (dict(dtype=7), "DTYPE"), (dict(act=3), "SHAPE"), (dict(x=NULL), "NULL_POINTER"),
                                           (dict(ld=4), "SHAPE"), (dict(gate=FAKE, gate_rows=3), "SHAPE"), (dict(gate=FAKE, gate_rows=0), "SHAPE"),
                                           (dict(gate=FAKE, gate_rows=2, ldgate=4), "SHAPE"), (dict(x=ctypes.c_void_p(4097)), "ALIGNMENT"),
                                           (dict(stats=ctypes.c_void_p(4100)), "ALIGNMENT"), (dict(y=NULL), "NULL_POINTER")])
def test_norm_refusals(built_library, change, status):
    assert refused(*norm(**change)) == "B200_ERR_" + status


def test_norm_backward_refusals(built_library):
    def call(rows=4, post=NULL, dpost=NULL, gate=NULL, dgate=NULL, gy=FAKE, ldgy=8, stats=FAKE):
        return refused("b200_gated_add_rms_norm_backward", gy, NULL, FAKE, FAKE, FAKE, post, gate, stats, FAKE, FAKE, FAKE, dpost, dgate, rows, 8, 1, ldgy, 8, 8, 8, 8, _lib.F32,
                       0, 1.0, 1.0, 0.0, FAKE, ctypes.c_size_t(0), NULL)
    assert call(post=FAKE) == "B200_ERR_NULL_POINTER"
    assert call(dgate=FAKE) == "B200_ERR_NULL_POINTER"
    assert call(gy=NULL) == "B200_ERR_NULL_POINTER"
    assert call(ldgy=4) == "B200_ERR_SHAPE"
    assert call(stats=ctypes.c_void_p(4100)) == "B200_ERR_ALIGNMENT"


def test_balance_refusals(built_library):
    def call(groups=1, tokens=4, experts=8, top_k=2, ld=8, dtype=_lib.F32, logits=FAKE, table=FAKE):
        return refused("b200_moe_balance_loss", logits, FAKE, NULL, FAKE, FAKE, FAKE, NULL, table, groups, tokens, experts, top_k, ld, dtype, FAKE, ctypes.c_size_t(0), NULL)
    assert call(experts=1025, ld=1025) == call(experts=0) == call(top_k=0) == call(top_k=9) == call(experts=64, ld=64, top_k=33) == "B200_ERR_SHAPE"
    assert call(groups=65536) == call(tokens=1 << 31) == call(tokens=1 << 30, top_k=2) == call(ld=4) == call(groups=-1) == "B200_ERR_SHAPE"
    assert call(dtype=5) == "B200_ERR_DTYPE"
    assert call(logits=NULL) == call(table=NULL) == "B200_ERR_NULL_POINTER"
    assert call(logits=ctypes.c_void_p(4098)) == "B200_ERR_ALIGNMENT"
    backward = ("b200_moe_balance_loss_backward", FAKE, NULL, NULL, FAKE, FAKE, FAKE, FAKE, 1, 4, 8, 8, 8, _lib.F32, NULL)
    assert refused(*backward) == "B200_ERR_NULL_POINTER"
    assert refused(*backward[:3], FAKE, *backward[4:11], 7, *backward[12:]) == "B200_ERR_SHAPE"


def test_embedding_refusals(built_library):
    def call(tokens=4, vocab=10, cols=8, ldw=8, ids=FAKE, weight=FAKE, wide=1, dtype=_lib.BF16):
        return refused("b200_embedding", ids, weight, FAKE, tokens, vocab, cols, ldw, 8, wide, dtype, 1.0, NULL)
    assert call(tokens=-1) == call(tokens=(1 << 30) + 1) == call(vocab=1 << 31) == call(cols=65535 * 128 + 1) == call(ldw=4) == "B200_ERR_SHAPE"
    assert call(ids=NULL) == call(weight=NULL) == "B200_ERR_NULL_POINTER"
    assert call(ids=ctypes.c_void_p(4100)) == call(weight=ctypes.c_void_p(4097)) == "B200_ERR_ALIGNMENT"
    assert call(dtype=9) == "B200_ERR_DTYPE"
    backward = ("b200_embedding_backward", FAKE, FAKE, FAKE, 4, 10, 8, 4, -1, 0, _lib.F32, 1.0, FAKE, ctypes.c_size_t(0), NULL)
    assert refused(*backward) == "B200_ERR_SHAPE"
    need = ctypes.c_size_t(0)
    _lib.call("b200_embedding_backward_scratch_bytes", 4, 10, 8, ctypes.byref(need))
    assert need.value >= 2 * 4 * 4 + 4


def test_empty_calls_touch_nothing(built_library):
    _lib.call("b200_gated_add_rms_norm", *[NULL] * 8, 0, 8, 0, 8, 8, 8, 8, 8, _lib.BF16, 0, 1.0, 1.0, 1e-6, 0.0, NULL)
    _lib.call("b200_moe_balance_loss_backward", *[NULL] * 7, 1, 0, 8, 8, 8, _lib.F32, NULL)
    _lib.call("b200_embedding", NULL, NULL, NULL, 0, 10, 8, 8, 8, 1, _lib.BF16, 1.0, NULL)
    _lib.call("b200_embedding_backward", NULL, NULL, NULL, 4, 0, 8, 8, -1, 1, _lib.BF16, 1.0, NULL, ctypes.c_size_t(0), NULL)
