"""Calls at the edges of the operators around the layers that need no GPU."""

import ctypes

import torch
from torch.autograd import forward_ad

from popcorn_b200 import _lib, autograd
from tests.test_block_ops import FAKE, NULL, refused


def test_embedding_tables_whose_row_counter_would_wrap_are_refused(built_library):
    need, most = ctypes.c_size_t(0), 2 ** 31 - 2 ** 16
    _lib.call("b200_embedding_backward_scratch_bytes", 4, most, 1, ctypes.byref(need))
    assert need.value >= most
    for vocab in (most + 1, 2 ** 31 - 1):
        assert refused("b200_embedding_backward_scratch_bytes", 4, vocab, 1, ctypes.byref(need)) == "B200_ERR_SHAPE"
        assert refused("b200_embedding", FAKE, FAKE, FAKE, 4, vocab, 1, 1, 1, 1, _lib.BF16, 1.0, NULL) == "B200_ERR_SHAPE"
        assert refused("b200_embedding_backward", FAKE, FAKE, FAKE, 4, vocab, 1, 1, -1, 1, _lib.BF16, 1.0, FAKE, ctypes.c_size_t(1 << 40), NULL) == "B200_ERR_SHAPE"


def test_a_tangent_counts_as_a_gradient():
    x = torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        for enabled in (True, False):
            with torch.set_grad_enabled(enabled):
                assert autograd._needs_grad(None, x, dual) and not autograd._needs_grad(x, None)
    assert not autograd._needs_grad(x) and autograd._needs_grad(x.requires_grad_(True))
