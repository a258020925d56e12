"""Memory that there is not: the call says so, and the next ones are none the worse for it."""

import ctypes as C

import pytest
import torch

import moe_reference as ref
from test_moe_gpu import check, prepared, tokens_of

pytestmark = pytest.mark.gpu


def test_a_layer_that_does_not_fit_leaves_later_calls_alone(qx):
    data, handle = torch.zeros(64, dtype=torch.uint8, device="cuda"), C.c_void_p()
    # (five terabytes; nothing is read before there is a place for it)
    status = qx.lib.qx_moe_prepare_dev(0, data.data_ptr(), data.data_ptr(), data.data_ptr(), 512, 32, 65536, 65536, None, C.byref(handle))
    assert status == qx.OUT_OF_MEMORY and not handle.value
    m = ref.layer(0, 4, 64, 32, seed=61)
    experts = prepared(qx, m)
    check(qx, m, tokens_of(m, 3, torch.float32), 2, experts=experts)


def test_a_workspace_that_does_not_fit_leaves_later_calls_alone(qx):
    handle = C.c_void_p()
    assert qx.lib.qx_workspace_create(1 << 44, C.byref(handle)) == qx.OUT_OF_MEMORY and not handle.value
    m = ref.layer(1, 4, 64, 32, seed=62)
    check(qx, m, tokens_of(m, 3, torch.float32), 2, experts=prepared(qx, m))
