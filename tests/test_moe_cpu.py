"""What mixture-of-experts layers refuse; shapes that the Python calls look at; the reference against itself."""

import ctypes as C

import numpy as np
import pytest
import torch

import moe_reference as ref


def served(qx, status):
    return status in (qx.OK, qx.DEVICE_ERROR)  # (there may be no device here)


def test_prepare_refuses(qx):
    data = np.zeros(1 << 16, np.uint8)
    handle = C.c_void_p()

    def call(fmt=0, gate=data, up=data, down=data, experts=2, shared=0, dim=64, inner=32, out=C.byref(handle)):
        address = [None if a is None else a.ctypes.data for a in (gate, up, down)]
        status = qx.lib.qx_moe_prepare(fmt, *address, experts, shared, dim, inner, out)
        if status == qx.OK:
            qx.lib.qx_moe_destroy(handle)
        return status

    assert served(qx, call())
    assert call(out=None) == qx.INVALID_ARGUMENT
    for name in ("gate", "up", "down"):
        assert call(**{name: None}) == qx.INVALID_ARGUMENT
    for fmt in (-1, 2):
        assert call(fmt=fmt) == qx.UNSUPPORTED_FORMAT
    for bad in (dict(experts=0), dict(experts=513), dict(shared=-1), dict(shared=33), dict(dim=0), dict(dim=48), dict(dim=-32),
                dict(dim=65568), dict(inner=0), dict(inner=31), dict(inner=65568)):
        assert call(**bad) == qx.INVALID_SHAPE


def test_apply_refuses_without_a_layer(qx):
    x = np.zeros((2, 64), np.float32)
    view, r = qx.RowsView(x.ctypes.data, 0, 64), qx.Router(x, 1).view
    assert qx.lib.qx_moe_apply(None, r, view, view, 2, 3, None, None) == qx.INVALID_ARGUMENT
    assert qx.lib.qx_moe_apply_dev(None, r, view, view, 2, 3, None, None, None, None) == qx.INVALID_ARGUMENT


def test_the_header_and_the_binding_agree(qx):
    assert C.sizeof(qx.MoeRouterView) == 40


def test_python_calls_look_at_shapes(qx):
    experts = qx.Experts()
    raw = np.zeros(2 * 32 * 2 * 34, np.uint8)
    with pytest.raises(AssertionError):
        experts.prepare(0, raw, raw, raw[1:], 2, 64, 32)
    with pytest.raises(AssertionError):
        experts.prepare(0, raw, raw, raw, 3, 64, 32)
    weights, x = np.zeros((4, 64), np.float32), np.zeros((3, 64), np.float32)
    router = qx.Router(weights, 2)
    for bad in (dict(x=np.zeros((3, 32), np.float32)), dict(out=np.zeros((2, 64), np.float32)),
                dict(chosen=np.zeros((3, 1), np.int32)), dict(chosen=np.zeros((3, 2), np.int64)), dict(weights=np.zeros((2, 2), np.float32))):
        with pytest.raises(AssertionError):
            experts.apply(router, bad.pop("x", x), bad.pop("out", x), **bad)
    with pytest.raises(AssertionError):
        qx.Router(weights, 2, bias=np.zeros(3, np.float32))
    with pytest.raises(AssertionError):
        qx.Router(weights[:, ::2], 2)
    assert experts.apply(router, x, x) == qx.INVALID_ARGUMENT  # not prepared


def test_the_reference_against_differences_of_its_parts():
    """The reference's output is linear in the router's scale, and its blocks are what their bytes say."""
    for fmt in (0, 1):
        m = ref.layer(fmt, 5, 64, 32, 1)
        x = torch.randn(4, 64, generator=torch.Generator().manual_seed(1))
        one, _ = ref.apply(m, x, 2, scale=1.0, out_type=torch.float32)
        two, _ = ref.apply(m, x, 2, scale=2.0, out_type=torch.float32)
        none, _ = ref.apply(m, x, 2, scale=0.0, out_type=torch.float32)
        assert torch.allclose(two - none, 2 * (one - none), rtol=1e-12, atol=1e-12)
        b = m.raw[0].reshape(-1, 34 if fmt == 0 else 18)
        d = b[:, :2].copy().view(np.float16).astype(np.float64)
        if fmt == 0:
            values = b[:, 2:].copy().view(np.int8) * d
        else:
            values = (np.concatenate([b[:, 2:] & 15, b[:, 2:] >> 4], 1).astype(np.float64) - 8) * d
        assert np.array_equal(values.reshape(6, 32, 64), m.gate.numpy())
