"""What the joins between blocks refuse, and in which order; shapes that the Python calls look at."""

import ctypes as C

import numpy as np
import pytest


def view(qx, a, kind=0, stride=None):
    return qx.RowsView(None if a is None else a.ctypes.data, kind, a.shape[1] if stride is None else stride)


@pytest.fixture
def parts(qx):
    return [np.zeros((4, 24), np.float32) for _ in range(4)]


def call(qx, residual, block, joined, normed, pre=None, post=None, gate=None, scale=1.0, tokens=4, dim=24):
    return qx.lib.qx_residual_norm_dev(residual, block, post, gate, scale, joined, pre, normed, tokens, dim, None)


def served(qx, status):
    return status in (qx.OK, qx.DEVICE_ERROR)  # (there may be no device here)


def norm(qx, **changes):
    n = qx.Norm().view
    for name, value in changes.items():
        setattr(n, name, value)
    return n


def test_refusals(qx, parts):
    r, b, j, o = (view(qx, a) for a in parts)
    n = norm(qx)
    nothing = call(qx, r, b, j, o, n, tokens=0)
    assert served(qx, nothing)
    # shapes
    for tokens, dim in ((-1, 24), (4, 0), (4, -8), (4, 32769)):
        assert call(qx, r, b, j, o, n, tokens=tokens, dim=dim) == qx.INVALID_SHAPE
    assert call(qx, view(qx, parts[0], stride=-1), b, j, o, n) == qx.INVALID_SHAPE
    assert call(qx, view(qx, parts[0], stride=1 << 61), b, j, o, n) == qx.INVALID_SHAPE
    assert call(qx, r, b, view(qx, parts[2], stride=23), o, n) == qx.INVALID_SHAPE  # rows that overlap
    assert call(qx, r, b, view(qx, parts[2], stride=0), o, n) == qx.INVALID_SHAPE
    # types
    for bad in (-1, 3):
        assert call(qx, view(qx, parts[0], bad), b, j, o, n) == qx.UNSUPPORTED_FORMAT
        assert call(qx, r, b, j, view(qx, parts[3], bad), n) == qx.UNSUPPORTED_FORMAT
        weight = norm(qx, type=bad, weight=parts[0].ctypes.data)
        assert call(qx, r, b, j, o, weight) == qx.UNSUPPORTED_FORMAT
    # operands that do not go together
    bad = qx.INVALID_ARGUMENT
    assert call(qx, None, None, j, o, n) == bad
    assert call(qx, r, b, None, None) == bad
    assert call(qx, r, b, j, o) == bad and call(qx, r, b, j, None, n) == bad  # a norm and its output come together
    assert call(qx, r, None, j, None, post=n) == bad and call(qx, r, None, j, None, gate=b) == bad
    assert call(qx, r, b, j, None, scale=float("inf")) == bad and call(qx, r, b, j, None, scale=float("nan")) == bad
    for changes in (dict(kind=2), dict(eps=-1e-6), dict(eps=float("nan")), dict(offset=float("inf")),
                    dict(weight=parts[0].ctypes.data + 2), dict(bias=parts[0].ctypes.data + 1)):
        assert call(qx, r, b, j, o, norm(qx, **changes)) == bad and call(qx, r, b, j, None, None, norm(qx, **changes)) == bad
    # places
    null = qx.RowsView(None, 0, 24)
    odd = qx.RowsView(parts[0].ctypes.data + 2, 0, 24)
    for x in (null, odd):
        assert call(qx, x, b, j, o, n) == bad and call(qx, r, x, j, o, n) == bad and call(qx, r, b, x, o, n) == bad
        assert call(qx, r, b, j, x, n) == bad and call(qx, r, b, j, o, n, gate=x) == bad
    assert call(qx, r, b, j, j, n) == bad  # both outputs at one place
    assert call(qx, r, b, view(qx, parts[0], stride=25), o, n) == bad  # a read view's place, but another view
    assert call(qx, r, b, view(qx, parts[0], 1, 24), o, n) == bad
    assert call(qx, r, b, j, o, n, gate=qx.RowsView(parts[3].ctypes.data, 0, 0)) == bad


def test_the_header_and_the_binding_agree(qx):
    assert C.sizeof(qx.RowsView) == 24 and C.sizeof(qx.NormView) == 32


def test_python_calls_look_at_shapes(qx, parts):
    r, b, j, o = parts
    n = qx.Norm(np.ones(24, np.float32))
    assert served(qx, qx.residual_norm(r, b, j, o, n, n, np.ones((1, 24), np.float32)))

    def refused(*operands, **more):
        with pytest.raises(AssertionError):
            qx.residual_norm(*operands, **more)

    refused(r, b[:3], j, o, n)
    refused(r, b[:, :23], j, o, n)
    refused(r, b, j[:2], o, n)
    refused(r, b, j, o, qx.Norm(np.ones(23, np.float32)))
    refused(r, b, j, o, n, gate=np.ones((3, 24), np.float32))
    refused(r, np.zeros((24, 8), np.float32).T[:4], j, o, n)  # columns are not rows
    with pytest.raises(AssertionError):
        qx.Norm(np.ones(24, np.float32), np.ones(23, np.float32))
    with pytest.raises(AssertionError):
        qx.Norm(np.ones((2, 24), np.float32))
    with pytest.raises(AssertionError):
        qx.Norm(np.ones(48, np.float32)[::2])
    with pytest.raises((AssertionError, RuntimeError)):  # (without a device torch says so first)
        qx.residual_norm_dev(r, b, j, o, n)
