"""What attention of drafted trees refuses."""

import ctypes as C

import numpy as np
import pytest


def int32(*values):
    return np.array(values, np.int32)


@pytest.fixture
def parts(qx):
    codes = [np.zeros((4, 2, 16, 32), np.int8) for _ in "kv"]
    cache = qx.KVCache(*codes, *[np.zeros((4, 2), np.float32) for _ in "kv"])
    batch = qx.KVBatch(int32(20, 5), np.array([[0, 1], [2, 3]], np.int32), 32, int32(0, 2, 3), 3, 2)
    return cache, batch, np.zeros((3, 4, 32), np.float32), np.zeros(3, np.int64)


def test_refusals(qx, parts):
    cache, batch, q, seen = parts
    view = qx.HeadsView(q.ctypes.data, 0, 4, 128, 32)

    def call(window=0, mask=seen.ctypes.data, max_tokens=2, scale=1.0, heads=view):
        b = qx.KVBatchView.from_buffer_copy(batch.view)
        b.max_tokens = max_tokens
        return qx.lib.qx_kv_tree_attention_dev(cache.view, b, heads, heads, None, scale, window, mask, None, None)

    assert call(max_tokens=65) == qx.INVALID_SHAPE
    for window in (-1, 1, 63):
        assert call(window=window) == qx.INVALID_ARGUMENT
    assert call(mask=None) == qx.INVALID_ARGUMENT
    assert call(mask=seen.ctypes.data + 4) == qx.INVALID_ARGUMENT
    assert call(scale=float("nan")) == qx.INVALID_ARGUMENT
    assert call(heads=qx.HeadsView(q.ctypes.data, 0, 3, 128, 32)) == qx.INVALID_SHAPE
    assert call(heads=qx.HeadsView(q.ctypes.data, 3, 4, 128, 32)) == qx.UNSUPPORTED_FORMAT


def test_host_calls_look_at_what_the_arrays_say(qx, parts):
    cache, batch, q, seen = parts
    assert cache.tree_attention(batch, q, q, seen) in (qx.OK, qx.DEVICE_ERROR)  # (there may be no device here)
    assert cache.tree_attention(batch, q, q, seen, window=10) == qx.INVALID_ARGUMENT
    wrong = qx.KVBatch(int32(20, 5), np.array([[0, 1], [2, 9]], np.int32), 32, int32(0, 2, 3), 3, 2)
    assert cache.tree_attention(wrong, q, q, seen) in (qx.OK, qx.DEVICE_ERROR)  # (block 9 is behind the text)
    wrong = qx.KVBatch(int32(20, 5), np.array([[0, 9], [2, 3]], np.int32), 32, int32(0, 2, 3), 3, 2)
    assert cache.tree_attention(wrong, q, q, seen) == qx.INVALID_ARGUMENT
    wrong = qx.KVBatch(int32(20, 40), np.array([[0, 1], [2, 3]], np.int32), 32, int32(0, 2, 3), 3, 2)
    assert cache.tree_attention(wrong, q, q, seen) == qx.INVALID_ARGUMENT


def test_python_calls_look_at_shapes(qx, parts):
    cache, batch, q, seen = parts
    for bad in (seen[:2], seen.astype(np.int32), seen.reshape(3, 1)):
        with pytest.raises(AssertionError):
            cache.tree_attention(batch, q, q, bad)
    with pytest.raises(AssertionError):
        cache.tree_attention(batch, q[:2], q, seen)
    assert C.sizeof(C.c_ulonglong) == seen.itemsize
