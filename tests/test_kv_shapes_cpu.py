"""The Python calls of rotation, cache and attention look at the shapes of what they are given: the library sees
addresses and counts only, and a kernel would follow them past an array's end."""

import numpy as np
import pytest
import torch


def int32(*values):
    return np.array(values, np.int32)


def arrays(blocks=4, heads=2, size=16, dim=32):
    return [np.zeros((blocks, heads, size, dim), np.int8) for _ in "kv"] + [np.zeros((blocks, heads), np.float32) for _ in "kv"]


@pytest.fixture
def parts(qx):
    cache = qx.KVCache(*arrays())
    batch = qx.KVBatch(int32(20, 5), np.array([[0, 1], [2, 3]], np.int32), 32, int32(0, 2, 3), 3, 2)
    return cache, batch, np.zeros((3, 2, 32), np.float32), np.zeros((3, 4, 32), np.float32)


def refused(call):
    with pytest.raises(AssertionError):
        call()


def served(qx, status):
    return status in (qx.OK, qx.DEVICE_ERROR)


def test_batches(qx):
    lengths, table, begin = int32(20, 5), np.zeros((2, 2), np.int32), int32(0, 2, 3)
    for bad in ((lengths, table[:1], begin), (lengths, table, begin[:2]), (lengths, table.reshape(-1), begin),
                (lengths.reshape(1, 2), table, begin), (lengths, table, begin.reshape(1, 3)), (lengths, table[:, :, None], begin)):
        refused(lambda: qx.KVBatch(bad[0], bad[1], 32, bad[2], 3, 2))
    refused(lambda: qx.KVBatch(lengths, table[:1], 32, None, 4, 2))
    # buffers for more sequences than the call has are fine
    more = qx.KVBatch(lengths[:1], table, 32, begin, 3, 2)
    assert more.view.sequences == 1 and more.view.table_stride == 2
    qx.KVBatch(lengths, table, 32, None, 4, 2)


def test_append(qx, parts):
    cache, batch, x, q = parts
    rope, at = qx.Rope(32), np.zeros(3, np.int64)
    assert served(qx, cache.append(batch, x, x, rope, q, q, at))
    for k, v in ((x[:2], x), (x, x[:2]), (x[..., :16], x), (x, np.zeros((3, 2, 48), np.float32))):
        refused(lambda: cache.append(batch, k, v))
    for a, b in ((q[:2], q), (q, q[:2]), (q[..., :16], q), (q, np.zeros((3, 4, 64), np.float32))):
        refused(lambda: cache.append(batch, x, x, rope, a, b))
    refused(lambda: cache.append(batch, x, x, rope, positions=at[:2]))
    longer = np.zeros((5, 2, 32), np.float32)  # rows behind the call's
    assert served(qx, cache.append(batch, longer, longer, rope, positions=np.zeros(5, np.int64)))


def test_read(qx, parts):
    cache, batch, x, _ = parts
    assert served(qx, cache.read(batch, x, None)) and served(qx, cache.read(batch, None, x.copy()))
    for bad in (x[:2], x[..., :16], np.zeros((3, 2, 48), np.float32)):
        refused(lambda: cache.read(batch, bad, x))
        refused(lambda: cache.read(batch, x, bad))


def test_attention(qx, parts):
    cache, batch, _, q = parts
    out, lse = q.copy(), np.zeros((3, 4), np.float32)
    assert served(qx, cache.attention(batch, q, out, lse=lse))
    for bad in (q[:2], q[..., :16], np.zeros((3, 4, 48), np.float32)):
        refused(lambda: cache.attention(batch, bad, out))
        refused(lambda: cache.attention(batch, q, bad))
    for bad in (lse[:2], lse[:, :2].copy(), lse.T.copy(), np.zeros((3, 5), np.float32), lse.reshape(-1)):
        refused(lambda: cache.attention(batch, q, out, lse=bad))


def test_rotation(qx):
    rope, x, at = qx.Rope(32), np.zeros((3, 2, 48), np.float32), np.zeros(3, np.int64)
    assert served(qx, rope.apply(x, x.copy(), at))
    for y in (x[:2], x[:, :1], x[..., :32], np.zeros((4, 2, 48), np.float32), np.zeros((3, 2, 64), np.float32)):
        refused(lambda: rope.apply(x, y, at))
    refused(lambda: rope.apply(x, x, at[:2]))


def test_elements_of_another_size_than_their_type(qx, parts):
    """16-bit arrays named as f32 would be read to twice their length."""
    cache, batch, x, q = parts
    narrow_q, narrow, at = np.zeros(q.shape, np.uint16), np.zeros(x.shape, np.uint16), np.zeros(3, np.int64)
    for kind, a, b in ((qx.F32, narrow_q, narrow), (qx.BF16, q, x)):
        refused(lambda: cache.attention(batch, a, a, kind=kind))
        refused(lambda: cache.append(batch, b, b, kind=kind))
        refused(lambda: cache.read(batch, b, None, kind=kind))
        refused(lambda: qx.Rope(32).apply(b, b, at, kind=kind))
    assert served(qx, cache.attention(batch, narrow_q, narrow_q, kind=qx.BF16))


class Elsewhere:
    """What a call on the device looks at of a tensor, without one."""

    def __init__(self, *shape, dtype=torch.float32):
        self.like = torch.empty(shape, dtype=dtype)
        self.shape, self.dtype, self.stride = self.like.shape, dtype, self.like.stride

    def get_device(self):
        return 0

    def data_ptr(self):
        return 4096

    def is_contiguous(self):
        return True


def test_device_calls(qx, monkeypatch):
    """The `_dev` calls refuse the same before the library is called."""
    called = []
    for name in ("qx_kv_append_dev", "qx_kv_read_dev", "qx_kv_attention_dev", "qx_rope_apply_dev"):
        monkeypatch.setattr(qx.lib, name, lambda *a, name=name: called.append(name) or qx.OK)
    monkeypatch.setattr(qx, "_device", lambda: 0)
    monkeypatch.setattr(qx, "_stream", lambda: 0)
    E, i8, i32, i64 = Elsewhere, torch.int8, torch.int32, torch.int64
    cache = qx.KVCache(E(4, 2, 16, 32, dtype=i8), E(4, 2, 16, 32, dtype=i8), E(4, 2), E(4, 2))
    refused(lambda: qx.KVBatch(E(2, dtype=i32), E(1, 2, dtype=i32), 32, E(3, dtype=i32), 3, 2))
    refused(lambda: qx.KVBatch(E(2, dtype=i32), E(2, 2, dtype=i32), 32, E(2, dtype=i32), 3, 2))
    batch = qx.KVBatch(E(2, dtype=i32), E(2, 2, dtype=i32), 32, E(3, dtype=i32), 3, 2)
    x, q, at, rope = E(3, 2, 32), E(3, 4, 32), E(3, dtype=i64), qx.Rope(32)
    assert cache.append_dev(batch, x, x, rope, q, q, at) == cache.read_dev(batch, x, None) == qx.OK
    assert cache.attention_dev(batch, q, q, lse=E(3, 4)) == rope.apply_dev(x, x, at) == qx.OK
    assert called == ["qx_kv_append_dev", "qx_kv_read_dev", "qx_kv_attention_dev", "qx_rope_apply_dev"]
    for bad in (E(2, 2, 32), E(3, 2, 16), E(3, 2, 64)):
        refused(lambda: cache.append_dev(batch, bad, x))
        refused(lambda: cache.append_dev(batch, x, bad))
        refused(lambda: cache.read_dev(batch, bad, None))
        refused(lambda: cache.read_dev(batch, None, bad))
        refused(lambda: rope.apply_dev(x, bad, at))
    for bad in (E(2, 4, 32), E(3, 4, 16), E(3, 4, 64)):
        refused(lambda: cache.append_dev(batch, x, x, rope, bad, q))
        refused(lambda: cache.append_dev(batch, x, x, rope, q, bad))
        refused(lambda: cache.attention_dev(batch, bad, q))
        refused(lambda: cache.attention_dev(batch, q, bad))
    for bad in (E(2, 4), E(4, 3), E(3, 2), E(12)):
        refused(lambda: cache.attention_dev(batch, q, q, lse=bad))
    refused(lambda: cache.append_dev(batch, x, x, rope, positions=E(2, dtype=i64)))
    refused(lambda: rope.apply_dev(x, x, E(2, dtype=i64)))
    assert len(called) == 4


def test_more_rows_than_32_bits_count_on_the_host(qx):
    """Sequences of max_tokens rows each, without token_begin: their first rows would wrap."""
    cache = qx.KVCache(*arrays())
    batch = qx.KVBatch(np.zeros(3, np.int32), np.zeros((3, 2), np.int32), 32, None, 3 << 30, 1 << 30)
    q, out = np.zeros((1, 2, 32), np.float32), np.zeros((1, 2, 32), np.float32)
    views = qx.heads_view(q, token_stride=0), qx.heads_view(out, token_stride=64)
    assert qx.lib.qx_kv_attention(cache.view, batch.view, *views, None, 1.0, 1, 0) == qx.INVALID_SHAPE
