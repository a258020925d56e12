"""Host-pointer forms on views that lie between each other in one array: each output's elements come back, nothing else
of the array changes."""

import numpy as np
import pytest
import torch

from test_kv_attention_gpu import filled
from test_kv_cache_gpu import batch_of, on_device, table_of, typed

pytestmark = pytest.mark.gpu


def parts(qx, size=32, heads=2, dim=64):
    cache, table = filled(20, heads, size, dim), table_of(2, 10, 20)
    lengths, new = [300, 20], [37, 20]
    batch, begin, rows = batch_of(qx, table, lengths, new, behind=2)
    host_batch = qx.KVBatch(np.array(lengths, np.int32), table, 300, begin, rows, 37)
    return on_device(qx, cache), qx.KVCache(*cache.codes, *cache.scales), batch, host_batch, rows


@pytest.mark.parametrize("order", ["k v", "v k", "heads outside tokens", "heads in turn"])
def test_read_into_slices_of_one_array(qx, order):
    heads, dim = 2, 64
    dev, host, batch, host_batch, rows = parts(qx)
    want = [torch.full((rows, heads, dim), 4.0, device="cuda") for _ in "kv"]
    assert dev.read_dev(batch, *want) == qx.OK
    shape = (2 * heads + 1, rows, dim) if order == "heads outside tokens" else (rows, 2 * heads + 1, dim)
    wide = np.full(shape, 4.0, np.float32)
    turned = wide.transpose(1, 0, 2) if order == "heads outside tokens" else wide
    k, v = (turned[:, 0:4:2], turned[:, 1:4:2]) if order == "heads in turn" else (turned[:, :2], turned[:, 2:4])
    if order == "v k":
        k, v = v, k
    assert host.read(host_batch, k, v) == qx.OK, qx.last_error()
    for name, got, come in (("k", k, want[0]), ("v", v, want[1])):
        assert np.array_equal(got, come.cpu().numpy()), name
    assert (turned[:, 4] == 4).all()


@pytest.mark.parametrize("k_first", [True, False])
def test_read_of_two_types_into_records(qx, k_first):
    """Records of f32 and f16 rows, the f16 ones at their start: the f32 ones are on boundaries of 4 bytes, no more."""
    heads, dim = 2, 64
    dev, host, batch, host_batch, rows = parts(qx)
    want = [torch.zeros(rows, heads, dim, dtype=t, device="cuda") for t in (torch.float32, torch.float16)]
    want = want if k_first else want[::-1]
    assert dev.read_dev(batch, *want) == qx.OK
    record = np.dtype([("head", np.float16), ("narrow", np.float16, (heads, dim)), ("tail", np.float16), ("wide", np.float32, (heads, dim))])
    assert record.itemsize % 4 == 0 and record.fields["wide"][1] % 4 == 0
    data = np.zeros(rows, record)
    wide, narrow = data["wide"], data["narrow"]
    views = (wide, narrow) if k_first else (narrow, wide)
    assert host.read(host_batch, *views) == qx.OK, qx.last_error()
    for got, come in zip(views, want):
        assert np.array_equal(got, come.cpu().numpy())
    assert not data["head"].any() and not data["tail"].any()


@pytest.mark.parametrize("place", ["a part of its own", "in place"])
def test_append_and_attention_in_one_packed_array(qx, place):
    """What a program does on the device, on the host: q, k and v parts of one array, queries turned in place or
    into a part of their own, the output and its log-sum-exp beside them."""
    heads, dim, q_heads = 2, 64, 4
    dev, host, batch, host_batch, rows = parts(qx)
    rope = qx.Rope(dim)
    packed = typed((rows, 3 * q_heads + 2 * heads, dim), torch.float32, 3)
    here, there = packed.numpy().copy(), packed.cuda()
    cut = lambda a: (a[:, :4], a[:, 4:6], a[:, 6:8], a[:, 8:12], a[:, 12:16])  # noqa: E731
    for a, call, attend, b in ((here, host.append, host.attention, host_batch), (there, dev.append_dev, dev.attention_dev, batch)):
        q, k, v, spare, out = cut(a)
        turned = q if place == "in place" else spare
        assert call(b, k, v, rope, q, turned) == qx.OK, qx.last_error()
        assert attend(b, turned, out) == qx.OK, qx.last_error()
    assert np.array_equal(here, there.cpu().numpy())
