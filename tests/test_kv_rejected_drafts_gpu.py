"""What drafts that are rejected leave in the cache, and how a program goes without: the block in which they began, copied
before and put back after."""

import pytest
import torch

from test_kv_cache_gpu import table_of, typed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kept", [33, 47, 48])
def test_a_block_that_is_put_back(qx, kept):
    """Blocks of 16 tokens; ten drafts, far louder than the text, begin inside a block or (48) with one and end in the next."""
    heads, dim, size = 2, 64, 16
    table = torch.from_numpy(table_of(1, 4, 5)).cuda()
    k, v = (typed((kept + 3, heads, dim), torch.bfloat16, i).cuda() for i in (1, 2))
    loud_k, loud_v = (typed((10, heads, dim), torch.bfloat16, i, 50.0).cuda() for i in (3, 4))

    def append(cache, length, keys, values):
        n = len(keys)
        batch = qx.KVBatch(torch.tensor([length], dtype=torch.int32, device="cuda"), table, 64,
                           torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, n)
        qx.check(cache.append_dev(batch, keys, values), "append")

    def contents(cache):
        whole = qx.KVBatch(torch.tensor([kept + 3], dtype=torch.int32, device="cuda"), table, 64,
                           torch.tensor([0, kept + 3], dtype=torch.int32, device="cuda"), kept + 3, kept + 3)
        out = [torch.empty(kept + 3, heads, dim, device="cuda") for _ in "kv"]
        qx.check(cache.read_dev(whole, *out), "read")
        torch.cuda.synchronize()
        qx.check(qx.lib.qx_check_device_errors(), "read")
        return out

    results = []
    for drafts, put_back in ((False, False), (True, False), (True, True)):
        cache = qx.KVCache.empty(5, heads, size, dim)
        append(cache, kept, k[:kept], v[:kept])
        if drafts:
            block = int(table[0, kept // size])
            before = [a[block].clone() for a in cache.arrays]
            append(cache, kept + 10, loud_k, loud_v)
            if put_back:
                for a, old in zip(cache.arrays, before):
                    a[block] = old
        append(cache, kept + 3, k[kept:], v[kept:])
        results.append(contents(cache))
    never, traces, restored = results
    for a, b in zip(never, restored):
        assert torch.equal(a, b)
    # without that, the text's part of the block is as coarse as the loudest draft asked for
    first = kept // size * size
    for a, b in zip(never, traces):
        assert torch.equal(a[:first], b[:first])
        assert torch.equal(a[first:], b[first:]) == (kept % size == 0)
