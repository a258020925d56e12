"""Block scales at the ends of their range, in a cache that somebody else filled too: zero and tiny ones beside codes
that are not zero."""

import numpy as np
import pytest
import torch

from kv_reference import Cache
from test_kv_attention_gpu import BF16, F32
from test_kv_cache_gpu import append_both, on_device, table_of, typed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [16, 128])
@pytest.mark.parametrize("before", [0.0, -0.0, 2.0 ** -149, 2.0 ** -110])
@pytest.mark.parametrize("spread", [[1.0], [0.0, 1.0], [1e-35, 0.0, 1.0]])
def test_append_beside_codes_without_a_scale(qx, dtype, size, before, spread):
    """Older codes of a block whose scale is zero, or is too small and becomes zero, count as zeros whatever they are."""
    heads, dim = 2, 64
    cache, table = Cache(6, heads, size, dim), table_of(2, 3, 6)  # (codes of every kind)
    for i in range(2):
        cache.scales[i][:] = before
    dev, lengths = on_device(qx, cache), [size + 5, 9]
    for step, by in enumerate(spread):
        lengths = [t + 2 for t in lengths]
        k, v = (typed((4, heads, dim), dtype, 10 * step + i, by) for i in range(2))
        append_both(qx, dev, cache, table, lengths, [2, 2], k, v)
        torch.cuda.synchronize()
        for i in range(2):
            assert np.array_equal(dev.arrays[2 + i].cpu().numpy(), cache.scales[i])
            for s, t in enumerate(lengths):
                for p in range((t - 1) // size * size, t):
                    block = table[s, p // size]
                    got = dev.arrays[i][block, :, p % size].cpu().numpy().astype(np.float64)
                    scale = cache.scales[i][block].astype(np.float64)[:, None]
                    assert np.array_equal(got * scale, cache.codes[i][block, :, p % size] * scale), (step, "kv"[i], p)
    same_codes = [(dev.arrays[i].cpu().numpy(), cache.codes[i]) for i in range(2)]
    for s, t in enumerate(lengths):  # (scales are numbers now: the codes too are the rule's)
        block, kept = table[s, (t - 1) // size], (t - 1) % size + 1
        for got, want in same_codes:
            assert np.array_equal(got[block, :, :kept], want[block, :, :kept])
