"""Queries at the ends of what their types hold."""

import math

import numpy as np
import pytest
import torch

from test_kv_attention_gpu import BF16, F16, F32, check, filled
from test_kv_cache_gpu import batch_of, on_device, table_of, typed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("new", [4, 130, 700])
@pytest.mark.parametrize("sign", [1, -1])
def test_a_query_that_is_no_number_gives_no_number(qx, dtype, value, new, sign):
    """... also where the codes of all keys that its row sees take the infinity the same way, to weights of zero say; and
    the other rows keep their bits."""
    cache, table = filled(48, 1, 16, 64), table_of(1, 48, 48)
    cache.codes[0][:, :, :, 7] = sign * (np.abs(cache.codes[0][:, :, :, 7].astype(np.int32)) % 127 + 1)
    dev, q = on_device(qx, cache), typed((new, 2, 64), dtype, 3)
    batch, _, _ = batch_of(qx, table, [new], [new])
    clean, got = (torch.full((new, 2, 64), 3.0, dtype=dtype, device="cuda") for _ in "ab")
    before, lse = (torch.zeros(new, 2, device="cuda") for _ in "ab")
    assert dev.attention_dev(batch, q.cuda(), clean, lse=before) == qx.OK
    bad = torch.zeros(new, 2, dtype=torch.bool, device="cuda")
    for row, head in ((0, 0), (1, 1), (new - 1, 0)):
        q[row, head, 7], bad[row, head] = value, True
    assert dev.attention_dev(batch, q.cuda(), got, lse=lse) == qx.OK
    assert bool(got[bad].isnan().all()) and bool(lse[bad].isnan().all())
    assert torch.equal(got[~bad], clean[~bad]) and torch.equal(lse[~bad], before[~bad])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [4, 130])
def test_a_query_that_is_no_number_and_sees_no_key(qx, dtype, new):
    """More rows than tokens: what sees nothing gives zeros, whatever its query."""
    cache, table = filled(4, 1, 16, 64), table_of(1, 4, 4)
    q = typed((new, 2, 64), dtype, 3)
    q[0, 0, 7], q[1, 1, 3] = math.inf, math.nan
    batch, _, _ = batch_of(qx, table, [new - 2 if new < 10 else 40], [new])
    out, lse = torch.full((new, 2, 64), 3.0, dtype=dtype, device="cuda"), torch.zeros(new, 2, device="cuda")
    assert on_device(qx, cache).attention_dev(batch, q.cuda(), out, lse=lse) == qx.OK
    assert bool((out[:2] == 0).all()) and bool((lse[:2] == -math.inf).all())


@pytest.mark.parametrize("dtype,above", [(F32, 2.0 ** 12), (F32, 2.0 ** 30), (F16, 2.0 ** 12), (BF16, 2.0 ** 12), (BF16, 2.0 ** 30)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 5, 200])
def test_one_element_far_above_its_row(qx, dtype, above, dim, new):
    """... where the keys hold zeros, so that the small elements make the scores: they are rounded to 2^-22 of the large
    one (the tolerance counts that), and to nothing else."""
    cache, table = filled(20, 2, 32, dim), table_of(1, 20, 20)
    cache.codes[0][:, :, :, 5] = 0
    q = typed((new, 4, dim), dtype, 11).double()
    q[:, :, 5] = above
    check(qx, cache, on_device(qx, cache), table, [600], [new], q.to(dtype))


@pytest.mark.parametrize("new", [1, 3, 200])
def test_bits_of_a_session_may_follow_its_neighbours(qx, new):
    """What stays: the tolerance, and the bits of the same call made again."""
    cache, table = filled(600, 8, 32, 64), table_of(12, 50, 600)
    dev, q = on_device(qx, cache), typed((12 * new, 32, 64), BF16, 2)
    for others in (1600, 700, new):
        lengths = [1500] + [others] * 11
        first, lse = check(qx, cache, dev, table, lengths, [new] * 12, q)
        again, lse_again = check(qx, cache, dev, table, lengths, [new] * 12, q)
        assert torch.equal(first, again) and torch.equal(lse, lse_again)
