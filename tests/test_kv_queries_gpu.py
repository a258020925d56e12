"""Queries at the ends of what their types hold."""

import math

import numpy as np
import pytest
import torch

from test_kv_attention_gpu import BF16, F16, F32, filled
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
