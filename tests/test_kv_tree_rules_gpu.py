"""Trees on both sides of the sizes that choose a kernel: 16 rows of a kv head and more, texts and windows around 1024 keys;
and masks that leave rows without a key where two softmax groups share a tile's keys."""

import numpy as np
import pytest
import torch

from test_kv_attention_gpu import filled
from test_kv_cache_gpu import on_device, table_of, typed
from test_kv_tree_gpu import BF16, F16, check, tables, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group,drafts", [(1, 16), (1, 17), (2, 12), (1, 47), (3, 16), (16, 1), (17, 1)])
@pytest.mark.parametrize("length,window", [(1023, 0), (1024, 0), (5000, 0), (5000, 64), (5000, 959), (5000, 960), (3001, 2000)])
def test_both_sides_of_the_prompt_kernel(qx, dtype, group, drafts, length, window):
    rng = np.random.default_rng(group * drafts + length)
    width = -(-length // 64)
    cache, table = filled(width + 8, 2, 64, 128, seed=window), tables(rng, 2, width, width + 8)
    trees = [tree(rng, drafts), tree(rng, max(1, drafts // 2))]
    q = typed((drafts + len(trees[1]) + 1, 2 * group, 128), dtype, drafts)
    check(qx, cache, on_device(qx, cache), table, [length, length // 3], trees, q, window, behind=1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("group", [1, 2, 6])
@pytest.mark.parametrize("front", [0, 3, 140])
def test_masks_of_every_kind_on_odd_numbers_of_tiles(qx, dtype, dim, group, front):
    """60 drafts, so one tile of rows, partly filled (60 or 120), or three; the first 60 to 200 keys lie in either half of a
    tile of keys. With nothing in front of the drafts rows see no key, or keys of one half only."""
    drafts, rng = 60, np.random.default_rng(dim + group + front)
    masks = [int(rng.integers(0, 1 << 60)) for _ in range(drafts)]
    masks[0] = masks[7] = masks[59] = 0
    masks[1], masks[2], masks[3] = (1 << 60) - 1, 1 << 59, 1
    masks[4:7] = [(1 << 30) - 1, (1 << 60) - (1 << 40), 1 << 20]
    cache, table = filled(16, 2, 32, dim), table_of(2, 8, 16)
    q = typed((2 * drafts, 2 * group, dim), dtype, 3)
    check(qx, cache, on_device(qx, cache), table, [drafts + front, drafts], [masks, masks[::-1]], q, junk=(1 << 64) - 1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [2, 6])
def test_rows_without_keys_beside_long_texts(qx, dtype, group):
    """Several chunks of keys, joined; one sequence sees all of its text, one only drafts, one nothing."""
    drafts, rng = 60, np.random.default_rng(group)
    cache, table = filled(130, 2, 32, 128), tables(rng, 3, 120, 130)
    trees = [tree(rng, drafts), [1 << i for i in range(drafts)], [0] * drafts]
    q = typed((3 * drafts, 2 * group, 128), dtype, 5)
    check(qx, cache, on_device(qx, cache), table, [3700, drafts, drafts], trees, q)
