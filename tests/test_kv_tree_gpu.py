"""Attention of drafted trees over the paged 8-bit cache against softmax over named keys in 64 bits: types, head sizes,
groups, one to 64 drafts, blocks of every size, windows, chains and arbitrary masks, rows that see nothing, ragged batches
on the streamed and the prompt kernel, scales that are no numbers in blocks that only others see; and a verification
step run as a whole."""

import math

import numpy as np
import pytest
import torch

from kv_reference import Cache, attention_tolerance, rotated
from test_kv_attention_gpu import filled
from test_kv_cache_gpu import batch_of, on_device, table_of, typed

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def attention(q, k, v, scale, seen):
    """One sequence in f64 over the keys that `seen` [n, length] names: output, ln of the sums, and what the tolerances want
    (magnitudes of values, weighted and plainly summed, and the largest sum of |scale q k| of a row)."""
    group, dim = q.shape[1] // k.shape[1], q.shape[2]
    qq = q.transpose(0, 1)
    kk, vv = (t.repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))
    s = (scale * (qq @ kk.transpose(1, 2))).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)
    spread = abs(scale) * (qq.abs() @ kk.abs().transpose(1, 2)).amax(-1)
    spread = spread + abs(scale) * qq.abs().amax(-1) * kk.abs().sum(-1).amax(-1)[:, None] * 2 / (dim / 16 + 22)
    return ((p @ vv).transpose(0, 1), lse.T, ((p @ vv.abs()).transpose(0, 1), (seen.double() @ vv.abs()).transpose(0, 1)), spread.T)


def signed(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)


def named(masks, length, window):
    """[n, length]: the keys that the rows with these masks see."""
    n = len(masks)
    seen = torch.zeros(n, length, dtype=torch.bool)
    for i, m in enumerate(masks):
        mine = [j for j in range(n) if m >> j & 1]
        place = length - n + len(mine) - 1
        first = max(0, place - window + 1) if window else 0
        seen[i, first:length - n] = True
        seen[i, [length - n + j for j in mine]] = True
    return seen


def tree(rng, n):
    """Masks of a random tree: a draft hangs on an earlier one or on the text."""
    masks = []
    for i in range(n):
        parent = int(rng.integers(-1, i)) if i else -1
        masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
    return masks


def tables(rng, sequences, width, blocks):
    """Sequences that share blocks, which attention only reads."""
    return np.stack([rng.permutation(blocks)[:width] for _ in range(sequences)]).astype(np.int32)


def check(qx, cache, dev, table, lengths, trees, q, window=0, scale=None, behind=0, junk=0):
    """`junk`: bits of rows that a sequence does not have, set in every mask."""
    heads, dim = q.shape[1], q.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    new = [len(t) for t in trees]
    batch, begin, rows = batch_of(qx, table, lengths, new, behind)
    masks = [m | (junk << n & (1 << 64) - 1) for t, n in zip(trees, new) for m in t] + [0] * behind
    out = torch.full(q.shape, 11.0, dtype=q.dtype, device="cuda")
    lse = torch.full((rows, heads), 11.0, device="cuda")
    qx.check(dev.tree_attention_dev(batch, q.cuda(), out, signed(masks).cuda(), scale, window, lse), "tree attention")
    torch.cuda.synchronize()
    assert qx.lib.qx_check_device_errors() == qx.OK, qx.last_error()
    for s, (t, n) in enumerate(zip(lengths, new)):
        k, v = (torch.from_numpy(cache.values(i, table[s], t)) for i in range(2))
        own = slice(int(begin[s]), int(begin[s]) + n)
        want, sums, magnitude, spread = attention(q[own].double(), k, v, scale, named(trees[s], t, window))
        limit, lse_limit = attention_tolerance(want, sums, magnitude, spread, q.dtype, dim, t)
        got, got_lse = out[own].cpu().double(), lse[own].cpu().double()
        off = (got - want).abs() / limit
        assert off.numel() == 0 or float(off.max()) <= 1, (s, float(off.max()))
        empty = sums == -math.inf
        assert bool((got_lse[empty] == -math.inf).all()) and bool((got[empty] == 0).all())
        assert bool(((got_lse - sums).abs()[~empty] <= lse_limit[~empty]).all())
    assert bool((out[int(begin[-1]):] == 11).all()) and bool((lse[int(begin[-1]):] == 11).all())
    return out, lse


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("drafts", [1, 7, 64])
def test_head_sizes(qx, dtype, dim, drafts):
    rng = np.random.default_rng(dim + drafts)
    cache, table = filled(30, 2, 32, dim), table_of(2, 15, 30)
    trees = [tree(rng, drafts), tree(rng, max(1, drafts // 2))]
    check(qx, cache, on_device(qx, cache), table, [400, 77], trees, typed((drafts + len(trees[1]) + 2, 6, dim), dtype, dim), behind=2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("length,drafts", [(1, 1), (5, 5), (64, 64), (65, 64), (17, 3), (31, 16), (32, 1), (33, 20), (97, 33), (128, 63),
                                           (129, 2), (300, 40), (1024, 64), (4133, 48)])
def test_where_drafts_meet_tiles_and_blocks(qx, dtype, size, length, drafts):
    rng = np.random.default_rng(length + drafts)
    width = -(-length // size)
    cache, table = filled(width + 1, 2, size, 64), table_of(1, width, width + 1)
    check(qx, cache, on_device(qx, cache), table, [length], [tree(rng, drafts)], typed((drafts, 8, 64), dtype, length))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("window", [0, 64, 100, 1000])
def test_ragged_batches_groups_and_windows(qx, dtype, group, window):
    rng = np.random.default_rng(group + window)
    lengths, drafts = [900, 40, 333, 64, 12], [30, 1, 64, 17, 0]
    cache, table = filled(90, 2, 16, 128), tables(rng, 5, 60, 90)
    check(qx, cache, on_device(qx, cache), table, lengths, [tree(rng, n) for n in drafts],
          typed((sum(drafts) + 3, 2 * group, 128), dtype, group), window, behind=3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("drafts", [6, 60])
def test_masks_of_every_kind(qx, dtype, drafts):
    """Not trees: arbitrary masks, empty ones, all ones, bits of rows that are not there, drafts that do not see themselves;
    and with nothing in front of the drafts, rows that see no key at all."""
    rng = np.random.default_rng(drafts)
    masks = [int(rng.integers(0, 1 << 62)) & (1 << drafts) - 1 for _ in range(drafts)]
    masks[0], masks[1], masks[2] = 0, (1 << drafts) - 1, 1 << drafts - 1
    cache, table = filled(16, 2, 32, 64), table_of(2, 8, 16)
    q = typed((2 * drafts, 8, 64), dtype, 3)
    check(qx, cache, on_device(qx, cache), table, [200, drafts], [masks, masks], q, junk=(1 << 64) - 1)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("drafts", [5, 64])
def test_a_chain_is_causal_attention(qx, dtype, drafts):
    cache, table = filled(50, 4, 16, 96), tables(np.random.default_rng(1), 3, 40, 50)
    dev, lengths = on_device(qx, cache), [600, 64, 333]
    q = typed((3 * drafts, 8, 96), dtype, 5)
    chain = [(2 << i) - 1 for i in range(drafts)]
    for length in lengths:  # (the masks of causal attention in a window)
        place, key = torch.arange(length - drafts, length)[:, None], torch.arange(length)
        causal = (key <= place) & ((key > place - 100) | (key >= length - drafts))
        assert torch.equal(named(chain, length, 100), causal)
    check(qx, cache, dev, table, lengths, [chain] * 3, q, window=100)


def test_more_rows_than_tokens(qx):
    """A sequence whose first drafts stand in front of its first token: they have no keys, and nobody sees them."""
    cache, table = filled(4, 1, 16, 64), table_of(1, 4, 4)
    dev, q = on_device(qx, cache), typed((6, 2, 64), F32, 1)
    masks = [(2 << i) - 1 for i in range(6)]
    batch, _, _ = batch_of(qx, table, [4], [6], 0)
    out, lse = torch.empty(6, 2, 64, device="cuda"), torch.empty(6, 2, device="cuda")
    qx.check(dev.tree_attention_dev(batch, q.cuda(), out, signed(masks).cuda(), None, 0, lse), "tree attention")
    torch.cuda.synchronize()
    qx.check(qx.lib.qx_check_device_errors(), "tree attention")
    assert bool((out[:2] == 0).all()) and bool((lse[:2] == -math.inf).all())
    k, v = (torch.from_numpy(cache.values(i, table[0], 4)) for i in range(2))
    seen = torch.tril(torch.ones(4, 4, dtype=torch.bool))
    want, sums, magnitude, spread = attention(q[2:].double(), k, v, 0.125, seen)
    limit, _ = attention_tolerance(want, sums, magnitude, spread, F32, 64, 4)
    assert bool(((out[2:].cpu().double() - want).abs() <= limit).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("drafts", [12, 64])
def test_blocks_that_hold_no_numbers_spoil_who_sees_them_only(qx, dtype, drafts):
    """The drafts of one branch lie in a block of their own, whose scales are NaN."""
    size = 16
    cache, table = filled(12, 2, size, 64), table_of(1, 12, 12)
    length = 3 * size + drafts  # the drafts begin a block
    bad = drafts // size * size - size if drafts > size else 0  # the first draft of that block
    first, last = bad, min(bad + size, drafts)
    for scales in cache.scales:
        scales[table[0, (3 * size + first) // size]] = np.nan
    inside = [i for i in range(drafts) if first <= i < last]
    outside = [i for i in range(drafts) if i not in inside]
    masks = [0] * drafts
    for i in range(drafts):
        of = inside if i in inside else outside
        masks[i] = sum(1 << j for j in of if j <= i)
    q = typed((drafts, 4, 64), dtype, 9)
    batch, _, _ = batch_of(qx, table, [length], [drafts], 0)
    out, lse = torch.empty(drafts, 4, 64, dtype=dtype, device="cuda"), torch.empty(drafts, 4, device="cuda")
    dev = on_device(qx, cache)
    qx.check(dev.tree_attention_dev(batch, q.cuda(), out, signed(masks).cuda(), None, 0, lse), "tree attention")
    torch.cuda.synchronize()
    qx.check(qx.lib.qx_check_device_errors(), "tree attention")
    assert bool(out[inside].isnan().all()) and bool(out[outside].isfinite().all()) and bool(lse[outside].isfinite().all())


@pytest.mark.parametrize("dtype", [F32, F16])
def test_host_buffers_strides_and_outputs_over_queries(qx, dtype):
    rng = np.random.default_rng(2)
    cache, table = filled(20, 2, 16, 64), table_of(2, 10, 20)
    dev, lengths, trees = on_device(qx, cache), [150, 60], [tree(rng, 20), tree(rng, 9)]
    q = typed((29, 8, 64), dtype, 4)
    want, sums = check(qx, cache, dev, table, lengths, trees, q)
    masks = signed([m for t in trees for m in t])
    # a slice of a packed projection, the outputs in its place
    packed = torch.zeros(29, 12, 64, dtype=dtype, device="cuda")
    packed[:, :8] = q.cuda()
    batch, begin, _ = batch_of(qx, table, lengths, [20, 9], 0)
    qx.check(dev.tree_attention_dev(batch, packed[:, :8], packed[:, :8], masks.cuda()), "tree attention")
    assert torch.equal(packed[:, :8], want) and bool((packed[:, 8:] == 0).all())
    host = qx.KVCache(*cache.codes, *cache.scales)
    arrays = qx.KVBatch(np.array(lengths, np.int32), np.ascontiguousarray(table, np.int32), 150, np.array([0, 20, 29], np.int32), 29, 20)
    a, lse = q.numpy().copy(), np.zeros((29, 8), np.float32)
    out = np.zeros_like(a)
    qx.check(host.tree_attention(arrays, a, out, masks.numpy(), lse=lse), "tree attention")
    assert np.array_equal(out, want.cpu().numpy()) and np.array_equal(lse, sums.cpu().numpy())


def test_captured_with_masks_that_change(qx):
    rng = np.random.default_rng(6)
    cache, table = filled(50, 2, 32, 128), tables(rng, 4, 40, 50)
    dev, lengths = on_device(qx, cache), [1000, 700, 1200, 64]
    q = typed((4 * 16, 8, 128), BF16, 7).cuda()
    batch, _, _ = batch_of(qx, table, lengths, [16] * 4, 0)
    masks = torch.zeros(64, dtype=torch.int64, device="cuda")
    out, once = torch.empty_like(q), torch.empty_like(q)
    qx.check(dev.tree_attention_dev(batch, q, out, masks), "tree attention")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qx.check(dev.tree_attention_dev(batch, q, out, masks), "tree attention")
    for _ in range(2):
        new = signed([m for _ in range(4) for m in tree(rng, 16)]).cuda()
        masks.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        qx.check(dev.tree_attention_dev(batch, q, once, new), "tree attention")
        assert torch.equal(out, once)
    qx.check(qx.lib.qx_check_device_errors(), "tree attention")


def test_many_sessions_on_a_balanced_launch(qx):
    rng = np.random.default_rng(8)
    lengths = [int(n) for n in rng.integers(64, 3000, 40)]
    cache = filled(600, 4, 32, 128)
    table = tables(rng, len(lengths), 100, 600)
    trees = [tree(rng, int(rng.integers(1, 5))) for _ in lengths]
    check(qx, cache, on_device(qx, cache), table, lengths, trees, typed((sum(map(len, trees)), 16, 128), BF16, 1))


def test_a_verification_step(qx):
    """Two sessions, three steps of drafts each: a tree is appended with the positions of its depths, attended to, and one
    of its paths is appended again in the drafts' place; the next step goes on behind that. Each step's attention is
    compared with 64 bits over the cache's own contents."""
    heads, kv_heads, dim, size = 8, 2, 64, 32
    gen, rng = torch.Generator().manual_seed(5), np.random.default_rng(5)
    rope = qx.Rope(dim)
    cache = qx.KVCache.empty(16, kv_heads, size, dim)
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8)
    kept = [50, 33]  # tokens that stay

    def batch_at(lengths, new):
        begin = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
        return qx.KVBatch(torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, 256, begin, sum(new), max(new))

    def projected(rows):
        return torch.randn(rows, heads + 2 * kv_heads, dim, generator=gen).bfloat16().cuda().split([heads, kv_heads, kv_heads], 1)

    q, k, v = projected(sum(kept))
    qx.check(cache.append_dev(batch_at(kept, kept), k, v, rope, q, q), "append")
    for _ in range(3):
        trees = [tree(rng, 13), tree(rng, 6)]
        new = [len(t) for t in trees]
        lengths = [a + b for a, b in zip(kept, new)]
        batch, (q, k, v) = batch_at(lengths, new), projected(sum(new))
        depth = torch.tensor([a + bin(m).count("1") - 1 for a, t in zip(kept, trees) for m in t], device="cuda")
        turned, out = torch.empty_like(q), torch.empty(sum(new), heads, dim, dtype=torch.bfloat16, device="cuda")
        qx.check(cache.append_dev(batch, k, v, rope, q, turned, depth), "append")
        want = rotated(q.cpu().double(), depth.tolist(), rope.view.frequency[:dim // 2])
        assert float((turned.cpu().double() - want).abs().max()) <= 2.0 ** -8 * 6 + 1e-4
        masks = signed([m for t in trees for m in t]).cuda()
        qx.check(cache.tree_attention_dev(batch, turned, out, masks), "tree attention")
        keys, values = (torch.empty(sum(lengths), kv_heads, dim, device="cuda") for _ in "kv")
        qx.check(cache.read_dev(batch_at(lengths, lengths), keys, values), "read")
        torch.cuda.synchronize()
        qx.check(qx.lib.qx_check_device_errors(), "step")
        row = key = 0
        paths = []
        for t, n, length in zip(trees, new, lengths):
            kk, vv = (x[key:key + length].cpu().double() for x in (keys, values))
            exact, sums, magnitude, spread = attention(turned[row:row + n].cpu().double(), kk, vv, dim ** -0.5, named(t, length, 0))
            limit, _ = attention_tolerance(exact, sums, magnitude, spread, BF16, dim, length)
            assert bool(((out[row:row + n].cpu().double() - exact).abs() <= limit).all())
            leaf = max(range(n), key=lambda i: bin(t[i]).count("1"))
            paths.append([row + j for j in range(n) if t[leaf] >> j & 1])
            row, key = row + n, key + length
        kept = [a + len(path) for a, path in zip(kept, paths)]
        rows = torch.tensor([r for path in paths for r in path], device="cuda")
        qx.check(cache.append_dev(batch_at(kept, [len(path) for path in paths]), k[rows], v[rows], rope), "append")
    torch.cuda.synchronize()
    qx.check(qx.lib.qx_check_device_errors(), "steps")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group,drafts,length,dim,window", [(6, 64, 700, 128, 0), (6, 47, 129, 64, 0), (5, 63, 2600, 128, 1000), (8, 33, 50, 80, 64)])
def test_three_tiles_of_rows(qx, dtype, group, drafts, length, dim, window):
    rng = np.random.default_rng(group + length)
    cache, table = filled(100, 2, 32, dim), tables(rng, 2, 90, 100)
    trees = [tree(rng, drafts), tree(rng, drafts // 3)]
    check(qx, cache, on_device(qx, cache), table, [length, drafts // 3 + 5], trees, typed((drafts + drafts // 3, 2 * group, dim), dtype, length), window)
