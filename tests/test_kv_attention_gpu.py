"""Attention over the paged 8-bit cache against softmax(scale q K^T) V in 64 bits: types, head sizes, groups,
lengths from nothing to thousands, masks, ragged batches, strides, splits, blocks that hold NaN, what may run
beside what; and a decoder layer's attention half run as a whole."""

import ctypes as C
import math

import numpy as np
import pytest
import torch

from kv_reference import Cache, attention, attention_tolerance, rotated
from test_kv_cache_gpu import batch_of, on_device, table_of, typed

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def filled(blocks, heads, size, dim, seed=0):
    """A cache of codes and scales of every kind."""
    rng = np.random.default_rng(seed)
    cache = Cache(blocks, heads, size, dim, seed)
    cache.codes = [np.clip(rng.normal(0, 42, (blocks, heads, size, dim)).round(), -127, 127).astype(np.int8) for _ in "kv"]
    cache.scales = [(rng.random((blocks, heads)) * 0.03 + 0.005).astype(np.float32) for _ in "kv"]
    return cache


def check(qx, cache, dev, table, lengths, new, q, causal=True, window=0, scale=None, behind=0, call=None):
    """Runs it, compares every row and that nobody else's rows are touched; returns output and lse."""
    heads, dim = q.shape[1], q.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    batch, begin, rows = batch_of(qx, table, lengths, new, behind)
    out = torch.full(q.shape, 11.0, dtype=q.dtype, device="cuda")
    lse = torch.full((rows, heads), 11.0, device="cuda")
    if call is None:
        assert dev.attention_dev(batch, q.cuda(), out, scale, causal, window, lse) == qx.OK, qx.last_error()
    else:
        call(batch, q.cuda(), out, lse)
    torch.cuda.synchronize()
    assert qx.lib.qx_check_device_errors() == qx.OK, qx.last_error()
    for s, (t, n) in enumerate(zip(lengths, new)):
        k, v = (torch.from_numpy(cache.values(i, table[s], t)) for i in range(2))
        rows_of = slice(int(begin[s]), int(begin[s]) + n)
        want, sums, magnitude, spread = attention(q[rows_of].double(), k, v, scale, causal, window)
        limit, lse_limit = attention_tolerance(want, sums, magnitude, spread, q.dtype, dim, t)
        got, got_lse = out[rows_of].cpu().double(), lse[rows_of].cpu().double()
        off = (got - want).abs() / limit
        assert off.numel() == 0 or float(off.max()) <= 1, (s, float(off.max()), off.argmax())
        empty = sums == -math.inf
        assert bool((got_lse[empty] == -math.inf).all()) and bool((got[empty] == 0).all())
        assert bool(((got_lse - sums).abs()[~empty] <= lse_limit[~empty]).all())
    assert bool((out[int(begin[-1]):] == 11).all()) and bool((lse[int(begin[-1]):] == 11).all())
    return out, lse


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 128, 144, 192, 256])
def test_head_sizes(qx, dtype, dim):
    cache, table = filled(40, 2, 32, dim), table_of(2, 20, 40)
    check(qx, cache, on_device(qx, cache), table, [600, 77], [3, 1], typed((5, 6, dim), dtype, dim), behind=1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 1024, 4133])
def test_single_tokens(qx, dtype, size, length):
    width = -(-length // size)
    cache, table = filled(width + 1, 2, size, 64), table_of(1, width, width + 1)
    check(qx, cache, on_device(qx, cache), table, [length], [1], typed((1, 8, 64), dtype, length))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group,new", [(1, 1), (1, 17), (3, 5), (5, 7), (7, 1), (8, 1), (8, 4), (16, 1), (16, 3), (20, 2), (40, 1)])
def test_groups_and_runs_of_tokens(qx, dtype, group, new):
    cache, table = filled(24, 2, 64, 128), table_of(2, 12, 24)
    check(qx, cache, on_device(qx, cache), table, [700, 33], [new, min(new, 2)], typed((new + min(new, 2), 2 * group, 128), dtype, group))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 7), (True, 64), (True, 100), (False, 50), (True, 5000)])
@pytest.mark.parametrize("size", [16, 64])
def test_masks(qx, dtype, causal, window, size):
    """A prompt, a chunk behind a prefix, a single token and a sequence of nothing in one batch."""
    width = 400 // size + 1
    cache, table = filled(4 * width, 2, size, 64), table_of(4, width, 4 * width)
    lengths, new = [130, 400, 260, 0], [130, 45, 1, 0]
    check(qx, cache, on_device(qx, cache), table, lengths, new, typed((sum(new) + 4, 4, 64), dtype, 3), causal, window, behind=4)


@pytest.mark.parametrize("causal", [True, False])
def test_rows_that_see_nothing(qx, causal):
    """More rows than tokens (an empty cache among them): zeros and -infinity where no key is seen."""
    cache, table = filled(8, 1, 16, 32), table_of(3, 2, 8)
    check(qx, cache, on_device(qx, cache), table, [0, 3, 20], [4, 9, 30], typed((43, 2, 32), F32, 1), causal)
    check(qx, cache, on_device(qx, cache), table, [0, 3, 20], [4, 9, 30], typed((43, 2, 32), BF16, 1), causal, window=2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 96, 256])
@pytest.mark.parametrize("group", [1, 4, 6])
def test_prompts(qx, dtype, dim, group):
    cache, table = filled(36, 2, 64, dim), table_of(3, 12, 36)
    lengths, new = [300, 517, 700], [300, 200, 129]
    check(qx, cache, on_device(qx, cache), table, lengths, new, typed((sum(new) + 1, 2 * group, dim), dtype, 5), behind=1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,size,group,new", [(128, 16, 8, 100), (64, 128, 2, 300), (16, 32, 1, 70), (112, 64, 3, 257)])
@pytest.mark.parametrize("window", [0, 900])
def test_chunks_of_a_prompt_behind_a_long_prefix(qx, dtype, dim, size, group, new, window):
    """Few row tiles and many keys: the keys are split among CTAs and joined."""
    width = -(-6100 // size)
    cache, table = filled(width, 1, size, dim), table_of(1, width, width)
    dev = on_device(qx, cache)
    for length in (6100, 2049, 513 + new):
        check(qx, cache, dev, table, [length], [new], typed((new, group, dim), dtype, length), True, window)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [63, 64, 65, 127, 128, 129, 255, 256, 257, 513])
def test_tiles_of_rows(qx, dtype, rows):
    """Row counts at and around the tiles, one query head per kv head, prompts of exactly that length and longer."""
    cache, table = filled(30, 2, 64, 64), table_of(2, 15, 30)
    check(qx, cache, on_device(qx, cache), table, [rows, rows + 130], [rows, rows - 60], typed((2 * rows - 60, 2, 64), dtype, rows))


@pytest.mark.parametrize("scale", [0.0, -0.125, 2.0])
def test_scales_of_a_prompts_scores(qx, scale):
    cache, table = filled(10, 2, 32, 64), table_of(1, 10, 10)
    check(qx, cache, on_device(qx, cache), table, [310], [310], typed((310, 2, 64), BF16, 9), scale=scale)


def test_value_scales_far_apart_in_a_prompt(qx):
    """Blocks whose value scales differ by 2^40, are zero or lie under the smallest that append makes: the weights
    carry them, so the tolerance goes by the largest scale of the keys that a row sees."""
    size, n = 16, 150
    cache, table = filled(10, 1, size, 64), table_of(1, 10, 10)
    for block, factor in ((0, 2.0 ** -40), (2, 0.0), (3, 2.0 ** 20), (5, 2.0 ** -110), (7, 2.0 ** 45)):
        cache.scales[1][table[0, block]] *= np.float32(factor)
    cache.scales[0][table[0, 4]] = 0.0
    dev, q = on_device(qx, cache), typed((n, 2, 64), BF16, 4)
    batch, _, _ = batch_of(qx, table, [n], [n])
    out = torch.empty(n, 2, 64, dtype=BF16, device="cuda")
    assert dev.attention_dev(batch, q.cuda(), out) == qx.OK
    k, v = (torch.from_numpy(cache.values(i, table[0], n)) for i in range(2))
    want, sums, magnitude, spread = attention(q.double(), k, v, 0.125, True, 0)
    limit, _ = attention_tolerance(want, sums, magnitude, spread, BF16, 64, n)
    scales = torch.from_numpy(cache.scales[1][table[0, np.arange(n) // size], 0].astype(np.float64))
    largest = torch.cummax(scales, 0).values  # of the keys up to each row
    limit = limit + ((2.0 ** -36 + 2.0 ** -60) * 127 * n * largest)[:, None, None]
    assert float(((out.cpu().double() - want).abs() / limit).max()) <= 1


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scales_of_scores(qx, dtype):
    """Peaked, flat, negative and zero scores' scales."""
    cache, table = filled(10, 2, 32, 64), table_of(1, 10, 10)
    dev = on_device(qx, cache)
    for scale in (0.0, -0.125, 2.0, 1e-6):
        check(qx, cache, dev, table, [310], [2], typed((2, 4, 64), dtype, 9), scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_queries_of_every_magnitude(qx, dtype):
    """Rows of zeros, of tiny and of huge values: each is brought to 16 bits by a power of two of its own."""
    cache, table = filled(10, 1, 32, 64), table_of(1, 10, 10)
    q = typed((8, 2, 64), dtype, 2).double()
    for row, factor in enumerate([0.0, 1e-7, 1e-4, 1.0, 30.0, 300.0, 1e-5, 1.0]):
        q[row] *= factor
    q[7, 1, 0] = 500.0  # one element far above the rest
    check(qx, cache, on_device(qx, cache), table, [310], [8], q.to(dtype), scale=0.01)


def test_scales_far_apart(qx):
    """Neighbouring blocks of 16 whose scales differ by 2^40 share a tile."""
    cache, table = filled(6, 1, 16, 64), table_of(1, 6, 6)
    cache.scales[1][table[0, 1]] *= 2.0 ** -40
    cache.scales[1][table[0, 3]] = 0.0
    cache.scales[0][table[0, 2]] = 0.0
    for dtype in (F32, BF16):
        check(qx, cache, on_device(qx, cache), table, [90], [2], typed((2, 2, 64), dtype, 4))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("which", [0, 1])
def test_blocks_that_are_no_numbers(qx, dtype, size, which):
    """Rows that see a block whose scale is NaN give NaN; rows whose masks hide it (causal, window) do not notice."""
    dim, n, window = 64, 6 * size, size
    cache, table = filled(8, 1, size, dim), table_of(1, 6, 8)
    dev = on_device(qx, cache)
    q = typed((n, 2, dim), dtype, 6)
    batch, _, _ = batch_of(qx, table, [n], [n])
    clean = torch.empty(n, 2, dim, dtype=dtype, device="cuda")
    assert dev.attention_dev(batch, q.cuda(), clean, window=window) == qx.OK
    dev.arrays[2 + which][int(table[0, 2])] = float("nan")
    for unused in set(range(8)) - set(table[0].tolist()):
        dev.arrays[2][unused] = dev.arrays[3][unused] = float("nan")
    got = torch.empty_like(clean)
    assert dev.attention_dev(batch, q.cuda(), got, window=window) == qx.OK
    rows = torch.arange(n, device="cuda")
    sees = (rows >= 2 * size) & (rows - window + 1 < 3 * size)
    assert bool(got[sees].isnan().all()), "a row that sees the block"
    assert torch.equal(got[~sees], clean[~sees]), "a row that does not"


def test_a_query_that_is_no_number_stays_in_its_row(qx):
    cache, table = filled(8, 2, 32, 64), table_of(1, 8, 8)
    dev = on_device(qx, cache)
    for dtype in (F32, F16, BF16):
        q = typed((5, 4, 64), dtype, 6)
        batch, _, _ = batch_of(qx, table, [200], [5])
        clean, got = (torch.empty(5, 4, 64, dtype=dtype, device="cuda") for _ in range(2))
        assert dev.attention_dev(batch, q.cuda(), clean) == qx.OK
        q[2, 1, 7], q[3, 0, 0] = float("nan"), float("inf")
        assert dev.attention_dev(batch, q.cuda(), got) == qx.OK
        bad = torch.zeros(5, 4, dtype=torch.bool, device="cuda")
        bad[2, 1] = bad[3, 0] = True
        assert bool(got[bad].isnan().all()) and torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("dtype,offset", [(F32, 1), (F16, 3), (BF16, 1), (BF16, 8)])
@pytest.mark.parametrize("new", [2, 150])
def test_strided_views(qx, dtype, offset, new):
    """Queries and output with heads outside tokens, odd row lengths, off every boundary."""
    heads, dim = 4, 64
    cache, table = filled(10, 2, 32, dim), table_of(1, 10, 10)
    dev = on_device(qx, cache)
    q = typed((new, heads, dim), dtype, 8)

    def call(batch, q_dev, out, lse):
        pitch = dim + 3
        store = [torch.full((heads * new * pitch + 16,), 5.0, dtype=dtype, device="cuda") for _ in range(2)]
        views = [s.as_strided((new, heads, dim), (pitch, new * pitch, 1), offset) for s in store]
        views[0].copy_(q_dev)
        assert dev.attention_dev(batch, views[0], views[1], lse=lse) == qx.OK
        out.copy_(views[1])
        views[1].fill_(5.0)
        assert bool((store[1] == 5.0).all())  # nothing beside the view was written

    check(qx, cache, dev, table, [310], [new], q, call=call)


def test_long_contexts_split_and_joined(qx):
    """Lengths at and around the chunks that a call is split into."""
    cache, table = filled(330, 1, 64, 64), table_of(1, 330, 330)
    dev = on_device(qx, cache)
    for length in (127, 128, 129, 8191, 8192, 8193, 21000):
        for dtype in (F32, BF16):
            check(qx, cache, dev, table, [length], [1], typed((1, 4, 64), dtype, length))
    check(qx, cache, dev, table, [21000], [2], typed((2, 4, 64), BF16, 1), window=9000)


def test_bounds_above_the_lengths(qx):
    """max_length and max_tokens are bounds: the launch is sized by them, the result is not."""
    cache, table = filled(64, 2, 64, 128), table_of(2, 32, 64)
    dev = on_device(qx, cache)
    q = typed((3, 8, 128), BF16, 1)
    lengths = torch.tensor([90, 700], dtype=torch.int32, device="cuda")
    begin = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    for most, longest in ((2, 700), (2, 2048), (3, 1000), (500, 2048)):
        def call(batch, q_dev, out, lse):
            wide = qx.KVBatch(lengths, torch.from_numpy(table).cuda(), longest, begin, 3, most)
            assert dev.attention_dev(wide, q_dev, out, lse=lse) == qx.OK
        check(qx, cache, dev, table, [90, 700], [1, 2], q, call=call)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_prefix(qx, dtype):
    """Sequences that read the same blocks."""
    cache, table = filled(20, 2, 32, 64), table_of(1, 10, 20).repeat(3, 0)
    table[1, 5:], table[2, 2:] = np.arange(5), np.arange(8)
    check(qx, cache, on_device(qx, cache), table, [300, 280, 190], [1, 3, 1], typed((5, 4, 64), dtype, 1))


def test_the_same_bits_every_time(qx):
    cache, table = filled(600, 2, 64, 128), table_of(3, 200, 600)
    dev = on_device(qx, cache)
    batch, _, rows = batch_of(qx, table, [12000, 3000, 64], [1, 5, 64])
    q = typed((rows, 16, 128), BF16, 1).cuda()
    first, again = torch.empty_like(q), torch.empty_like(q)
    assert dev.attention_dev(batch, q, first) == qx.OK
    for _ in range(20):
        assert dev.attention_dev(batch, q, again) == qx.OK
        assert torch.equal(first, again)


@pytest.mark.parametrize("what", ["block past the cache", "block below zero", "length past the bound", "rows past the bound",
                                  "rows past the views", "rows backwards"])
@pytest.mark.parametrize("new", [2, 40])
def test_a_batch_that_contradicts_itself_is_reported(qx, what, new):
    """Nothing is followed out of the cache; the other sequence is served; a block that is not there is not seen."""
    size, dim = 16, 64
    lengths, longest, most = [70, 50], 128, new
    cache, table = filled(12, 2, size, dim), table_of(2, 5, 12)
    begin = np.array([0, new, 2 * new], np.int32)
    if what == "block past the cache":
        table[0, 1] = 12
    elif what == "block below zero":
        table[0, 1] = -3
    elif what == "length past the bound":
        lengths[0], longest = 81, 80
    elif what == "rows past the bound":
        begin[:] = 0, new + 1, 2 * new
    elif what == "rows past the views":
        begin[:] = 2 * new, 3 * new, 4 * new
    else:
        begin[:] = new, 0, new
    dev = on_device(qx, cache)
    q = typed((2 * new, 4, dim), BF16, 1)
    out = torch.full((2 * new, 4, dim), 3.0, dtype=BF16, device="cuda")
    longest = min(longest, 80)
    batch = qx.KVBatch(torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.from_numpy(table).cuda(), longest,
                       torch.from_numpy(begin).cuda(), 2 * new, most)
    assert dev.attention_dev(batch, q.cuda(), out) == qx.OK
    torch.cuda.synchronize()
    assert qx.lib.qx_check_device_errors() == qx.DEVICE_ERROR
    assert qx.lib.qx_check_device_errors() == qx.OK
    if what != "rows past the views":
        a, b = int(begin[1]), int(begin[2])
        k, v = (torch.from_numpy(cache.values(i, table[1], 50)) for i in range(2))
        want, sums, magnitude, spread = attention(q[a:b].double(), k, v, dim ** -0.5, True, 0)
        limit, _ = attention_tolerance(want, sums, magnitude, spread, BF16, dim, 50)
        assert bool(((out[a:b].cpu().double() - want).abs() <= limit).all())
    if "block" in what:
        table[0, 1] = 0  # (any block: its tokens are masked)
        k, v = (torch.from_numpy(cache.values(i, table[0], 70)) for i in range(2))
        want, sums, magnitude, spread = attention(q[:new].double(), k, v, dim ** -0.5, True, 0, missing=range(16, 32))
        limit, _ = attention_tolerance(want, sums, magnitude, spread, BF16, dim, 70)
        assert bool(((out[:new].cpu().double() - want).abs() <= limit).all())
    elif what in ("length past the bound", "rows past the views"):
        assert bool((out[:new] == 3).all())


def test_captured_and_beside_each_other(qx):
    """Two captured steps with a workspace each, replayed on two streams at once, lengths changing in between."""
    cache, table = filled(300, 2, 64, 128), table_of(1, 300, 300)
    dev = on_device(qx, cache)
    tables = torch.from_numpy(table).cuda()
    sides = []
    for i in range(2):
        workspace = C.c_void_p()
        assert qx.lib.qx_workspace_create(64 << 20, C.byref(workspace)) == qx.OK
        lengths = torch.tensor([5000 + i], dtype=torch.int32, device="cuda")
        q = typed((1, 16, 128), BF16, i).cuda()
        out, want = torch.empty_like(q), torch.empty_like(q)
        batch = qx.KVBatch(lengths, tables, 19000, None, 1, 1)
        held = qx.lib.qx_workspace_capacity(workspace)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert dev.attention_dev(batch, q, out, workspace=workspace) == qx.OK
        assert qx.lib.qx_workspace_capacity(workspace) == held
        sides.append((graph, lengths, q, out, want, batch, workspace, torch.cuda.Stream()))
    for step in range(10):
        for _, lengths, q, _, want, batch, workspace, _ in sides:
            lengths.fill_(100 + 1777 * step)
            q.normal_()
            assert dev.attention_dev(batch, q, want) == qx.OK  # (the default workspace)
        torch.cuda.synchronize()
        for graph, *_, stream in sides:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, _, out, want, *_ in sides:
            assert torch.equal(out, want)
    for side in sides:
        qx.lib.qx_workspace_destroy(side[6])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_host_buffers(qx, dtype):
    cache, table = filled(20, 2, 32, 64), table_of(2, 10, 20)
    lengths, new = [300, 20], [2, 20]
    dev, host = on_device(qx, cache), qx.KVCache(*cache.codes, *cache.scales)
    batch, begin, rows = batch_of(qx, table, lengths, new, behind=1)
    q = typed((rows, 4, 64), dtype, 1)
    kind = qx.F32 if dtype == F32 else qx.BF16
    raw = q.numpy() if dtype == F32 else q.view(torch.int16).numpy().view(np.uint16)
    out, lse = np.zeros_like(raw), np.full((rows, 4), 2.0, np.float32)
    host_batch = qx.KVBatch(np.array(lengths, np.int32), table, 300, begin, rows, 20)
    assert host.attention(host_batch, raw, out, lse=lse, kind=kind) == qx.OK, qx.last_error()
    want, want_lse = torch.zeros(rows, 4, 64, dtype=dtype, device="cuda"), torch.full((rows, 4), 2.0, device="cuda")
    assert dev.attention_dev(batch, q.cuda(), want, lse=want_lse) == qx.OK
    got = torch.from_numpy(out if dtype == F32 else out.view(np.int16)).view(dtype)
    assert torch.equal(got, want.cpu()) and np.array_equal(lse, want_lse.cpu().numpy())


def test_no_rows_no_sequences(qx):
    cache, table = filled(4, 1, 16, 32), table_of(1, 2, 4)
    dev = on_device(qx, cache)
    q = torch.full((0, 2, 32), 1.0, device="cuda")
    nobody = torch.zeros(0, dtype=torch.int32, device="cuda")
    for batch in (qx.KVBatch(nobody, torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 32, None, 0, 1),
                  qx.KVBatch(nobody.new_zeros(1), torch.from_numpy(table).cuda(), 32, nobody.new_zeros(2), 0, 0)):
        assert dev.attention_dev(batch, q, q) == qx.OK
        assert dev.append_dev(batch, q[:, :1], q[:, :1]) == qx.OK
        assert dev.read_dev(batch, q[:, :1], q[:, :1]) == qx.OK


@pytest.mark.parametrize("fmt_name", ["Q4_0", "Q8_0"])
def test_the_attention_half_of_a_decoder_layer(qx, wl, fmt_name):
    """What a program runs per token: fused q + k + v projection, rotation and append in one call, attention, the
    output projection; a prompt first, then tokens one by one, against the same chain in 64 bits on the projections'
    own outputs."""
    fmt = getattr(qx, fmt_name)
    hidden, q_heads, kv_heads, dim, size = 512, 8, 2, 64, 16
    low, high = (0.002, 0.04) if fmt == qx.Q4_0 else (0.001, 0.02)
    rows = [q_heads * dim, kv_heads * dim, kv_heads * dim]
    packed = [wl.packed_blocks(fmt, n, hidden, low, high, seed=i) for i, n in enumerate(rows)]
    qkv, projection = qx.PackedWeights(), qx.PackedWeights()
    assert qkv.prepare_fused(fmt, packed, rows, hidden) == qx.OK
    last = wl.packed_blocks(fmt, hidden, q_heads * dim, low, high, seed=9)
    assert projection.prepare(fmt, last, hidden, q_heads * dim) == qx.OK
    weights = qx.qgemv_unpack(fmt, last, hidden, q_heads * dim)[1].astype(np.float64)
    rope = qx.Rope(dim, qx.ROPE_HALVES, 10000.0)
    dev, table = qx.KVCache.empty(6, kv_heads, size, dim), table_of(1, 4, 6)
    tables = torch.from_numpy(table).cuda()
    length, k_all, v_all = 0, [], []
    for step, n in enumerate([21, 1, 1, 3, 1]):
        x = typed((n, hidden), F32, step).cuda()
        q, k, v = (torch.empty(n, h, dim, device="cuda") for h in (q_heads, kv_heads, kv_heads))
        qx.check(qkv.qgemm_fused_dev(x, [q, k, v], n), "qkv")
        length += n
        batch = qx.KVBatch(torch.tensor([length], dtype=torch.int32, device="cuda"), tables, 64, None, n, n)
        turned, mixed = torch.empty_like(q), torch.empty_like(q)
        y = torch.empty(n, hidden, device="cuda")
        qx.check(dev.append_dev(batch, k, v, rope, q, turned), "append")
        qx.check(dev.attention_dev(batch, turned, mixed), "attention")
        qx.check(projection.qgemm_dev(mixed.view(n, -1), y, n), "projection")
        torch.cuda.synchronize()
        at, f = list(range(length - n, length)), rope.view.frequency[:dim // 2]
        k_all.append(rotated(k.cpu().double(), at, f))
        v_all.append(v.cpu().double())
        keys, values = torch.cat(k_all), torch.cat(v_all)
        want, *_ = attention(rotated(q.cpu().double(), at, f), keys, values, dim ** -0.5, True, 0)
        # Every cached element is off by at most half a step of its block's scale for each time that the scale
        # grew (here at most 16 tokens to a block: in all less than the scale, max / 127, itself), which moves a
        # score by |q| . that and an output by the value's own error and twice the scores' share of the values.
        step_k, step_v = float(keys.abs().max()) / 127, float(values.abs().max()) / 127
        moved = float(q.abs().sum(-1).max()) * dim ** -0.5 * step_k
        assert float((mixed.cpu().double() - want).abs().max()) <= step_v + 2 * moved * float(values.abs().max())
        # and exactly, against the cache's own contents
        got_k, got_v = (torch.empty(length, kv_heads, dim, device="cuda") for _ in "kv")
        whole = qx.KVBatch(batch.arrays[0], tables, 64, None, length, length)
        qx.check(dev.read_dev(whole, got_k, got_v), "read")
        close, sums, magnitude, spread = attention(turned.cpu().double(), got_k.cpu().double(), got_v.cpu().double(), dim ** -0.5, True, 0)
        limit, _ = attention_tolerance(close, sums, magnitude, spread, F32, dim, length)
        # (read rounds code * scale to f32: half a step of every key and value)
        limit = limit + 2.0 ** -23 * (1 + 2 * spread)[..., None] * magnitude[0]
        assert bool(((mixed.cpu().double() - close).abs() <= limit).all())
        # the projection: activations to 2^-23 of their block of 32, f32 sums of the blocks
        flat = mixed.cpu().double().view(n, -1).numpy()
        envelope = np.abs(flat).reshape(n, -1, 32).max(-1).repeat(32, -1)
        loose = 2.0 ** -22 * envelope + (flat.shape[1] / 32 + 8) * 2.0 ** -23 * np.abs(flat)
        assert np.all(np.abs(y.cpu().numpy() - flat @ weights.T) <= loose @ np.abs(weights).T)
    assert qx.lib.qx_check_device_errors() == qx.OK
