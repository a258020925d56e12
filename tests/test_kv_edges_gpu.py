"""Attention, append and rotation at the ends of what their documentation allows: windows as wide as whole numbers go,
many ragged sessions in one launch, types that differ, outputs in the queries' place, other streams, captured and
replayed calls beside each other."""

import ctypes as C

import numpy as np
import pytest
import torch

from test_kv_attention_gpu import BF16, F16, F32, check, filled
from test_kv_cache_gpu import batch_of, on_device, table_of, typed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [9, 130])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 40])
def test_windows_wider_than_any_context(qx, dtype, causal, new, window):
    """... with rows in front of the first token: their positions are negative."""
    cache, table = filled(16, 2, 16, 64), table_of(2, 8, 16)
    q = typed((2 * new, 4, 64), dtype, new)
    wide, _ = check(qx, cache, on_device(qx, cache), table, [new - 6, 120], [new, new], q, causal, window)
    none, _ = check(qx, cache, on_device(qx, cache), table, [new - 6, 120], [new, new], q, causal, 0)
    assert torch.equal(wide, none)


def ragged(sequences, longest, most, seed):
    """Lengths and new tokens: nothing, one, a few, many, as long as it goes."""
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, 300, sequences)
    lengths[rng.integers(0, sequences, 3)] = 0, 1, longest
    new = rng.integers(0, most + 1, sequences)
    new[rng.integers(0, sequences, 2)] = 0, most
    return lengths.tolist(), new.tolist()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,kv_heads,group,sequences,most", [(128, 8, 4, 40, 1), (64, 10, 3, 33, 5), (256, 2, 4, 60, 1),
                                                             (80, 2, 8, 128, 1), (64, 40, 1, 2, 7), (144, 1, 5, 65, 3)])
@pytest.mark.parametrize("window", [0, 150])
def test_many_ragged_sessions_in_one_launch(qx, dtype, dim, kv_heads, group, sequences, most, window):
    """Bounds far above the lengths give each CTA a piece of the line of all sessions and heads; the same workspace
    serves one call after the other, of other lengths."""
    size, longest, bound = 32, 1500, 9600
    width = bound // size
    cache = filled(300, kv_heads, size, dim)
    table = np.random.default_rng(dim).integers(0, 300, (sequences, width)).astype(np.int32)  # (blocks may be shared)
    dev = on_device(qx, cache)
    for seed in range(2):
        lengths, new = ragged(sequences, longest, most, seed)

        def call(batch, q, out, lse):
            wide = qx.KVBatch(torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.from_numpy(table).cuda(), bound,
                              torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda"),
                              q.shape[0], most)
            for _ in range(3):
                out.fill_(11), lse.fill_(11)
                assert dev.attention_dev(wide, q, out, window=window, lse=lse) == qx.OK, qx.last_error()
        check(qx, cache, dev, table, lengths, new, typed((sum(new) + 2, kv_heads * group, dim), dtype, seed), True, window,
              behind=2, call=call)


@pytest.mark.parametrize("dim,size,group,new", [(128, 16, 8, 100), (64, 128, 2, 300), (16, 32, 1, 100), (112, 64, 3, 257)])
@pytest.mark.parametrize("window", [0, 900])
def test_f32_chunks_of_a_prompt_behind_a_long_prefix(qx, dim, size, group, new, window):
    width = -(-6100 // size)
    cache, table = filled(width, 1, size, dim), table_of(1, width, width)
    dev = on_device(qx, cache)
    for length in (6100, 2049, 513 + new):
        check(qx, cache, dev, table, [length], [new], typed((new, group, dim), F32, length), True, window)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows", [16, 17, 47, 48, 49, 95, 96, 97])
def test_row_counts_at_which_other_kernels_take_over(qx, dtype, rows):
    cache, table = filled(30, 2, 64, 128), table_of(2, 15, 30)
    check(qx, cache, on_device(qx, cache), table, [rows, 900], [rows, 3], typed((rows + 3, 2, 128), dtype, rows))


@pytest.mark.parametrize("lengths,new", [([300, 40], [1, 1]), ([5000], [1]), ([300, 200], [130, 97]), ([5000], [60])])
@pytest.mark.parametrize("offset", [0, 1])
def test_outputs_of_another_type(qx, lengths, new, offset):
    """The output is the same f32 result rounded once to its own type, whatever the queries' is and wherever it lies."""
    cache, table = filled(160, 2, 32, 96), table_of(1, 157, 160).repeat(len(lengths), 0)
    dev = on_device(qx, cache)
    batch, _, rows = batch_of(qx, table, lengths, new)
    for from_type in (F32, F16, BF16):
        q = typed((rows, 8, 96), from_type, 5).cuda()
        exact = torch.zeros(rows, 8, 96, device="cuda")
        assert dev.attention_dev(batch, q, exact) == qx.OK
        for to_type in (F32, F16, BF16):
            flat = torch.zeros(rows * 8 * 96 + 8, dtype=to_type, device="cuda")
            out = flat[offset:offset + exact.numel()].view(exact.shape)
            assert dev.attention_dev(batch, q, out) == qx.OK, qx.last_error()
            assert torch.equal(out, exact.to(to_type)), (from_type, to_type)
            assert bool((flat[:offset] == 0).all()) and bool((flat[offset + exact.numel():] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths,new", [([300, 40], [1, 1]), ([6000], [1]), ([300, 200], [130, 97]), ([6000], [60])])
def test_the_output_in_the_queries_place(qx, dtype, lengths, new):
    cache, table = filled(200, 2, 32, 128), table_of(1, 188, 200).repeat(len(lengths), 0)
    dev = on_device(qx, cache)
    batch, _, rows = batch_of(qx, table, lengths, new)
    q = typed((rows, 8, 128), dtype, 5).cuda()
    want = torch.zeros_like(q)
    assert dev.attention_dev(batch, q, want) == qx.OK and dev.attention_dev(batch, q, q) == qx.OK
    assert torch.equal(q, want)


def test_captured_sessions_beside_each_other(qx):
    """Two captured decode steps of many sessions (append and attention), a workspace and a cache each, replayed at the
    same time on two streams while lengths grow; a third runs uncaptured on a stream of its own."""
    sequences, heads, dim, size, bound = 40, 8, 128, 32, 8192
    rope = qx.Rope(dim)
    rng = np.random.default_rng(7)
    sides = []
    for i in range(3):
        cache = filled(sequences * 6, heads, size, dim, i)
        dev = on_device(qx, cache)
        table = np.zeros((sequences, bound // size), np.int32)
        table[:, :6] = rng.permutation(sequences * 6).reshape(sequences, 6)
        lengths = torch.tensor(rng.integers(1, 150, sequences), dtype=torch.int32, device="cuda")
        batch = qx.KVBatch(lengths, torch.from_numpy(table).cuda(), bound, None, sequences, 1)
        qkv = typed((sequences, 6 * heads, dim), BF16, i).cuda()
        q, k, v = qkv[:, :4 * heads], qkv[:, 4 * heads:5 * heads], qkv[:, 5 * heads:]
        turned, out = torch.empty_like(q), torch.empty(sequences, 4 * heads, dim, dtype=BF16, device="cuda")
        workspace = C.c_void_p()
        assert qx.lib.qx_workspace_create(256 << 20, C.byref(workspace)) == qx.OK

        def step(dev=dev, batch=batch, q=q, k=k, v=v, turned=turned, out=out, workspace=workspace):
            assert dev.append_dev(batch, k, v, rope, q, turned) == qx.OK
            assert dev.attention_dev(batch, turned, out, workspace=workspace) == qx.OK
        sides.append((step, dev, cache, table, lengths, qkv, out, torch.cuda.Stream(), workspace))
    torch.cuda.synchronize()
    graphs = []
    for side in sides[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            side[0]()
        graphs.append(graph)
    for turn in range(6):
        for i, (step, *_, lengths, qkv, out, stream, _) in enumerate(sides):
            with torch.cuda.stream(stream):
                lengths.add_(1)
                qkv.normal_()
                if i < 2:
                    graphs[i].replay()
                else:
                    step()
        torch.cuda.synchronize()
        assert qx.lib.qx_check_device_errors() == qx.OK
        for step, dev, cache, table, lengths, qkv, out, stream, _ in sides:  # (the same once more, by itself)
            got = out.clone()
            step()
            torch.cuda.synchronize()
            assert torch.equal(out, got), turn
    for side in sides:
        qx.lib.qx_workspace_destroy(side[-1])


@pytest.mark.parametrize("k_type,v_type", [(F32, BF16), (F16, F32), (BF16, F16)])
@pytest.mark.parametrize("new", [[1, 1, 0], [40, 7, 65]])
def test_keys_and_values_of_different_types(qx, k_type, v_type, new):
    """... give the same bits as two appends of one type each."""
    lengths = [90, 7, 130]
    k, v = typed((sum(new) + 1, 2, 64), k_type, 1).cuda(), typed((sum(new) + 1, 2, 64), v_type, 2).cuda()
    caches = [on_device(qx, filled(20, 2, 32, 64, 3)) for _ in range(2)]
    table = table_of(3, 5, 20)
    batch, _, _ = batch_of(qx, table, lengths, new, 1)
    assert caches[0].append_dev(batch, k, v, qx.Rope(32)) == qx.OK
    assert caches[1].append_dev(batch, k.float(), v.float(), qx.Rope(32)) == qx.OK  # (exact)
    for a, b in zip(caches[0].arrays, caches[1].arrays):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_nobody_beside_many_queries(qx, dtype):
    """More tokens than the append kernel turns by itself: the queries' own launch leaves rows behind the batch alone."""
    lengths, new = [900, 30, 64, 2000], [400, 30, 0, 700]
    rows = sum(new) + 3
    cache, table = filled(300, 1, 32, 64, 3), table_of(4, 63, 300)
    batch, _, _ = batch_of(qx, table, lengths, new, 3)
    k = typed((rows, 1, 64), dtype, 1).cuda()
    q = typed((rows, 3, 64), dtype, 2).cuda()
    out = torch.full_like(q, 7.0)
    positions = torch.cat([torch.arange(t - n, t) for t, n in zip(lengths, new)] + [torch.zeros(3, dtype=torch.int64)]).cuda()
    rope = qx.Rope(64)
    want = torch.empty_like(q)
    assert rope.apply_dev(q, want, positions) == qx.OK
    assert on_device(qx, cache).append_dev(batch, k, k, rope, q, out) == qx.OK
    assert torch.equal(out[:-3], want[:-3]) and bool((out[-3:] == 7).all())


@pytest.mark.parametrize("lengths,new", [([900, 70, 300], [1, 1, 1]), ([900], [1]), ([900, 200], [60, 200])])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_blocks_past_two_gigabytes(qx, lengths, new, dtype):
    """Few blocks of a cache of 2.4 GB of codes each for keys and values, the last ones: the same as in a small cache."""
    size, dim, heads, count = 128, 128, 2, 74000  # 32 KB of codes a block
    small, table = filled(16, heads, size, dim), table_of(len(lengths), 8 if len(lengths) < 3 else 5, 16)
    width = -(-max(lengths) // size)
    table = np.resize(table, (len(lengths), width)).astype(np.int32)
    near = on_device(qx, small)
    far = qx.KVCache.empty(count, heads, size, dim)
    for to, come in zip(far.arrays, near.arrays):
        to[count - 16:] = come
    batch, _, rows = batch_of(qx, table, lengths, new)
    moved, _, _ = batch_of(qx, table + (count - 16), lengths, new)
    q = typed((rows, 4, dim), dtype, 3).cuda()
    want, got = torch.zeros_like(q), torch.zeros_like(q)
    assert near.attention_dev(batch, q, want) == qx.OK and far.attention_dev(moved, q, got) == qx.OK
    torch.cuda.synchronize()
    assert qx.lib.qx_check_device_errors() == qx.OK and bool((want != 0).any())
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", [3, 60])
def test_views_past_two_gigabytes(qx, new):
    """Heads whose rows lie so far apart that their offsets pass 32 bits, in every operator."""
    heads, dim, size = 2, 64, 32
    stride = ((1 << 31) // (new - 1) + 4096) // 64 * 64  # elements: the last row lies behind 2^31
    room = torch.zeros((new - 1) * stride + heads * dim, dtype=BF16, device="cuda")
    wide = room.as_strided((new, heads, dim), (stride, dim, 1))
    x = typed((new, heads, dim), BF16, 1).cuda()
    wide.copy_(x)
    cache, table = filled(8, heads, size, dim), table_of(1, 4, 8)
    batch, _, _ = batch_of(qx, table, [100], [new])
    rope, positions = qx.Rope(dim), torch.arange(new, device="cuda")
    for turned in (lambda src, dst: rope.apply_dev(src, dst, positions),
                   lambda src, dst: on_device(qx, cache).append_dev(batch, x, x, rope, src, dst),
                   lambda src, dst: on_device(qx, cache).attention_dev(batch, src, dst),
                   lambda src, dst: on_device(qx, cache).read_dev(batch, dst, None)):
        want, got = torch.zeros_like(x), torch.zeros_like(x)
        assert turned(x, want) == qx.OK and turned(wide, got) == qx.OK, qx.last_error()
        assert torch.equal(got, want) and bool((want != 0).any())
        assert turned(x, wide) == qx.OK, qx.last_error()
        assert torch.equal(wide, want)
        wide.copy_(x)
    near, far = (on_device(qx, cache) for _ in range(2))
    assert near.append_dev(batch, x, x) == qx.OK and far.append_dev(batch, wide, wide) == qx.OK
    for a, b in zip(near.arrays, far.arrays):
        assert torch.equal(a, b)
