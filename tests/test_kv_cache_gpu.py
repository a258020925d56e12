"""The paged 8-bit cache: codes and scales bit for bit against the rule in 64 bits, in one go and token by
token, ragged batches, strides, blocks that hold NaN, batches that contradict themselves; read; host buffers."""

import numpy as np
import pytest
import torch

from kv_reference import Cache, rotated

pytestmark = pytest.mark.gpu


def on_device(qx, cache):
    return qx.KVCache(*[torch.from_numpy(a.copy()).cuda() for a in cache.codes + cache.scales])


def same(qx, dev, cache):
    torch.cuda.synchronize()
    assert qx.lib.qx_check_device_errors() == qx.OK, qx.last_error()
    for i in range(2):
        got, want = dev.arrays[2 + i].cpu().numpy(), cache.scales[i]
        assert np.array_equal(got, want, equal_nan=True), f"scales of {'kv'[i]}"
        got, want = dev.arrays[i].cpu().numpy(), cache.codes[i]
        # (the codes of a block without a scale say nothing)
        there = np.isfinite(cache.scales[i])[:, :, None, None] | np.zeros(want.shape, bool)
        assert np.array_equal(got[there], want[there]), f"codes of {'kv'[i]}"


def table_of(sequences, width, blocks, seed=0):
    """`width` blocks for every sequence, in random order."""
    order = np.random.default_rng(seed).permutation(blocks).astype(np.int32)
    return order[:sequences * width].reshape(sequences, width).copy()


def batch_of(qx, table, lengths, new, behind=0):
    """(KVBatch on the device, begin, rows): `new` tokens of every sequence packed, rows of nobody behind them."""
    begin = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    rows = int(begin[-1]) + behind
    dev = qx.KVBatch(torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.from_numpy(table).cuda(),
                     max(lengths), torch.from_numpy(begin).cuda(), rows, max(new))
    return dev, begin, rows


def append_both(qx, dev, cache, table, lengths, new, k, v, behind=0, **more):
    """The same append on the device and by the rule. `k`, `v`: packed rows, on the CPU."""
    batch, begin, rows = batch_of(qx, table, lengths, new, behind)
    assert k.shape[0] == rows
    assert dev.append_dev(batch, k.cuda(), v.cuda(), **more) == qx.OK, qx.last_error()
    for s, (t, n) in enumerate(zip(lengths, new)):
        for which, x in enumerate((k, v)):
            cache.append(which, table[s], t - n, x[begin[s]:begin[s] + n].double().numpy())
    return batch, begin


def typed(shape, dtype, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * spread).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size,dim,heads", [(16, 16, 1), (32, 64, 3), (64, 128, 8), (128, 256, 2), (16, 80, 2), (64, 96, 1)])
def test_prompts_then_tokens(qx, dtype, size, dim, heads):
    """Prompts of unequal lengths, then steps of 1, 2 and 5 tokens that grow the scales of the last blocks."""
    cache, table = Cache(40, heads, size, dim), table_of(4, 8, 40)
    dev, lengths = on_device(qx, cache), [0, 0, 0, 0]
    for step, new in enumerate([[1, size, 3 * size + size // 2, 0], [1, 0, 1, 1], [2, 2, 2, 0], [5, 0, size + 5, 1], [1, 1, 1, 1]]):
        lengths = [t + n for t, n in zip(lengths, new)]
        k, v = (typed((sum(new) + 3, heads, dim), dtype, 10 * step + i, 0.5 + step % 3) for i in range(2))
        append_both(qx, dev, cache, table, lengths, new, k, v, behind=3)
        same(qx, dev, cache)


def test_a_growing_scale_moves_older_codes(qx):
    """Every token louder than the last: all older codes of the block are moved each time, halves to even."""
    cache, table = Cache(3, 2, 16, 16), table_of(1, 2, 3)
    dev = on_device(qx, cache)
    for i in range(20):
        k, v = (typed((1, 2, 16), torch.float32, 5 * i + j, 1.1 ** i) for j in range(2))
        if i == 7:  # twice the scale: every odd code is a tie
            top = cache.scales[0][table[0, 0]].max() * 127 * 2
            k[:] = float(top)
        append_both(qx, dev, cache, table, [i + 1], [1], k, v)
        same(qx, dev, cache)


def test_halves_and_the_largest_code(qx):
    """Elements next to and on the halves between two codes, where a product with the inverse would round wrongly."""
    rng = np.random.default_rng(3)
    for scale in (1.0, 0.3, 1.7e-20, 3.1e30):
        top = np.float32(127 * np.float32(scale))
        s = np.float64(np.float32(np.float64(top) / 127))
        halves = ((rng.integers(-127, 126, 4096) + 0.5) * s).astype(np.float32)
        near = np.concatenate([halves, np.nextafter(halves, np.float32(np.inf)), np.nextafter(halves, -np.float32(np.inf))])
        x = torch.from_numpy(near[:3 * 4096].reshape(-1, 1, 256)).clamp(-float(top), float(top))
        x[::16, 0, 0] = float(top)
        cache, table = Cache(3, 1, 16, 256), table_of(1, 3, 3)
        dev, n = on_device(qx, cache), x.shape[0]
        append_both(qx, dev, cache, table, [n], [n], x, x.flip(0))
        same(qx, dev, cache)


def test_zeros_and_tiny_values(qx):
    cache, table = Cache(4, 1, 16, 32), table_of(1, 4, 4)
    dev = on_device(qx, cache)
    x = torch.zeros(64, 1, 32)
    x[16:32] = 1e-40   # below the smallest scale: zeros
    x[32:48] = 1e-28   # 1e-28 / 127 = 7.874e-31, just below 2^-100 = 7.889e-31: zeros too
    x[48:, 0, 3] = 127 * 2.0 ** -100
    append_both(qx, dev, cache, table, [64], [64], x, -x)
    same(qx, dev, cache)
    assert sorted(cache.scales[0][:, 0] > 0) == [False, False, False, True]


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_value_that_is_no_number_takes_its_block_and_head(qx, value):
    cache, table = Cache(6, 3, 16, 32), table_of(1, 4, 6)
    dev = on_device(qx, cache)
    k, v = typed((40, 3, 32), torch.float32, 1), typed((40, 3, 32), torch.float32, 2)
    k[20, 1, 5] = value
    append_both(qx, dev, cache, table, [40], [40], k, v)
    same(qx, dev, cache)
    assert np.isnan(cache.scales[0][table[0, 1], 1])
    assert np.isfinite(cache.scales[0][table[0]][[0, 0, 2, 2], [0, 1, 0, 1]]).all() and np.isfinite(cache.scales[1][table[0, :3]]).all()
    # and stays, until the block is begun anew
    append_both(qx, dev, cache, table, [41], [1], k[:1], v[:1])
    same(qx, dev, cache)
    append_both(qx, dev, cache, table, [33], [33], k[:33].nan_to_num(0, 0, 0), v[:33])
    same(qx, dev, cache)
    assert np.isfinite(cache.scales[0][table[0, :3]]).all()


@pytest.mark.parametrize("dtype,offset", [(torch.float32, 1), (torch.float16, 1), (torch.bfloat16, 8)])
def test_strided_inputs(qx, dtype, offset):
    """Slices of a packed projection, rows of odd lengths, broadcast heads."""
    size, dim, heads, n = 16, 48, 2, 21
    cache, table = Cache(4, heads, size, dim), table_of(1, 2, 4)
    dev = on_device(qx, cache)
    k, v = typed((n, heads, dim), dtype, 1), typed((n, 1, dim), dtype, 2).expand(n, heads, dim)
    store = torch.zeros(n * 301 + offset, dtype=dtype, device="cuda")
    k_dev = store.as_strided((n, heads, dim), (301, 100, 1), offset)
    k_dev.copy_(k)
    batch, begin, _ = batch_of(qx, table, [n], [n])
    assert dev.append_dev(batch, k_dev, v[:, :1].cuda().expand(n, heads, dim)) == qx.OK
    for which, x in enumerate((k, v)):
        cache.append(which, table[0], 0, x.double().numpy())
    same(qx, dev, cache)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("given", [False, True])
def test_rotation_on_the_way(qx, dtype, interleaved, given):
    """Keys rotated without a rounding in between: scales to f32's precision, codes of the rotated value but for
    those next to a half; the queries have the bits of qx_rope_apply."""
    size, dim, heads, lengths, new = 64, 128, 4, [70, 300], [3, 129]
    rope = qx.Rope(64, interleaved, 10000.0, dict(kind=qx.ROPE_LINEAR, factor=3.0))
    cache, table = Cache(12, heads, size, dim), table_of(2, 5, 12)
    for i in range(2):
        cache.scales[i][:] = 0.0  # blocks that hold older tokens: all of them zero
        cache.codes[i][:] = 0
    dev = on_device(qx, cache)
    batch, begin, rows = batch_of(qx, table, lengths, new, behind=2)
    k, v, q = typed((rows, heads, dim), dtype, 1), typed((rows, heads, dim), dtype, 2), typed((rows, 12, dim), dtype, 3)
    place = torch.cat([torch.arange(t - n, t) for t, n in zip(lengths, new)] + [torch.zeros(2, dtype=torch.int64)])
    at = place * 1000 + 7 if given else place
    q_out = torch.full((rows, 12, dim), 5.0, dtype=dtype, device="cuda")
    assert dev.append_dev(batch, k.cuda(), v.cuda(), rope, q.cuda(), q_out, at.cuda() if given else None) == qx.OK
    torch.cuda.synchronize()
    assert qx.lib.qx_check_device_errors() == qx.OK
    alone = torch.empty_like(q_out)
    qx.check(rope.apply_dev(q.cuda(), alone, at.cuda()), "rope")
    assert torch.equal(q_out[:-2], alone[:-2]) and bool((q_out[-2:] == 5).all())
    turned = rotated(k.double(), at.tolist(), rope.view.frequency[:32], interleaved=interleaved).numpy()
    for s, (t, n) in enumerate(zip(lengths, new)):
        cache.append(0, table[s], t - n, turned[begin[s]:begin[s] + n])
        cache.append(1, table[s], t - n, v[begin[s]:begin[s] + n].double().numpy())
    scales = dev.arrays[2].cpu().numpy()
    # rotated values are within 24 u of 2 max |x| (tests of the rotation), scales one rounding more
    slack = 24 * 2.0 ** -24 * 2 * float(k.double().abs().max())
    for s, (t, n) in enumerate(zip(lengths, new)):
        for p in range(t - n, t):
            block = table[s, p // size]
            assert np.all(np.abs(scales[block] - cache.scales[0][block]) <= slack / 127 + 2.0 ** -23 * scales[block])
            got = dev.arrays[0][block, :, p % size].cpu().numpy().astype(np.float64) * scales[block][:, None].astype(np.float64)
            want = turned[begin[s] + p - (t - n)]
            assert np.all(np.abs(got - want) <= scales[block][:, None] * 0.5 * (1 + 2.0 ** -20) + 4 * slack)
    values = dev.arrays[3].cpu().numpy()
    assert np.array_equal(values, cache.scales[1]) and np.array_equal(dev.arrays[1].cpu().numpy(), cache.codes[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size,dim", [(16, 16), (64, 128), (32, 80), (128, 256)])
def test_read(qx, dtype, size, dim):
    heads, lengths, new = 3, [5, 0, 2 * size + 3, size], [5, 0, size + 1, 0]
    cache, table = Cache(16, heads, size, dim, seed=4), table_of(4, 4, 16)
    cache.scales = [np.random.default_rng(i).random((16, heads), np.float32) for i in range(2)]
    dev = on_device(qx, cache)
    batch, begin, rows = batch_of(qx, table, lengths, new, behind=2)
    wide = torch.full((rows, heads + 2, dim), 7.0, dtype=dtype, device="cuda")  # k inside wider rows
    v = torch.full((rows, heads, dim + 1), 7.0, dtype=dtype, device="cuda")     # v off every boundary
    assert dev.read_dev(batch, wide[:, 1:1 + heads], v[..., 1:]) == qx.OK
    only = torch.zeros(rows, heads, dim, dtype=dtype, device="cuda")
    assert dev.read_dev(batch, None, only) == qx.OK
    torch.cuda.synchronize()
    assert qx.lib.qx_check_device_errors() == qx.OK
    for s, (t, n) in enumerate(zip(lengths, new)):
        rows_of = slice(int(begin[s]), int(begin[s]) + n)
        for which, got in ((0, wide[:, 1:1 + heads]), (1, v[..., 1:]), (1, only)):
            want = torch.from_numpy(cache.values(which, table[s], t)[t - n:]).float().to(dtype)  # (code * scale: f32 rounds once)
            assert torch.equal(got[rows_of].cpu(), want)
    assert bool((wide[:, 0] == 7).all()) and bool((wide[:, -1] == 7).all()) and bool((v[..., 0] == 7).all())
    assert bool((wide[-2:] == 7).all()) and bool((v[-2:] == 7).all())


def test_codes_past_two_gigabytes(qx):
    """Block numbers whose byte offsets need more than 32 bits."""
    blocks, heads, size, dim = 70000, 2, 128, 128
    codes = [torch.zeros(blocks, heads, size, dim, dtype=torch.int8, device="cuda") for _ in "kv"]
    scales = [torch.zeros(blocks, heads, device="cuda") for _ in "kv"]
    dev = qx.KVCache(*codes, *scales)
    table = np.array([[69999, 3], [65536, 65535]], np.int32)
    k, v = typed((200, heads, dim), torch.bfloat16, 1), typed((200, heads, dim), torch.bfloat16, 2)
    batch, begin, _ = batch_of(qx, table, [140, 60], [140, 60])
    assert dev.append_dev(batch, k.cuda(), v.cuda()) == qx.OK
    out = [torch.empty(200, heads, dim, device="cuda") for _ in "kv"]
    assert dev.read_dev(batch, *out) == qx.OK
    small = Cache(4, heads, size, dim)
    local = np.array([[0, 1], [2, 3]], np.int32)
    for s, (t, a) in enumerate(((140, 0), (60, 140))):
        for which, x in enumerate((k, v)):
            small.append(which, local[s], 0, x[a:a + t].double().numpy())
            want = torch.from_numpy(small.values(which, local[s], t)).float()
            assert torch.equal(out[which][a:a + t].cpu(), want)
    for blocks_of in (69999, 65536):
        assert float(scales[0][blocks_of].min()) > 0
    assert int((scales[0].sum(1) > 0).sum()) == 3


@pytest.mark.parametrize("what", ["block past the cache", "block below zero", "length past the bound", "rows past the bound",
                                  "rows past the views", "rows backwards", "more rows than tokens"])
def test_a_batch_that_contradicts_itself_is_reported(qx, what):
    """The other sequence is served, nothing is written out of place, and the report comes once."""
    size, dim, heads = 16, 32, 2
    lengths, new, most, longest = [20, 10], [20, 10], 20, 32
    table = np.array([[0, 1], [2, 3]], np.int32)
    begin = np.array([0, 20, 30], np.int32)
    if what == "block past the cache":
        table[0, 1] = 6
    elif what == "block below zero":
        table[0, 1] = -1
    elif what == "length past the bound":
        lengths[0] = 33
    elif what == "rows past the bound":
        most = 19
    elif what == "rows past the views":
        begin[:] = 20, 40, 50
    elif what == "rows backwards":
        begin[:] = 10, 0, 10
    else:
        lengths[0] = 19
    cache = Cache(6, heads, size, dim)
    cache.scales = [np.full((6, heads), 9.0, np.float32) for _ in "kv"]
    dev = on_device(qx, cache)
    tensors = [torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.from_numpy(table).cuda(), torch.from_numpy(begin).cuda()]
    batch = qx.KVBatch(tensors[0], tensors[1], longest, tensors[2], 30, most)
    k, v = typed((30, heads, dim), torch.float32, 1), typed((30, heads, dim), torch.float32, 2)
    for call in ("append", "read", "append"):
        if call == "append":
            assert dev.append_dev(batch, k.cuda(), v.cuda()) == qx.OK
        else:
            assert dev.read_dev(batch, *[torch.zeros(30, heads, dim, device="cuda") for _ in "kv"]) == qx.OK
        torch.cuda.synchronize()
        assert qx.lib.qx_check_device_errors() == qx.DEVICE_ERROR
        assert ("block" if "block" in what else "sequence") in qx.last_error()
        assert qx.lib.qx_check_device_errors() == qx.OK
    if what != "rows past the views":
        first = int(begin[1])
        cache.append(0, table[1], 0, k[first:first + 10].double().numpy())
        cache.append(1, table[1], 0, v[first:first + 10].double().numpy())
    if "block" in what:  # the blocks of the sequence that are there
        cache.append(0, table[0], 0, k[:16].double().numpy())
        cache.append(1, table[0], 0, v[:16].double().numpy())
    same(qx, dev, cache)


def test_captured(qx):
    """A captured step reads lengths and blocks anew at every replay."""
    size, dim, heads = 16, 64, 2
    cache, table = Cache(8, heads, size, dim), table_of(2, 4, 8)
    dev = on_device(qx, cache)
    k, v = (torch.zeros(2, heads, dim, device="cuda") for _ in "kv")
    lengths = torch.tensor([1, 15], dtype=torch.int32, device="cuda")
    batch = qx.KVBatch(lengths, torch.from_numpy(table).cuda(), 64, None, 2, 1)
    seed_k, seed_v = typed((14, heads, dim), torch.float32, 7), typed((14, heads, dim), torch.float32, 8)
    append_both(qx, dev, cache, table, [0, 14], [0, 14], seed_k, seed_v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert dev.append_dev(batch, k, v) == qx.OK
    for step in range(20):
        a, b = typed((2, heads, dim), torch.float32, 100 + step), typed((2, heads, dim), torch.float32, 200 + step)
        k.copy_(a)
        v.copy_(b)
        graph.replay()
        for s in range(2):
            cache.append(0, table[s], int(lengths[s]) - 1, a[s:s + 1].double().numpy())
            cache.append(1, table[s], int(lengths[s]) - 1, b[s:s + 1].double().numpy())
        lengths += 1
        same(qx, dev, cache)


@pytest.mark.parametrize("rope_on", [False, True])
def test_host_buffers(qx, rope_on):
    """The same bits as the device forms; blocks that the batch does not name are not touched."""
    size, dim, heads, lengths, new = 32, 48, 2, [40, 7, 0], [10, 7, 0]
    cache, table = Cache(9, heads, size, dim), table_of(3, 2, 9)
    cache.scales = [np.random.default_rng(i).random((9, heads), np.float32) for i in range(2)]
    dev, host = on_device(qx, cache), qx.KVCache(*[a.copy() for a in cache.codes + cache.scales])
    batch, begin, rows = batch_of(qx, table, lengths, new, behind=1)
    host_batch = qx.KVBatch(np.array(lengths, np.int32), table, 64, begin, rows, max(new))
    rope = qx.Rope(32) if rope_on else None
    k, v, q = (typed((rows, h, dim), torch.float32, i) for i, h in enumerate((heads, heads, 4)))
    q_out = torch.full((rows, 4, dim), 3.0)
    q_dev = q_out.cuda()
    more = ((rope, q.cuda(), q_dev), (rope, q.numpy(), q_out.numpy())) if rope_on else ((), ())
    assert dev.append_dev(batch, k.cuda(), v.cuda(), *more[0]) == qx.OK
    assert host.append(host_batch, k.numpy(), v.numpy(), *more[1]) == qx.OK, qx.last_error()
    torch.cuda.synchronize()
    for a, b in zip(dev.arrays, host.arrays):
        assert np.array_equal(a.cpu().numpy(), b)
    assert torch.equal(q_dev.cpu(), q_out)
    out = [np.full((rows, heads, dim), 4.0, np.float32) for _ in "kv"]
    out_dev = [torch.full((rows, heads, dim), 4.0, device="cuda") for _ in "kv"]
    assert host.read(host_batch, *out) == qx.OK, qx.last_error()
    assert dev.read_dev(batch, *out_dev) == qx.OK
    for a, b in zip(out_dev, out):
        assert np.array_equal(a.cpu().numpy(), b)
    assert (out[0][-1] == 4).all()
