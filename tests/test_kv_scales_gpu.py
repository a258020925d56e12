"""Block scales at the ends of their range, in a cache that somebody else filled too: zero and tiny ones beside codes
that are not zero, neighbours far apart, masks that hide the larger one."""

import numpy as np
import pytest
import torch

from kv_reference import Cache, attention, attention_tolerance
from test_kv_attention_gpu import BF16, F16, F32, filled
from test_kv_cache_gpu import append_both, batch_of, on_device, table_of, typed

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


def compare(qx, cache, table, lengths, new, q, window=0, missing=None):
    """Causal attention with an f32 output (values of any magnitude fit) and its lse, row by row; `missing`: keys without
    a weight in any precision."""
    heads, dim = q.shape[1:]
    batch, begin, rows = batch_of(qx, table, lengths, new)
    out, lse = torch.full((rows, heads, dim), 3.0, device="cuda"), torch.full((rows, heads), 3.0, device="cuda")
    assert on_device(qx, cache).attention_dev(batch, q.cuda(), out, window=window, lse=lse) == qx.OK, qx.last_error()
    for s, (t, n) in enumerate(zip(lengths, new)):
        at = slice(int(begin[s]), int(begin[s]) + n)
        k, v = (torch.from_numpy(cache.values(i, table[s], t)) for i in range(2))
        want, sums, magnitude, _ = attention(q[at].double(), k, v, dim ** -0.5, True, window, missing or ())
        if missing:
            k[list(missing)] = 0  # (their products are no part of the others' scores)
        *_, spread = attention(q[at].double(), k, v, dim ** -0.5, True, window)
        limit, lse_limit = attention_tolerance(want, sums, magnitude, spread, q.dtype, dim, t)
        off, lse_off = (out[at].cpu().double() - want).abs() / limit, (lse[at].cpu().double() - sums).abs() / lse_limit
        assert float(off.max()) <= 1 and float(lse_off.max()) <= 1, (s, float(off.max()), float(lse_off.max()))


SHAPES = pytest.mark.parametrize("dim,group,new", [(64, 1, 1), (128, 4, 1), (64, 3, 5), (256, 2, 3), (96, 5, 2)])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@SHAPES
@pytest.mark.parametrize("factor", [2.0 ** 20, 2.0 ** 45])
@pytest.mark.parametrize("where", ["in front of the window", "behind the mask"])
def test_a_hidden_block_leaves_its_neighbour_its_bits(qx, dtype, dim, group, new, factor, where):
    """Two blocks of 16 share a tile of keys, and a mask hides the one with the larger scale: the tolerance goes by what
    a row sees."""
    size = 16
    cache, table = filled(30, 2, size, dim), table_of(3, 10, 30)
    if where == "in front of the window":  # the rows stand at the ends of blocks 3, 5 and 7
        lengths, window = [6 * size, 4 * size, 8 * size], 8
        for row in table:
            cache.scales[1][row[0::2]] *= np.float32(factor)
    else:  # only the last row sees the first token of the last block
        lengths, window = [5 * size + 1, 3 * size + 1, 7 * size + 1], 0
        for row, t in zip(table, lengths):
            cache.scales[1][row[t // size]] *= np.float32(factor)
    q = typed((3 * new, 2 * group, dim), dtype, 4)
    compare(qx, cache, table, lengths, [new] * 3, q, window)
    compare(qx, cache, table[:1], lengths[:1], [new], q[:new], window)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@SHAPES
def test_a_block_that_weighs_nothing_leaves_its_neighbour_its_bits(qx, dtype, dim, group, new):
    """The louder of two blocks of 16 in a tile is seen, with scores so far below the others' that its weights are zero in
    any precision: what is left is attention without it."""
    size, n = 16, 90
    cache, table = filled(6, 1, size, dim), table_of(1, 6, 6)
    q = typed((new, group, dim), dtype, 4).abs() + 1
    quiet = table[0, 2]
    cache.codes[0][quiet], cache.scales[0][quiet] = -127, 2000.0 / dim / dim ** -0.5 / 127  # scores of -2000 and below
    cache.scales[1][quiet] *= np.float32(2.0 ** 40)
    k = torch.from_numpy(cache.values(0, table[0], n))
    scores = dim ** -0.5 * (q.double().transpose(0, 1) @ k[:, 0].T)
    assert float((scores[..., 2 * size:3 * size].amax(-1) - scores[..., :2 * size].amax(-1)).max()) < -700  # (of e)
    compare(qx, cache, table, [n], [new], q, missing=range(2 * size, 3 * size))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@SHAPES
@pytest.mark.parametrize("length", [16, 17, 90])
def test_values_of_two_blocks_without_a_scale_are_zeros(qx, dtype, dim, group, new, length):
    cache, table = filled(6, 1, 16, dim), table_of(1, 6, 6)
    cache.scales[1][:] = 0.0
    batch, _, _ = batch_of(qx, table, [length], [new])
    out = torch.full((new, group, dim), 3.0, device="cuda")
    assert on_device(qx, cache).attention_dev(batch, typed((new, group, dim), dtype, 3).cuda(), out) == qx.OK
    assert bool((out == 0).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", [16, 64])
@pytest.mark.parametrize("scale", [0.0, -0.0])
@pytest.mark.parametrize("length,new", [(200, 130), (3000, 130)])
def test_values_of_a_prompt_without_a_scale_are_zeros(qx, dtype, size, scale, length, new):
    """Beside blocks that have one, too: rows that see none of those give zeros, the others what those give."""
    width = -(-length // size)
    cache, table = filled(width, 1, size, 64), table_of(1, width, width)
    cache.scales[1][:] = scale
    q = typed((new, 2, 64), dtype, 3)
    out = torch.full((new, 2, 64), 3.0, device="cuda")
    batch, _, _ = batch_of(qx, table, [length], [new])
    assert on_device(qx, cache).attention_dev(batch, q.cuda(), out) == qx.OK
    assert bool((out == 0).all())
    cache.scales[1][table[0, (length - 20) // size]] = 0.01
    compare(qx, cache, table, [length], [new], q)
    first = (length - 20) // size * size - (length - new)
    assert on_device(qx, cache).attention_dev(batch, q.cuda(), out) == qx.OK
    assert bool((out[:max(0, first)] == 0).all()) and bool((out[max(0, first) + 1:] != 0).any())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", [16, 64, 128])
@pytest.mark.parametrize("first,then", [(0.0, 2.0 ** 14), (0.0, 2.0 ** 40), (2.0 ** -90, 2.0 ** 40), (2.0 ** -60, 2.0 ** 60)])
@pytest.mark.parametrize("length,new", [(400, 400), (700, 130)])
def test_quiet_values_in_front_of_loud_ones(qx, dtype, size, first, then, length, new):
    """The first 128 keys' values are zero or tiny against all others: their weights count like any."""
    width = -(-length // size)
    cache, table = filled(width, 1, size, 64), table_of(1, width, width)
    cache.scales[1][:] *= np.float32(then)
    cache.scales[1][table[0, :128 // size]] = first
    compare(qx, cache, table, [length], [new], typed((new, 2, 64), dtype, 3))


def rounded_logarithms(around, sign):
    """A scale whose logarithm f32 rounds up (1) or down (-1) the most."""
    mantissas = np.float32(2.0) ** around * np.linspace(1, 1.999, 100001).astype(np.float32)
    exact = np.log2(mantissas.astype(np.float64))
    return mantissas[np.argmax(sign * (exact.astype(np.float32).astype(np.float64) - exact))]


U = 2.0 ** -23


@pytest.mark.parametrize("dim,size", [(64, 16), (128, 64)])
@pytest.mark.parametrize("around", [-90, -66, -40, 40, 66])
@pytest.mark.parametrize("sign", [1, -1])
def test_f32_prompts_keep_the_bits_of_value_scales(qx, dim, size, around, sign):
    """Every row sees its own key alone. Its weight is held as two f16 halves, 2 u, and meets the code in two products,
    1 u; the inverse of the scale, its product with the weight, the quotient of the largest scale and the sum, and the
    product with that are rounded, 0.5 u each."""
    cache, table = filled(-(-300 // size), 1, size, dim), table_of(1, -(-300 // size), -(-300 // size))
    cache.scales[1][:] = rounded_logarithms(around, sign)
    batch, _, _ = batch_of(qx, table, [300], [200])
    out = torch.zeros(200, 2, dim, device="cuda")
    assert on_device(qx, cache).attention_dev(batch, typed((200, 2, dim), F32, 3).cuda(), out, window=1) == qx.OK
    want = torch.from_numpy(cache.values(1, table[0], 300)[100:])
    assert float(((out.cpu().double() - want).abs() / want.abs().clamp_min(2.0 ** -120)).max()) <= 5 * U


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("by", [2.0 ** -90, 2.0 ** 112])
@pytest.mark.parametrize("sequences,length,new", [(1, 90, 1), (1, 6000, 2), (1, 20000, 1), (40, 900, 1), (2, 300, 150), (1, 6000, 100)])
def test_values_of_any_magnitude(qx, dtype, by, sequences, length, new):
    """Whole rows, rows in parts joined by either kernel, the balanced line: no sum leaves f32's range before the output
    does."""
    size, dim = 32, 64
    width = -(-length // size)
    cache, table = filled(width, 2, size, dim), table_of(1, width, width).repeat(sequences, 0)  # (all the same blocks)
    cache.scales[1][:] *= np.float32(by)
    compare(qx, cache, table, [length] * sequences, [new] * sequences, typed((sequences * new, 4, dim), dtype, 3))
