"""Rotary positions, the 8-bit key-value cache and attention over it, without a GPU: what the entry points
refuse, in which order, and the frequencies of qx_rope_init against their formulas."""

import ctypes as C
import math

import numpy as np
import pytest
import torch


def cache_arrays(blocks=4, heads=2, size=16, dim=32):
    return [np.zeros((blocks, heads, size, dim), np.int8) for _ in "kv"] + [np.zeros((blocks, heads), np.float32) for _ in "kv"]


def int32(*values):
    return np.array(values, np.int32)


@pytest.fixture
def parts(qx):
    cache = qx.KVCache(*cache_arrays())
    batch = qx.KVBatch(int32(20, 5), np.array([[0, 1], [2, 3]], np.int32), 32, int32(0, 2, 3), 3, 2)
    x = np.zeros((3, 2, 32), np.float32)
    q = np.zeros((3, 4, 32), np.float32)
    return cache, batch, x, q


def served(qx, status):
    """All checks passed: the call went on to look for a device."""
    return status in (qx.OK, qx.DEVICE_ERROR)


# ---- rotary positions ---------------------------------------------------------------------

def test_frequencies(qx):
    plain = qx.Rope(64, qx.ROPE_INTERLEAVED, 10000.0).view
    assert (plain.rotary_dim, plain.style, plain.amplitude) == (64, qx.ROPE_INTERLEAVED, 1.0)
    base = [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert np.allclose(plain.frequency[:32], base, rtol=1e-14)
    assert all(v == 0 for v in plain.frequency[32:])
    linear = qx.Rope(64, scaling=dict(kind=qx.ROPE_LINEAR, factor=4.0)).view
    assert np.allclose(linear.frequency[:32], np.array(base) / 4, rtol=1e-14)
    assert linear.amplitude == 1.0


def test_banded_frequencies(qx):
    view = qx.Rope(128, base=500000.0, scaling=dict(kind=qx.ROPE_BANDS, factor=8.0, trained=8192, slow=1.0, fast=4.0)).view
    kept = divided = between = 0
    for i in range(64):
        f = 500000.0 ** (-2 * i / 128)
        turns = 8192 * f / (2 * math.pi)
        if turns >= 4:
            want, kept = f, kept + 1
        elif turns <= 1:
            want, divided = f / 8, divided + 1
        else:
            w = (turns - 1) / 3
            want, between = (1 - w) * f / 8 + w * f, between + 1
        assert view.frequency[i] == pytest.approx(want, rel=1e-13)
    assert kept and divided and between and view.amplitude == 1.0


def test_ramped_frequencies(qx):
    factor, trained, base, dim = 16.0, 4096, 10000.0, 128
    view = qx.Rope(dim, base=base, scaling=dict(kind=qx.ROPE_RAMP, factor=factor, trained=trained, slow=1.0, fast=32.0)).view
    at = lambda turns: dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = math.floor(at(32)), math.ceil(at(1))
    for i in range(dim // 2):
        f = base ** (-2 * i / dim)
        cut = min(1, max(0, (i - low) / (high - low)))
        assert view.frequency[i] == pytest.approx(f / factor * cut + f * (1 - cut), rel=1e-13)
    assert view.amplitude == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-15)
    assert qx.Rope(dim, scaling=dict(kind=qx.ROPE_RAMP, factor=0.5, trained=trained, slow=1, fast=32)).view.amplitude == 1.0


def test_rope_init_refusals(qx):
    view = qx.RopeView()
    init = lambda d=64, s=0, b=1e4, k=None, r=C.byref(view): qx.lib.qx_rope_init(r, d, s, b, k)  # noqa: E731
    for dim in (0, -2, 63, 258):
        assert init(d=dim) == qx.INVALID_SHAPE
    assert init(s=2) == qx.UNSUPPORTED_FORMAT
    assert init(k=qx.RopeScaling(4, 1, 1, 1, 2)) == qx.UNSUPPORTED_FORMAT
    assert init(r=None) == qx.INVALID_ARGUMENT
    for base in (1.0, 0.0, -5.0, math.inf, math.nan):
        assert init(b=base) == qx.INVALID_ARGUMENT
    for scaling in ((1, 0.0, 1, 1, 2), (1, math.nan, 1, 1, 2), (2, 8, 0, 1, 4), (2, 8, 100, 4, 4), (3, 8, 100, 0, 4),
                    (3, 8, math.inf, 1, 4), (2, 8, 100, 1, math.inf)):
        assert init(k=qx.RopeScaling(*scaling)) == qx.INVALID_ARGUMENT, scaling
    assert init(d=256) == qx.OK


def test_rope_apply_refusals(qx):
    rope, x, at = qx.Rope(32), np.zeros((3, 2, 48), np.float32), np.zeros(3, np.int64)
    H = qx.heads_view
    call = lambda r=rope.view, a=None, b=None, p=at.ctypes.data, t=3, d=48: qx.lib.qx_rope_apply(  # noqa: E731
        r, a or H(x), b or H(x), p, t, d, 0)
    assert served(qx, call())
    assert call(t=-1) == qx.INVALID_SHAPE
    assert call(d=0) == qx.INVALID_SHAPE
    assert call(d=30) == qx.INVALID_SHAPE  # smaller than the rotary part
    assert call(r=None) == qx.INVALID_ARGUMENT
    assert qx.lib.qx_rope_apply(rope.view, None, H(x), at.ctypes.data, 3, 48, 0) == qx.INVALID_ARGUMENT
    assert call(p=None) == qx.INVALID_ARGUMENT
    assert call(a=H(x, kind=3)) == qx.UNSUPPORTED_FORMAT
    assert call(a=H(x, kind=qx.F16)) == qx.UNSUPPORTED_FORMAT  # not y's type
    assert call(a=H(x, heads=0)) == qx.INVALID_SHAPE
    assert call(a=H(x, heads=1)) == qx.INVALID_SHAPE  # not y's heads
    assert call(a=H(x, token_stride=-1)) == qx.INVALID_SHAPE
    y = np.zeros((3, 2, 48), np.float32)
    assert call(b=H(y, token_stride=40)) == qx.INVALID_SHAPE  # overlaps itself
    assert call(b=H(y, head_stride=0)) == qx.INVALID_SHAPE
    assert call(b=H(y, token_stride=90)) == qx.INVALID_SHAPE
    assert served(qx, call(a=H(x, token_stride=0, head_stride=0), b=H(y)))  # one head for all: read only
    assert call(a=H(x, token_stride=0)) == qx.INVALID_ARGUMENT  # in place through another view
    assert call(b=H(y, token_stride=1 << 62)) == qx.INVALID_SHAPE
    odd = H(y)
    odd.data += 2
    assert call(b=odd) == qx.INVALID_ARGUMENT
    bad = qx.Rope(32)
    bad.view.frequency[3] = math.nan
    assert call(r=bad.view) == qx.INVALID_ARGUMENT
    bad = qx.Rope(32)
    bad.view.rotary_dim = 31
    assert call(r=bad.view) == qx.INVALID_SHAPE
    bad.view.rotary_dim, bad.view.style = 32, 7
    assert call(r=bad.view) == qx.UNSUPPORTED_FORMAT
    assert served(qx, call(t=0, p=None))


# ---- cache and batch ----------------------------------------------------------------------

def each_call(qx, cache, batch, x, q):
    """(name, call) of the three host-pointer operators."""
    H = qx.heads_view
    return [("append", lambda c=cache, b=batch: qx.lib.qx_kv_append(c, b, H(x), H(x), None, None, None, None)),
            ("read", lambda c=cache, b=batch: qx.lib.qx_kv_read(c, b, H(x), H(x.copy()))),
            ("attention", lambda c=cache, b=batch: qx.lib.qx_kv_attention(c, b, H(q), H(q), None, 1.0, 1, 0))]


def test_cache_refusals(qx, parts):
    cache, batch, x, q = parts
    for name, call in each_call(qx, cache.view, batch.view, x, q):
        assert served(qx, call()), name
        assert call(c=None) == qx.INVALID_ARGUMENT, name
        assert call(b=None) == qx.INVALID_ARGUMENT, name
        for field, values, status in (("blocks", (0, -1, 1 << 40), qx.INVALID_SHAPE), ("kv_heads", (0, -1), qx.INVALID_SHAPE),
                                      ("block_tokens", (0, 8, 48, 256), qx.INVALID_SHAPE),
                                      ("head_dim", (0, 8, 40, 272), qx.INVALID_SHAPE),
                                      ("k_codes", (None, cache.view.k_codes + 8), qx.INVALID_ARGUMENT),
                                      ("v_codes", (None, cache.view.v_codes + 1), qx.INVALID_ARGUMENT),
                                      ("k_scales", (None, cache.view.k_scales + 2), qx.INVALID_ARGUMENT),
                                      ("v_scales", (None,), qx.INVALID_ARGUMENT)):
            for value in values:
                bad = qx.KVCacheView.from_buffer_copy(cache.view)
                setattr(bad, field, value)
                assert call(c=bad) == status, (name, field, value)


def test_batch_refusals(qx, parts):
    cache, batch, x, q = parts
    for name, call in each_call(qx, cache.view, batch.view, x, q):
        for field, values, status in (("sequences", (-1,), qx.INVALID_SHAPE), ("tokens", (-1,), qx.INVALID_SHAPE),
                                      ("max_tokens", (-1, 0x7FFFFFFF), qx.INVALID_SHAPE),
                                      ("max_length", (-1, 33, 0x7FFFFFFF), qx.INVALID_SHAPE),
                                      ("table_stride", (-1, 1, 1 << 62), qx.INVALID_SHAPE),
                                      ("lengths", (None,), qx.INVALID_ARGUMENT),
                                      ("block_table", (None,), qx.INVALID_ARGUMENT)):
            for value in values:
                bad = qx.KVBatchView.from_buffer_copy(batch.view)
                setattr(bad, field, value)
                assert call(b=bad) == status, (name, field, value)
        even = qx.KVBatchView.from_buffer_copy(batch.view)
        even.token_begin = None
        assert call(b=even) == qx.INVALID_SHAPE, name  # two sequences of two tokens in three rows
        even.max_tokens = 1
        assert served(qx, call(b=even)), name


@pytest.mark.parametrize("what", ["block past the cache", "block below zero", "length below zero", "length past the bound",
                                  "rows past the bound", "rows past the views", "rows backwards", "rows before the first",
                                  "more rows than tokens"])
def test_contents_of_a_batch_are_checked_on_the_host(qx, parts, what):
    cache, _, x, q = parts
    lengths, table, begin, most = int32(20, 5), np.array([[0, 1], [2, 3]], np.int32), int32(0, 2, 3), 2
    if what == "block past the cache":
        table[0, 1] = 4
    elif what == "block below zero":
        table[1, 0] = -1
    elif what == "length below zero":
        lengths[1] = -1
    elif what == "length past the bound":
        lengths[0] = 33
    elif what == "rows past the bound":
        begin[:] = 0, 3, 3
    elif what == "rows past the views":
        begin[:] = 0, 2, 4
    elif what == "rows backwards":
        begin[:] = 0, 2, 1
    elif what == "rows before the first":
        begin[:] = -1, 1, 3
    else:
        lengths[0] = 1
    batch = qx.KVBatch(lengths, table, 32, begin, 3, most)
    for name, call in each_call(qx, cache.view, batch.view, x, q):
        if what == "more rows than tokens" and name == "attention":
            assert served(qx, call())  # (rows that see nothing)
        else:
            assert call() == qx.INVALID_ARGUMENT, name


def test_blocks_behind_a_length_are_not_looked_at(qx, parts):
    cache, _, x, q = parts
    batch = qx.KVBatch(int32(16, 0), np.array([[1, 99], [-7, 99]], np.int32), 32, int32(0, 3, 3), 3, 3)
    for name, call in each_call(qx, cache.view, batch.view, x, q):
        assert served(qx, call()), name


def test_written_blocks_belong_to_one_sequence(qx, parts):
    cache, _, x, q = parts
    shared = np.array([[0, 1], [0, 1]], np.int32)
    for lengths, fine in ((int32(18, 17), False), (int32(18, 16), False), (int32(32, 32), False)):
        batch = qx.KVBatch(lengths, shared, 32, int32(0, 1, 2), 3, 2)
        results = dict((name, call()) for name, call in each_call(qx, cache.view, batch.view, x, q))
        assert results["append"] == qx.INVALID_ARGUMENT
        assert served(qx, results["read"]) and served(qx, results["attention"])
    # a shared full prefix, blocks of one's own behind it
    batch = qx.KVBatch(int32(18, 17), np.array([[0, 1], [0, 2]], np.int32), 32, int32(0, 2, 3), 3, 2)
    assert served(qx, each_call(qx, cache.view, batch.view, x, q)[0][1]())


def test_append_refusals(qx, parts):
    cache, batch, x, q = parts
    H, rope = qx.heads_view, qx.Rope(32)
    call = lambda k=None, v=None, r=None, a=None, b=None: qx.lib.qx_kv_append(  # noqa: E731
        cache.view, batch.view, k or H(x), v or H(x), r, None, a, b)
    assert qx.lib.qx_kv_append(cache.view, batch.view, None, H(x), None, None, None, None) == qx.INVALID_ARGUMENT
    assert call(k=H(q)) == qx.INVALID_SHAPE  # four heads
    assert call(v=H(x, heads=1)) == qx.INVALID_SHAPE
    assert call(k=H(x, kind=5)) == qx.UNSUPPORTED_FORMAT
    assert call(r=qx.Rope(24).view) == qx.INVALID_SHAPE  # not whole units of 16
    assert call(r=qx.Rope(48).view) == qx.INVALID_SHAPE  # larger than the head
    assert call(a=H(q)) == qx.INVALID_ARGUMENT  # a query without a place for it
    assert call(a=H(q), b=H(q)) == qx.INVALID_ARGUMENT  # and without a rotation
    assert call(r=rope.view, a=H(q), b=H(x)) == qx.INVALID_SHAPE
    assert call(r=rope.view, a=H(q), b=H(q, kind=qx.BF16)) == qx.UNSUPPORTED_FORMAT
    assert served(qx, call(r=rope.view, a=H(q), b=H(q)))
    assert served(qx, call(k=H(x, token_stride=0, head_stride=0)))


def test_read_and_attention_refusals(qx, parts):
    cache, batch, x, q = parts
    H = qx.heads_view
    assert qx.lib.qx_kv_read(cache.view, batch.view, H(q), None) == qx.INVALID_SHAPE
    assert qx.lib.qx_kv_read(cache.view, batch.view, None, H(x, head_stride=8)) == qx.INVALID_SHAPE
    assert served(qx, qx.lib.qx_kv_read(cache.view, batch.view, H(x), None))
    call = lambda a=None, b=None, scale=1.0, window=0: qx.lib.qx_kv_attention(  # noqa: E731
        cache.view, batch.view, a or H(q), b or H(q), None, scale, 1, window)
    assert call(a=H(q, heads=3), b=H(q, heads=3)) == qx.INVALID_SHAPE  # no multiple of the kv heads
    assert call(b=H(x)) == qx.INVALID_SHAPE
    assert call(a=H(q, kind=9)) == qx.UNSUPPORTED_FORMAT
    for scale in (math.inf, math.nan):
        assert call(scale=scale) == qx.INVALID_ARGUMENT
    assert call(window=-1) == qx.INVALID_ARGUMENT
    assert served(qx, call(b=H(q.copy(), kind=qx.F32), window=1 << 40))


def test_device_forms_check_the_same_shapes(qx, parts):
    cache, batch, x, q = parts
    H, bad = qx.heads_view, qx.KVCacheView.from_buffer_copy(cache.view)
    bad.block_tokens = 20
    assert qx.lib.qx_kv_append_dev(bad, batch.view, H(x), H(x), None, None, None, None, None) == qx.INVALID_SHAPE
    assert qx.lib.qx_kv_read_dev(bad, batch.view, H(x), H(x), None) == qx.INVALID_SHAPE
    assert qx.lib.qx_kv_attention_dev(bad, batch.view, H(q), H(q), None, 1.0, 1, 0, None, None) == qx.INVALID_SHAPE
    assert qx.lib.qx_rope_apply_dev(qx.Rope(32).view, H(x), H(x), None, 3, 32, 0, None) == qx.INVALID_ARGUMENT


def test_arrays_off_their_boundaries_are_refused(qx, parts):
    """Positions, batch arrays and lse that start inside an element, by both forms."""
    cache, batch, x, q = parts
    H, rope, room = qx.heads_view, qx.Rope(32), np.zeros(64, np.uint8)
    odd = room.ctypes.data + 4
    odd += 8 - odd % 8 + 2
    for field in ("token_begin", "lengths", "block_table"):
        bad = qx.KVBatchView.from_buffer_copy(batch.view)
        setattr(bad, field, odd)
        for name, call in each_call(qx, cache.view, batch.view, x, q):
            assert call(b=bad) == qx.INVALID_ARGUMENT, (name, field)
        assert qx.lib.qx_kv_append_dev(cache.view, bad, H(x), H(x), None, None, None, None, None) == qx.INVALID_ARGUMENT
        assert qx.lib.qx_kv_read_dev(cache.view, bad, H(x), H(x), None) == qx.INVALID_ARGUMENT
        assert qx.lib.qx_kv_attention_dev(cache.view, bad, H(q), H(q), None, 1.0, 1, 0, None, None) == qx.INVALID_ARGUMENT
    for at in (odd, odd + 2):
        assert qx.lib.qx_kv_append(cache.view, batch.view, H(x), H(x), rope.view, at, None, None) == qx.INVALID_ARGUMENT
        assert qx.lib.qx_kv_append_dev(cache.view, batch.view, H(x), H(x), rope.view, at, None, None, None) == qx.INVALID_ARGUMENT
        assert qx.lib.qx_rope_apply(rope.view, H(x), H(x), at, 3, 32, 0) == qx.INVALID_ARGUMENT
        assert qx.lib.qx_rope_apply_dev(rope.view, H(x), H(x), at, 3, 32, 0, None) == qx.INVALID_ARGUMENT
    assert qx.lib.qx_kv_attention(cache.view, batch.view, H(q), H(q), odd, 1.0, 1, 0) == qx.INVALID_ARGUMENT
    assert qx.lib.qx_kv_attention_dev(cache.view, batch.view, H(q), H(q), odd, 1.0, 1, 0, None, None) == qx.INVALID_ARGUMENT


def test_an_output_that_begins_where_the_queries_do_is_the_same_view(qx, parts):
    cache, batch, x, q = parts
    H = qx.heads_view
    call = lambda b: qx.lib.qx_kv_attention(cache.view, batch.view, H(q), b, None, 1.0, 1, 0)  # noqa: E731
    assert served(qx, call(H(q)))
    assert call(H(q, kind=qx.BF16)) == qx.INVALID_ARGUMENT
    assert call(H(q, token_stride=2 * q.shape[1] * q.shape[2])) == qx.INVALID_ARGUMENT


def test_arrays_of_another_element_type_are_refused(qx, parts):
    """The library sees addresses only; the Python calls look at what lies there."""
    cache, batch, x, q = parts
    lengths, table, begin = batch.arrays
    for wrong in ((lengths.astype(np.int64), table, begin), (lengths, table.astype(np.int64), begin),
                  (lengths, table, begin.astype(np.uint32))):
        with pytest.raises(AssertionError):
            qx.KVBatch(wrong[0], wrong[1], 32, wrong[2], 3, 2)
    k_codes, v_codes, k_scales, v_scales = cache.arrays
    for wrong in ((k_codes.view(np.uint8), v_codes, k_scales, v_scales), (k_codes, v_codes, k_scales, v_scales.astype(np.float64)),
                  (k_codes, v_codes[:2], k_scales, v_scales), (k_codes, v_codes, k_scales, v_scales[:, :1])):
        with pytest.raises(AssertionError):
            qx.KVCache(*wrong)
    rope, at = qx.Rope(32), np.arange(3, dtype=np.int32)
    with pytest.raises(AssertionError):
        rope.apply(x, x, at)
    with pytest.raises(AssertionError):
        cache.append(batch, x, x, rope, positions=at)
    with pytest.raises(AssertionError):
        cache.attention(batch, q, q, lse=np.zeros((3, q.shape[1])))


def test_arrays_in_another_place_are_refused(qx, parts, monkeypatch):
    """Host arrays never reach a `_dev` call, nor tensors of another device: the kernel would follow their addresses."""
    cache, batch, x, q = parts
    at = np.arange(3)
    monkeypatch.setattr(qx, "_device", lambda: 0)
    for call in (lambda: qx.Rope(32).apply_dev(x, x, at), lambda: cache.append_dev(batch, x, x),
                 lambda: cache.read_dev(batch, x, x), lambda: cache.attention_dev(batch, q, q)):
        with pytest.raises(AssertionError):
            call()
    elsewhere = qx.KVBatch(*batch.arrays[:2], 32, batch.arrays[2], 3, 2)
    elsewhere.device = 1  # (as if its tensors lay there)
    for call in (lambda: cache.append(elsewhere, x, x), lambda: cache.read(elsewhere, x, x),
                 lambda: cache.attention(elsewhere, q, q)):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(AssertionError):
        qx.heads_view(torch.zeros(3, 2, 32), device=0)  # (a tensor of the host)
    with pytest.raises(AssertionError):
        qx.KVBatch(batch.arrays[0], torch.from_numpy(batch.arrays[1]), 32, batch.arrays[2], 3, 2)
