"""Norms, gate and residual sum between two blocks against the 64-bit formula: every type, widths from one element to
the most, norms of both kinds on either side, strides and alignments, broadcast gates, in place, host buffers."""

import numpy as np
import pytest
import torch

from kv_reference import HALF_STEP

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24  # half a step of f32, relative


def normed(v, kind, weight, bias, eps, offset):
    """-> the norm of rows in 64 bits, and the size of the terms of its last sum."""
    if kind:
        v = v - v.mean(1, keepdim=True)
    v = v / (v.square().mean(1, keepdim=True) + eps).sqrt()
    v = v if weight is None else v * (weight.double() + offset)
    return (v, v.abs()) if bias is None else (v + bias.double(), v.abs() + bias.double().abs())


def depth(dim):
    """Roundings that an element of a row's sum passes through: 8 in its vector, 8 vectors, 10 of the threads."""
    return 26


def check(residual, block, joined, out, pre=None, post=None, gate=None, scale=1.0):
    """`pre`, `post`: (kind, weight, bias, eps, offset). The limits count the roundings of f32 arithmetic, u each.

    A norm: sums of n positive terms are off by depth(n) u relative, the root by half of that; with the division, the
    root, the mean's and eps's sum 6 u more; the products 3 u and the weight's offset 1 u. A layer norm takes a mean that
    is off by depth u of the row's mean magnitude m: that moves v by as much, and the norm by as much over its deviation.
    The norm in front sees joined with its own error e: that moves it by e / deviation, and its statistics by as much
    relative again, which the same bound counts for an element of the size of the row's largest."""
    residual, block, gate = (None if t is None else t.cpu().double() for t in (residual, block, gate))
    u, e, dim = None, 0.0, (residual if block is None else block).shape[1]

    def apply(v, e, norm):
        kind, weight, bias, eps, offset = norm
        y, size = normed(v, kind, None if weight is None else weight.cpu(), None if bias is None else bias.cpu(), eps, offset)
        centred = v - v.mean(1, keepdim=True) if kind else v
        inverse = 1 / (centred.square().mean(1, keepdim=True) + eps).sqrt()
        moved = e + (depth(dim) * U * v.abs().mean(1, keepdim=True) + 2 * U * v.abs() if kind else 0.0)
        factor = 1.0 if weight is None else (weight.cpu().double() + offset).abs()
        relative = (depth(dim) / 2 + 12) * U
        # the statistics' own change: the root mean square of the elements' changes over that of the elements
        spread = (moved * torch.ones_like(v)).square().mean(1, keepdim=True).sqrt() * inverse
        return y, size * (relative + spread) + moved * inverse * factor

    if block is not None:
        u = block
        if post is not None:
            u, e = apply(u, 0.0, post)
        if gate is not None:
            u, e = u * gate, e * gate.abs() + U * (u * gate).abs()
        u, e = scale * u, abs(scale) * e + 2 * U * (scale * u).abs()
    total = residual if u is None else u if residual is None else residual + u
    e = e + 2 * U * total.abs()
    if joined is not None:
        off = (joined.cpu().double() - total).abs() - (HALF_STEP[joined.dtype] * total.abs() + e + least(joined.dtype))
        assert float(off.max()) <= 0, f"joined {float(off.max())}"
    if out is not None:
        y, e = apply(total, e, pre)
        off = (out.cpu().double() - y).abs() - (HALF_STEP[out.dtype] * (y.abs() + e) + e + least(out.dtype))
        assert float(off.max()) <= 0, f"normed {float(off.max())}"


def least(dtype):
    """Half of the smallest step of a type, where its values run out of exponents."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134


def operands(tokens, dim, dtype, stream=None, seed=1):
    gen = torch.Generator().manual_seed(seed)
    loud = torch.where(torch.rand(dim, generator=gen) < 0.02, 30.0, 1.0)
    residual = (torch.randn(tokens, dim, generator=gen) * loud + 0.3).to(stream or dtype).cuda()
    block = torch.randn(tokens, dim, generator=gen).to(dtype).cuda()
    weight, bias, gate = ((torch.randn(n, dim, generator=gen) * 0.3 + m).to(dtype).cuda() for n, m in ((1, 1), (1, 0), (tokens, 0.5)))
    return residual, block, weight[0], bias[0], gate


def like(t, dtype=None):
    return torch.full(t.shape, float("nan"), dtype=dtype or t.dtype, device="cuda")


def norms(qx, *specs):
    return [None if s is None else qx.Norm(s[1], s[2], s[0], s[3], s[4]) for s in specs]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("tokens,dim", [(1, 1), (3, 2), (2, 7), (5, 8), (1, 31), (9, 64), (4, 257), (33, 256), (3, 1000), (2, 1153),
                                        (2, 4096), (3, 4104), (1, 8193), (2, 16384), (2, 20001), (1, 32768)])
def test_against_the_formula(qx, dtype, kind, tokens, dim):
    residual, block, weight, bias, gate = operands(tokens, dim, dtype)
    joined, out = like(residual), like(block)
    pre, post = (kind, weight, bias, 1e-6, 0.0), (kind, bias, None, 1e-5, 1.0)
    a, b = norms(qx, pre, post)
    qx.check(qx.residual_norm_dev(residual, block, joined, out, a, b, gate, 0.7), "residual norm")
    check(residual, block, joined, out, pre, post, gate, 0.7)
    # without what may be left out
    joined, out = like(residual), like(block)
    qx.check(qx.residual_norm_dev(residual, block, joined, out, a), "residual norm")
    check(residual, block, joined, out, pre)
    plain = (kind, None, None, 1e-6, 0.0)
    out = like(block)
    qx.check(qx.residual_norm_dev(residual, None, None, out, *norms(qx, plain)), "residual norm")
    check(residual, None, None, out, plain)
    joined = like(residual)
    qx.check(qx.residual_norm_dev(None, block, joined, None, None, b, gate, -2.0), "residual norm")
    check(None, block, joined, None, None, post, gate, -2.0)


@pytest.mark.parametrize("stream", TYPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out_type", TYPES)
def test_types_beside_each_other(qx, stream, dtype, out_type):
    residual, block, weight, bias, gate = operands(6, 520, dtype, stream)
    joined, out = like(residual), like(block, out_type)
    pre = (0, weight.float(), bias.float(), 1e-6, 0.0)
    post = (1, weight.half(), None, 1e-6, 0.0)
    qx.check(qx.residual_norm_dev(residual, block, joined, out, *norms(qx, pre, post), gate.float()), "residual norm")
    check(residual, block, joined, out, pre, post, gate.float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,width", [(0, 96), (1, 96), (3, 99), (8, 104), (4, 100)])
def test_strides_and_alignment(qx, dtype, offset, width):
    """Rows inside wider ones, data that starts off a 16-byte boundary, one row for all tokens; what lies between rows stays."""
    tokens, dim = 7, 96
    residual, block, weight, bias, gate = operands(tokens, dim, dtype)
    stores = [torch.full((tokens * width + offset + 8,), 5.0, dtype=dtype, device="cuda") for _ in range(4)]
    r, b, joined, out = (s.as_strided((tokens, dim), (width, 1), offset) for s in stores)
    r.copy_(residual)
    b.copy_(block)
    w = torch.cat([bias[:offset], weight])[offset:]
    pre, post = (0, w, None, 1e-6, 0.0), (1, weight, bias, 1e-6, 0.0)
    qx.check(qx.residual_norm_dev(r, b, joined, out, *norms(qx, pre, post), gate[:1]), "residual norm")
    check(residual, block, joined, out, pre, post, gate[:1])
    for s, view in zip(stores[2:], (joined, out)):
        view.fill_(5.0)
        assert bool((s == 5.0).all())
    one = residual[:1].expand(tokens, dim)
    qx.check(qx.residual_norm_dev(one, b, joined, out, *norms(qx, pre)), "residual norm")
    check(one, block, joined, out, pre)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [100, 4096, 20000])
def test_in_place(qx, dtype, dim):
    """joined over the residual, normed over the block's output, and the other way round: the same bits."""
    residual, block, weight, bias, gate = operands(5, dim, dtype)
    pre, post = norms(qx, (0, weight, bias, 1e-6, 0.0), (0, weight, None, 1e-6, 0.0))
    joined, out = like(residual), like(block)
    qx.check(qx.residual_norm_dev(residual, block, joined, out, pre, post, gate), "residual norm")
    for swap in (False, True):
        r, b = residual.clone(), block.clone()
        qx.check(qx.residual_norm_dev(r, b, b if swap else r, r if swap else b, pre, post, gate), "residual norm")
        assert torch.equal(b if swap else r, joined) and torch.equal(r if swap else b, out)
    r, g = residual.clone(), gate.clone()
    qx.check(qx.residual_norm_dev(r, block, r, g, pre, post, g), "residual norm")
    assert torch.equal(r, joined) and torch.equal(g, out)


@pytest.mark.parametrize("dim", [48, 1024, 5120])
def test_a_row_has_the_same_bits_in_every_batch(qx, dim):
    residual, block, weight, bias, gate = operands(300, dim, torch.bfloat16, torch.float32)
    pre, post = norms(qx, (1, weight, bias, 1e-6, 0.0), (0, weight, None, 1e-6, 0.0))
    joined, out = like(residual), like(block)
    qx.check(qx.residual_norm_dev(residual, block, joined, out, pre, post, gate), "residual norm")
    for t in (0, 7, 299):
        j, o = like(residual[:1]), like(block[:1])
        qx.check(qx.residual_norm_dev(residual[t:t + 1], block[t:t + 1], j, o, pre, post, gate[t:t + 1]), "residual norm")
        assert torch.equal(j[0], joined[t]) and torch.equal(o[0], out[t])


def test_rows_of_zeros_infinities_and_nan(qx):
    """Zeros give zeros (eps keeps them) or, with eps 0, NaN as the formula does; what is no number stays in its row."""
    residual = torch.zeros(5, 64, device="cuda")
    residual[1] = torch.linspace(1, 2, 64)
    residual[2, 3] = float("inf")
    residual[3, 3] = float("nan")
    out = like(residual)
    qx.check(qx.residual_norm_dev(residual, None, None, out, qx.Norm(eps=1e-6)), "residual norm")
    assert bool((out[0] == 0).all()) and bool(out[1].isfinite().all()) and bool((out[4] == 0).all())
    assert bool(out[2, 3].isnan()) and bool((out[2, :3] == 0).all()) and bool(out[3].isnan().all())
    qx.check(qx.residual_norm_dev(residual, None, None, out, qx.Norm(eps=0.0)), "residual norm")
    assert bool(out[0].isnan().all()) and bool(out[1].isfinite().all())
    # a constant row is its mean: nothing but the bias is left of it
    residual[:] = 3.0
    bias = torch.linspace(-1, 1, 64, device="cuda")
    qx.check(qx.residual_norm_dev(residual, None, None, out, qx.Norm(None, bias, qx.NORM_LAYER)), "residual norm")
    assert torch.equal(out, bias.expand(5, 64))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_host_buffers(qx, dtype):
    residual, block, weight, bias, gate = operands(6, 90, dtype)
    pre, post = (0, weight, bias, 1e-6, 0.0), (1, weight, None, 1e-6, 0.5)
    joined, out = like(residual), like(block)
    qx.check(qx.residual_norm_dev(residual, block, joined, out, *norms(qx, pre, post), gate), "residual norm")
    r, b, w, c, g = (t.cpu().numpy() for t in (residual, block, weight, bias, gate))
    a, z = qx.Norm(w, c, 0, 1e-6), qx.Norm(w, None, 1, 1e-6, 0.5)
    store = np.full((6, 2, 95), 7, r.dtype)  # the two outputs in each other's gaps
    qx.check(qx.residual_norm(r, b, store[:, 0, :90], store[:, 1, :90], a, z, g), "residual norm")
    assert np.array_equal(store[:, 0, :90], joined.cpu().numpy()) and np.array_equal(store[:, 1, :90], out.cpu().numpy())
    assert bool((store[:, :, 90:] == 7).all())
    qx.check(qx.residual_norm(r, b, r, b, a, z, g), "residual norm")  # in place
    assert np.array_equal(r, joined.cpu().numpy()) and np.array_equal(b, out.cpu().numpy())


def test_streams_and_graphs(qx):
    residual, block, weight, bias, gate = operands(40, 2048, torch.bfloat16)
    pre = qx.Norm(weight)
    joined, out, want = like(residual), like(block), [like(residual), like(block)]
    qx.check(qx.residual_norm_dev(residual, block, *want, pre), "residual norm")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        qx.check(qx.residual_norm_dev(residual, block, joined, out, pre), "residual norm")
    side.synchronize()
    assert torch.equal(joined, want[0]) and torch.equal(out, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qx.check(qx.residual_norm_dev(residual, block, joined, out, pre), "residual norm")
        qx.check(qx.residual_norm_dev(joined, out, joined, out, pre), "residual norm")
    qx.check(qx.residual_norm_dev(*want, *want, pre), "residual norm")
    for _ in range(2):
        joined.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(joined, want[0]) and torch.equal(out, want[1])


def test_past_two_gigabytes(qx):
    """Rows whose offsets pass 32 bits."""
    tokens, dim = 3, 64
    far = (1 << 31) // 2 + 8  # elements between rows
    store = torch.zeros(2 * far + dim, dtype=torch.float16, device="cuda")
    view = store.as_strided((tokens, dim), (far, 1))
    residual, block, weight, bias, gate = operands(tokens, dim, torch.float16)
    view.copy_(residual)
    out, spec = like(block), (0, weight, None, 1e-6, 0.0)
    qx.check(qx.residual_norm_dev(view, block, view, out, *norms(qx, spec)), "residual norm")
    check(residual, block, view, out, spec)
