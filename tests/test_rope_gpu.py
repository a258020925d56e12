"""Rotary positions against the 64-bit formula: layouts, partly rotated heads, head sizes and rotary parts of
every kind, strides and alignments, far positions, in place, the gradient, host buffers."""

import numpy as np
import pytest
import torch

from kv_reference import HALF_STEP, rotated

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def tolerance(y, x, amplitude, dtype):
    """Half a step of the type, and for the f32 arithmetic: {cos, sin} within 6 ulp of 1 (half a turn rounded to
    f32, two ulps of the functions, the amplitude's product) and three roundings, u = 2^-24 each, on products of
    no more than |a| + |b| <= 2 max |x|."""
    return HALF_STEP[dtype] * y.abs() + 12 * 2.0 ** -24 * 2 * x.abs().amax() * amplitude


def close(got, want, x, amplitude=1.0):
    limit = tolerance(want, x, amplitude, got.dtype)
    off = (got.cpu().double() - want).abs() - limit
    assert float(off.max()) <= 0, float(off.max())


def inputs(tokens, heads, dim, dtype, far=1 << 20, seed=1):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=gen).to(dtype)
    return x, torch.randint(0, far, (tokens,), generator=gen)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,heads,dim,rotary", [(1, 1, 16, 16), (3, 5, 64, 64), (7, 3, 128, 64), (2, 40, 128, 128),
                                                     (5, 2, 80, 32), (33, 2, 96, 96), (2, 3, 256, 256), (4, 3, 40, 20),
                                                     (3, 2, 7, 2), (2, 2, 66, 50), (9, 1, 33, 32)])
def test_against_the_formula(qx, dtype, interleaved, tokens, heads, dim, rotary):
    rope = qx.Rope(rotary, interleaved, 500000.0, dict(kind=qx.ROPE_RAMP, factor=8.0, trained=4096, slow=1, fast=32))
    x, at = inputs(tokens, heads, dim, dtype)
    y = torch.full((tokens, heads, dim), float("nan"), dtype=dtype, device="cuda")
    qx.check(rope.apply_dev(x.cuda(), y, at.cuda()), "rope")
    want = rotated(x.double(), at.tolist(), rope.view.frequency[:rotary // 2], rope.view.amplitude, interleaved)
    close(y, want, x, rope.view.amplitude)
    assert torch.equal(y[..., rotary:].cpu(), x[..., rotary:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rotary", [(64, 32), (64, 64), (36, 12)])
def test_in_place_in_a_packed_projection(qx, dtype, dim, rotary):
    rope = qx.Rope(rotary)
    x, at = inputs(50, 12, dim, dtype)
    packed = x.cuda()
    qx.check(rope.apply_dev(packed[:, :9], packed[:, :9], at.cuda()), "rope")
    close(packed[:, :9], rotated(x[:, :9].double(), at.tolist(), rope.view.frequency[:rotary // 2]), x)
    assert torch.equal(packed[:, 9:].cpu(), x[:, 9:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 3, 8])
def test_strides_and_alignment(qx, dtype, offset):
    """Heads outside tokens, rows of odd lengths, data that starts off a 16-byte boundary, broadcast inputs."""
    rope, (tokens, heads, dim) = qx.Rope(32), (11, 3, 48)
    x, at = inputs(tokens, heads, dim, dtype)
    store = torch.zeros(heads * tokens * 51 + 64, dtype=dtype, device="cuda")
    view = store[offset:].as_strided((tokens, heads, dim), (51, tokens * 51, 1), offset)
    view.copy_(x)
    y = torch.zeros(tokens, heads, dim + 5, dtype=dtype, device="cuda")[..., :dim]
    qx.check(rope.apply_dev(view, y, at.cuda()), "rope")
    close(y, rotated(x.double(), at.tolist(), rope.view.frequency[:16]), x)
    one = x[:1, :1].cuda().expand(tokens, heads, dim)
    qx.check(rope.apply_dev(one, y, at.cuda()), "rope")
    close(y, rotated(x[:1, :1].double().expand(tokens, heads, dim), at.tolist(), rope.view.frequency[:16]), x)


def test_far_positions(qx):
    """The angle of position 2^31 - 1 is as exact as that of position 0, and negative ones turn the other way."""
    rope = qx.Rope(64, base=10000.0)
    x, _ = inputs(6, 2, 64, torch.float32)
    at = torch.tensor([0, 1, -5, 1 << 24, (1 << 24) + 1, (1 << 31) - 1])
    y = torch.empty(6, 2, 64, device="cuda")
    qx.check(rope.apply_dev(x.cuda(), y, at.cuda()), "rope")
    close(y, rotated(x.double(), at.tolist(), rope.view.frequency[:32]), x)


@pytest.mark.parametrize("interleaved", [0, 1])
def test_gradient(qx, interleaved):
    """`inverse` gives dL/dx of dL/dy: against the transposed formula, against differences of the kernel itself
    (the map is linear: a unit step in x changes L by the gradient), and as the way back."""
    rope = qx.Rope(32, interleaved, 10000.0, dict(kind=qx.ROPE_RAMP, factor=4.0, trained=64, slow=1, fast=8))
    x, at = inputs(5, 3, 40, torch.float32, far=1000)
    up, _ = inputs(5, 3, 40, torch.float32, seed=2)
    at_dev, f, amplitude = at.cuda(), rope.view.frequency[:16], rope.view.amplitude
    grad, y, moved, back = (torch.empty(5, 3, 40, device="cuda") for _ in range(4))
    qx.check(rope.apply_dev(up.cuda(), grad, at_dev, inverse=True), "rope")
    close(grad, rotated(up.double(), at.tolist(), f, amplitude, interleaved, inverse=True), up, amplitude)
    qx.check(rope.apply_dev(x.cuda(), y, at_dev), "rope")
    for d in (0, 1, 15, 16, 31, 39):
        step = x.clone()
        step[:, :, d] += 1
        qx.check(rope.apply_dev(step.cuda(), moved, at_dev), "rope")
        change = ((moved.double() - y.double()).cpu() * up.double()).sum(-1)
        # each of the 40 elements of both passes is off by the tolerance above at most
        limit = 2 * 40 * 12 * 2.0 ** -24 * 2 * (x.abs().amax() + 1) * amplitude * up.abs().amax() + 2.0 ** -23 * 8
        assert float((change - grad[:, :, d].double().cpu()).abs().max()) <= limit
    qx.check(rope.apply_dev(y, back, at_dev, inverse=True), "rope")
    scale = torch.ones(40, dtype=torch.float64)
    scale[:32] = amplitude ** 2
    assert float((back.double().cpu() - x.double() * scale).abs().max()) <= 60 * 2.0 ** -24 * 4 * float(x.abs().amax()) * amplitude ** 2


@pytest.mark.parametrize("tokens", [1, 5000])
def test_many_tokens_and_heads(qx, tokens):
    """Every row of a long call has the bits of a call of its own (angles are per token)."""
    rope, (x, at) = qx.Rope(128), inputs(tokens, 24, 128, torch.bfloat16)
    x, at = x.cuda(), at.cuda()
    y, one = torch.empty_like(x), torch.empty_like(x[:1])
    qx.check(rope.apply_dev(x, y, at), "rope")
    for t in {0, tokens // 2, tokens - 1}:
        qx.check(rope.apply_dev(x[t:t + 1], one, at[t:t + 1]), "rope")
        assert torch.equal(one[0], y[t])


def test_nothing_to_rotate(qx):
    empty = torch.empty(0, 2, 32, device="cuda")
    assert qx.Rope(32).apply_dev(empty, empty, torch.empty(0, dtype=torch.int64, device="cuda")) == qx.OK


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_host_buffers(qx, dtype, in_place):
    rope, (x, at) = qx.Rope(64), inputs(9, 4, 96, dtype)
    kind = qx.F32 if dtype == torch.float32 else qx.BF16
    raw = x.numpy().copy() if dtype == torch.float32 else x.view(torch.int16).numpy().view(np.uint16).copy()
    out = raw if in_place else np.zeros_like(raw)
    assert rope.apply(raw[:, 1:3], out[:, 1:3], at.numpy(), kind=kind) == qx.OK, qx.last_error()
    got = torch.from_numpy(out.view(np.int16) if dtype != torch.float32 else out).view(dtype)
    close(got[:, 1:3], rotated(x[:, 1:3].double(), at.tolist(), rope.view.frequency[:32]), x)
    rest = x if in_place else torch.zeros_like(x)
    assert torch.equal(got[:, 0], rest[:, 0]) and torch.equal(got[:, 3], rest[:, 3])
