"""Mixture-of-experts layers against the 64-bit formula: formats, types, widths, counts of tokens and experts, routers of
every kind, strides, in place, host buffers, streams, graphs, workspaces; what is no number stays in its row."""

import ctypes as C
import threading

import numpy as np
import pytest
import torch

import moe_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def prepared(qx, m, host=False):
    experts = qx.Experts()
    if host:
        status = experts.prepare(m.fmt, *m.raw, m.experts, m.dim, m.inner, m.shared)
    else:
        status = experts.prepare_dev(m.fmt, *(torch.from_numpy(r).cuda() for r in m.raw), m.experts, m.dim, m.inner, m.shared)
    qx.check(status, "prepare")
    return experts


def router(qx, m, top, sigmoid=False, biased=False, normalise=True, scale=1.0):
    return qx.Router(m.router.cuda(), top, qx.SCORE_SIGMOID if sigmoid else qx.SCORE_SOFTMAX, m.bias.cuda() if biased else None,
                     normalise, scale)


def tokens_of(m, tokens, dtype, seed=5):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(tokens, m.dim, generator=gen).to(dtype)


def check(qx, m, x, top, out_type=None, experts=None, activation=3, **kind):
    out_type = out_type or x.dtype
    experts = experts or prepared(qx, m)
    out = torch.full(x.shape, float("nan"), dtype=out_type, device="cuda")
    chosen = torch.full((len(x), top), -1, dtype=torch.int32, device="cuda")
    weights = torch.full((len(x), top), float("nan"), device="cuda")
    qx.check(experts.apply_dev(router(qx, m, top, **kind), x.cuda(), out, activation, chosen, weights), "apply")
    torch.cuda.synchronize()
    qx.check(qx.lib.qx_check_device_errors(), "apply")
    picks = chosen.cpu().long()
    _, shares, shares_off = ref.route(m, x, top, chosen=picks, **kind)
    assert bool(((weights.cpu().double() - shares).abs() <= shares_off).all())
    want, limit = ref.apply(m, x, top, activation, out_type=out_type, chosen=picks, **kind)
    off = (out.cpu().double() - want).abs() - limit
    assert float(off.max()) <= 0, float(off.max())
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("tokens,experts,top,dim,inner", [(1, 1, 1, 32, 32), (1, 4, 2, 64, 96), (2, 8, 8, 96, 64), (5, 16, 3, 288, 160),
                                                          (7, 5, 2, 1120, 224), (33, 8, 2, 256, 288), (64, 20, 4, 160, 128),
                                                          (3, 130, 6, 128, 64), (130, 6, 2, 96, 96), (1, 512, 32, 64, 32)])
def test_against_the_formula(qx, dtype, fmt, tokens, experts, top, dim, inner):
    m = ref.layer(fmt, experts, dim, inner, seed=tokens)
    check(qx, m, tokens_of(m, tokens, dtype), top)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("shared", [0, 1, 3])
def test_routers(qx, sigmoid, biased, normalise, shared):
    m = ref.layer(1, 24, 256, 96, shared, seed=3, router=torch.bfloat16)
    check(qx, m, tokens_of(m, 11, torch.bfloat16), 5, sigmoid=sigmoid, biased=biased, normalise=normalise, scale=2.5)


@pytest.mark.parametrize("activation", range(5))
def test_activations(qx, activation):
    m = ref.layer(0, 6, 128, 64, 1, seed=4)
    check(qx, m, tokens_of(m, 9, torch.float32) * 2, 2, activation=activation)


@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("out_type", TYPES)
@pytest.mark.parametrize("router_type", TYPES)
def test_types_beside_each_other(qx, x_type, out_type, router_type):
    m = ref.layer(1, 12, 192, 96, seed=6, router=router_type)
    check(qx, m, tokens_of(m, 10, x_type), 3, out_type)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_token_on_one_expert(qx, dtype):
    """More tokens of an expert than a unit of work takes, and experts that have none."""
    m = ref.layer(0, 9, 160, 96, seed=7)
    x = tokens_of(m, 70, dtype).abs()
    m.router[:] = -m.router.abs()
    m.router[4] = m.router[4].abs()
    m.router[6] = m.router[6].abs() / 2
    check(qx, m, x, 2)


def test_equal_scores_go_to_the_lower_expert(qx):
    m = ref.layer(0, 40, 64, 32, seed=8)
    m.router[:] = 0
    m.router[7] = m.router[33] = m.router[39] = 1.0
    x = torch.ones(3, 64)
    chosen = torch.empty(3, 5, dtype=torch.int32, device="cuda")
    out = torch.empty(3, 64, device="cuda")
    qx.check(prepared(qx, m).apply_dev(router(qx, m, 5), x.cuda(), out, chosen=chosen), "apply")
    assert chosen.cpu().tolist() == [[7, 33, 39, 0, 1]] * 3


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", [0, 1])
def test_a_token_has_the_same_bits_beside_any_others(qx, dtype, fmt):
    m = ref.layer(fmt, 10, 320, 128, 1, seed=9)
    x, experts = tokens_of(m, 150, dtype), prepared(qx, m)
    out = check(qx, m, x, 3, experts=experts)
    for t in (0, 5, 127, 128, 149):
        one = torch.empty(1, m.dim, dtype=dtype, device="cuda")
        qx.check(experts.apply_dev(router(qx, m, 3), x[t:t + 1].cuda(), one), "apply")
        assert torch.equal(one[0], out[t])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,width", [(0, 128), (1, 96), (3, 99), (8, 104)])
def test_strides_and_alignment(qx, dtype, offset, width):
    m = ref.layer(1, 7, 96, 64, seed=10)
    x, experts = tokens_of(m, 12, dtype), prepared(qx, m)
    want = check(qx, m, x, 2, experts=experts)
    stores = [torch.full((12 * width + offset,), 7.0, dtype=dtype, device="cuda") for _ in "xy"]
    view, out = (s.as_strided((12, 96), (width, 1), offset) for s in stores)
    view.copy_(x)
    weights = torch.zeros(7 * 96 + 1, device="cuda")[1:].view(7, 96).copy_(m.router)  # off a 16-byte boundary
    qx.check(experts.apply_dev(qx.Router(weights, 2), view, out), "apply")
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert bool((stores[1] == 7.0).all())
    one = x[:1].cuda().expand(12, 96)  # the same token again and again
    qx.check(experts.apply_dev(qx.Router(weights, 2), one, out), "apply")
    assert torch.equal(out, want[:1].expand(12, 96))
    qx.check(experts.apply_dev(qx.Router(weights, 2), view, view), "apply")  # in place
    assert torch.equal(view, want)


def test_what_is_no_number_stays_in_its_row(qx):
    m = ref.layer(1, 6, 96, 64, 1, seed=11)
    x, experts, r = tokens_of(m, 6, torch.float32).cuda(), prepared(qx, m), router(qx, m, 2)
    want, out = torch.empty_like(x), torch.empty_like(x)
    qx.check(experts.apply_dev(r, x, want), "apply")
    bad = x.clone()
    bad[1, 5], bad[3, 70] = float("nan"), float("inf")
    qx.check(experts.apply_dev(r, bad, out), "apply")
    torch.cuda.synchronize()
    qx.check(qx.lib.qx_check_device_errors(), "apply")
    assert bool(out[1].isnan().all()) and not bool(out[3].isfinite().any())
    for t in (0, 2, 4, 5):
        assert torch.equal(out[t], want[t])


@pytest.mark.parametrize("size", [2.0 ** -30, 2.0 ** -20, 2.0 ** 40])
def test_small_and_large_activations(qx, size):
    """A bilinear layer (no activation) of x times a power of two is the square of that times the layer: to the last bit in f32."""
    m = ref.layer(0, 4, 128, 96, seed=12)
    x, experts, r = tokens_of(m, 5, torch.float32).cuda(), prepared(qx, m), qx.Router(torch.zeros(4, 128, device="cuda"), 4)
    want, out = torch.empty_like(x), torch.empty_like(x)
    qx.check(experts.apply_dev(r, x, want, qx.ACT_NONE), "apply")
    qx.check(experts.apply_dev(r, x * size, out, qx.ACT_NONE), "apply")
    assert torch.equal(out, want * size * size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_host_buffers(qx, dtype):
    m = ref.layer(1, 9, 128, 64, 1, seed=13)
    x = tokens_of(m, 8, dtype)
    want = check(qx, m, x, 3, biased=True).cpu().numpy()
    experts = prepared(qx, m, host=True)
    a, store = x.numpy(), np.full((8, 140), 3, x.numpy().dtype)
    chosen, weights = np.zeros((8, 3), np.int32), np.zeros((8, 3), np.float32)
    r = qx.Router(m.router.numpy(), 3, bias=m.bias.numpy())
    qx.check(experts.apply(r, a, store[:, :128], chosen=chosen, weights=weights), "apply")
    assert np.array_equal(store[:, :128], want) and bool((store[:, 128:] == 3).all())
    ref.route(m, x, 3, biased=True, chosen=torch.from_numpy(chosen).long())
    qx.check(experts.apply(r, a, a), "apply")
    assert np.array_equal(a, want)


def workspace(qx, size=1 << 24):
    handle = C.c_void_p()
    qx.check(qx.lib.qx_workspace_create(size, C.byref(handle)), "workspace")
    return handle


def test_two_streams_with_a_workspace_each(qx):
    """Calls that run at the same time, each with all of the card's thread blocks."""
    m = ref.layer(1, 16, 1024, 512, seed=14)
    experts, r = prepared(qx, m), router(qx, m, 4)
    xs = [tokens_of(m, n, torch.bfloat16, n).cuda() for n in (40, 7)]
    want = [torch.empty_like(x) for x in xs]
    for x, w in zip(xs, want):
        qx.check(experts.apply_dev(r, x, w), "apply")
    torch.cuda.synchronize()
    streams, spaces = [torch.cuda.Stream() for _ in xs], [workspace(qx) for _ in xs]
    outs = [[torch.empty_like(x) for _ in range(20)] for x in xs]
    for i in range(20):
        for x, out, stream, space in zip(xs, outs, streams, spaces):
            with torch.cuda.stream(stream):
                qx.check(experts.apply_dev(r, x, out[i], workspace=space), "apply")
    torch.cuda.synchronize()
    qx.check(qx.lib.qx_check_device_errors(), "apply")
    for out, w in zip(outs, want):
        assert all(torch.equal(o, w) for o in out)
    for space in spaces:
        qx.lib.qx_workspace_destroy(space)


def test_captured_and_replayed_with_other_inputs(qx):
    m = ref.layer(0, 12, 256, 128, 1, seed=15)
    experts, r, space = prepared(qx, m), router(qx, m, 3), workspace(qx)
    x, out = tokens_of(m, 20, torch.float16).cuda(), torch.empty(20, 256, dtype=torch.float16, device="cuda")
    qx.check(experts.apply_dev(r, x, out, workspace=space), "apply")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qx.check(experts.apply_dev(r, x, out, workspace=space), "apply")
        qx.check(experts.apply_dev(r, out, out, workspace=space), "apply")
    for seed in (1, 2):
        new = tokens_of(m, 20, torch.float16, seed)
        x.copy_(new)
        graph.replay()
        once = torch.empty_like(out)
        torch.cuda.synchronize()
        qx.check(experts.apply_dev(r, new.cuda(), once), "apply")
        qx.check(experts.apply_dev(r, once, once), "apply")
        assert torch.equal(out, once)
    qx.check(qx.lib.qx_check_device_errors(), "apply")
    qx.lib.qx_workspace_destroy(space)


def test_prepared_from_the_host_and_from_the_device_are_the_same(qx):
    for fmt in (0, 1):
        m = ref.layer(fmt, 3, 96, 160, 1, seed=16)
        x = tokens_of(m, 4, torch.float32).cuda()
        outs = []
        for host in (False, True):
            outs.append(torch.empty_like(x))
            qx.check(prepared(qx, m, host).apply_dev(router(qx, m, 2), x, outs[-1]), "apply")
        assert torch.equal(*outs)


def test_codes_of_every_value(qx):
    """Blocks that hold each code that the formats have (-128 among them), against exact sums."""
    for fmt, codes in ((0, 256), (1, 16)):
        m = ref.layer(fmt, 1, 256, 256, seed=17)
        blocks = [r.reshape(-1, qx.BLOCK_BYTES[fmt]).copy() for r in m.raw]
        for b, name in zip(blocks, ("gate", "up", "down")):
            order = (np.arange(b.shape[0] * 32) * 37 + 11) % codes
            raw = order.reshape(-1, 32).astype(np.uint8)
            d = b[:, :2].copy().view(np.float16).astype(np.float64)
            if fmt == 0:
                b[:, 2:], values = raw, raw.view(np.int8).astype(np.float64)
            else:
                b[:, 2:], values = raw[:, :16] | raw[:, 16:] << 4, raw.astype(np.float64) - 8
            setattr(m, name, torch.from_numpy((values * d).reshape(1, 256, 256)))
        m.raw = tuple(b.reshape(-1) for b in blocks)
        check(qx, m, tokens_of(m, 3, torch.float32), 1)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_scores_far_below_their_bias(qx, sigmoid):
    """Experts that are chosen for a large bias, with scores down to 1e-20: their weights are those of the scores."""
    m = ref.layer(0, 12, 64, 32, seed=31)
    m.router = m.router * 12
    m.bias = torch.linspace(-40, 50, 12)
    for normalise in (False, True):
        check(qx, m, tokens_of(m, 9, torch.float32), 4, sigmoid=sigmoid, biased=True, normalise=normalise)


def test_scores_that_all_lie_far_below_zero(qx):
    """sigmoid(l) of about e^-150 runs out of f32; normalised weights are quotients of such."""
    m = ref.layer(1, 6, 64, 32, seed=32)
    x = tokens_of(m, 5, torch.float32)
    x[:, 0] = 8.0
    m.router[:, 0] = -20.0
    assert float((x.double() @ m.router.double().T).max()) < -140
    check(qx, m, x, 3, sigmoid=True)


@pytest.mark.parametrize("fmt,experts,dim,inner,shared,top,tokens", [(0, 512, 64, 32, 32, 32, 70), (1, 2, 65536, 32, 0, 1, 2), (0, 2, 32, 65536, 0, 1, 3)])
def test_the_largest_layers(qx, fmt, experts, dim, inner, shared, top, tokens):
    """As many experts, chosen and shared ones, and as wide rows as there may be."""
    m = ref.layer(fmt, experts, dim, inner, shared, seed=33)
    check(qx, m, tokens_of(m, tokens, torch.float32), top)


def test_one_token_for_all(qx):
    m = ref.layer(1, 6, 64, 96, seed=34)
    check(qx, m, tokens_of(m, 1, torch.bfloat16).expand(5, 64), 2)
    x, out = tokens_of(m, 1, torch.float32).cuda().expand(5, 64), torch.zeros(5, 64, device="cuda")
    qx.check(prepared(qx, m).apply_dev(router(qx, m, 2), x, out), "apply")
    assert all(torch.equal(row, out[0]) for row in out)


def test_threads_with_a_stream_and_workspace_each(qx):
    m = ref.layer(1, 16, 512, 256, 1, seed=35)
    experts, r = prepared(qx, m), router(qx, m, 4)
    x = tokens_of(m, 9, torch.bfloat16).cuda()
    want = torch.empty_like(x)
    qx.check(experts.apply_dev(r, x, want), "apply")
    torch.cuda.synchronize()
    wrong = []

    def work():
        space, stream = workspace(qx), torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                out = torch.empty_like(x)
                status = experts.apply_dev(r, x, out, workspace=space)
                stream.synchronize()
                if status != qx.OK or not torch.equal(out, want):
                    wrong.append(status)
        qx.lib.qx_workspace_destroy(space)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    qx.check(qx.lib.qx_check_device_errors(), "apply")
    assert not wrong
