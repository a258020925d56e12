"""Router weights whose scores run low: quotients of scores that f32 or even 64 bits no longer hold, chosen by a bias or by
themselves, against logarithms of the scores in 64 bits."""

import pytest
import torch

import moe_reference as ref
from test_moe_gpu import prepared, router, tokens_of

pytestmark = pytest.mark.gpu
U = ref.U


def far_layer(targets, lifted, dtype=torch.float32, seed=41):
    """A layer whose experts' logits lie about `targets`, a bias for the choice of `lifted` experts in an order of their own,
    and its tokens."""
    m = ref.layer(1, len(targets), 64, 32, seed=seed)
    x = tokens_of(m, 7, dtype)
    x[:, 0] = 8.0
    m.router[:, 0] = torch.tensor(targets) / 8
    m.bias = torch.full((len(targets),), -50.0)
    for place, expert in enumerate(lifted):
        m.bias[expert] = 40.0 - 3 * place  # (far apart: scores are no more than 1)
    return m, x


def shares(m, x, chosen, sigmoid, normalise, scale):
    """The weights of `chosen` from logarithms, and how far they may be off: as moe_reference.route has it, and half of the
    smallest step of f32."""
    x, w = x.double(), m.router.double()
    logits, off = x @ w.T, 36 * U * (x.abs() @ w.abs().T)
    log = torch.nn.functional.logsigmoid(logits) if sigmoid else torch.log_softmax(logits, 1)
    log = log.gather(1, chosen)
    if normalise:
        log = log - torch.logsumexp(log, 1, keepdim=True)
    weights = scale * log.exp()
    return weights, weights * (2 * off.amax(1, keepdim=True) + (8 + 4 * logits.abs().amax(1, keepdim=True)) * U) + 2.0 ** -150


def check(qx, m, x, top, sigmoid, biased, normalise, scale=2.5):
    out = torch.full(x.shape, float("nan"), device="cuda")
    chosen = torch.full((len(x), top), -1, dtype=torch.int32, device="cuda")
    weights = torch.full((len(x), top), float("nan"), device="cuda")
    kind = dict(sigmoid=sigmoid, biased=biased, normalise=normalise, scale=scale)
    qx.check(prepared(qx, m).apply_dev(router(qx, m, top, **kind), x.cuda(), out, chosen=chosen, weights=weights), "apply")
    torch.cuda.synchronize()
    qx.check(qx.lib.qx_check_device_errors(), "apply")
    picks = chosen.cpu().long()
    if biased:
        assert picks.tolist() == [m.bias.argsort(descending=True)[:top].tolist()] * len(x)
    else:
        ref.route(m, x, top, chosen=picks)  # (logits and scores have one order)
    want, limit = shares(m, x, picks, sigmoid, normalise, scale)
    off = (weights.cpu().double() - want).abs() - limit
    assert float(off.max()) <= 0, float(off.max())
    assert bool(out.isfinite().all())
    return weights


RANGES = [(-60.0, -95.0), (-79.0, -100.0), (-90.0, -150.0), (-100.0, -108.0), (-110.0, -111.0), (-600.0, -1500.0)]


@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("top", [1, 2, 5])
@pytest.mark.parametrize("first,last", RANGES)
def test_sigmoids_chosen_by_a_bias(qx, first, last, top, normalise):
    m, x = far_layer(torch.linspace(first, last, 9).tolist(), [3, 7, 1, 8, 0])
    check(qx, m, x, top, True, True, normalise)


@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("top", [1, 2, 5])
@pytest.mark.parametrize("first,last", RANGES)
def test_softmax_scores_lifted_past_far_larger_logits(qx, first, last, top, normalise):
    m, x = far_layer([5.0] + torch.linspace(first, last, 9).tolist() + [3.0], [4, 1, 9, 6, 2])
    check(qx, m, x, top, False, True, normalise)


@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_scores_of_both_sides_of_the_range(qx, dtype, normalise):
    """Scores near one beside such as f32 does not hold."""
    m, x = far_layer([3.0, -120.0, -2.0, -140.0, 0.5, -95.0], [1, 0, 3, 4], dtype)
    for sigmoid in (False, True):
        check(qx, m, x, 4, sigmoid, True, normalise)


@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("top", [1, 3, 6])
@pytest.mark.parametrize("first,last", RANGES)
def test_sigmoids_without_a_bias(qx, first, last, top, normalise):
    """Among them the largest just inside of what f32 holds and the others outside."""
    m, x = far_layer(torch.linspace(first, last, 9).tolist(), [])
    check(qx, m, x, top, True, False, normalise)


@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("scale", [1.0, 1e30])
def test_softmax_without_a_bias(qx, scale, normalise):
    """Experts far below the largest, with a scale that makes plain numbers of their weights."""
    m, x = far_layer([5.0, -60.0, -75.0, -90.0, -98.0, -120.0], [])
    m.raw[2].reshape(-1, 18)[:, :2] = 0  # (down projections of zeros: outputs that fit)
    check(qx, m, x, 6, False, False, normalise, scale)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_one_expert_takes_the_whole_weight(qx, sigmoid, biased):
    m, x = far_layer([1.0, -200.0, -300.0], [2])
    assert bool((check(qx, m, x, 1, sigmoid, biased, True) == 2.5).all())
