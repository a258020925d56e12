"""A mixture-of-experts layer in 64 bits, with how far f32 sums and the stated roundings may move it."""

from types import SimpleNamespace

import numpy as np
import torch

from kv_reference import HALF_STEP

U = 2.0 ** -24  # half a step of f32, relative
SILU = 3


def quantised(rng, fmt, *shape):
    """GGUF blocks (0: q8_0, 1: q4_0) of normal values of variance 1 / columns -> (bytes, their values in 64 bits)."""
    rows = int(np.prod(shape[:-1]))
    w = rng.standard_normal((rows, shape[-1] // 32, 32)) / np.sqrt(shape[-1])
    if fmt == 0:
        d = (np.abs(w).max(-1, keepdims=True) / 127).astype(np.float16)
        codes = np.clip(np.rint(w / d), -128, 127).astype(np.int8)
        raw, values = codes.view(np.uint8), codes
    else:
        d = (np.take_along_axis(w, np.abs(w).argmax(-1)[..., None], -1) / -8).astype(np.float16)
        codes = np.clip(np.floor(w / d + 8.5), 0, 15).astype(np.uint8)
        raw, values = codes[..., :16] | codes[..., 16:] << 4, codes.astype(np.int8) - 8
    packed = np.concatenate([d.view(np.uint8), raw], -1).reshape(-1)
    return packed, torch.from_numpy((values * d.astype(np.float64)).reshape(shape))


def activate(g, kind):
    if kind == 1:
        return 0.5 * g * (1 + torch.erf(g / 2 ** 0.5))
    if kind == 2:
        return torch.nn.functional.gelu(g, approximate="tanh")
    if kind == 3:
        return g * torch.sigmoid(g)
    if kind == 4:
        return torch.relu(g) ** 2
    return g


def layer(fmt, experts, dim, inner, shared=0, seed=0, router=torch.float32):
    rng = np.random.default_rng(seed)
    count = experts + shared
    gate, up, down = (quantised(rng, fmt, count, *s) for s in ((inner, dim), (inner, dim), (dim, inner)))
    weights = torch.from_numpy(rng.standard_normal((experts, dim)) * 1.5 / np.sqrt(dim)).to(router)
    bias = torch.from_numpy(rng.standard_normal(experts) * 0.1).float()
    return SimpleNamespace(fmt=fmt, experts=experts, dim=dim, inner=inner, shared=shared, raw=(gate[0], up[0], down[0]),
                           gate=gate[1], up=up[1], down=down[1], router=weights, bias=bias)


def route(m, x, top, sigmoid=False, biased=False, normalise=True, scale=1.0, chosen=None):
    """-> chosen [tokens, top], their weights, and how far those may be off. `chosen` given: that choice is looked at (two
    experts may lie closer together than sums in f32 tell apart) and taken."""
    x, w = x.double(), m.router.double()
    logits = x @ w.T
    # exact products, 32 a sum in f32 (f32 and f16 operands: their terms' products too, which are no larger) as MMAs take them, in
    # 2 .. 18 steps that cut off, 2 u of no more than the products' magnitudes each, then 64 bits
    off = 36 * U * (x.abs() @ w.abs().T)
    score = torch.sigmoid(logits) if sigmoid else torch.softmax(logits, 1)
    # (a logit that is off by o moves every score's share by no more than 2 o relative)
    key, key_off = (score + m.bias.double(), 2 * off.amax(1, keepdim=True) * score) if biased else (logits, off)
    order = key.sort(dim=1, descending=True, stable=True).indices[:, :top]
    if chosen is None:
        chosen = order
    else:
        assert bool((chosen.sort(1).values.diff(dim=1) > 0).all()) and 0 <= int(chosen.min()) <= int(chosen.max()) < m.experts
        # the j-th largest of keys that are off by o at most moves by o at most, and the one found there is off by o itself
        moved = (key.gather(1, chosen) - key.gather(1, order)).abs()
        assert bool((moved <= 2 * key_off.amax(1, keepdim=True)).all()), "another choice"
    picked = score.gather(1, chosen)
    weights = scale * (picked / picked.sum(1, keepdim=True) if normalise else picked)
    # (exponents are rounded to f32: u of their size moves a score by as much, relative; exp, sums and quotients 8 u)
    return chosen, weights, weights.abs() * (2 * off.amax(1, keepdim=True) + (8 + 4 * logits.abs().amax(1, keepdim=True)) * U)


def apply(m, x, top, activation=SILU, sigmoid=False, biased=False, normalise=True, scale=1.0, out_type=None, chosen=None):
    """-> the layer's output, and the limit of |kernel - output|, both in 64 bits.

    Inputs and inner activations are digits under a power of two: off by 2^-15 (16-bit x) or 2^-23 of the largest of their
    block of 32, or 2^-103. The sums of a block are exact. Then, in f32: two digits are joined, the block's factors are
    multiplied, and their product added, four roundings, one behind the other in eight parts, which three additions join:
    a matrix product of k columns is off by (k / 32 / 8 + 12) u of the sum of its terms' magnitudes at most. Those of the
    digits are no more than |x| and 2^-6 of the block's largest. The activation's slope is below 1.13 (its argument is off, and
    a few u of itself); relu^2 has a slope of 2 g."""
    chosen, weights, weights_off = route(m, x, top, sigmoid, biased, normalise, scale, chosen)
    kept = 2.0 ** -23 if x.dtype == torch.float32 else 2.0 ** -15
    x = x.double()

    def largest(v):  # of each block of 32, spread over it
        return v.abs().unflatten(1, (-1, 32)).amax(2, keepdim=True).expand(-1, -1, 32).flatten(1)

    def product(v, v_off, w):
        """v @ w.T where v is off by v_off, and how far it is off."""
        size = v.abs() + v_off + 2.0 ** -6 * largest(v.abs() + v_off)
        return v @ w.T, (v_off + U * (v.shape[1] / 256 + 12) * size) @ w.abs().T

    x_off = kept * largest(x) + 2.0 ** -103
    out, limit = torch.zeros_like(x), torch.zeros_like(x)
    for e in range(m.experts + m.shared):
        if e < m.experts:
            rows, place = (chosen == e).nonzero(as_tuple=True)
            w, w_off = weights[rows, place, None], weights_off[rows, place, None]
        else:
            rows, w, w_off = torch.arange(len(x)), torch.ones(len(x), 1, dtype=torch.float64), 0.0
        if not len(rows):
            continue
        v, v_off = x[rows], x_off[rows]
        g, g_off = product(v, v_off, m.gate[e])
        u, u_off = product(v, v_off, m.up[e])
        f = activate(g, activation)
        slope = 2 * (g.abs() + g_off) if activation == 4 else 1.13
        f_off = slope * g_off + 8 * U * (f.abs() + g.abs())
        a = f * u
        a_off = f_off * u.abs() + (f.abs() + f_off) * u_off + U * a.abs()
        a_off = a_off + kept * largest(a.abs() + a_off) + 2.0 ** -103
        y, y_off = product(a, a_off, m.down[e])
        out[rows] += w * y
        limit[rows] += w.abs() * y_off + w_off * (y.abs() + y_off) + (top + m.shared + 1) * U * (w * y).abs()
    return out, limit + HALF_STEP[out_type] * (out.abs() + limit) + (2.0 ** -25 if out_type == torch.float16 else 2.0 ** -134)
