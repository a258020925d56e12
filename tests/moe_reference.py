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
    # eight products a sum in f32 (eight roundings of no more than the products' magnitudes), then 64 bits
    off = 8 * U * (x.abs() @ w.abs().T)
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
    return chosen, weights, weights.abs() * (2 * off.amax(1, keepdim=True) + 2 * U)


def apply(m, x, top, activation=SILU, sigmoid=False, biased=False, normalise=True, scale=1.0, out_type=None, chosen=None):
    """-> the layer's output, and the limit of |kernel - output|, both in 64 bits.

    Roundings of a sum of n terms: n u of the sum of their magnitudes at most, whatever the order; a product with a block
    is one sum of 32 products inside an MMA (rounded or cut: 2 u a step, in four steps), two multiplications with scales, and the
    blocks are added one behind the other, in two halves. So a matrix product of k columns is off by
    (k / 32 + 12) * 2 u of sum |w x| at most. Inputs: 16-bit ones are exact, f32 ones are taken to 2^-22 of themselves, or
    2^-38 of their block's largest. The activation's slope is below 1.13 (its argument is off, and a few u of itself);
    relu^2 has a slope of 2 g. The inner activations are rounded to 2^-11 (16-bit x) or 2^-22 of themselves."""
    chosen, weights, weights_off = route(m, x, top, sigmoid, biased, normalise, scale, chosen)
    wide = x.dtype == torch.float32
    kept, least = (2.0 ** -22, 2.0 ** -38) if wide else (0.0, 2.0 ** -38)
    inner_kept = 2.0 ** -22 if wide else 2.0 ** -11
    x = x.double()

    def largest(v):  # of each block of 32, spread over it
        return v.abs().unflatten(1, (-1, 32)).amax(2, keepdim=True).expand(-1, -1, 32).flatten(1)

    x_off = kept * x.abs() + least * largest(x)
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
        sums = 2 * U * (m.dim / 32 + 12)
        g, u = v @ m.gate[e].T, v @ m.up[e].T
        g_off = v.abs() @ m.gate[e].abs().T * sums + v_off @ m.gate[e].abs().T
        u_off = v.abs() @ m.up[e].abs().T * sums + v_off @ m.up[e].abs().T
        f = activate(g, activation)
        slope = 2 * (g.abs() + g_off) if activation == 4 else 1.13
        f_off = slope * g_off + 8 * U * (f.abs() + g.abs())
        a = f * u
        a_off = f_off * u.abs() + (f.abs() + f_off) * u_off + U * a.abs()
        a_off = a_off + inner_kept * (a.abs() + a_off) + least * largest(a)
        y = a @ m.down[e].T
        y_off = a_off @ m.down[e].abs().T + (a.abs() + a_off) @ m.down[e].abs().T * (2 * U * (m.inner / 32 + 12))
        out[rows] += w * y
        limit[rows] += w.abs() * y_off + w_off * (y.abs() + y_off) + (top + m.shared + 1) * U * (w * y).abs()
    return out, limit + HALF_STEP[out_type] * (out.abs() + limit) + (2.0 ** -25 if out_type == torch.float16 else 2.0 ** -134)
