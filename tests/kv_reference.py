"""Plain 64-bit restatements, token by token, of the operators between the qkv projection and the output
projection: rotary positions, the paged 8-bit key-value cache, attention over it. What the tests compare
the kernels with."""

import math

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rotated(x, positions, frequency, amplitude=1.0, interleaved=False, inverse=False):
    """x [tokens, heads, dim] f64 and positions [tokens] -> the rotated heads, f64."""
    y = x.clone()
    r = 2 * len(frequency)
    for t, position in enumerate(positions):
        for i, f in enumerate(frequency):
            c, s = math.cos(position * f) * amplitude, math.sin(position * f) * amplitude * (-1 if inverse else 1)
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
            y[t, :, a], y[t, :, b] = x[t, :, a] * c - x[t, :, b] * s, x[t, :, a] * s + x[t, :, b] * c
    return y


def half_even(num, den):
    """num / den rounded half to even: the quotient of two f64 values of at most 32 bits each is far enough from a
    half where it is none."""
    return np.rint(num / den)


class Cache:
    """[blocks, heads, block_tokens, dim] int8 codes and [blocks, heads] f32 scales, numpy."""

    def __init__(self, blocks, heads, size, dim, seed=0):
        rng = np.random.default_rng(seed)
        # (what a block held before is of no consequence: not even NaN)
        self.codes = [rng.integers(-128, 128, (blocks, heads, size, dim), dtype=np.int8) for _ in "kv"]
        self.scales = [np.full((blocks, heads), np.nan, np.float32) for _ in "kv"]
        self.size = size

    def append(self, which, table, first, x):
        """x [tokens, heads, dim] f64: new tokens of one sequence from position `first` on."""
        size = self.size
        n, heads, _ = x.shape
        for index in range(first // size, (first + n - 1) // size + 1 if n else 0):
            block, begin = table[index], index * size
            a, b = max(first, begin), min(first + n, begin + size)
            new = x[a - first:b - first]
            for h in range(heads):
                kept = a - begin
                old = np.float32(self.scales[which][block, h]) if kept else np.float32(0)
                scale = max(np.float32(np.float64(np.abs(new[:, h]).max()) / 127.0), old)
                if not np.isfinite(new[:, h]).all() or not np.isfinite(old):
                    self.scales[which][block, h] = np.nan
                    continue
                if scale < 2.0 ** -100:
                    scale = np.float32(0)
                self.scales[which][block, h] = scale
                codes = self.codes[which][block, h]
                if scale == 0:
                    codes[kept:b - begin] = 0
                    continue
                if kept:
                    codes[:kept] = half_even(codes[:kept].astype(np.float64) * np.float64(old), np.float64(scale))
                codes[kept:b - begin] = np.clip(half_even(new[:, h], np.float64(scale)), -127, 127)

    def values(self, which, table, length):
        """[length, heads, dim] f64"""
        out = []
        for p in range(length):
            block = table[p // self.size]
            out.append(self.codes[which][block, :, p % self.size].astype(np.float64) *
                       self.scales[which][block].astype(np.float64)[:, None])
        return np.stack(out) if out else np.zeros((0,) + self.codes[0].shape[1::2])


def attention(q, k, v, scale, causal, window, missing=()):
    """One sequence, f64: q [n, q_heads, dim], k and v [length, kv_heads, dim]. Returns the output, ln of the sums
    and, for the tolerances, the magnitudes of the values, weighted and plainly summed over the keys seen, and the
    largest sum of |scale q k| of a row."""
    n, heads, dim = q.shape
    length, kv_heads, _ = k.shape
    group = heads // kv_heads
    kk, vv = k.repeat_interleave(group, 1).transpose(0, 1), v.repeat_interleave(group, 1).transpose(0, 1)
    qq = q.transpose(0, 1)
    s = scale * (qq @ kk.transpose(1, 2))
    place = torch.arange(length - n, length)[:, None]
    key = torch.arange(length)[None]
    seen = torch.ones(n, length, dtype=torch.bool)
    if causal:
        seen &= key <= place
    if window:
        seen &= key > place - window
    seen[:, list(missing)] = False
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1) if length else torch.full((heads, n), -math.inf, dtype=torch.float64)
    p = torch.where(seen, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)
    spread = (abs(scale) * (qq.abs() @ kk.abs().transpose(1, 2))).amax(-1) if length else torch.zeros(heads, n)
    if length:  # (2^-22 of the row's largest query element, in units of the tolerances' 2^-23)
        spread = spread + abs(scale) * qq.abs().amax(-1) * kk.abs().sum(-1).amax(-1)[:, None] * 2 / (dim / 16 + 22)
    magnitude = (p @ vv.abs()).transpose(0, 1), (seen.double() @ vv.abs()).transpose(0, 1)
    return (p @ vv).transpose(0, 1), lse.T, magnitude, spread.T


def attention_tolerance(out, lse, magnitude, spread, dtype, dim, length):
    """Bounds on |kernel - exact|, per output element and per entry of lse. With u = 2^-23:
      scores   products of queries, rounded to 2^-22 of their row's largest magnitude (the second term of `spread`),
               and exact codes, summed in f32 (each of the dim / 16 MMAs may truncate), three multiplications:
               (dim / 16 + 22) u of the sum of magnitudes, at most;
      weights  exp2 to 2 u, its argument (up to `spread` * 1.44 away from the maximum) to one rounding: inside
               the next term;
      a score that is off by d takes d of its weight with it, and d of the sum: 2 d;
      weights are rounded to f16 (11 significant bits: a weight in [2^e, 2^(e+1)) is off by half of 2^(e-10) at
               most, so 2^-11 of each where it stands at 2^e; the values are exact) or, for f32, to a pair of which
               the second takes what the first leaves, 2^-11 of it, again to 2^-11: 2^-22, and to no less than
               the smallest step of f16, 2^-24, held times 2^12 against the row's largest weight: half of that,
               2^-37, of every value seen, however small its weight (the sum of weights is the largest one or more).
               Long prompts of 16-bit queries hold weight times value scale times 2^11, against the largest such
               product: 2^-36 of every code under the largest scale seen, with value scales that are within a
               factor of eight of each other (as they are where this is called) 2^-33 of every value;
      sums of at most `length` weights and of the tiles, each addition u: (length / 32 + 64) u of the magnitudes;
      one rounding to the output's type."""
    u = 2.0 ** -23
    score = (dim / 16 + 22) * u * spread + 4 * u
    rounded = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    sums = (length / 32 + 64) * u
    weighted, plain = magnitude
    smallest = 2.0 ** -37 if dtype == torch.float32 else 2.0 ** -33
    return (HALF_STEP[dtype] * out.abs() + (2 * score + rounded + sums)[..., None] * weighted + smallest * plain + 1e-37,
            score + sums + 2 * u * lse.abs())
