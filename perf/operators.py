"""The operators between a decoder layer's qkv projection and its output projection, as timed cases:

  rope    rotary positions on query and key heads: both pair layouts, part of the head, scaled for
          long contexts
  append  new keys and values quantised into a paged cache of 8-bit codes with one f32 scale per
          (block of tokens, kv head), optionally rotated on the way, and the touched blocks read
          back as values
  attend  attention of packed ragged queries over that cache: single tokens, speculated runs,
          chunks of a prompt, whole prompts; causal, windowed or neither

`run` computes them from elementary torch operations, or (own = True) through the library's entry
points. Block 0 of every cache is the padding block that serving programs keep: no sequence owns it.
"""

from __future__ import annotations

import functools
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------------------

def listed():
    return [
        # rotation of one decode step's queries and keys, 32 sessions far into a stretched context
        dict(name="rope_step_bf16", kind="rope", type="bf16", tokens=32, heads=40, dim=128, rotary=128,
             style="halves", scaling="ramp", first=100000, packed=True),
        # a long prompt's queries and keys, half of each head rotated, inside the packed projection
        dict(name="rope_prompt_f16", kind="rope", type="f16", tokens=8191, heads=40, dim=128, rotary=64,
             style="interleaved", scaling="none", first=0, packed=True),
        # one decode step of 64 sessions: keys rotated and appended, queries rotated in the same call
        dict(name="append_step_bf16", kind="append", type="bf16", seqs=64, tokens=1, ragged=False, length=2048,
             q_heads=32, kv_heads=8, dim=128, block=64, rope="halves", scaling="bands"),
        # three prompts of unequal lengths behind cached prefixes, f32 as the projections give it
        dict(name="append_prompt_f32", kind="append", type="f32", seqs=3, tokens=4096, ragged=True, length=5000,
             q_heads=32, kv_heads=8, dim=128, block=32, rope="none", scaling="none"),
        # the smallest call: one token of one short session on f32 projections
        dict(name="attend_one_f32", kind="attend", type="f32", seqs=1, tokens=1, ragged=False, length=1000,
             q_heads=32, kv_heads=8, dim=128, block=64, causal=True, window=0, packed=False),
        # one decode step of a full batch, lengths spread
        dict(name="attend_step_bf16", kind="attend", type="bf16", seqs=32, tokens=1, ragged=False, length=8192,
             q_heads=32, kv_heads=8, dim=128, block=64, causal=True, window=0, packed=True),
        # one token behind a very long context, split over the whole card
        dict(name="attend_long_bf16", kind="attend", type="bf16", seqs=1, tokens=1, ragged=False, length=131072,
             q_heads=64, kv_heads=8, dim=128, block=128, causal=True, window=0, packed=False),
        # speculated runs of up to five tokens, three query heads to a kv head, sliding window
        dict(name="attend_draft_f16", kind="attend", type="f16", seqs=8, tokens=5, ragged=True, length=16384,
             q_heads=24, kv_heads=8, dim=64, block=16, causal=True, window=4096, packed=True),
        # two prompts of unequal lengths, causal
        dict(name="attend_prompt_bf16", kind="attend", type="bf16", seqs=2, tokens=4096, ragged=True, length=4096,
             q_heads=32, kv_heads=8, dim=128, block=64, causal=True, window=0, packed=True),
        # a chunk of a long prompt behind what is cached of it
        dict(name="attend_chunk_f16", kind="attend", type="f16", seqs=1, tokens=1024, ragged=False, length=16384,
             q_heads=32, kv_heads=8, dim=128, block=32, causal=True, window=0, packed=False),
        # short texts read in both directions in f32, one kv head per query head, an odd head size
        dict(name="attend_text_f32", kind="attend", type="f32", seqs=4, tokens=500, ragged=True, length=500,
             q_heads=16, kv_heads=16, dim=96, block=64, causal=False, window=0, packed=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "attend", "attend", "attend"])
    typ = rng.choice(["f32", "f16", "bf16", "bf16"])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    if kind == "rope":
        heads = rng.choice([1, 8, 24, 40, 72])
        tokens = _log(rng, 1, 8191 * 40 * 128 // (heads * dim) // (2 if typ == "f32" else 1))
        return dict(kind=kind, type=typ, tokens=tokens, heads=heads, dim=dim,
                    rotary=rng.choice([dim, dim, dim // 2, 32]), style=rng.choice(["halves", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "bands", "ramp"]), first=rng.randrange(1 << 20),
                    packed=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 8, 8, 16])
    block = rng.choice([16, 32, 64, 128])
    step = rng.random() < 0.6
    if kind == "append":
        row = kv_heads * dim
        seqs = _log(rng, 1, 128) if step else rng.randint(1, 6)
        tokens = rng.randint(1, 4) if step else _log(rng, 8, max(9, 8 * 1024 * 1024 // (row * seqs)))
        rope = "none" if typ == "f32" else rng.choice(["none", "halves", "interleaved"])
        return dict(kind=kind, type=typ, seqs=seqs, tokens=tokens, ragged=rng.random() < 0.6,
                    length=tokens + rng.randint(0, 3000), q_heads=kv_heads * min(group, 8), kv_heads=kv_heads, dim=dim,
                    block=block, rope=rope, scaling=rng.choice(["none", "linear", "bands", "ramp"]))
    row = kv_heads * dim
    if step:
        seqs = _log(rng, 1, 64)
        tokens = rng.choice([1, 1, 1, 2, 5])
        length = tokens + _log(rng, 1, max(16, min(131072, 100 * 1024 * 1024 // (row * seqs))))
    else:
        seqs = rng.randint(1, 4)
        tokens = _log(rng, 8, 2048)
        if typ == "f32":
            tokens = min(tokens, 700)
        while seqs * tokens * kv_heads * group * dim > 2048 * 32 * 128 * 2:
            tokens = tokens * 2 // 3
        most = 200_000_000 // (seqs * tokens * kv_heads * group) * 128 // dim
        length = tokens + (0 if rng.random() < 0.5 else rng.randint(0, max(1, min(16384, most) - tokens)) if most > tokens else 0)
    return dict(kind=kind, type=typ, seqs=seqs, tokens=tokens, ragged=rng.random() < 0.6, length=length,
                q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, block=block, causal=rng.random() < 0.8,
                window=rng.choice([0, 0, 0, 128, 1000, 4096]), packed=rng.random() < 0.5)


def _lengths(case):
    """New tokens and lengths (those included) of every sequence, and rows behind the last one."""
    seqs, tokens, length = case["seqs"], case["tokens"], case["length"]
    mixed = case["ragged"] or seqs > 1
    new = [max(1, tokens - (tokens * 4 * i) // (7 * seqs)) if case["ragged"] else tokens for i in range(seqs)]
    total = [max(n, length - (length * 6 * i) // (7 * seqs) - 7 * (i % 3)) if mixed else length for i, n in enumerate(new)]
    return new, total, (5 if case["ragged"] else 0)


def _pairs(case):
    """(query, key) pairs that the masks leave, and keys that any query sees, over all sequences."""
    pairs = keys = 0
    for n, total in zip(*_lengths(case)[:2]):
        if not case["causal"] and not case["window"]:
            pairs, keys = pairs + n * total, keys + total
            continue
        w = case["window"] or total + 1
        first = total - n
        top = [(first + 1), total] if case["causal"] else [total, total]
        # sum over p = first .. total - 1 of (last seen + 1) - max(0, p - w + 1)
        seen = (top[0] + top[1]) * n // 2
        a = max(first, w - 1)
        cut = (total - 1 - a + 1) * ((a - w + 1) + (total - 1 - w + 1)) // 2 if a < total else 0
        pairs, keys = pairs + seen - cut, keys + total - max(0, first - w + 1)
    return pairs, keys


def work(case):
    size = torch.empty(0, dtype=TYPES[case["type"]]).element_size()
    if case["kind"] == "rope":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * values * size + 8 * case["tokens"], "flops": 3 * values * case["rotary"] / case["dim"]}
    row = case["kv_heads"] * case["dim"]
    new, total, _ = _lengths(case)
    if case["kind"] == "append":
        read_back = sum(_tail(case, n, t) for n, t in zip(new, total))
        old = read_back - sum(new)
        rotated = 2 * sum(new) * case["q_heads"] * case["dim"] * size if case["rope"] != "none" else 0
        # new keys and values in, their codes out, the older codes of the touched blocks, values out
        return {"bytes": 2 * row * (sum(new) * (size + 1) + old + read_back * size) + rotated,
                "flops": 4 * row * sum(new)}
    pairs, keys = _pairs(case)
    scales = 8 * case["kv_heads"] * (keys // case["block"] + 1)
    return {"bytes": 2 * row * keys + scales + 2 * sum(new) * case["q_heads"] * case["dim"] * size,
            "flops": 4 * case["dim"] * case["q_heads"] * pairs}


def _tail(case, n, total):
    """Tokens of a sequence from the first block that its new tokens touch to its end."""
    return total - (total - n) // case["block"] * case["block"]


# ---- inputs -----------------------------------------------------------------------------

BASE, TRAINED = 500000.0, 8192


def _frequencies(rotary, scaling):
    """Angles per position of the rotary // 2 pairs, and the amplitude."""
    f = [BASE ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    if scaling == "linear":
        return [v / 4.0 for v in f], 1.0
    if scaling == "bands":  # by how often a pair turns over the trained length: 1 .. 4 blends
        turns = [TRAINED * v / (2 * math.pi) for v in f]
        keep = [min(1.0, max(0.0, (t - 1.0) / 3.0)) for t in turns]
        return [(1 - k) * v / 8.0 + k * v for k, v in zip(keep, f)], 1.0
    if scaling == "ramp":  # linear in the pair's index between the pairs that turn 32 times and once
        at = [rotary * math.log(TRAINED / (r * 2 * math.pi)) / (2 * math.log(BASE)) for r in (32.0, 1.0)]
        low, high = max(0, math.floor(at[0])), min(rotary - 1, math.ceil(at[1]))
        span = high - low if high > low else 0.001
        cut = [min(1.0, max(0.0, (i - low) / span)) for i in range(len(f))]
        return [v / 16.0 * c + v * (1 - c) for c, v in zip(cut, f)], 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _heads(gen, tokens, heads, others, dim, dtype, packed):
    """`heads` heads of every token: alone, or in front of `others` in a packed projection's rows."""
    wide = torch.randn(tokens, heads + (others if packed else 0), dim, generator=gen, device="cuda")
    return wide.to(dtype)[:, :heads]


def _quantised(gen, blocks, heads, block, dim):
    """Codes [blocks, heads, block, dim] and scales [blocks, heads] of normal values, some heads louder."""
    loud = torch.rand(1, heads, 1, 1, generator=gen, device="cuda") * 1.5 + 0.5
    codes = torch.empty(blocks, heads, block, dim, dtype=torch.int8, device="cuda")
    scales = torch.empty(blocks, heads, device="cuda")
    some = max(1, (1 << 26) // (heads * block * dim))
    for b in range(0, blocks, some):
        x = torch.randn(min(some, blocks - b), heads, block, dim, generator=gen, device="cuda") * loud
        s = x.abs().amax((2, 3)) / 127.0
        scales[b:b + some] = s
        codes[b:b + some] = (x / s[:, :, None, None]).round().clamp(-127, 127).to(torch.int8)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    state = {"case": dict(case)}
    if case["kind"] == "rope":
        tokens = case["tokens"]
        state["x"] = _heads(gen, tokens, case["heads"], 8, case["dim"], dtype, case["packed"])
        step = torch.randint(0, 4, (tokens,), generator=gen, device="cuda")
        state["positions"] = case["first"] + torch.cumsum(step, 0)
        state["frequencies"] = _frequencies(case["rotary"], case["scaling"])
        return state
    new, total, behind = _lengths(case)
    rows = sum(new) + behind
    row = case["block"]
    width = max(-(-t // row) for t in total) + 1
    blocks = sum(-(-t // row) for t in total) + 1
    order = (torch.randperm(blocks - 1, generator=gen, device="cuda") + 1).to(torch.int32)
    table = torch.zeros(case["seqs"], width, dtype=torch.int32, device="cuda")
    at = 0
    for i, t in enumerate(total):
        n = -(-t // row)
        table[i, :n] = order[at:at + n]
        at += n
    state["k_codes"], state["k_scales"] = _quantised(gen, blocks, case["kv_heads"], row, case["dim"])
    state["v_codes"], state["v_scales"] = _quantised(gen, blocks, case["kv_heads"], row, case["dim"])
    state["table"] = table
    state["lengths"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    state["begin"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    state["rows"], state["max_new"], state["max_length"] = rows, max(new), max(total)
    qkv = torch.randn(rows, case["q_heads"] + 2 * case["kv_heads"], case["dim"], generator=gen, device="cuda").to(dtype)
    q, k, v = qkv.split([case["q_heads"], case["kv_heads"], case["kv_heads"]], 1)
    if case["kind"] == "append":
        state["q"], state["k"], state["v"] = q, k, v
        state["q_out"] = torch.zeros(rows, case["q_heads"], case["dim"], dtype=dtype, device="cuda")
        state["frequencies"] = _frequencies(case["dim"], case["scaling"])
        tails = [_tail(case, n, t) for n, t in zip(new, total)]
        state["tail_begin"] = torch.tensor([sum(tails[:i]) for i in range(len(tails) + 1)], dtype=torch.int32, device="cuda")
        state["tail_rows"], state["max_tail"] = sum(tails), max(tails)
    else:
        state["q"] = q if case["packed"] else q.contiguous()
        state["out"] = torch.zeros(rows, case["q_heads"], case["dim"], dtype=dtype, device="cuda")
    return state


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "rope":
        return _rope(state["case"]["style"], state["x"].float(), state["positions"], state["frequencies"]).to(state["x"].dtype)
    return _append(state) if kind == "append" else _attend(state)


def _rope(style, x, positions, frequencies):
    """x [tokens, heads, dim] f32, rotated. The angles are taken in 64 bits: far positions lose them in 32."""
    f, amplitude = frequencies
    f = torch.tensor(f, dtype=torch.float64, device=x.device)
    angle = positions.double()[:, None] * f
    cos, sin = (t.float()[:, None, :] * amplitude for t in (angle.cos(), angle.sin()))
    half = f.numel()
    y = x.clone()
    if style == "halves":
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, a * sin + b * cos
    return y


def _rows(begin, rows):
    """For packed rows: the sequence of each, its index in there, and whether it belongs to one at all."""
    at = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(begin[1:].contiguous(), at.to(torch.int32), right=True)
    inside = seq < begin.numel() - 1
    seq = seq.clamp(max=begin.numel() - 2)
    return seq, at - begin[seq], inside


def _places(state, begin, rows):
    """Position, block and slot of every packed row; rows behind the last sequence get the padding block."""
    seq, index, inside = _rows(begin, rows)
    first = state["lengths"] - (begin[1:] - begin[:-1])
    position = torch.where(inside, first[seq] + index, 0).long()
    block = torch.where(inside, state["table"][seq, position // state["case"]["block"]], 0).long()
    return position, block, position % state["case"]["block"], inside


def _append(state):
    case = state["case"]
    position, block, slot, inside = _places(state, state["begin"], state["rows"])
    k, v, q = state["k"].float(), state["v"].float(), None
    if case["rope"] != "none":
        q = state["q_out"]
        rotated = _rope(case["rope"], state["q"].float(), position, state["frequencies"]).to(q.dtype)
        q.copy_(torch.where(inside[:, None, None], rotated, q))
        k = _rope(case["rope"], k, position, state["frequencies"])
    first = state["lengths"] - (state["begin"][1:] - state["begin"][:-1])
    last = state["table"][torch.arange(case["seqs"], device="cuda"), (first // case["block"]).long()].long()
    held = torch.where(first % case["block"] > 0, last, 0)  # the block that a sequence's older tokens end in
    _append_one(k, block, slot, held, state["k_codes"], state["k_scales"])
    _append_one(v, block, slot, held, state["v_codes"], state["v_scales"])
    tail = state["tail_begin"]
    _, block, slot, _ = _places(state, tail, state["tail_rows"])
    out = [(c[block, :, slot].float() * s[block][..., None]).to(TYPES[case["type"]])
           for c, s in ((state["k_codes"], state["k_scales"]), (state["v_codes"], state["v_scales"]))]
    return out if q is None else out + [q]


def _append_one(x, block, slot, held, codes, scales):
    kept = torch.zeros_like(scales)
    kept[held] = scales[held]
    kept[0] = 0  # (the padding block)
    # (the divisor on the device: by a number, torch multiplies with its rounded reciprocal instead)
    new = torch.zeros_like(scales).index_reduce_(0, block, x.abs().amax(2), "amax") / torch.full((), 127.0, device="cuda")
    new = torch.maximum(kept, new)
    # quotients in 64 bits: in 32 those next to a half fall on its wrong side
    step = torch.where(new > 0, new, 1.0).double()
    values = codes[held].double() * kept[held][:, :, None, None]
    codes[held] = (values / step[held][:, :, None, None]).round().to(torch.int8)
    codes[block, :, slot] = (x.double() / step[block][..., None]).round().clamp(-127, 127).to(torch.int8)
    scales.scatter_(0, block[:, None].expand(-1, scales.shape[1]), new[block])


def _attend(state):
    case = state["case"]
    group, most, length = case["q_heads"] // case["kv_heads"], state["max_new"], state["max_length"]
    begin, lengths, table = state["begin"].long(), state["lengths"].long(), state["table"].long()
    seq, index, inside = _rows(state["begin"], state["rows"])
    # queries padded to [sequence, kv head, group, new token, dim]
    at = (begin[:-1, None] + torch.arange(most, device="cuda")).clamp(max=state["rows"] - 1)
    q = state["q"][at].float().view(case["seqs"], most, case["kv_heads"], group, case["dim"]).permute(0, 2, 3, 1, 4)
    width = -(-length // case["block"])

    def values(codes, scales):
        x = codes[table[:, :width]].float() * scales[table[:, :width]][..., None, None]
        return x.transpose(1, 2).flatten(2, 3)  # [sequence, kv head, token, dim]

    s = torch.matmul(q, values(state["k_codes"], state["k_scales"])[:, :, None].transpose(-1, -2)) * case["dim"] ** -0.5
    position = ((lengths - (begin[1:] - begin[:-1]))[:, None] + torch.arange(most, device="cuda"))[:, :, None]
    key = torch.arange(s.shape[-1], device="cuda")
    seen = key < lengths[:, None, None]
    if case["causal"]:
        seen = seen & (key <= position)
    if case["window"]:
        seen = seen & (key > position - case["window"])
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, values(state["v_codes"], state["v_scales"])[:, :, None]) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, index.clamp(max=most - 1)]  # packed rows again
    out = state["out"]
    out.copy_(torch.where(inside[:, None, None], o.to(out.dtype), out))
    return out


# ---- the library's calls ----------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _library():
    import __graft_entry__
    return __graft_entry__.load_package()


@functools.lru_cache(maxsize=64)
def _plan(rotary, style, scaling):
    """The rotation that a program keeps for a model."""
    qx = _library()
    more = {"none": None, "linear": dict(kind=qx.ROPE_LINEAR, factor=4.0),
            "bands": dict(kind=qx.ROPE_BANDS, factor=8.0, trained=TRAINED, slow=1.0, fast=4.0),
            "ramp": dict(kind=qx.ROPE_RAMP, factor=16.0, trained=TRAINED, slow=1.0, fast=32.0)}[scaling]
    return qx.Rope(rotary, qx.ROPE_HALVES if style == "halves" else qx.ROPE_INTERLEAVED, BASE, more)


def _own(state):
    qx, case = _library(), state["case"]
    if case["kind"] == "rope":
        y = torch.empty(state["x"].shape, dtype=state["x"].dtype, device="cuda")
        qx.check(_plan(case["rotary"], case["style"], case["scaling"]).apply_dev(state["x"], y, state["positions"]), "rope")
        return y
    cache = qx.KVCache(state["k_codes"], state["v_codes"], state["k_scales"], state["v_scales"])
    batch = qx.KVBatch(state["lengths"], state["table"], state["max_length"], state["begin"], state["rows"], state["max_new"])
    if case["kind"] == "attend":
        qx.check(cache.attention_dev(batch, state["q"], state["out"], causal=case["causal"], window=case["window"]), "attention")
        return state["out"]
    rope = None if case["rope"] == "none" else _plan(case["dim"], case["rope"], case["scaling"])
    q, q_out = (None, None) if rope is None else (state["q"], state["q_out"])
    qx.check(cache.append_dev(batch, state["k"], state["v"], rope, q, q_out), "append")
    k, v = (torch.empty(state["tail_rows"], case["kv_heads"], case["dim"], dtype=TYPES[case["type"]], device="cuda") for _ in "kv")
    tail = qx.KVBatch(state["lengths"], state["table"], state["max_length"], state["tail_begin"], state["tail_rows"], state["max_tail"])
    qx.check(cache.read_dev(tail, k, v), "read")
    return [k, v] if q_out is None else [k, v, q_out]


# ---- 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rope":
        return _turned(case["style"], state["x"], state["positions"].tolist(), state["frequencies"])
    new, total, _ = _lengths(case)
    return (_exact_append if case["kind"] == "append" else _exact_attend)(case, state, new, total)


def _turned(style, x, positions, frequencies):
    f, amplitude = frequencies
    turn = torch.outer(torch.tensor(positions, dtype=torch.float64), torch.tensor(f, dtype=torch.float64)).cuda()
    turn = torch.polar(torch.full_like(turn, amplitude), turn)[:, None]
    x = x.double()
    r = 2 * len(f)
    if style == "halves":
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
        parts = [z.real, z.imag]
    else:
        z = torch.view_as_complex(x[..., :r].unflatten(-1, (-1, 2)).contiguous()) * turn
        parts = [torch.view_as_real(z).flatten(-2)]
    return torch.cat(parts + [x[..., r:]], -1)


def _exact_append(case, state, new, total):
    size, heads, dim = case["block"], case["kv_heads"], case["dim"]
    q = state["q_out"].double()
    tails, sources = [[], []], [state["k"].double(), state["v"].double()]
    at = 0
    for i, (n, t) in enumerate(zip(new, total)):
        rows, places = slice(at, at + n), list(range(t - n, t))
        at += n
        here = [s[rows] for s in sources]
        if case["rope"] != "none":
            here[0] = _turned(case["rope"], state["k"][rows], places, state["frequencies"])
            q[rows] = _turned(case["rope"], state["q"][rows], places, state["frequencies"])
        first = (t - n) // size
        kept = (t - n) - first * size
        for x, codes, scales, tail in zip(here, ("k_codes", "v_codes"), ("k_scales", "v_scales"), tails):
            block = int(state["table"][i, first])
            old = state[codes][block].double()[:, :kept].transpose(0, 1)  # [token, head, dim]
            before = state[scales][block].double() if kept else torch.zeros(heads, dtype=torch.float64, device="cuda")
            blocks = -(-(kept + n) // size)
            whole = torch.zeros(blocks * size, heads, dim, dtype=torch.float64, device="cuda")
            whole[kept:kept + n] = x
            s = (whole.view(blocks, size, heads, dim).abs().amax((1, 3)) / 127).float().double()  # (scales are f32)
            s[0] = torch.maximum(s[0], before)
            each = s.repeat_interleave(size, 0)[..., None]
            whole = (whole / torch.where(each > 0, each, 1)).round().clamp(-127, 127)
            whole[:kept] = (old * torch.where(s[0] > 0, before / s[0], 0)[None, :, None]).round()
            tail.append((whole * each)[:kept + n])
    out = [torch.cat(t) for t in tails]
    return out if case["rope"] == "none" else out + [q]


def _exact_attend(case, state, new, total):
    if 4 * case["dim"] * case["q_heads"] * sum(n * t for n, t in zip(new, total)) > 2e12:
        return None
    size, group = case["block"], case["q_heads"] // case["kv_heads"]
    out = state["out"].double()
    at = 0
    for i, (n, t) in enumerate(zip(new, total)):
        place = torch.arange(t - n, t, device="cuda")[:, None]
        key = torch.arange(t, device="cuda")
        hidden = torch.zeros(n, t, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= key > place
        if case["window"]:
            hidden |= key <= place - case["window"]
        blocks = state["table"][i, :-(-t // size)].long()
        for h in range(case["kv_heads"]):
            k, v = ((state[c][blocks, h].double() * state[s][blocks, h].double()[:, None, None]).flatten(0, 1)[:t]
                    for c, s in (("k_codes", "k_scales"), ("v_codes", "v_scales")))
            for g in range(h * group, (h + 1) * group):
                s = state["q"][at:at + n, g].double() @ k.T / math.sqrt(case["dim"])
                out[at:at + n, g] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
        at += n
    return out
