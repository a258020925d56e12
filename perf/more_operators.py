"""The operators around a decoder layer's projections for a few rows at a time, as timed cases:

  join  what lies between two blocks: the norm behind a block, its gate and residual scale, the sum
        with the residual stream, the norm in front of the next block
  moe   a mixture-of-experts feed-forward layer: router, choice of experts, their products with q8_0
        or q4_0 weights, weighted sum
  tree  attention of a tree of drafted tokens over the paged 8-bit cache: each draft sees what is in
        front of the drafts, its ancestors and itself

`run` computes them from elementary torch operations, or (own = True) through the library's entry
points.
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
        # one token of one session between two blocks: latency
        dict(name="join_token_bf16", kind="join", type="bf16", stream="bf16", tokens=1, dim=4096, norm="rms", post=False,
             gate="none", offset=0.0, scale=1.0),
        # a decode step of 64 sessions, norms on both sides of the block, f32 residual stream
        dict(name="join_sandwich_f16", kind="join", type="f16", stream="f32", tokens=64, dim=5120, norm="rms", post=True,
             gate="vector", offset=1.0, scale=0.7),
        # a prompt: bandwidth
        dict(name="join_prompt_bf16", kind="join", type="bf16", stream="bf16", tokens=8192, dim=4096, norm="rms", post=False,
             gate="none", offset=0.0, scale=1.0),
        # texts through an encoder with layer norms, gated by the token, an odd width
        dict(name="join_text_f32", kind="join", type="f32", stream="f32", tokens=1500, dim=1153, norm="layer", post=True,
             gate="token", offset=0.0, scale=0.5),
        # one token of one session, eight of 64 experts: the latency of a decode step
        dict(name="moe_token_q4_bf16", kind="moe", type="bf16", format="q4_0", tokens=1, dim=2048, inner=1024, experts=64,
             shared=0, top=8, score="softmax", bias=False, normalise=True, scale=1.0),
        # eight drafted tokens, two shared experts, scores by sigmoid with a bias for the choice
        dict(name="moe_draft_q8_f16", kind="moe", type="f16", format="q8_0", tokens=8, dim=2048, inner=1408, experts=64,
             shared=2, top=6, score="sigmoid", bias=True, normalise=True, scale=2.5),
        # a decode step of 64 sessions: nearly every expert is touched
        dict(name="moe_step_q4_bf16", kind="moe", type="bf16", format="q4_0", tokens=64, dim=4096, inner=1536, experts=128,
             shared=0, top=8, score="softmax", bias=False, normalise=True, scale=1.0),
        # f32 activations as the projections give them, few large experts, widths off the powers of two
        dict(name="moe_f32_q8", kind="moe", type="f32", format="q8_0", tokens=5, dim=1120, inner=2016, experts=8,
             shared=1, top=2, score="softmax", bias=False, normalise=False, scale=1.0),
        # a small tree behind a short text, f32
        dict(name="tree_one_f32", kind="tree", type="f32", seqs=1, nodes=9, ragged=False, length=1500, q_heads=32, kv_heads=8,
             dim=128, block=64, window=0, packed=False),
        # the trees of a batch of sessions, lengths spread
        dict(name="tree_step_bf16", kind="tree", type="bf16", seqs=16, nodes=16, ragged=True, length=8192, q_heads=32,
             kv_heads=8, dim=128, block=64, window=0, packed=True),
        # wide trees, small heads, a sliding window
        dict(name="tree_wide_f16", kind="tree", type="f16", seqs=6, nodes=63, ragged=True, length=12000, q_heads=24, kv_heads=8,
             dim=64, block=16, window=4096, packed=True),
        # one tree behind a very long text
        dict(name="tree_long_bf16", kind="tree", type="bf16", seqs=1, nodes=48, ragged=False, length=131072, q_heads=64,
             kv_heads=8, dim=128, block=128, window=0, packed=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["join", "moe", "moe", "tree", "tree"])
    typ = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "join":
        dim = rng.choice([_log(rng, 64, 16384), 32 * _log(rng, 4, 512)])
        return dict(kind=kind, type=typ, stream=rng.choice([typ, "f32"]), tokens=_log(rng, 1, min(8192, 8192 * 2048 // dim)),
                    dim=dim, norm=rng.choice(["rms", "rms", "layer"]), post=rng.random() < 0.5,
                    gate=rng.choice(["none", "vector", "token"]), offset=rng.choice([0.0, 1.0]),
                    scale=rng.choice([1.0, 0.25, 1.4]))
    if kind == "moe":
        experts = rng.choice([4, 8, 16, 32, 60, 64, 128, 256])
        shared = rng.choice([0, 0, 1, 2])
        fmt = rng.choice(["q4_0", "q4_0", "q8_0"])
        dim, most = 32 * _log(rng, 8, 160), (4096 if fmt == "q4_0" else 2048) * 128 * 1536
        inner = 32 * _log(rng, 4, max(5, min(256, most // ((experts + shared) * dim * 32))))
        return dict(kind=kind, type=typ, format=fmt, tokens=_log(rng, 1, 64), dim=dim, inner=inner, experts=experts,
                    shared=shared, top=min(experts, rng.choice([1, 2, 4, 6, 8])),
                    score=rng.choice(["softmax", "softmax", "sigmoid"]), bias=rng.random() < 0.3,
                    normalise=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]))
    dim = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    seqs = _log(rng, 1, 32)
    nodes = min(_log(rng, 2, 64), 8 * 64 // kv_heads, max(2, 512 // seqs))
    length = nodes + _log(rng, 1, max(16, min(65536, 12 * 1024 * 1024 * 8 // (kv_heads * dim * seqs))))
    return dict(kind=kind, type=typ, seqs=seqs, nodes=nodes, ragged=rng.random() < 0.6, length=length,
                q_heads=kv_heads * rng.choice([1, 2, 3, 4, 4, 8]), kv_heads=kv_heads, dim=dim,
                block=rng.choice([16, 32, 64, 128]), window=rng.choice([0, 0, 128, 1000, 4096]), packed=rng.random() < 0.5)


def _lengths(case):
    """Drafts and lengths (those included) of every sequence, and rows behind the last one."""
    seqs, nodes, length = case["seqs"], case["nodes"], case["length"]
    new = [max(1, nodes - (nodes * 3 * i) // (5 * seqs)) if case["ragged"] else nodes for i in range(seqs)]
    total = [max(n, length - (length * 5 * i) // (7 * seqs) - 5 * (i % 4)) if seqs > 1 else length for i, n in enumerate(new)]
    return new, total, (3 if case["ragged"] else 0)


def work(case):
    size = torch.empty(0, dtype=TYPES[case["type"]]).element_size()
    if case["kind"] == "join":
        wide = torch.empty(0, dtype=TYPES[case["stream"]]).element_size()
        values = case["tokens"] * case["dim"]
        gate = values * size if case["gate"] == "token" else 0
        return {"bytes": values * 2 * (size + wide) + gate, "flops": 12 * values}
    if case["kind"] == "moe":
        tokens, experts = case["tokens"], case["experts"]
        touched = experts * (1 - (1 - case["top"] / experts) ** tokens) + case["shared"]
        weights = 3 * case["dim"] * case["inner"]
        return {"bytes": touched * weights * (18 if case["format"] == "q4_0" else 34) / 32 + experts * case["dim"] * 2 +
                2 * tokens * case["dim"] * size,
                "flops": 2 * tokens * ((case["top"] + case["shared"]) * weights + experts * case["dim"])}
    new, total, _ = _lengths(case)
    window = case["window"] or max(total)
    keys = sum(min(t, window + n) for n, t in zip(new, total))
    pairs = sum(n * min(t, window) for n, t in zip(new, total))
    return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] + 2 * sum(new) * case["q_heads"] * case["dim"] * size,
            "flops": 4 * case["dim"] * case["q_heads"] * pairs}


# ---- inputs -----------------------------------------------------------------------------

EPS = 1e-6


def _blocks(gen, fmt, *shape):
    """GGUF blocks of normal values of variance 1 / columns: bytes [..., rows, columns / 32 * block bytes]."""
    w = torch.randn(*shape[:-1], shape[-1] // 32, 32, generator=gen, device="cuda") * shape[-1] ** -0.5
    if fmt == "q8_0":
        d = (w.abs().amax(-1, keepdim=True) / 127).half()
        codes = (w / d.float()).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    else:  # the element of the largest magnitude becomes code 0, and 8 stands for zero
        d = (w.gather(-1, w.abs().argmax(-1, keepdim=True)) / -8).half()
        codes = (w / d.float()).add_(8.5).floor_().clamp_(0, 15).to(torch.uint8)
        codes = codes[..., :16] | codes[..., 16:] << 4
    return torch.cat([d.view(torch.uint8), codes], -1).flatten(-2)


def _quantised(gen, blocks, heads, block, dim):
    """Codes [blocks, heads, block, dim] and scales [blocks, heads] of normal values, some heads louder."""
    loud = torch.rand(1, heads, 1, 1, generator=gen, device="cuda") * 1.5 + 0.5
    x = torch.randn(blocks, heads, block, dim, generator=gen, device="cuda") * loud
    s = x.abs().amax((2, 3)) / 127.0
    return (x / s[:, :, None, None]).round_().clamp_(-127, 127).to(torch.int8), s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    state = {"case": dict(case)}

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda") * scale + mean

    if case["kind"] == "join":
        tokens, dim = case["tokens"], case["dim"]
        # some channels of a residual stream are far louder than the others
        loud = torch.where(torch.rand(dim, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
        state["residual"] = (normal(tokens, dim) * loud).to(TYPES[case["stream"]])
        state["block"] = normal(tokens, dim, scale=0.5).to(dtype)
        mean = 1.0 - case["offset"]
        state["pre"] = normal(dim, scale=0.1, mean=mean).to(dtype)
        state["post"] = normal(dim, scale=0.1, mean=mean).to(dtype) if case["post"] else None
        biased = case["norm"] == "layer"
        state["pre_bias"] = normal(dim, scale=0.1).to(dtype) if biased else None
        state["post_bias"] = normal(dim, scale=0.1).to(dtype) if biased and case["post"] else None
        state["gate"] = None
        if case["gate"] != "none":
            state["gate"] = normal(tokens if case["gate"] == "token" else 1, dim, scale=0.3, mean=0.5).to(dtype)
        return state
    if case["kind"] == "moe":
        dim, inner, experts = case["dim"], case["inner"], case["experts"]
        count = experts + case["shared"]
        state["x"] = normal(case["tokens"], dim).to(dtype)
        state["router"] = normal(experts, dim, scale=1.5 * dim ** -0.5).to(torch.bfloat16)
        state["bias"] = normal(experts, scale=0.05) if case["bias"] else None
        state["gate"], state["up"] = (_blocks(gen, case["format"], count, inner, dim) for _ in range(2))
        state["down"] = _blocks(gen, case["format"], count, dim, inner)
        if own:  # the weights as a program keeps them
            state["layer"] = _experts(state)
        return state
    new, total, behind = _lengths(case)
    rows, size = sum(new) + behind, case["block"]
    blocks = sum(-(-t // size) for t in total) + 1
    order = (torch.randperm(blocks - 1, generator=gen, device="cuda") + 1).to(torch.int32)
    table = torch.zeros(case["seqs"], max(-(-t // size) for t in total) + 1, dtype=torch.int32, device="cuda")
    at = 0
    for i, t in enumerate(total):
        n = -(-t // size)
        table[i, :n] = order[at:at + n]
        at += n
    state["k_codes"], state["k_scales"] = _quantised(gen, blocks, case["kv_heads"], size, case["dim"])
    state["v_codes"], state["v_scales"] = _quantised(gen, blocks, case["kv_heads"], size, case["dim"])
    state["table"] = table
    state["lengths"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    state["begin"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    state["rows"], state["max_new"], state["max_length"] = rows, max(new), max(total)
    # a tree's drafts hang on earlier ones, the late ones more often; the first on the text itself
    pick = torch.rand(rows, generator=gen, device="cuda").tolist()
    seen = []
    for n in new:
        first = len(seen)
        for i in range(n):
            parent = min(i - 1, int((1 - pick[first + i] ** 2) * (i + 1)) - 1)
            seen.append((seen[first + parent] if parent >= 0 else 0) | 1 << i)
    seen += [0] * behind
    state["seen"] = torch.tensor([m - (1 << 64) if m >> 63 else m for m in seen], dtype=torch.int64, device="cuda")
    heads = case["q_heads"] + (2 * case["kv_heads"] if case["packed"] else 0)
    state["q"] = normal(rows, heads, case["dim"]).to(dtype)[:, :case["q_heads"]]
    state["out"] = torch.zeros(rows, case["q_heads"], case["dim"], dtype=dtype, device="cuda")
    return state


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    return {"join": _join, "moe": _moe, "tree": _tree}[state["case"]["kind"]](state)


def _norm(case, x, weight, bias):
    if case["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (weight.float() + case["offset"])
    return x if bias is None else x + bias.float()


def _join(state):
    case = state["case"]
    u = state["block"].float()
    if case["post"]:
        u = _norm(case, u, state["post"], state["post_bias"])
    if state["gate"] is not None:
        u = u * state["gate"].float()
    joined = state["residual"].float() + case["scale"] * u
    return [joined.to(state["residual"].dtype), _norm(case, joined, state["pre"], state["pre_bias"]).to(state["block"].dtype)]


def _values(fmt, blocks):
    """The values of GGUF blocks, f32 [..., rows, columns]."""
    b = blocks.unflatten(-1, (-1, 34 if fmt == "q8_0" else 18))
    d, codes = b[..., :2].contiguous().view(torch.float16).float(), b[..., 2:]
    if fmt == "q8_0":
        w = codes.contiguous().view(torch.int8).float()
    else:
        w = torch.cat([codes & 15, codes >> 4], -1).float() - 8
    return (w * d).flatten(-2)


def _moe(state):
    case = state["case"]
    x, fmt = state["x"].float(), case["format"]
    # (logits and scores in 64 bits: two experts may lie next to each other on both sides of the choice)
    logits = x.double() @ state["router"].double().T
    if case["score"] == "softmax":
        score = (logits - logits.amax(-1, keepdim=True)).exp()
        score = score / score.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + (-logits).exp())
    key = logits if state["bias"] is None else score + state["bias"].double()
    chosen = key.sort(dim=-1, descending=True, stable=True).indices[:, :case["top"]]
    weight = score.gather(1, chosen)
    if case["normalise"]:
        weight = weight / weight.sum(-1, keepdim=True)
    share = torch.zeros(case["tokens"], case["experts"] + case["shared"], device="cuda")
    share.scatter_(1, chosen, (weight * case["scale"]).float())
    share[:, case["experts"]:] = 1
    gate, up = (torch.matmul(x, _values(fmt, state[name]).transpose(1, 2)) for name in ("gate", "up"))
    inner = gate / (1 + (-gate).exp()) * up
    each = torch.matmul(inner, _values(fmt, state["down"]).transpose(1, 2))
    return (share.T[:, :, None] * each).sum(0).to(state["x"].dtype)


def _tree(state):
    case = state["case"]
    group, most, length = case["q_heads"] // case["kv_heads"], state["max_new"], state["max_length"]
    begin, lengths, table = state["begin"].long(), state["lengths"].long(), state["table"].long()
    count = begin[1:] - begin[:-1]
    # queries padded to [sequence, kv head, group, draft, dim]
    at = (begin[:-1, None] + torch.arange(most, device="cuda")).clamp(max=state["rows"] - 1)
    q = state["q"][at].float().view(case["seqs"], most, case["kv_heads"], group, case["dim"]).permute(0, 2, 3, 1, 4)
    width = -(-length // case["block"])

    def values(codes, scales):
        x = codes[table[:, :width]].float() * scales[table[:, :width]][..., None, None]
        return x.transpose(1, 2).flatten(2, 3)  # [sequence, kv head, token, dim]

    s = torch.matmul(q, values(state["k_codes"], state["k_scales"])[:, :, None].transpose(-1, -2)) * case["dim"] ** -0.5
    bits = state["seen"][at][..., None] >> torch.arange(64, device="cuda") & 1
    place = (lengths - count)[:, None] + bits.sum(-1) - 1  # of a draft in its text
    key = torch.arange(s.shape[-1], device="cuda")
    draft = key - (lengths - count)[:, None]  # [sequence, key]
    seen = (draft < 0)[:, None, :].expand(-1, most, -1)
    if case["window"]:
        seen = seen & (key > place[..., None] - case["window"])
    named = bits.gather(2, draft.clamp(0, 63)[:, None, :].expand(-1, most, -1)) > 0
    seen = seen | (named & (draft >= 0)[:, None, :] & (draft < count[:, None])[:, None, :])
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, values(state["v_codes"], state["v_scales"])[:, :, None]) / p.sum(-1, keepdim=True)
    # packed rows again; those behind the last sequence stay as they are
    row = torch.arange(state["rows"], device="cuda")
    seq = torch.searchsorted(begin[1:].contiguous(), row, right=True)
    inside = seq < case["seqs"]
    seq = seq.clamp(max=case["seqs"] - 1)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, (row - begin[seq]).clamp(max=most - 1)]
    out = state["out"]
    out.copy_(torch.where(inside[:, None, None], o.to(out.dtype), out))
    return out


# ---- the library's calls ----------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _library():
    import __graft_entry__
    return __graft_entry__.load_package()


def _experts(state):
    qx, case = _library(), state["case"]
    layer = qx.Experts()
    qx.check(layer.prepare_dev(qx.Q8_0 if case["format"] == "q8_0" else qx.Q4_0, state["gate"], state["up"], state["down"],
                               case["experts"], case["dim"], case["inner"], case["shared"]), "experts")
    return layer


def _own(state):
    qx, case = _library(), state["case"]
    if case["kind"] == "join":
        residual, block = state["residual"], state["block"]
        joined, normed = torch.empty_like(residual), torch.empty_like(block)
        kind = qx.NORM_LAYER if case["norm"] == "layer" else qx.NORM_RMS
        pre = qx.Norm(state["pre"], state["pre_bias"], kind, EPS, case["offset"])
        post = qx.Norm(state["post"], state["post_bias"], kind, EPS, case["offset"]) if case["post"] else None
        qx.check(qx.residual_norm_dev(residual, block, joined, normed, pre, post, state["gate"], case["scale"]), "join")
        return [joined, normed]
    if case["kind"] == "moe":
        out = torch.empty_like(state["x"])
        router = qx.Router(state["router"], case["top"], qx.SCORE_SOFTMAX if case["score"] == "softmax" else qx.SCORE_SIGMOID,
                           state["bias"], case["normalise"], case["scale"])
        qx.check(state["layer"].apply_dev(router, state["x"], out), "experts")
        return out
    cache = qx.KVCache(state["k_codes"], state["v_codes"], state["k_scales"], state["v_scales"])
    batch = qx.KVBatch(state["lengths"], state["table"], state["max_length"], state["begin"], state["rows"], state["max_new"])
    qx.check(cache.tree_attention_dev(batch, state["q"], state["out"], state["seen"], window=case["window"]), "tree attention")
    return state["out"]


# ---- 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"join": _exact_join, "moe": _exact_moe, "tree": _exact_tree}[case["kind"]](case, state)


def _exact_join(case, state):
    def norm(v, name):
        w, b = state[name].double() + case["offset"], state[name + "_bias"]
        if case["norm"] == "layer":
            v = (v - v.mean(1, True)) / (v.var(1, unbiased=False, keepdim=True) + EPS).sqrt()
        else:
            v = v / ((v ** 2).sum(1, True) / case["dim"] + EPS).sqrt()
        return v * w + (0 if b is None else b.double())

    v = state["block"].double()
    v = norm(v, "post") if case["post"] else v
    v = v if state["gate"] is None else v * state["gate"].double()
    joined = state["residual"].double() + case["scale"] * v
    return [joined, norm(joined, "pre")]


def _exact_moe(case, state):
    step, experts, top = (34 if case["format"] == "q8_0" else 18), case["experts"], case["top"]

    def matrix(name, e):
        raw = state[name][e].unflatten(1, (-1, step))
        d = raw[:, :, :2].contiguous().view(torch.float16).double()
        q = raw[:, :, 2:]
        if case["format"] == "q8_0":
            q = q.contiguous().view(torch.int8).double()
        else:
            q = torch.cat([q % 16, q // 16], 2).double() - 8
        return (q * d).flatten(1)

    x = state["x"].double()
    logits = x @ state["router"].double().T
    score = logits.softmax(1) if case["score"] == "softmax" else logits.sigmoid()
    rank = score if state["bias"] is None else score + state["bias"].double()
    out = torch.zeros_like(x)
    weights = torch.zeros(case["tokens"], experts + case["shared"], dtype=torch.float64, device="cuda")
    for t in range(case["tokens"]):
        pick = rank[t].topk(top).indices
        w = score[t, pick]
        weights[t, pick] = case["scale"] * (w / w.sum() if case["normalise"] else w)
    weights[:, experts:] = 1
    for e in range(experts + case["shared"]):
        rows = weights[:, e].nonzero()[:, 0]
        if len(rows):
            g = x[rows] @ matrix("gate", e).T
            y = (torch.nn.functional.silu(g) * (x[rows] @ matrix("up", e).T)) @ matrix("down", e).T
            out[rows] += weights[rows, e, None] * y
    return out


def _exact_tree(case, state):
    new, total, _ = _lengths(case)
    size, group = case["block"], case["q_heads"] // case["kv_heads"]
    out = state["out"].double()
    masks = state["seen"].tolist()
    at = 0
    for i, (n, t) in enumerate(zip(new, total)):
        hidden = torch.ones(n, t, dtype=torch.bool)
        for r in range(n):
            mine = [j for j in range(n) if masks[at + r] >> j & 1]
            place = t - n + len(mine) - 1
            hidden[r, max(0, place - case["window"] + 1) if case["window"] else 0:t - n] = False
            hidden[r, [t - n + j for j in mine]] = False
        hidden = hidden.cuda()
        blocks = state["table"][i, :-(-t // size)].long()
        for h in range(case["kv_heads"]):
            k, v = ((state[c][blocks, h].double() * state[s][blocks, h].double()[:, None, None]).flatten(0, 1)[:t]
                    for c, s in (("k_codes", "k_scales"), ("v_codes", "v_scales")))
            for g in range(h * group, (h + 1) * group):
                s = state["q"][at:at + n, g].double() @ k.T / math.sqrt(case["dim"])
                out[at:at + n, g] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
        at += n
    return out
