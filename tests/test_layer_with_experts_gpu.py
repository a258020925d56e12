"""What a program runs for the drafts of several sessions: per layer a residual norm, the fused projection, rotation and
append, attention over trees of drafts, the output projection, a residual norm with the norm behind the block, a
mixture-of-experts layer. Two layers as one captured graph, replayed over other activations, trees and lengths; each of
the three operators is compared with 64 bits on what stood in front of it."""

import numpy as np
import pytest
import torch

import moe_reference as ref
from kv_reference import attention_tolerance
from test_kv_tree_gpu import attention, named, signed, tree
from test_moe_gpu import prepared, router
from test_residual_norm_gpu import check as check_norm

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV_HEADS, DIM, SIZE, TOP = 256, 8, 2, 64, 16, 2


class Layer:
    def __init__(self, qx, fmt, dtype, rows, seed):
        rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.experts_values = ref.layer(fmt, 8, HIDDEN, 160, shared=1, seed=seed)
        self.experts, self.router = prepared(qx, self.experts_values), router(qx, self.experts_values, TOP, biased=True)
        heads = [HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM]
        packed = [ref.quantised(rng, fmt, n, HIDDEN)[0] for n in heads]
        self.qkv, self.projection = qx.PackedWeights(), qx.PackedWeights()
        qx.check(self.qkv.prepare_fused(fmt, packed, heads, HIDDEN), "qkv")
        qx.check(self.projection.prepare(fmt, ref.quantised(rng, fmt, HIDDEN, HEADS * DIM)[0], HIDDEN, HEADS * DIM), "projection")
        self.weights = [(torch.randn(HIDDEN, generator=gen) * 0.3 + 1).to(dtype).cuda() for _ in range(3)]
        self.first, self.behind, self.second = (qx.Norm(w) for w in self.weights)
        self.cache = qx.KVCache.empty(16, KV_HEADS, SIZE, DIM)

        def rows_of(*shape, kind=torch.float32):
            return torch.zeros(rows, *shape, dtype=kind, device="cuda")

        self.joined, self.normed, self.joined2 = rows_of(HIDDEN), rows_of(HIDDEN), rows_of(HIDDEN)
        self.q, self.k, self.v, self.mixed = (rows_of(n, DIM) for n in (HEADS, KV_HEADS, KV_HEADS, HEADS))
        self.attended, self.normed2, self.out = rows_of(HIDDEN), rows_of(HIDDEN, kind=dtype), rows_of(HIDDEN, kind=dtype)
        self.chosen = torch.zeros(rows, TOP, dtype=torch.int32, device="cuda")

    def run(self, qx, residual, block, batch, rope, depth, masks):
        rows = len(residual)
        qx.check(qx.residual_norm_dev(residual, block, self.joined, self.normed, self.first), "first norm")
        qx.check(self.qkv.qgemm_fused_dev(self.normed, [self.q, self.k, self.v], rows), "qkv")
        qx.check(self.cache.append_dev(batch, self.k, self.v, rope, self.q, self.q, depth), "append")
        qx.check(self.cache.tree_attention_dev(batch, self.q, self.mixed, masks), "attention")
        qx.check(self.projection.qgemm_dev(self.mixed.view(rows, -1), self.attended, rows), "projection")
        qx.check(qx.residual_norm_dev(self.joined, self.attended, self.joined2, self.normed2, self.second, self.behind, None, 0.5),
                 "second norm")
        qx.check(self.experts.apply_dev(self.router, self.normed2, self.out, chosen=self.chosen), "experts")

    def compare(self, qx, residual, block, table, lengths, trees, dtype):
        specs = [(0, w, None, 1e-6, 0.0) for w in self.weights]
        check_norm(residual, block, self.joined, self.normed, specs[0])
        check_norm(self.joined, self.attended, self.joined2, self.normed2, specs[2], specs[1], None, 0.5)
        want, limit = ref.apply(self.experts_values, self.normed2.cpu(), TOP, biased=True, out_type=dtype,
                                chosen=self.chosen.cpu().long())
        assert bool(((self.out.cpu().double() - want).abs() <= limit).all())
        keys, values = (torch.empty(sum(lengths), KV_HEADS, DIM, device="cuda") for _ in "kv")
        begin = torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32, device="cuda")
        whole = qx.KVBatch(torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, 80, begin, sum(lengths), max(lengths))
        qx.check(self.cache.read_dev(whole, keys, values), "read")
        row = key = 0
        for t, length in zip(trees, lengths):
            n = len(t)
            kk, vv = (x[key:key + length].cpu().double() for x in (keys, values))
            exact, sums, magnitude, spread = attention(self.q[row:row + n].cpu().double(), kk, vv, DIM ** -0.5, named(t, length, 0))
            limit, _ = attention_tolerance(exact, sums, magnitude, spread, torch.float32, DIM, length)
            # (read rounds code * scale to f32: half a step of every key and value)
            limit = limit + 2.0 ** -23 * (1 + 2 * spread)[..., None] * magnitude[0]
            assert bool(((self.mixed[row:row + n].cpu().double() - exact).abs() <= limit).all())
            row, key = row + n, key + length


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_layers_for_drafts_as_a_graph(qx, dtype, fmt):
    rng, gen = np.random.default_rng(7), torch.Generator().manual_seed(7)
    new, kept = [7, 1, 4], [37, 5, 60]
    rows, lengths = sum(new), [a + b for a, b in zip(kept, new)]
    table = torch.arange(16, dtype=torch.int32, device="cuda")[torch.tensor([[0, 1, 2, 3, 4], [5, 6, 7, 8, 9], [10, 11, 12, 13, 14]])]
    rope, layers = qx.Rope(DIM), [Layer(qx, fmt, dtype, rows, seed) for seed in (1, 2)]
    begin = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    batch = qx.KVBatch(length, table, 80, begin, rows, max(new))
    masks, depth = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.zeros(rows, dtype=torch.int64, device="cuda")
    hidden, block = torch.zeros(rows, HIDDEN, device="cuda"), torch.zeros(rows, HIDDEN, dtype=torch.float32, device="cuda")

    def fill():
        trees = [tree(rng, n) for n in new]
        masks.copy_(signed([m for t in trees for m in t]))
        depth.copy_(torch.tensor([int(a) - n + bin(m).count("1") - 1 for a, n, t in zip(length.tolist(), new, trees) for m in t]))
        hidden.copy_(torch.randn(rows, HIDDEN, generator=gen))
        block.copy_(torch.randn(rows, HIDDEN, generator=gen))
        return trees

    def step():
        layers[0].run(qx, hidden, block, batch, rope, depth, masks)
        layers[1].run(qx, layers[0].joined2, layers[0].out, batch, rope, depth, masks)

    text = sum(kept)
    text_begin = torch.tensor([0] + list(np.cumsum(kept)), dtype=torch.int32, device="cuda")
    text_batch = qx.KVBatch(torch.tensor(kept, dtype=torch.int32, device="cuda"), table, 80, text_begin, text, max(kept))
    for layer in layers:
        k, v = (torch.randn(text, KV_HEADS, DIM, generator=gen).cuda() for _ in "kv")
        qx.check(layer.cache.append_dev(text_batch, k, v, rope), "text")
    fill()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        trees = fill()
        before = [[a.clone() for a in layer.cache.arrays] for layer in layers]
        graph.replay()
        torch.cuda.synchronize()
        qx.check(qx.lib.qx_check_device_errors(), "layers")
        layers[0].compare(qx, hidden, block, table, length.tolist(), trees, dtype)
        layers[1].compare(qx, layers[0].joined2, layers[0].out, table, length.tolist(), trees, dtype)
        # the same without the graph
        kept_out = [layer.out.clone() for layer in layers]
        for layer, arrays in zip(layers, before):
            for a, b in zip(layer.cache.arrays, arrays):
                a.copy_(b)
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(layer.out, out) for layer, out in zip(layers, kept_out))
        length += torch.tensor([2, 1, 3], dtype=torch.int32, device="cuda")
