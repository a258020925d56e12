// Attention over the paged 8-bit cache: which kernel a call takes, how its keys are cut, and the kernel that joins
// chunks. (The streamed kernel: qx_attention_streamed.cuh; that for prompts: qx_attention_tc.cu.)

#include "qx_attention_streamed.cuh"

namespace qx {
namespace kv {
namespace {

// Rows per sequence from which queries take the prompt kernel (f32 ones, of half as many rows per CTA and twice the
// products: later). Streamed | prompt kernel, us: f16, 4 sequences of 4096 keys, 32 rows 37 | 40, 48 rows 48 | 41, 192
// rows 101 | 54; one of 16384 keys, 48 rows 42 | 41; f32, 4 of 4096 keys, 64 rows 84 | 87, 100 rows 96 | 90; 16 whole
// texts of 64 tokens 25 | 29, of 100 tokens 40 | 32.
constexpr long long kPromptFrom = 48, kPromptFromWide = 96;
// Trees of 16-bit rows: as soon as the streamed kernel would read the codes more than once, over texts that are not short.
// Streamed | prompt kernel, us, 24 (44) rows of 128 elements: 16 sequences of 8192 keys 132 | 107 (169 | 107), 4 of 4096 39 | 27 (49 |
// 27), one of 16384 32 | 27 (40 | 27), 4 of 600 16.6 | 18.4 (17.1 | 18.6); of 64 elements, 32 rows, 4 of 4096 24.5 | 24.1.
constexpr long long kPromptFromTree = 17, kPromptFromTreeKeys = 1024;
// Trees whose rows fill one or three tiles of 128 take CTAs of one such tile, two softmax groups sharing its keys; of CTAs with
// two tiles the last would have one to itself. One tile | two tiles a CTA, us, bf16 unless it says f16: 16 sequences of 64 rows, up
// to 8192 keys 107 | 149; 384 rows, 131072 keys 273 | 306; 4 of 320 rows, 8192 keys 109 | 117; 8 of 384 rows, up to 4096 keys
// 57 | 73; one of 384 f16 rows of 64 elements, 16384 keys 45 | 52. An even number: 6 of 189 f16 rows of 64 elements, 4096 keys
// 58 | 44; 4 of 192 rows, 4096 keys 47 | 44. Five tiles, each of which would convert every code: one session of 16384 keys 90 | 84, of
// 131072 537 | 452, 8 of 4096 121 | 106, 16 of 2000 130 | 109, f16 rows of 64 elements 79 | 73; the other way round where CTAs of two
// tiles leave much of the card empty, as 96 of them do (4 of 8192 116 | 177).
constexpr long long kSpreadTiles = 3;

// Joins the chunks of one row, in an order that their number fixes: the threads are cut into parts, a thread of part i
// takes four head elements of chunks i, i + parts, ..., with several chunks' loads under way before it uses the first.
// Few chunks take 128 threads, many 512 (54 chunks of 64 rows: 14 us with 128 threads, one load after the other).
constexpr int kJoinThreads = 512, kJoinBatch = 4;
template <bool kTree>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ AttentionParams p) {
  __shared__ float4 shared[kJoinThreads];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int r = static_cast<int>(blockIdx.x % p.tile_rows);
  const long long tile_index = blockIdx.x / p.tile_rows;
  const int row_tile = static_cast<int>(tile_index % p.row_tiles);
  const int head = static_cast<int>(tile_index / p.row_tiles % p.kv_heads);
  const int s = static_cast<int>(tile_index / p.row_tiles / p.kv_heads);
  const long long first = tile_index * p.splits * p.tile_rows + r;  // chunk c: + c * tile_rows
  const float2* const stats = reinterpret_cast<const float2*>(p.statistics) + first;
  const int vectors = p.dim / 4, parts = blockDim.x / vectors;
  const int part = threadIdx.x / vectors, at = threadIdx.x % vectors;
  const float4* const sums = reinterpret_cast<const float4*>(p.partial + first * p.dim) + at;
  Rows rows;
  if (!rows_of<kTree>(p, s, row_tile * p.tile_rows, p.tile_rows, &rows) || r >= rows.count) return;
  const int used = splits_used(p, rows);
  if (used == 1) return;
  float top = -INFINITY, sum = 0.0f;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int c0 = part < parts ? part : used; c0 < used; c0 += kJoinBatch * parts) {
    float2 stat[kJoinBatch];
    float4 x[kJoinBatch];
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) {
      const long long c = c0 + i * parts;
      stat[i] = c < used ? stats[c * p.tile_rows] : make_float2(-INFINITY, 0.0f);
      x[i] = c < used ? sums[c * p.tile_rows * vectors] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) {
      const float most = fmaxf(top, stat[i].x), base = most == -INFINITY ? 0.0f : most;
      const float keep = exp2_fast(top - base), weight = exp2_fast(stat[i].x - base);
      top = most;
      sum = fmaf(sum, keep, stat[i].y * weight);
      v.x = fmaf(v.x, keep, x[i].x * weight);
      v.y = fmaf(v.y, keep, x[i].y * weight);
      v.z = fmaf(v.z, keep, x[i].z * weight);
      v.w = fmaf(v.w, keep, x[i].w * weight);
    }
  }
  shared[threadIdx.x] = v;
  __shared__ float2 part_stats[kJoinThreads / 4];  // (at most: head sizes start at 16)
  if (at == 0 && part < parts) part_stats[part] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.x >= vectors) return;
  const int token = (rows.first + r) / p.group, member = (rows.first + r) % p.group;
  const long long out_head = static_cast<long long>(head) * p.group + member;
  top = -INFINITY;
  for (int q = 0; q < parts; ++q) top = fmaxf(top, part_stats[q].x);
  const float base = top == -INFINITY ? 0.0f : top;
  sum = 0.0f;
  v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int q = 0; q < parts; ++q) {
    const float weight = exp2_fast(part_stats[q].x - base);
    const float4 x = shared[q * vectors + threadIdx.x];
    sum = fmaf(part_stats[q].y, weight, sum);
    v.x = fmaf(x.x, weight, v.x);
    v.y = fmaf(x.y, weight, v.y);
    v.z = fmaf(x.z, weight, v.z);
    v.w = fmaf(x.w, weight, v.w);
  }
  const float inverse = sum == 0.0f ? 0.0f : exp2f(p.shift) / sum;
  const long long to = (rows.row + token) * p.out.token_stride + out_head * p.out.head_stride + 4 * threadIdx.x;
  store_one(p.out.data, p.out.type, to, v.x * inverse);
  store_one(p.out.data, p.out.type, to + 1, v.y * inverse);
  store_one(p.out.data, p.out.type, to + 2, v.z * inverse);
  store_one(p.out.data, p.out.type, to + 3, v.w * inverse);
  if (threadIdx.x == 0 && p.lse != nullptr) {
    p.lse[(rows.row + token) * p.out.heads + out_head] =
        sum == 0.0f ? -INFINITY : (top + log2f(sum) - p.shift) * 0.69314718055994531f;
  }
}

// The same for trees and few chunks: a CTA takes every `stride`th row of a tile, dim / 4 threads to a row, each all of its chunks
// in their order. (Six trees of 63 drafts, 189 rows, three chunks: 22 us with a thread block per row, which most of these are
// too small for.)
constexpr int kTreeJoinThreads = 256, kTreeJoinSplits = 32;
struct TreeJoin {
  AttentionParams attention;
  int stride;
};
__global__ void __launch_bounds__(kTreeJoinThreads) tree_join_kernel(const __grid_constant__ TreeJoin j) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const AttentionParams& p = j.attention;
  const int first_row = static_cast<int>(blockIdx.x % j.stride);
  const long long tile_index = blockIdx.x / j.stride;
  const int row_tile = static_cast<int>(tile_index % p.row_tiles);
  const int head = static_cast<int>(tile_index / p.row_tiles % p.kv_heads);
  const int s = static_cast<int>(tile_index / p.row_tiles / p.kv_heads);
  Rows rows;
  if (!rows_of<true>(p, s, row_tile * p.tile_rows, p.tile_rows, &rows)) return;
  const int used = splits_used(p, rows);
  if (used == 1) return;
  const int vectors = p.dim / 4, count = (rows.count - first_row + j.stride - 1) / j.stride * vectors;
  for (int i = threadIdx.x; i < count; i += kTreeJoinThreads) {
    const int r = first_row + i / vectors * j.stride, at = i % vectors;
    const long long first = tile_index * p.splits * p.tile_rows + r;
    float top = -INFINITY, sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int kBatch = 8;  // loads under way
    for (int c0 = 0; c0 < used; c0 += kBatch) {
      float2 stat[kBatch];
      float4 x[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        stat[b] = make_float2(-INFINITY, 0.0f);
        x[b] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c0 + b < used) {
          const long long from = first + static_cast<long long>(c0 + b) * p.tile_rows;
          stat[b] = __ldcg(reinterpret_cast<const float2*>(p.statistics) + from);
          x[b] = __ldcg(reinterpret_cast<const float4*>(p.partial + from * p.dim) + at);
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const float most = fmaxf(top, stat[b].x), base = most == -INFINITY ? 0.0f : most;
        const float keep = exp2_fast(top - base), weight = exp2_fast(stat[b].x - base);
        top = most;
        sum = fmaf(sum, keep, stat[b].y * weight);
        v.x = fmaf(v.x, keep, x[b].x * weight);
        v.y = fmaf(v.y, keep, x[b].y * weight);
        v.z = fmaf(v.z, keep, x[b].z * weight);
        v.w = fmaf(v.w, keep, x[b].w * weight);
      }
    }
    const float inverse = sum == 0.0f ? 0.0f : exp2f(p.shift) / sum;
    const int token = (rows.first + r) / p.group, member = (rows.first + r) % p.group;
    const long long out_row = rows.row + token, out_head = static_cast<long long>(head) * p.group + member;
    const long long to = out_row * p.out.token_stride + out_head * p.out.head_stride + 4 * at;
    store_one(p.out.data, p.out.type, to, v.x * inverse);
    store_one(p.out.data, p.out.type, to + 1, v.y * inverse);
    store_one(p.out.data, p.out.type, to + 2, v.z * inverse);
    store_one(p.out.data, p.out.type, to + 3, v.w * inverse);
    if (at == 0 && p.lse != nullptr) {
      p.lse[out_row * p.out.heads + out_head] = sum == 0.0f ? -INFINITY : (top + log2f(sum) - p.shift) * 0.69314718055994531f;
    }
  }
}

}  // namespace

qx_status check_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                          const float* lse, float scale, long long window) {
  QX_TRY(check_cache(cache));
  QX_TRY(check_batch(cache, batch));
  QX_TRY(check_heads(q, batch->tokens, cache->head_dim, false));
  QX_TRY(check_heads(out, batch->tokens, cache->head_dim, true));
  if (q->heads != out->heads || q->heads % cache->kv_heads != 0) return QX_STATUS_INVALID_SHAPE;
  if (static_cast<__int128>(batch->max_tokens) * (q->heads / cache->kv_heads) > 0x7FFFFFFF - 4096) {
    return QX_STATUS_INVALID_SHAPE;
  }
  if (!std::isfinite(scale) || window < 0 || !on_boundary(lse)) return QX_STATUS_INVALID_ARGUMENT;
  if (q->data == out->data && batch->tokens > 0 &&
      (q->type != out->type || q->token_stride != out->token_stride || q->head_stride != out->head_stride)) {
    return QX_STATUS_INVALID_ARGUMENT;  // (the queries' place, but another view)
  }
  return QX_STATUS_OK;
}

qx_status check_tree_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                               const float* lse, float scale, long long window, const uint64_t* seen) {
  QX_TRY(check_attention(cache, batch, q, out, lse, scale, window));
  if (batch->max_tokens > kTreeRows) return QX_STATUS_INVALID_SHAPE;
  // (a narrower window could hide drafts from one another by how deep they are, which masks do not say)
  if (window != 0 && window < kTreeRows) return QX_STATUS_INVALID_ARGUMENT;
  return (batch->tokens > 0 && seen == nullptr) || !on_boundary(seen) ? QX_STATUS_INVALID_ARGUMENT : QX_STATUS_OK;
}

qx_status launch_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                           float* lse, float scale, int causal, long long window, const uint64_t* tree, DeviceContext* ctx,
                           qx_workspace* workspace, cudaStream_t stream) {
  if (batch->sequences == 0 || batch->max_tokens == 0 || batch->tokens == 0) return QX_STATUS_OK;
  AttentionParams p{};
  p.batch = device_batch(cache, batch, ctx->error_dev);
  p.k_codes = cache->k_codes;
  p.v_codes = cache->v_codes;
  p.k_scales = cache->k_scales;
  p.v_scales = cache->v_scales;
  p.kv_heads = cache->kv_heads;
  p.block_tokens = cache->block_tokens;
  while ((1 << p.block_shift) < p.block_tokens) ++p.block_shift;
  p.dim = cache->head_dim;
  p.q = device_heads(q);
  p.out = device_heads(out);
  p.lse = lse;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.causal = causal != 0;
  p.tree = tree;
  p.window = static_cast<int>(std::min<long long>(window, 0x7FFFFFFF));
  p.group = q->heads / cache->kv_heads;
  const long long most_rows = static_cast<long long>(batch->max_tokens) * p.group;
  const bool wide = q->type == QX_STORAGE_F32;
  const long long tree_keys = p.window > 0 ? std::min<long long>(batch->max_length, static_cast<long long>(p.window) + kTreeRows) : batch->max_length;
  const bool long_tree = tree != nullptr && tree_keys >= kPromptFromTreeKeys;
  const bool prompt = cache->head_dim <= 128 && most_rows >= (wide ? kPromptFromWide : long_tree ? kPromptFromTree : kPromptFrom);
  const long long spread_tiles = (most_rows + kPromptRowsSpread - 1) / kPromptRowsSpread;
  const bool spread = prompt && tree != nullptr && !wide && spread_tiles <= kSpreadTiles && spread_tiles % 2 == 1;
  p.tile_rows = prompt ? (wide ? kPromptRowsWide : spread ? kPromptRowsSpread : kPromptRows) : most_rows <= 8 ? 8 : 16;
  p.shift = prompt ? kPromptShift : kShift;
  p.row_tiles = static_cast<int>((most_rows + p.tile_rows - 1) / p.tile_rows);
  const long long items = static_cast<long long>(batch->sequences) * cache->kv_heads * p.row_tiles;
  // Most keys that a tile can see.
  long long range = batch->max_length;
  if (p.window > 0 && tree != nullptr) range = std::min<long long>(range, static_cast<long long>(p.window) + kTreeRows);
  else if (p.window > 0 && p.causal) range = std::min<long long>(range, static_cast<long long>(p.window) + p.tile_rows);
  range += 31;  // (from a multiple of 32 on)
  // Chunks: one sequence fills the card with one round of equal chunks; several, of lengths that only the
  // device knows, get half as many again (measured with 1 | 1.5 | 3 | 6 rounds, us: 32 sessions of 1200 to 8192
  // 87 | 84 | 85 | 85, of up to 2000 31 | 34 | 38 | 38, 8 sessions of up to 20000 64 | 58 | 57 | 67). No chunk is
  // below a tile per warp (in the prompt kernel, four tiles): then the joining would cost more than the keys.
  const int dp = cache->head_dim <= 64 ? 64 : cache->head_dim <= 128 ? 128 : 256;
  const auto streamed = [&](bool balanced, long long grid) {
    return tree == nullptr ? launch_sized<false>(p, dp, wide, balanced, grid, stream) : launch_tree_streamed(p, dp, wide, balanced, grid, stream);
  };
  const long long slots = static_cast<long long>(ctx->prop.multiProcessorCount) * (prompt ? 1 : streamed_ctas(dp, p.tile_rows / 8));
  // Balanced: several sequences; items enough that each has few parts to join (by one CTA, at about 0.15 us a part), and
  // not so many that whole ones even out by themselves; tiles enough per CTA that finding its piece pays. Balanced |
  // chunks, us, 128 elements, 8 kv heads: 32 sessions of up to 8192 64.5 | 76.5, 2048 26.6 | 29.4, 1024 20.0 | 20.8, 700
  // 18.8 | 18.3, 512 15.9 | 12.5; 12 of up to 2000 16.2 | 15.3; 64 of up to 8192 116 | 129, 100 175 | 161.
  const long long counters = static_cast<long long>(batch->sequences) * cache->kv_heads;
  const long long item_tiles = (range + kTile - 1) / kTile, units = counters * (item_tiles + kItemCost);
  if (!prompt && p.row_tiles == 1 && batch->sequences > 1 && batch->sequences <= kBalancedSequences && counters >= slots / 16 &&
      counters <= slots + slots / 2 && counters * item_tiles >= 16 * slots && units < (1LL << 31)) {
    // Two parts per CTA; behind the arrival counters, which the kernel leaves at zero.
    const long long grid = std::min(slots, (units + kLeastPiece - 1) / kLeastPiece);
    const size_t rows = 2 * static_cast<size_t>(grid) * p.tile_rows;
    const size_t sums = align_up(rows * cache->head_dim * sizeof(float), 256);
    QX_TRY(workspace->reserve(kWorkspaceCounterBytes + sums + rows * 2 * sizeof(float)));
    p.counters = static_cast<int*>(workspace->base);
    p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace->base) + kWorkspaceCounterBytes);
    p.statistics = p.partial + sums / sizeof(float);
    return streamed(true, grid);
  }
  const bool one_round = batch->sequences == 1 || prompt;
  const long long wanted = one_round ? std::max(1LL, slots / items) : (3 * slots / 2 + items - 1) / items;
  const long long unit = prompt ? 128 : kTile;
  const long long least = prompt ? 512 : kTile * kWarps * (batch->sequences == 1 ? 1 : 2);
  const long long chunk = (std::max((range + wanted - 1) / wanted, least) + unit - 1) / unit * unit;
  p.chunk = static_cast<int>(chunk);
  p.splits = static_cast<int>(std::max(1LL, (range + chunk - 1) / chunk));
  if (p.splits > 1) {
    const size_t rows = static_cast<size_t>(items) * p.splits * p.tile_rows;
    const size_t sums = align_up(rows * cache->head_dim * sizeof(float), 256);
    // (behind the arrival counters that other kernels keep at the workspace's start)
    QX_TRY(workspace->reserve(kWorkspaceCounterBytes + sums + rows * 2 * sizeof(float)));
    p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace->base) + kWorkspaceCounterBytes);
    p.statistics = p.partial + sums / sizeof(float);
    // few parts are joined by the last CTA to arrive, which saves a launch (2 us of the host's time; on the device 1000
    // keys of 8 kv heads take 7.7 us either way); many by a kernel that spreads them out (8 kv heads of 8 rows, 4000 keys
    // 11.4 us | joined by the last CTA 14.1, 8000 keys 13.0 | 18.3)
    if (!prompt && p.splits <= 16 && items <= static_cast<long long>(kWorkspaceCounterBytes / sizeof(int))) {
      p.counters = static_cast<int*>(workspace->base);
    }
  }
  const long long grid = items * p.splits;
  QX_TRY(prompt ? launch_prompt(p, wide, spread, grid, stream) : streamed(false, grid));
  if (p.splits <= 1 || p.counters != nullptr) return QX_STATUS_OK;
  if (tree != nullptr && p.splits <= kTreeJoinSplits) {
    // two CTAs per SM, of a thread's worth of rows at least
    const int most = std::max(1, p.tile_rows * (p.dim / 4) / kTreeJoinThreads);
    const int stride = static_cast<int>(std::min<long long>(most, std::max(1LL, 2LL * ctx->prop.multiProcessorCount / items)));
    return launch_behind(tree_join_kernel, items * stride, kTreeJoinThreads, 0, stream, TreeJoin{p, stride});
  }
  return launch_behind(tree == nullptr ? join_kernel<false> : join_kernel<true>, items * p.tile_rows, p.splits <= 16 ? 128 : kJoinThreads, 0, stream, p);
}

}  // namespace kv
}  // namespace qx

using namespace qx;

extern "C" qx_status qx_kv_attention_dev(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q,
                                         const qx_heads* out, float* lse_dev, float scale, int causal, long long window,
                                         qx_workspace* workspace, void* stream) {
  QX_TRY(kv::check_attention(cache, batch, q, out, lse_dev, scale, window));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  if (workspace == nullptr) workspace = &ctx->workspace;
  if (workspace->device != ctx->device) return QX_STATUS_INVALID_ARGUMENT;
  return kv::launch_attention(cache, batch, q, out, lse_dev, scale, causal, window, nullptr, ctx, workspace,
                              static_cast<cudaStream_t>(stream));
}

extern "C" qx_status qx_kv_tree_attention_dev(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q,
                                              const qx_heads* out, float* lse_dev, float scale, long long window,
                                              const uint64_t* seen_dev, qx_workspace* workspace, void* stream) {
  QX_TRY(kv::check_tree_attention(cache, batch, q, out, lse_dev, scale, window, seen_dev));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  if (workspace == nullptr) workspace = &ctx->workspace;
  if (workspace->device != ctx->device) return QX_STATUS_INVALID_ARGUMENT;
  return kv::launch_attention(cache, batch, q, out, lse_dev, scale, 1, window, seen_dev, ctx, workspace,
                              static_cast<cudaStream_t>(stream));
}
