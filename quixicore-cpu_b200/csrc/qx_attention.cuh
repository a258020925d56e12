// What the attention kernels over the 8-bit cache share: parameters and the range of keys that a tile of
// rows sees.
#pragma once

#include "qx_kv.cuh"

namespace qx {
namespace kv {

struct AttentionParams {
  Batch batch;
  const int8_t* k_codes;
  const int8_t* v_codes;
  const float* k_scales;
  const float* v_scales;
  int kv_heads, block_tokens, block_shift, dim;  // (block_tokens = 1 << block_shift)
  Heads q, out;
  float* lse;
  float scale_log2;  // scale * log2(e)
  int causal, window;
  const uint64_t* tree;  // [row of the views] drafts that it sees; NULL: no trees
  int group;         // query heads per kv head
  int tile_rows;     // rows of a tile
  int row_tiles, splits, chunk;
  float shift;       // log2 of what sums of weights carry (and those of weights times values do not)
  float* partial;    // [tile][split][rows][dim] sums, then [tile][split][rows] {maximum, sum}
  float* statistics;
  int* counters;     // [item] CTAs that have written a part, zero between calls; NULL: another kernel joins
};

// A tile's rows are (token, query head of the group) pairs of one sequence and kv head, token major.
struct Rows {
  long long row;       // of the sequence's first token in the views
  int n, length;       // tokens with rows, tokens in the cache
  int first, count;    // rows of this tile
  int low, high;       // keys [low, high) that any of them sees, low on a multiple of 32
};

// The first key that a row at `position` sees. (No difference with more than 31 bits: positions of rows that a sequence
// has beyond its tokens are negative, a window may be as wide as whole numbers go.)
__device__ __forceinline__ int first_seen(const AttentionParams& p, int position) {
  return p.window > 0 && position >= p.window ? position - p.window + 1 : 0;
}

// kTree: the sequence's rows are drafts, row i sees those in front of them and draft j where bit j of its mask says so. Its
// position is the one behind as many drafts as it sees, itself among them.
constexpr int kTreeRows = 64;
__device__ __forceinline__ uint64_t drafts_of(const AttentionParams& p, const Rows& r, int token) {
  return p.tree[r.row + token] & (r.n >= kTreeRows ? ~0ull : (1ull << r.n) - 1);
}
// Which of the kKeys (16 or 32) keys from `key` on a row sees: bit i, key + i. `low`: its first key; `start`: the first draft.
template <int kKeys>
__device__ __forceinline__ uint32_t seen_of(uint64_t drafts, int key, int start, int low) {
  constexpr uint32_t kAll = static_cast<uint32_t>((1ull << kKeys) - 1);
  const int in = key - start;  // (the drafts end the text: nothing is behind them)
  uint32_t seen = in >= kTreeRows ? 0u : in >= 0 ? static_cast<uint32_t>(drafts >> in)
                  : in > -kKeys ? static_cast<uint32_t>(drafts << -in) | ((1u << -in) - 1) : kAll;
  const int hidden = min(max(low - key, 0), kKeys);
  return seen & kAll & static_cast<uint32_t>(~((1ull << hidden) - 1));
}

template <bool kTree = false>
__device__ __forceinline__ bool rows_of(const AttentionParams& p, int s, int first, int most, Rows* r, bool each = false) {
  Sequence q;
  if (!sequence_of(p.batch, s, false, &q, each)) return false;
  const long long total = static_cast<long long>(q.n) * p.group;
  if (first >= total) return false;
  r->row = q.row;
  r->n = q.n;
  r->length = q.length;
  r->first = first;
  r->count = static_cast<int>(min(static_cast<long long>(most), total - first));
  const int start = q.length - q.n;  // (negative where the sequence has more rows than tokens)
  const int position0 = kTree ? start - 1 : start + first / p.group, position1 = start + (first + r->count - 1) / p.group;
  r->high = max(0, p.causal && !kTree ? min(q.length, position1 + 1) : q.length);
  r->low = first_seen(p, position0) & ~31;
  r->low = min(r->low, r->high);
  return true;
}
__device__ __forceinline__ int splits_used(const AttentionParams& p, const Rows& r) {
  return max(1, static_cast<int>((static_cast<long long>(r.high) - r.low + p.chunk - 1) / p.chunk));
}
// Keys [begin, end) of a chunk; false where there is nothing to do (chunk 0 always has: rows that see nothing).
__device__ __forceinline__ bool chunk_of(const AttentionParams& p, const Rows& r, int split, int* begin, int* end) {
  const long long at = r.low + static_cast<long long>(split) * p.chunk;
  if (split > 0 && at >= r.high) return false;
  *begin = static_cast<int>(at);
  *end = static_cast<int>(min(static_cast<long long>(r.high), at + p.chunk));
  return true;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows per CTA of the prompt kernel (qx_attention_tc.cu; f32 queries), and its shift: P is held times 2^11 .. 2^15
// there.
constexpr int kPromptRows = 256, kPromptRowsWide = 128, kPromptRowsSpread = 128;
constexpr float kPromptShift = 11.0f;
// `spread`: of trees, 16-bit queries, in tiles of 128 rows.
qx_status launch_prompt(const AttentionParams& p, bool wide, bool spread, long long grid, cudaStream_t stream);
// The streamed kernel for trees (qx_attention_tree.cu).
qx_status launch_tree_streamed(const AttentionParams& p, int dp, bool wide, bool balanced, long long grid, cudaStream_t stream);

}  // namespace kv
}  // namespace qx
