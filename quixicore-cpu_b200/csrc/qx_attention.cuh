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
  int kv_heads, block_tokens, dim;
  Heads q, out;
  float* lse;
  float scale_log2;  // scale * log2(e)
  int causal, window;
  int group;         // query heads per kv head
  int row_tiles, splits, chunk;
  float* partial;    // [tile][split][rows][dim] sums, then [tile][split][rows] {maximum, sum}
  float* statistics;
};

// A tile's rows are (token, query head of the group) pairs of one sequence and kv head, token major.
struct Rows {
  long long row;       // of the sequence's first token in the views
  int n, length;       // tokens with rows, tokens in the cache
  int first, count;    // rows of this tile
  int low, high;       // keys [low, high) that any of them sees, low on a multiple of 32
};

__device__ __forceinline__ bool rows_of(const AttentionParams& p, int s, int first, int most, Rows* r) {
  Sequence q;
  if (!sequence_of(p.batch, s, false, &q)) return false;
  const long long total = static_cast<long long>(q.n) * p.group;
  if (first >= total) return false;
  r->row = q.row;
  r->n = q.n;
  r->length = q.length;
  r->first = first;
  r->count = static_cast<int>(min(static_cast<long long>(most), total - first));
  const int start = q.length - q.n;  // (negative where the sequence has more rows than tokens)
  const int position0 = start + first / p.group, position1 = start + (first + r->count - 1) / p.group;
  r->high = max(0, p.causal ? min(q.length, position1 + 1) : q.length);
  r->low = p.window > 0 ? max(0, position0 - p.window + 1) & ~31 : 0;
  r->low = min(r->low, r->high);
  return true;
}
__device__ __forceinline__ int splits_used(const AttentionParams& p, const Rows& r) {
  return max(1, (r.high - r.low + p.chunk - 1) / p.chunk);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// P is held times 2^12 where it is rounded to 16 bits, so that weights down to 2^-26 keep all their bits;
// sums of P carry the same factor.
constexpr float kShift = 12.0f;

}  // namespace kv
}  // namespace qx
