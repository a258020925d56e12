// Attention over the paged 8-bit cache, streamed: the kernel for single tokens, short runs of tokens, f32
// queries and every head size. (Long prompts of 16-bit queries: qx_attention_tc.cu.)
//
// softmax(scale q K^T) V with K = ks * codes, V = vs * codes. The codes are exact in f16, so the products
// run on warp-level f16 MMAs with f32 sums and the scales are applied to the sums: one multiplication per
// score (ks) and one per 32 tokens and output element (vs). Queries enter as f16 times a power of two of
// their own per row: exact for f16 and bf16, hi + lo pairs (22 bits) for f32. Weights enter as f16 (a
// rounding of 2^-12 relative, no further than the 16-bit outputs' own), as hi + lo pairs for f32.
//
// Split. A CTA takes 16 rows (tokens x query heads of one kv head) and a chunk of the keys; its four warps
// take tiles of 32 keys in turn, each with a running maximum and sum of its own, and are joined at the end
// through shared memory. So one pass over the codes serves all heads of a group, and the card is filled by
// chunks where there are few rows; chunks are joined by a second, small kernel in a fixed order.
//
// Data movement. Each warp has a ring of three stages of its own (codes of 32 keys and values, their
// scales), filled by 16-byte asynchronous copies: two tiles in flight while a third is computed, nothing to
// wait for but the warp's own copies. Codes go from shared memory to MMA operands without a shuffle: the
// order of head elements inside a product, of keys inside P V and of output columns are free, so each lane
// takes the bytes that lie together (16 of a key row, 16 columns of four value rows) and turns them into
// f16 pairs by byte permutes (0x6400 | code + 128 is 1024 + code + 128). 16-byte pieces of a row are
// permuted among the eight bank groups so that these reads meet no conflicts for head sizes up to 128.
//
// Bound by HBM for long contexts: 2 * head_dim bytes per key and kv head, whatever the group.

#include <algorithm>
#include <cmath>

#include "qx_attention.cuh"

namespace qx {
namespace kv {


namespace {

// P is held times 2^12 where it is rounded to 16 bits, so that weights down to 2^-26 keep all their bits;
// sums of P carry the same factor.
constexpr float kShift = 12.0f;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kStages = 3, kTile = 32, kRows = 16;

// Rows per sequence from which 16-bit queries take the prompt kernel.
constexpr long long kPromptFrom = 64;

template <int DP>
struct Shape {
  static constexpr int kChunks = DP / 16;                      // 16-byte pieces of a row
  static constexpr int kStageBytes = 2 * kTile * DP + 32;      // keys, values, scales and flags
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kPitch = DP + 4;                        // floats per row when warps are joined
  static constexpr int kJoin = kWarps * kRows * (kPitch + 2) * 4;
  static constexpr int kQueries = kRows * DP * 2;              // f16 fragments, hi or lo
  static constexpr int kCtas = DP == 64 ? 4 : DP == 128 ? 2 : 1;
};
template <int DP, bool kWide>
constexpr int smem_bytes() {
  return std::max(Shape<DP>::kRing, Shape<DP>::kJoin) + Shape<DP>::kQueries * (kWide ? 2 : 1) + kRows * 4;
}

// Byte offset of 16-byte piece c of row r in a stage.
template <int DP>
__device__ __forceinline__ int piece(int r, int c) {
  if (DP == 64) {
    const int line = r >> 1;
    return line * 128 + ((((r & 1) * 4 + c) ^ (2 * (line & 3))) << 4);
  }
  if (DP == 128) return r * 128 + ((c ^ (r & 7)) << 4);
  return r * 256 + (c >> 3) * 128 + (((c & 7) ^ (r & 7)) << 4);
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
template <int kLeft>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Two of four biased codes (code + 128) as a pair of f16 codes.
template <int kPair>
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased) {
  const uint32_t raw = __byte_perm(biased, 0x64646464u, kPair == 0 ? 0x4140 : 0x4342);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&raw), __half2half2(__ushort_as_half(0x6480)));  // 1152
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pair_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What is left of a and b beside their f16 roundings.
__device__ __forceinline__ uint32_t rest_f16(float a, float b, uint32_t rounded) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
  return pair_f16(a - f.x, b - f.y);
}

template <int DP, bool kWide>
__global__ void __launch_bounds__(kThreads, Shape<DP>::kCtas) attention_kernel(const __grid_constant__ AttentionParams p) {
  using S = Shape<DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  uint8_t* const queries = smem + (S::kRing > S::kJoin ? S::kRing : S::kJoin);
  float* const row_factor = reinterpret_cast<float*>(queries + S::kQueries * (kWide ? 2 : 1));

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  long long index = blockIdx.x;
  const int split = static_cast<int>(index % p.splits);
  index /= p.splits;
  const long long tile_index = index;
  const int row_tile = static_cast<int>(index % p.row_tiles);
  index /= p.row_tiles;
  const int head = static_cast<int>(index % p.kv_heads), s = static_cast<int>(index / p.kv_heads);
  Rows rows;
  if (!rows_of(p, s, row_tile * kRows, kRows, &rows)) return;
  int begin, end;
  if (!chunk_of(p, rows, split, &begin, &end)) return;
  const int32_t* const table = p.batch.table + s * p.batch.table_stride;
  const int tiles = (end - begin + kTile - 1) / kTile;  // (zero or less: the rows see nothing)

  // ---- copies -------------------------------------------------------------------------------
  const uint32_t ring = sm100::smem_u32(smem) + warp * (kStages * S::kStageBytes);
  uint8_t* const ring_bytes = smem + warp * (kStages * S::kStageBytes);
  const int pieces = p.dim / 16;
  // Ids of the two blocks that a tile's halves lie in (the same one from 32 tokens per block on); -1: nothing to see.
  const auto ids_of = [&](int tile, int (&id)[2]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int token = begin + tile * kTile + 16 * half;
      id[half] = -1;
      if (tile < tiles && token < end) {
        const int block = table[token / p.block_tokens];
        if (block >= 0 && block < p.batch.blocks) id[half] = block;
        else if (lane == 0) sm100::report_error(p.batch.error, kErrorBlock);
      }
    }
  };
  const auto issue = [&](int tile, const int (&id)[2]) {
    const int stage = tile / kWarps % kStages;
    const uint32_t to = ring + stage * S::kStageBytes;
    float* const meta = reinterpret_cast<float*>(ring_bytes + stage * S::kStageBytes + 2 * kTile * DP);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int slot = (begin + tile * kTile + 16 * half) % p.block_tokens;
      if (lane == 0) reinterpret_cast<int*>(meta)[4 + half] = id[half] >= 0;
      if (id[half] < 0) {
        if (lane == 0) meta[half] = meta[2 + half] = 0.0f;
        continue;
      }
      const long long slice = static_cast<long long>(id[half]) * p.kv_heads + head;
      const long long at = (slice * p.block_tokens + slot) * p.dim;
      if (lane == 0) copy4(to + 2 * kTile * DP + 4 * half, p.k_scales + slice);
      if (lane == 1) copy4(to + 2 * kTile * DP + 8 + 4 * half, p.v_scales + slice);
#pragma unroll
      for (int i = 0; i < S::kChunks / 2; ++i) {
        const int item = i * 32 + lane, r = item / S::kChunks, c = item % S::kChunks;
        if (DP != p.dim && c >= pieces) continue;
        const int where = piece<DP>(16 * half + r, c);
        const long long from = at + r * p.dim + 16 * c;
        copy16(to + where, p.k_codes + from);
        copy16(to + kTile * DP + where, p.v_codes + from);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int next_ids[2];
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    ids_of(warp + i * kWarps, next_ids);
    if (warp + i * kWarps < tiles) issue(warp + i * kWarps, next_ids);
    else asm volatile("cp.async.commit_group;" ::: "memory");
  }
  ids_of(warp + (kStages - 1) * kWarps, next_ids);

  // ---- queries: f16 times a power of two that brings the row's largest magnitude to 2^7 .. 2^8 -------------
  for (int r = warp; r < kRows; r += kWarps) {
    float v[DP / 32];
    uint32_t top = 0;
    long long base = 0;
    if (r < rows.count) {
      const int token = (rows.first + r) / p.group, member = (rows.first + r) % p.group;
      base = (rows.row + token) * p.q.token_stride + (static_cast<long long>(head) * p.group + member) * p.q.head_stride;
    }
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
      const int d = i * 32 + lane;
      v[i] = r < rows.count && d < p.dim ? load_one(p.q.data, p.q.type, base + d) : 0.0f;
      top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top) >> 23;
    const int shift = top >= 255 ? 0 : min(120, max(-120, 134 - static_cast<int>(top)));
    const float factor = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
    if (lane == 0) row_factor[r] = __uint_as_float(static_cast<uint32_t>(127 - shift) << 23) * p.scale_log2;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
      const int d = i * 32 + lane, own_t = d / (DP / 4), rest = d % (DP / 4);
      const int at = ((rest / 4 * 32 + (r & 7) * 4 + own_t) * 4 + (rest % 4 >> 1) * 2 + (r >> 3)) * 2 + (rest & 1);
      const float x = v[i] * factor;
      const __half hi = __float2half_rn(x);
      reinterpret_cast<__half*>(queries)[at] = hi;
      if (kWide) reinterpret_cast<__half*>(queries + S::kQueries)[at] = __float2half_rn(x - __half2float(hi));
    }
  }
  __syncthreads();
  constexpr bool kResident = !kWide && DP <= 128;
  uint32_t resident[kResident ? DP / 16 : 1][4];
  if (kResident) {
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      const uint4 f = reinterpret_cast<const uint4*>(queries)[j * 32 + lane];
      resident[j][0] = f.x;
      resident[j][1] = f.y;
      resident[j][2] = f.z;
      resident[j][3] = f.w;
    }
  }
  const float factor0 = row_factor[g], factor1 = row_factor[g + 8];
  // keys [low, high) of this lane's two rows
  int low0 = 0, high0 = 0, low1 = 0, high1 = 0;
  {
    const int start = rows.length - rows.n;
    const auto bounds = [&](int r, int* low, int* high) {
      if (r >= rows.count) return;
      const int position = start + (rows.first + r) / p.group;
      *high = p.causal ? min(rows.length, position + 1) : rows.length;
      *low = p.window > 0 ? max(0, position - p.window + 1) : 0;
    };
    bounds(g, &low0, &high0);
    bounds(g + 8, &low1, &high1);
  }
  const int start = rows.length - rows.n, position0 = start + rows.first / p.group;
  const int position1 = start + (rows.first + rows.count - 1) / p.group;
  const int open_high = p.causal ? min(rows.length, position0 + 1) : rows.length;  // below: no key is hidden
  const int open_low = p.window > 0 ? max(0, position1 - p.window + 1) : 0;

  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float max0 = -INFINITY, max1 = -INFINITY, sum0 = 0.0f, sum1 = 0.0f;

  for (int tile = warp; tile < tiles; tile += kWarps) {
    const int ahead = tile + (kStages - 1) * kWarps;
    if (ahead < tiles) issue(ahead, next_ids);
    else asm volatile("cp.async.commit_group;" ::: "memory");
    ids_of(ahead + kWarps, next_ids);
    wait_copies<kStages - 1>();
    __syncwarp();
    const uint8_t* const keys = ring_bytes + tile / kWarps % kStages * S::kStageBytes;
    const uint8_t* const values = keys + kTile * DP;
    const float* const meta = reinterpret_cast<const float*>(values + kTile * DP);
    const int token0 = begin + tile * kTile;

    // ---- scores ---------------------------------------------------------------------------
    float score[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) score[n][0] = score[n][1] = score[n][2] = score[n][3] = 0.0f;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
      uint32_t w[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint4 f = *reinterpret_cast<const uint4*>(keys + piece<DP>(8 * n + g, DP / 64 * t + i));
        w[n][0] = f.x ^ 0x80808080u;
        w[n][1] = f.y ^ 0x80808080u;
        w[n][2] = f.z ^ 0x80808080u;
        w[n][3] = f.w ^ 0x80808080u;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = 4 * i + k;
        uint32_t a[4], low[4];
        if (kResident) {
          a[0] = resident[j % (DP / 16)][0];
          a[1] = resident[j % (DP / 16)][1];
          a[2] = resident[j % (DP / 16)][2];
          a[3] = resident[j % (DP / 16)][3];
        } else {
          const uint4 f = reinterpret_cast<const uint4*>(queries)[j * 32 + lane];
          a[0] = f.x;
          a[1] = f.y;
          a[2] = f.z;
          a[3] = f.w;
        }
        if (kWide) {
          const uint4 f = reinterpret_cast<const uint4*>(queries + S::kQueries)[j * 32 + lane];
          low[0] = f.x;
          low[1] = f.y;
          low[2] = f.z;
          low[3] = f.w;
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t b0 = codes_f16<0>(w[n][k]), b1 = codes_f16<1>(w[n][k]);
          mma16816(score[n], a, b0, b1);
          if (kWide) mma16816(score[n], low, b0, b1);
        }
      }
    }

    // ---- softmax --------------------------------------------------------------------------
    const float ks[2] = {meta[0], meta[1]}, vs[2] = {meta[2], meta[3]};
    const int present = (reinterpret_cast<const int*>(meta)[4] ? 1 : 0) | (reinterpret_cast<const int*>(meta)[5] ? 2 : 0);
    const bool open = token0 + kTile <= open_high && token0 >= open_low && present == 3;
    float top0 = -INFINITY, top1 = -INFINITY;
    bool seen0 = true, seen1 = true;  // whether the row sees any key of the tile
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float f0 = factor0 * ks[n >> 1], f1 = factor1 * ks[n >> 1];
      score[n][0] *= f0;
      score[n][1] *= f0;
      score[n][2] *= f1;
      score[n][3] *= f1;
    }
    if (!open) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = token0 + 8 * n + 2 * t + e;
          const bool there = present >> (n >> 1) & 1;
          if (!(there && key >= low0 && key < high0)) score[n][e] = -INFINITY;
          if (!(there && key >= low1 && key < high1)) score[n][2 + e] = -INFINITY;
        }
      }
      const auto sees = [&](int low, int high) {
        return ((present & 1) && low < token0 + 16 && high > max(token0, low)) ||
               ((present & 2) && low < token0 + 32 && high > max(token0 + 16, low));
      };
      seen0 = sees(low0, high0);
      seen1 = sees(low1, high1);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      top0 = fmaxf(top0, fmaxf(score[n][0], score[n][1]));
      top1 = fmaxf(top1, fmaxf(score[n][2], score[n][3]));
    }
#pragma unroll
    for (int h = 1; h <= 2; h <<= 1) {
      top0 = fmaxf(top0, __shfl_xor_sync(0xFFFFFFFFu, top0, h));
      top1 = fmaxf(top1, __shfl_xor_sync(0xFFFFFFFFu, top1, h));
    }
    top0 = fmaxf(top0, max0);
    top1 = fmaxf(top1, max1);
    // (a row that has seen nothing yet: weights exp2(-inf) = 0 against any finite maximum)
    const float base0 = top0 == -INFINITY ? 0.0f : top0, base1 = top1 == -INFINITY ? 0.0f : top1;
    const float keep0 = exp2_fast(max0 - base0), keep1 = exp2_fast(max1 - base1);
    max0 = top0;
    max1 = top1;
    sum0 *= keep0;
    sum1 *= keep1;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      score[n][0] = exp2_fast(score[n][0] - base0 + kShift);
      score[n][1] = exp2_fast(score[n][1] - base0 + kShift);
      score[n][2] = exp2_fast(score[n][2] - base1 + kShift);
      score[n][3] = exp2_fast(score[n][3] - base1 + kShift);
      sum0 += score[n][0] + score[n][1];
      sum1 += score[n][2] + score[n][3];
    }
    // One scale for the tile's values: the larger of its two blocks', the weights take the ratio. (Beside a scale
    // that is no number the larger is the other; with that at zero, any does.) A weight of zero that a mask has
    // made stays zero beside a scale that is no number.
    float scale = vs[0];
    if (p.block_tokens < kTile) {
      scale = fmaxf(vs[0], vs[1]);
      if (!(scale > 0.0f)) scale = 1.0f;
      if (vs[0] != scale || vs[1] != scale) {
        const float ratio[2] = {vs[0] / scale, vs[1] / scale};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = token0 + 8 * n + 2 * t + (e & 1);
            const bool visible = open || ((present >> (n >> 1) & 1) && key >= (e < 2 ? low0 : low1) && key < (e < 2 ? high0 : high1));
            score[n][e] = visible ? score[n][e] * ratio[n >> 1] : 0.0f;
          }
        }
      }
    }
    const float gain0 = seen0 ? scale : 0.0f, gain1 = seen1 ? scale : 0.0f;

    // ---- weights x values -----------------------------------------------------------------
    uint32_t weight[2][4], low_weight[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = score[2 * k + (e >> 1)][(e & 1) * 2], b = score[2 * k + (e >> 1)][(e & 1) * 2 + 1];
        weight[k][e] = pair_f16(a, b);
        if (kWide) low_weight[k][e] = rest_f16(a, b, weight[k][e]);
      }
    }
    constexpr int kWords = DP == 64 ? 2 : 4;  // of a value row per lane and load
#pragma unroll
    for (int i = 0; i < (DP == 256 ? 2 : 1); ++i) {
      uint32_t w[2][4][kWords];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 16 * k + 2 * t + (e & 1) + 8 * (e >> 1);
          if (DP == 64) {
            const uint2 f = *reinterpret_cast<const uint2*>(values + piece<DP>(r, g >> 1) + 8 * (g & 1));
            w[k][e][0] = f.x;
            w[k][e][1] = f.y;
          } else {
            const uint4 f = *reinterpret_cast<const uint4*>(values + piece<DP>(r, DP / 128 * g + i));
            w[k][e][0] = f.x;
            w[k][e][1] = f.y;
            w[k][e][kWords - 2] = f.z;
            w[k][e][kWords - 1] = f.w;
          }
        }
      }
#pragma unroll
      for (int word = 0; word < kWords; ++word) {
        float acc[4][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t x0 = __byte_perm(w[k][0][word], w[k][1][word], 0x5140) ^ 0x80808080u;
          const uint32_t x1 = __byte_perm(w[k][0][word], w[k][1][word], 0x7362) ^ 0x80808080u;
          const uint32_t y0 = __byte_perm(w[k][2][word], w[k][3][word], 0x5140) ^ 0x80808080u;
          const uint32_t y1 = __byte_perm(w[k][2][word], w[k][3][word], 0x7362) ^ 0x80808080u;
          const uint32_t b[4][2] = {{codes_f16<0>(x0), codes_f16<0>(y0)}, {codes_f16<1>(x0), codes_f16<1>(y0)},
                                    {codes_f16<0>(x1), codes_f16<0>(y1)}, {codes_f16<1>(x1), codes_f16<1>(y1)}};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            mma16816(acc[e], weight[k], b[e][0], b[e][1]);
            if (kWide) mma16816(acc[e], low_weight[k], b[e][0], b[e][1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float (&out)[4] = o[16 * i + 4 * word + e];
          out[0] = fmaf(acc[e][0], gain0, out[0] * keep0);
          out[1] = fmaf(acc[e][1], gain0, out[1] * keep0);
          out[2] = fmaf(acc[e][2], gain1, out[2] * keep1);
          out[3] = fmaf(acc[e][3], gain1, out[3] * keep1);
        }
      }
    }
    __syncwarp();  // the stage is free for the next copies
  }

  // ---- the four warps joined ---------------------------------------------------------------
#pragma unroll
  for (int h = 1; h <= 2; h <<= 1) {
    sum0 += __shfl_xor_sync(0xFFFFFFFFu, sum0, h);
    sum1 += __shfl_xor_sync(0xFFFFFFFFu, sum1, h);
  }
  wait_copies<0>();
  __syncthreads();
  float* const joined = reinterpret_cast<float*>(smem);
  float* const stats = joined + kWarps * kRows * S::kPitch;  // [warp][row] {maximum, sum}
  {
    // column n of output fragment i is head element DP / 8 * n + i
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float* const to = joined + (warp * kRows + g + (e >> 1) * 8) * S::kPitch + (2 * t + (e & 1)) * (DP / 8);
#pragma unroll
      for (int i = 0; i < DP / 8; i += 4) {
        *reinterpret_cast<float4*>(to + i) = make_float4(o[i][e], o[i + 1][e], o[i + 2][e], o[i + 3][e]);
      }
    }
    if (t == 0) {
      *reinterpret_cast<float2*>(stats + 2 * (warp * kRows + g)) = make_float2(max0, sum0);
      *reinterpret_cast<float2*>(stats + 2 * (warp * kRows + g + 8)) = make_float2(max1, sum1);
    }
  }
  __syncthreads();
  const bool whole = splits_used(p, rows) == 1;
  const int per_row = p.dim / 8;
  for (int i = threadIdx.x; i < rows.count * per_row; i += kThreads) {
    const int r = i / per_row, d = (i - r * per_row) * 8;
    float top = -INFINITY, sum = 0.0f, v[8], weight[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats[2 * (w * kRows + r)]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      weight[w] = exp2_fast(stats[2 * (w * kRows + r)] - base);
      sum += stats[2 * (w * kRows + r) + 1] * weight[w];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4* const from = reinterpret_cast<const float4*>(joined + (w * kRows + r) * S::kPitch + d);
      const float4 a = from[0], b = from[1];
      v[0] = fmaf(a.x, weight[w], v[0]);
      v[1] = fmaf(a.y, weight[w], v[1]);
      v[2] = fmaf(a.z, weight[w], v[2]);
      v[3] = fmaf(a.w, weight[w], v[3]);
      v[4] = fmaf(b.x, weight[w], v[4]);
      v[5] = fmaf(b.y, weight[w], v[5]);
      v[6] = fmaf(b.z, weight[w], v[6]);
      v[7] = fmaf(b.w, weight[w], v[7]);
    }
    if (!whole) {
      const long long at = (tile_index * p.splits + split) * kRows + r;
      float4* const to = reinterpret_cast<float4*>(p.partial + at * p.dim + d);
      to[0] = make_float4(v[0], v[1], v[2], v[3]);
      to[1] = make_float4(v[4], v[5], v[6], v[7]);
      if (d == 0) *reinterpret_cast<float2*>(p.statistics + 2 * at) = make_float2(top, sum);
      continue;
    }
    const int token = (rows.first + r) / p.group, member = (rows.first + r) % p.group;
    const long long out_head = static_cast<long long>(head) * p.group + member;
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= inverse;
    store8(p.out.data, p.out.type, p.out.vector, (rows.row + token) * p.out.token_stride + out_head * p.out.head_stride + d, v);
    if (p.lse != nullptr && d == 0) {
      p.lse[(rows.row + token) * p.out.heads + out_head] =
          sum == 0.0f ? -INFINITY : (top + log2f(sum) - kShift) * 0.69314718055994531f;
    }
  }
}

// Joins the chunks of one row, in their order: threads by four head elements, and by every fourth (or
// eighth) chunk.
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ AttentionParams p) {
  __shared__ float4 shared[kThreads];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int r = static_cast<int>(blockIdx.x % p.tile_rows);
  const long long tile_index = blockIdx.x / p.tile_rows;
  const int row_tile = static_cast<int>(tile_index % p.row_tiles);
  const int head = static_cast<int>(tile_index / p.row_tiles % p.kv_heads);
  const int s = static_cast<int>(tile_index / p.row_tiles / p.kv_heads);
  Rows rows;
  if (!rows_of(p, s, row_tile * p.tile_rows, p.tile_rows, &rows) || r >= rows.count) return;
  const int used = splits_used(p, rows);
  if (used == 1) return;
  const long long first = tile_index * p.splits * p.tile_rows + r;  // chunk c: + c * tile_rows
  const float2* const stats = reinterpret_cast<const float2*>(p.statistics) + first;
  const int lane = threadIdx.x & 31;
  float top = -INFINITY, sum = 0.0f;
  for (int c = lane; c < used; c += 32) top = fmaxf(top, stats[static_cast<long long>(c) * p.tile_rows].x);
#pragma unroll
  for (int h = 16; h >= 1; h >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, h));
  const float base = top == -INFINITY ? 0.0f : top;
  for (int c = lane; c < used; c += 32) {
    const float2 v = stats[static_cast<long long>(c) * p.tile_rows];
    sum += v.y * exp2_fast(v.x - base);
  }
#pragma unroll
  for (int h = 16; h >= 1; h >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, h);
  const int vectors = p.dim / 4, parts = kThreads / vectors;
  const int part = threadIdx.x / vectors, at = threadIdx.x % vectors;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (part < parts) {
    for (int c = part; c < used; c += parts) {
      const float weight = exp2_fast(stats[static_cast<long long>(c) * p.tile_rows].x - base);
      const float4 x = reinterpret_cast<const float4*>(p.partial + (first + static_cast<long long>(c) * p.tile_rows) * p.dim)[at];
      v.x = fmaf(x.x, weight, v.x);
      v.y = fmaf(x.y, weight, v.y);
      v.z = fmaf(x.z, weight, v.z);
      v.w = fmaf(x.w, weight, v.w);
    }
  }
  shared[threadIdx.x] = v;
  __syncthreads();
  const int token = (rows.first + r) / p.group, member = (rows.first + r) % p.group;
  const long long out_head = static_cast<long long>(head) * p.group + member;
  if (threadIdx.x < vectors) {
    for (int q = 1; q < parts; ++q) {
      const float4 x = shared[q * vectors + threadIdx.x];
      v.x += x.x;
      v.y += x.y;
      v.z += x.z;
      v.w += x.w;
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    const long long to = (rows.row + token) * p.out.token_stride + out_head * p.out.head_stride + 4 * threadIdx.x;
    store_one(p.out.data, p.out.type, to, v.x * inverse);
    store_one(p.out.data, p.out.type, to + 1, v.y * inverse);
    store_one(p.out.data, p.out.type, to + 2, v.z * inverse);
    store_one(p.out.data, p.out.type, to + 3, v.w * inverse);
  }
  if (threadIdx.x == 0 && p.lse != nullptr) {
    p.lse[(rows.row + token) * p.out.heads + out_head] =
        sum == 0.0f ? -INFINITY : (top + log2f(sum) - p.shift) * 0.69314718055994531f;
  }
}

template <int DP, bool kWide>
qx_status launch_streamed(const AttentionParams& p, long long grid, cudaStream_t stream) {
  static SmemOptIn opt_in;
  constexpr int bytes = smem_bytes<DP, kWide>();
  QX_TRY(opt_in.ensure(attention_kernel<DP, kWide>, bytes));
  return launch_behind(attention_kernel<DP, kWide>, grid, kThreads, bytes, stream, p);
}

}  // namespace

qx_status check_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                          float scale, long long window) {
  QX_TRY(check_cache(cache));
  QX_TRY(check_batch(cache, batch));
  QX_TRY(check_heads(q, batch->tokens, cache->head_dim, false));
  QX_TRY(check_heads(out, batch->tokens, cache->head_dim, true));
  if (q->heads != out->heads || q->heads % cache->kv_heads != 0) return QX_STATUS_INVALID_SHAPE;
  if (static_cast<__int128>(batch->max_tokens) * (q->heads / cache->kv_heads) > 0x7FFFFFFF - 4096) {
    return QX_STATUS_INVALID_SHAPE;
  }
  if (!std::isfinite(scale) || window < 0) return QX_STATUS_INVALID_ARGUMENT;
  return QX_STATUS_OK;
}

qx_status launch_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                           float* lse, float scale, int causal, long long window, DeviceContext* ctx,
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
  p.dim = cache->head_dim;
  p.q = device_heads(q);
  p.out = device_heads(out);
  p.lse = lse;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.causal = causal != 0;
  p.window = static_cast<int>(std::min<long long>(window, 0x7FFFFFFF));
  p.group = q->heads / cache->kv_heads;
  const long long most_rows = static_cast<long long>(batch->max_tokens) * p.group;
  const bool prompt = q->type != QX_STORAGE_F32 && cache->head_dim <= 128 && most_rows >= kPromptFrom;
  p.tile_rows = prompt ? kPromptRows : kRows;
  p.shift = prompt ? kPromptShift : kShift;
  p.row_tiles = static_cast<int>((most_rows + p.tile_rows - 1) / p.tile_rows);
  const long long items = static_cast<long long>(batch->sequences) * cache->kv_heads * p.row_tiles;
  // Most keys that a tile can see.
  long long range = batch->max_length;
  if (p.window > 0 && p.causal) range = std::min<long long>(range, static_cast<long long>(p.window) + p.tile_rows);
  range += 31;  // (from a multiple of 32 on)
  // Chunks: one sequence fills the card with one round of equal chunks; several, of lengths that only the
  // device knows, get four rounds of smaller ones, so that the SMs which end early take the next. No chunk is
  // below a tile per warp (in the prompt kernel, four tiles): then the joining would cost more than the keys.
  const int dp = cache->head_dim <= 64 ? 64 : cache->head_dim <= 128 ? 128 : 256;
  const long long slots = static_cast<long long>(ctx->prop.multiProcessorCount) * (prompt ? 1 : dp == 64 ? 4 : dp == 128 ? 2 : 1);
  const bool one_round = batch->sequences == 1 || prompt;
  const long long wanted = one_round ? std::max(1LL, slots / items) : (4 * slots + items - 1) / items;
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
  }
  const long long grid = items * p.splits;
  const bool wide = q->type == QX_STORAGE_F32;
  qx_status status;
  if (prompt) status = launch_prompt(p, grid, stream);
  else if (dp == 64) status = wide ? launch_streamed<64, true>(p, grid, stream) : launch_streamed<64, false>(p, grid, stream);
  else if (dp == 128) status = wide ? launch_streamed<128, true>(p, grid, stream) : launch_streamed<128, false>(p, grid, stream);
  else status = wide ? launch_streamed<256, true>(p, grid, stream) : launch_streamed<256, false>(p, grid, stream);
  QX_TRY(status);
  return p.splits > 1 ? launch_behind(join_kernel, items * p.tile_rows, kThreads, 0, stream, p) : QX_STATUS_OK;
}

}  // namespace kv
}  // namespace qx

using namespace qx;

extern "C" qx_status qx_kv_attention_dev(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q,
                                         const qx_heads* out, float* lse_dev, float scale, int causal, long long window,
                                         qx_workspace* workspace, void* stream) {
  QX_TRY(kv::check_attention(cache, batch, q, out, scale, window));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  return kv::launch_attention(cache, batch, q, out, lse_dev, scale, causal, window, ctx,
                              workspace != nullptr ? workspace : &ctx->workspace, static_cast<cudaStream_t>(stream));
}
