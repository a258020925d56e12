// Attention over the paged 8-bit cache for prompts: 16-bit queries, head sizes up to 128, many rows per
// sequence. The tensor-core form of qx_attention.cu.
//
// A CTA takes 256 rows (tokens x query heads of one kv head) as two tiles of 128 and walks the keys in tiles
// of 128. S = Q K^T and O += P V run on tcgen05.mma kind::f16 (M = 128, f32 accumulators in TMEM: S and O of
// both row tiles, 512 columns; P takes the place of its S). Roles:
//   warps 0-3, 4-7  softmax of row tile 0, 1: a thread owns a row, so maximum and sum need no shuffles
//   warps 8-11      codes -> f16: global memory to registers (a tile ahead) to shared memory, in the 128-byte
//                   swizzle; keys become a K-major operand and values an N-major one of the same layout, so
//                   nothing is transposed
//   warp 12         issues the MMAs: while one row tile's softmax runs, the other's products do
// (warps 13-15 fill up the last warpgroup: registers move by warpgroups, 192 to a softmax thread, which holds a
// whole row of S, and 64 to the others.)
//
// The codes are exact in f16 and so are the queries, times a power of two per row (f16 loses the bits of
// elements below 2^-32 of the row's largest). The scale of a key block multiplies the scores. The scale of a
// value block goes into the exponent of the weights: P = 2^(s + log2 vs - m), m following the largest s +
// log2 vs, so one f16 rounding (2^-11) holds for every mixture of scales; the sums of weights divide it out
// again, once per 16 keys, relative to the largest scale that the row has seen. (A scale more than 2^60 below
// that one counts as 2^-60 of it, so that no weight leaves f32's range on the way; that moves an output by 2^-53
// of the largest value.) A scale of zero takes its block's codes for zeros. m only follows when it has fallen 4 behind (a
// factor of 16): then the row's sum and O are scaled, in TMEM, by the row's own warp, which is rare after the first tiles.
//
// f32 queries (kWide) take one tile of 128 rows per CTA, whose queries and weights are f16 pairs, hi + lo, of 22 bits:
// the second tile's place in shared memory holds the low halves of the queries, the second half of S the low halves
// of the weights, and every product is two. A sum over all keys would lose f32's last bits to the MMA's own
// additions, so each tile's product goes to one of two buffers of O, and warps 4-7 add those up in registers, in
// f32, with the maxima's changes in between. S has the second row tile's place for the next tile of keys, so that it is
// ready when a softmax ends (2 x 1000 tokens, 4000 keys, 16 heads of 96 elements: 190 us without, 166 with).
//
// Measured: two prompts of up to 4096 bf16 tokens, 32 query heads on 8, 128 elements, causal: 303 us (208 GFLOP, 680
// TFLOP/s); 1024 f16 tokens behind 15360: 322 us (825 TFLOP/s); 4 texts of up to 500 f32 tokens, 16 heads of 96
// elements: 41.0 us. A tile of 128 keys takes 4600 cycles for both row tiles, where the MMAs alone take 2050 and the
// exponentials 2050: a row tile's S, softmax and P V follow one another, and only the other row tile runs beside them.
// A CTA's way in (11000 cycles: table, queries to operands, first keys) and out (6000) comes on top.
//
// Every wait is bounded; one that runs out raises the CTA's abort flag, all roles leave their loops, MMAs
// in flight are waited for (bounded) and TMEM is freed.

#include <algorithm>
#include <cmath>

#include "qx_attention.cuh"
#include "qx_tile_pipe.cuh"

namespace qx {
namespace kv {
namespace {

using namespace sm100;

constexpr int kRowTile = 128, kKeys = 128, kGroups = kKeys / 16;
constexpr int kConvertWarps = 4, kTcThreads = 512;
constexpr int kSoftmaxRegisters = 192, kOtherRegisters = 64;  // of 128 at launch: 256 * 192 + 256 * 64 = 512 * 128
constexpr int kMetaStages = 4;
static_assert(kPromptRows == 2 * kRowTile && kPromptRowsWide == kRowTile, "two tiles per CTA, f32: one");
constexpr int kKeepStages = 4;
constexpr float kBehind = 4.0f;
constexpr float kLeastLog = -100.0f;  // of a value scale: append makes no smaller one but zero, and smaller ones count as that
constexpr float kLeastScale = 7.8886090522101181e-31f;  // 2^-100

constexpr float kCarriedInverse = 1.0f / 2048.0f;  // 2^-kPromptShift
constexpr float kSpan = 60.0f;  // log2 of the largest ratio of value scales that is kept
constexpr float kSpanInverse = 1.1529215046068470e18f;  // 2^kSpan

// What the softmax needs to know about a tile of keys, by groups of 16.
struct Meta {
  float2 scales[kGroups];        // of the keys, and log2 of the values'
  float value_inverse[kGroups];  // of the values' scale
  int present[kGroups];
};

struct Barriers {
  uint64_t queries[2], key_full[2], key_empty[2], value_full[2], value_empty[2];
  uint64_t scores[2], halves[2], weights[2], sums[2], meta[kMetaStages], drain;
  uint64_t kept[kKeepStages], taken[2], gain;  // kWide: factors written, buffers of O read, last factors written
  uint32_t tmem_base;
  int abort_flag;
};

template <int DP>
struct TcShape {
  static constexpr int kOperand = kKeys * DP * 2;  // bytes of a tile of queries, keys or values
  static constexpr int kQueries = 0;
  static constexpr int kKeyRing = kQueries + 2 * kOperand;
  static constexpr int kValueRing = kKeyRing + 2 * kOperand;
  static constexpr int kMeta = kValueRing + 2 * kOperand;
  static constexpr int kKeep = kMeta + kMetaStages * static_cast<int>(sizeof(Meta));  // kWide: [stage][row], [row]
  static constexpr int kBars = kKeep + (kKeepStages + 1) * kRowTile * 4;
  static constexpr int kBytes = kBars + static_cast<int>(sizeof(Barriers)) + 1024;  // (the operands start on 1024)
};

// D[tmem] (+)= A[tmem] * B[smem], f16 operands, f32 accumulate.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Waits for the loads in flight and names the registers that they fill, so that nothing computed from those can
// be moved in front of the wait.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
// N-major operand in the 128-byte swizzle: rows (of K) of 128 bytes = 64 elements of N, groups of eight rows
// 1024 bytes apart (stride offset), the next 64 elements of N `next` bytes on (leading offset).
__device__ __forceinline__ uint64_t make_sw128_nmajor_desc(uint32_t smem_addr, uint32_t next) {
  uint64_t desc = 0;
  desc |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  desc |= static_cast<uint64_t>(next >> 4) << 16;
  desc |= static_cast<uint64_t>(1024 >> 4) << 32;
  desc |= static_cast<uint64_t>(1) << 46;
  desc |= static_cast<uint64_t>(2) << 61;
  return desc;
}

__device__ __forceinline__ unsigned long long fmaf2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float v;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}

// Sixteen codes to two 16-byte pieces of f16.
__device__ __forceinline__ void convert16(const uint4& codes, uint4* a, uint4* b) {
  a->x = tile::convert_bytes2<false>(codes.x, 0x4140);
  a->y = tile::convert_bytes2<false>(codes.x, 0x4342);
  a->z = tile::convert_bytes2<false>(codes.y, 0x4140);
  a->w = tile::convert_bytes2<false>(codes.y, 0x4342);
  b->x = tile::convert_bytes2<false>(codes.z, 0x4140);
  b->y = tile::convert_bytes2<false>(codes.z, 0x4342);
  b->z = tile::convert_bytes2<false>(codes.w, 0x4140);
  b->w = tile::convert_bytes2<false>(codes.w, 0x4342);
}

// What a softmax thread knows about its row.
struct RowState {
  float factor;       // of the raw scores, log2(e) in it
  int low, high;      // keys that the row sees
  float maximum, sum;
  float largest_log, largest;  // value scale that it has seen, and its log2
};

// One tile of scores to weights, in TMEM. `scores`: this warp's lanes of S, which P replaces; `sums`: of O. Keys
// share scales by `kUnit`s of 16 or 32.
// kOpen: no row of the warp has a hidden key. kHidden: some have; those scores become -infinity before anything else
// is done with them. kSpecial: besides, a scale is no plain number (zero, infinite, NaN), which would take -infinity
// to NaN: hidden keys are told apart at every step. (Two prompts of up to 4096, one of 1024 behind 15360, f32 texts
// of up to 500, us: kOpen and kSpecial alone 308, 321, 49.5; one form for the first two 327, 360, 46.7; these three 305, 322,
// 46.5.)
// kWide: the row's factor for what O holds so far goes to *keep_to instead.
enum Mask { kOpen, kHidden, kSpecial };
template <int DP, int kUnit, Mask kMask, bool kWide>
__device__ __forceinline__ void softmax_tile(uint32_t scores, uint32_t sums, const Meta& meta, RowState& row, int key0,
                                             bool first, uint64_t* first_half, float* keep_to) {
  constexpr int kUnits = kKeys / kUnit, kPerUnit = kUnit / 16;
  uint32_t s[4][32];
  tmem_ld_32x32(scores, s[0]);
  tmem_ld_32x32(scores + 32, s[1]);

  float factor[kUnits], log[kUnits], relative[kUnits];
  float largest = row.largest_log;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const float2 scales = meta.scales[u * kPerUnit];
    factor[u] = row.factor * scales.x;
    log[u] = scales.y;
    relative[u] = meta.value_inverse[u * kPerUnit];
    const int key = key0 + kUnit * u;
    const bool seen = kMask == kOpen || (meta.present[u * kPerUnit] != 0 && key < row.high && key + kUnit > row.low);
    largest = fmaxf(largest, seen ? log[u] : -INFINITY);
  }
  // The sum stands against the largest scale and the maximum. It follows both in one step: alone, a rise of the scale by
  // more than about 2^100 would take it past f32's range, where the maximum rises as far.
  float rise = 0.0f;
  if (largest > row.largest_log) {
    if (row.sum != 0.0f) rise = largest - row.largest_log;
    row.largest_log = largest;
    row.largest = exp2f(largest);
  }
  const float least = largest - kSpan;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    relative[u] = log[u] < least ? kSpanInverse : relative[u] * row.largest;
    log[u] = log[u] < least ? least : log[u];  // (no number stays none)
  }

  const auto hidden = [&](int key) { return key < row.low || key >= row.high; };
  const auto hide = [&](int c) {  // of 32 keys
    const int low = min(max(row.low - key0 - 32 * c, 0), 32), high = min(max(row.high - key0 - 32 * c, 0), 32);
    uint32_t seen = static_cast<uint32_t>((1ull << high) - 1) & ~static_cast<uint32_t>((1ull << low) - 1);
    if (meta.present[2 * c] == 0) seen &= 0xFFFF0000u;
    if (meta.present[2 * c + 1] == 0) seen &= 0xFFFFu;
    if (__all_sync(0xFFFFFFFFu, seen == 0xFFFFFFFFu)) return;
#pragma unroll
    for (int i = 0; i < 32; ++i) s[c][i] = (seen >> i & 1) != 0 ? s[c][i] : 0xFF800000u;
  };
  float top = -INFINITY;
  const auto top_of = [&](int u) {
    const bool present = kMask != kSpecial || meta.present[u * kPerUnit] != 0;
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // (four chains: one would wait for itself)
#pragma unroll
    for (int i = 0; i < kUnit; i += 2) {
      const int at = kUnit * u + i;
      const float a = __uint_as_float(s[at / 32][at % 32]), b = __uint_as_float(s[at / 32][at % 32 + 1]);
      float& chain = m[i / 2 % 4];
      if (kMask != kSpecial) {
        chain = max3(chain, a, b);
      } else {
        if (present && !hidden(key0 + at)) chain = fmaxf(chain, a);
        if (present && !hidden(key0 + at + 1)) chain = fmaxf(chain, b);
      }
    }
    const float most = fmaxf(max3(m[0], m[1], m[2]), m[3]);
    // (nothing seen: -infinity times a factor that may be zero or no number)
    top = fmaxf(top, kMask == kSpecial && most == -INFINITY ? -INFINITY : fmaf(most, factor[u], log[u]));
  };
  tmem_ld_wait_for(s[0]);
  tmem_ld_wait_for(s[1]);
  tmem_ld_32x32(scores + 64, s[2]);
  tmem_ld_32x32(scores + 96, s[3]);
  if (kMask == kHidden) {
    hide(0);
    hide(1);
  }
#pragma unroll
  for (int u = 0; u < kUnits / 2; ++u) top_of(u);
  tmem_ld_wait_for(s[2]);
  tmem_ld_wait_for(s[3]);
  if (kMask == kHidden) {
    hide(2);
    hide(3);
  }
#pragma unroll
  for (int u = kUnits / 2; u < kUnits; ++u) top_of(u);

  const bool behind = top > row.maximum + kBehind;  // (from -infinity on, any score is)
  if (kWide) {
    const float before = row.maximum;
    if (behind) row.maximum = top;
    const float moved = before == row.maximum ? 0.0f : before - row.maximum;
    *keep_to = exp2_fast(moved);
    rise += moved;
  } else if (__any_sync(0xFFFFFFFFu, behind)) {
    const float before = row.maximum;
    if (behind) row.maximum = top;
    const float moved = before == row.maximum ? 0.0f : before - row.maximum;
    const float keep = exp2_fast(moved);
    rise += moved;
    if (!first) {
#pragma unroll 1
      for (int c = 0; c < DP; c += 16) {
        uint32_t o[16];
        tmem_ld_32x16(sums + c, o);
        tmem_ld_wait_for(o);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
        tmem_st_32x16(sums + c, o);
      }
    }
  }
  if (rise != 0.0f) row.sum *= exp2_fast(rise);
  const float base = (row.maximum == -INFINITY ? 0.0f : row.maximum) - kPromptShift;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t p[16], low[16];
#pragma unroll
    for (int h = 0; h < 32 / kUnit; ++h) {
      const int u = c * (32 / kUnit) + h;
      const float add = log[u] - base;
      const unsigned long long f2 = tile::pack2(__float_as_uint(factor[u]), __float_as_uint(factor[u]));
      const unsigned long long c2 = tile::pack2(__float_as_uint(add), __float_as_uint(add));
      const bool present = kMask != kSpecial || meta.present[u * kPerUnit] != 0;
      unsigned long long sum2 = 0;
#pragma unroll
      for (int i = 0; i < kUnit; i += 2) {
        const int at = kUnit * h + i;
        const unsigned long long t2 = fmaf2(tile::pack2(s[c][at], s[c][at + 1]), f2, c2);
        uint32_t lo, hi;
        tile::unpack2(t2, lo, hi);
        float a = exp2_fast(__uint_as_float(lo)), b = exp2_fast(__uint_as_float(hi));
        if (kMask == kSpecial) {  // (behind exp2: also where the arguments are no numbers)
          a = !present || hidden(key0 + 32 * c + at) ? 0.0f : a;
          b = !present || hidden(key0 + 32 * c + at + 1) ? 0.0f : b;
        }
        const __half2 w = __floats2half2_rn(a, b);
        p[at / 2] = *reinterpret_cast<const uint32_t*>(&w);
        if (kWide) {
          const float2 rounded = __half22float2(w);
          const __half2 rest = __floats2half2_rn(a - rounded.x, b - rounded.y);
          low[at / 2] = *reinterpret_cast<const uint32_t*>(&rest);
        }
        sum2 = tile::addf2(sum2, tile::pack2(__float_as_uint(a), __float_as_uint(b)));
      }
      uint32_t lo, hi;
      tile::unpack2(sum2, lo, hi);
      const float sum = __uint_as_float(lo) + __uint_as_float(hi);
      // (a unit that is hidden as a whole may have a scale that is no number)
      if (kMask != kSpecial || sum != 0.0f) row.sum = fmaf(sum, relative[u], row.sum);
    }
    tmem_st_32x16(scores + 16 * c, p);
    if (kWide) tmem_st_32x16(scores + kKeys / 2 + 16 * c, low);
    if (!kWide && c == 1) {  // the product with the first half of the keys' values may begin
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(first_half);
    }
  }
  tmem_st_wait();
}

// A lane's way over rows of a view, from `row` of the sequence's on: where its row begins, in elements.
struct RowWalk {
  long long at, step, wrap;
  int member, by, group;
  __device__ __forceinline__ RowWalk(const Heads& view, const Rows& rows, int head, int group_, int row, int at_once)
      : group(group_) {
    const int token = row / group;
    member = row - token * group;
    at = (rows.row + token) * view.token_stride + (static_cast<long long>(head) * group + member) * view.head_stride;
    by = at_once % group;
    step = at_once / group * view.token_stride + by * view.head_stride;
    wrap = view.token_stride - group * view.head_stride;
  }
  __device__ __forceinline__ void next() {
    at += step;
    member += by;
    if (member >= group) {
      member -= group;
      at += wrap;
    }
  }
};

// 16 bytes of a row of an operand: c counts them. And of a row of f32 elements that lies where a pair's halves go: their
// pieces 2c and 2c + 1 where elements 8c .. 8c + 7 of the high and of the low halves do.
template <int DP, bool kWide>
__device__ __forceinline__ uint8_t* piece_at(uint8_t* tile, int r, int c) {
  const int chunk = kWide ? c >> 1 : c;
  return tile + (kWide ? (c & 1) * (kRowTile * DP * 2) : 0) + (chunk >> 3) * (kRowTile * 128) + r * 128 +
         (((chunk ^ r) & 7) << 4);
}

// 32 elements of a row of O, from element c of the head on, times `gain`, into the operand's place of that row ...
template <int DP, bool kWide>
__device__ __forceinline__ void stage_row(uint8_t* tile, int type, const uint32_t (&o)[32], float gain, int r, int c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = gain == 0.0f ? 0.0f : __uint_as_float(o[8 * i + e]) * gain;  // (O may be unset)
    if constexpr (kWide) {
      uint4 w[2];
      to_words<QX_STORAGE_F32>(v, w);
      *reinterpret_cast<uint4*>(piece_at<DP, true>(tile, r, c / 4 + 2 * i)) = w[0];
      *reinterpret_cast<uint4*>(piece_at<DP, true>(tile, r, c / 4 + 2 * i + 1)) = w[1];
    } else {
      uint4 w[1];
      if (type == QX_STORAGE_F16) to_words<QX_STORAGE_F16>(v, w);
      else to_words<QX_STORAGE_BF16>(v, w);
      *reinterpret_cast<uint4*>(piece_at<DP, false>(tile, r, c / 8 + i)) = w[0];
    }
  }
}
// ... from where the warp writes its 32 rows, runs of lanes to a row.
template <int DP, bool kWide>
__device__ __forceinline__ void write_rows(const AttentionParams& p, uint8_t* tile, const Rows& rows, int head, int warp_row) {
  constexpr int kElements = kWide ? 4 : 8, kLanes = DP / kElements, kAtOnce = 32 / kLanes;
  const int lane = threadIdx.x & 31, piece = lane % kLanes, first = lane / kLanes;
  __syncwarp();
  if (piece * kElements >= p.dim) return;
  RowWalk to(p.out, rows, head, p.group, rows.first + warp_row + first, kAtOnce);
#pragma unroll 1
  for (int r = first; r < 32; r += 8 * kAtOnce) {
    uint4 w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = *reinterpret_cast<const uint4*>(piece_at<DP, kWide>(tile, (warp_row & (kRowTile - 1)) + r + i * kAtOnce, piece));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (warp_row + r + i * kAtOnce < rows.count) {
        *reinterpret_cast<uint4*>(p.out.data + (to.at + piece * kElements) * (kWide ? 4 : 2)) = w[i];
      }
      to.next();
    }
  }
}
// The same elements by the row's own thread, to the partial results or to a view that is not as the above needs it.
__device__ __forceinline__ void write_row(const AttentionParams& p, const uint32_t (&o)[32], float gain, float* partial,
                                          long long to, int c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + 8 * i >= p.dim) break;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = gain == 0.0f ? 0.0f : __uint_as_float(o[8 * i + e]) * gain;
    if (partial == nullptr) {
      store8(p.out.data, p.out.type, p.out.vector, to + c + 8 * i, v);
    } else {
      store8_typed<QX_STORAGE_F32>(reinterpret_cast<uint8_t*>(partial), to + c + 8 * i, v);
    }
  }
}

template <int DP, int kUnit, bool kWide>
__global__ void __launch_bounds__(kTcThreads, 1) prompt_kernel(const __grid_constant__ AttentionParams p) {
  using S = TcShape<DP>;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  Meta* const meta = reinterpret_cast<Meta*>(smem + S::kMeta);
  float* const keep = reinterpret_cast<float*>(smem + S::kKeep);
  float* const gains = keep + kKeepStages * kRowTile;
  Barriers* const bars = reinterpret_cast<Barriers*>(smem + S::kBars);
  volatile int* const abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");

  const uint32_t index = blockIdx.x / p.splits;
  const int split = static_cast<int>(blockIdx.x - index * p.splits);
  const uint32_t by_head = index / p.row_tiles;
  // the last rows first: with a causal mask they see the most keys
  const int row_tile = p.row_tiles - 1 - static_cast<int>(index - by_head * p.row_tiles);
  const long long tile_index = static_cast<long long>(by_head) * p.row_tiles + row_tile;
  const int s = static_cast<int>(by_head / p.kv_heads), head = static_cast<int>(by_head - s * p.kv_heads);
  Rows rows;
  constexpr int kCtaRows = kWide ? kRowTile : 2 * kRowTile;
  if (!rows_of(p, s, row_tile * kCtaRows, kCtaRows, &rows)) return;
  int begin, end;
  if (!chunk_of(p, rows, split, &begin, &end)) return;
  const int tiles = max(0, (end - begin + kKeys - 1) / kKeys);
  const int row_tiles = !kWide && rows.count > kRowTile ? 2 : 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->queries[i], kRowTile);
      mbar_init(&bars->key_full[i], kConvertWarps);
      mbar_init(&bars->key_empty[i], 1);
      mbar_init(&bars->value_full[i], kConvertWarps);
      mbar_init(&bars->value_empty[i], 1);
      mbar_init(&bars->scores[i], 1);
      mbar_init(&bars->halves[i], 4);
      mbar_init(&bars->weights[i], 4);
      mbar_init(&bars->sums[i], 1);
    }
    for (int i = 0; i < kMetaStages; ++i) mbar_init(&bars->meta[i], kConvertWarps);
    for (int i = 0; i < kKeepStages; ++i) mbar_init(&bars->kept[i], 4);
    mbar_init(&bars->taken[0], 4);
    mbar_init(&bars->taken[1], 4);
    mbar_init(&bars->gain, 4);
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  bool ok = true;

  if (warp < 8) {
    // ---- softmax --------------------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
    const int which = warp >> 2;
    if (kWide && which == 1) {
      // ---- the tiles' products added up, f32 -------------------------------------------------
      const int r = threadIdx.x & 127;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      uint32_t total[DP / 32][32];
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
#pragma unroll
        for (int i = 0; i < 32; ++i) total[c][i] = 0;
      }
      for (int j = 0; ok && j < tiles; ++j) {
        ok = mbar_wait_warp(&bars->kept[j % kKeepStages], j / kKeepStages & 1, abort_flag) &&
             mbar_wait_warp(&bars->sums[j & 1], j >> 1 & 1, abort_flag);
        if (!ok) break;
        __syncwarp();
        tc_fence_after_sync();
        const float factor = keep[j % kKeepStages * kRowTile + r];
        const uint32_t product = tmem + lanes + 256 + (j & 1) * 128;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32(product + 32 * c, o);
          tmem_ld_wait_for(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            total[c][i] = __float_as_uint(fmaf(__uint_as_float(total[c][i]), factor, __uint_as_float(o[i])));
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->taken[j & 1]);
      }
      if (ok) ok = mbar_wait_warp(&bars->gain, 0, abort_flag);
      if (ok) {
        const int token = (rows.first + r) / p.group, member = (rows.first + r) % p.group;
        const bool whole = splits_used(p, rows) == 1;
        const long long at = (tile_index * p.splits + split) * kCtaRows + r;
        const long long out_head = static_cast<long long>(head) * p.group + member;
        const long long to = whole ? (rows.row + token) * p.out.token_stride + out_head * p.out.head_stride : at * p.dim;
        const bool staged = whole && p.out.type == QX_STORAGE_F32 && p.out.vector;  // (every product is done: so are the queries)
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          if (staged) stage_row<DP, true>(smem + S::kQueries, QX_STORAGE_F32, total[c], gains[r], r, 32 * c);
          else if (r < rows.count && 32 * c < p.dim) write_row(p, total[c], gains[r], whole ? nullptr : p.partial, to, 32 * c);
        }
        if (staged) write_rows<DP, true>(p, smem + S::kQueries, rows, head, (warp & 3) * 32);
      }
      if (!ok) {
        *abort_flag = 1;
        report_error(p.batch.error, 44);
      }
    } else if (which < row_tiles) {
      const int r = threadIdx.x & 127, in_tile = which * kRowTile + r;
      const bool real = in_tile < rows.count;
      const int start = rows.length - rows.n;
      const int token = (rows.first + in_tile) / p.group, member = (rows.first + in_tile) % p.group;
      const long long row_at = rows.row + token, out_head = static_cast<long long>(head) * p.group + member;
      RowState row;
      row.low = row.high = 0;
      row.maximum = -INFINITY;
      row.sum = 0.0f;
      row.largest_log = -INFINITY;
      row.largest = 0.0f;
      if (real) {
        row.high = p.causal ? min(rows.length, start + token + 1) : rows.length;
        row.low = first_seen(p, start + token);
      }
      // The queries: f16 times a power of two that brings the row's largest magnitude to 2^7 .. 2^8. A warp copies its
      // rows as they are to where their operands go, runs of lanes to a row; then each thread converts its own row in
      // place (f32: the 16-byte pieces 2c and 2c + 1 lie where the high and the low halves of elements 8c .. 8c + 7
      // go). Loops, not straight code: what runs once per CTA waits for its instructions at every line.
      {
        constexpr int kElements = kWide ? 4 : 8, kBytes = kWide ? 4 : 2, kLanes = DP / kElements, kAtOnce = 32 / kLanes;
        const int piece = lane % kLanes, d = piece * kElements, warp_row = which * kRowTile + (warp & 3) * 32;
        uint8_t* const tile = smem + S::kQueries + which * S::kOperand;
        RowWalk from(p.q, rows, head, p.group, rows.first + warp_row + lane / kLanes, kAtOnce);
        if (p.q.vector) {
#pragma unroll 8
          for (int i = lane / kLanes; i < 32; i += kAtOnce) {
            const bool there = warp_row + i < rows.count && d < p.dim;  // (or no bytes: zeros)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                         ::"r"(smem_u32(piece_at<DP, kWide>(tile, (warp & 3) * 32 + i, piece))),
                         "l"(p.q.data + (there ? from.at + d : 0) * kBytes), "r"(there ? 16 : 0)
                         : "memory");
            from.next();
          }
        } else {
#pragma unroll 1
          for (int i = lane / kLanes; i < 32; i += kAtOnce) {
            uint8_t* const to = piece_at<DP, kWide>(tile, (warp & 3) * 32 + i, piece);
            const bool there = warp_row + i < rows.count && d < p.dim;
#pragma unroll 1
            for (int e = 0; e < kElements; ++e) {
              if (kWide) reinterpret_cast<uint32_t*>(to)[e] = there ? reinterpret_cast<const uint32_t*>(p.q.data)[from.at + d + e] : 0;
              else reinterpret_cast<uint16_t*>(to)[e] = there ? reinterpret_cast<const uint16_t*>(p.q.data)[from.at + d + e] : 0;
            }
            from.next();
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        const bool f16 = p.q.type == QX_STORAGE_F16;
        const auto pair = [&](uint32_t w) {
          return f16 ? __half22float2(*reinterpret_cast<const __half2*>(&w)) : make_float2(bf16_low(w), bf16_high(w));
        };
        uint32_t top = 0;  // of the bit patterns without sign: they grow with the magnitude
#pragma unroll 4
        for (int c = 0; c < DP / 8; ++c) {
          const uint4 a = *reinterpret_cast<const uint4*>(piece_at<DP, false>(tile, r, c));
          if (kWide) {
            const uint4 b = *reinterpret_cast<const uint4*>(piece_at<DP, false>(tile, r, c) + S::kOperand);
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, w[e] & 0x7FFFFFFFu);
          } else {
            top = __vimax3_u16x2(top, a.x & 0x7FFF7FFFu, a.y & 0x7FFF7FFFu);
            top = __vimax3_u16x2(top, a.z & 0x7FFF7FFFu, a.w & 0x7FFF7FFFu);
          }
        }
        if (!kWide) top = __float_as_uint(pair(max(top & 0xFFFFu, top >> 16)).x);
        top >>= 23;
        const int shift = top >= 255 ? 0 : min(120, max(-120, 134 - static_cast<int>(top)));
        // (a negative scale turns the query's sign, so that larger raw scores are larger scores)
        const float up = copysignf(__uint_as_float(static_cast<uint32_t>(127 + shift) << 23), p.scale_log2);
        // (a row that holds a NaN or an infinity gives NaN: its products may all be -infinity, which reads as no key)
        row.factor = top >= 255 ? __uint_as_float(0x7FC00000u)
                                : __uint_as_float(static_cast<uint32_t>(127 - shift) << 23) * fabsf(p.scale_log2);
#pragma unroll 2
        for (int c = 0; c < DP / 8; ++c) {
          uint4* const at = reinterpret_cast<uint4*>(piece_at<DP, false>(tile, r, c));
          uint4* const low_at = reinterpret_cast<uint4*>(piece_at<DP, false>(tile, r, c) + S::kOperand);
          const uint4 first = *at, second = kWide ? *low_at : first;
          const uint32_t in[8] = {first.x, first.y, first.z, first.w, second.x, second.y, second.z, second.w};
          uint32_t high[4], low[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = kWide ? make_float2(__uint_as_float(in[2 * i]), __uint_as_float(in[2 * i + 1])) : pair(in[i]);
            const __half2 h = __floats2half2_rn(v.x * up, v.y * up);
            high[i] = *reinterpret_cast<const uint32_t*>(&h);
            if (kWide) {
              const float2 rounded = __half22float2(h);
              const __half2 rest = __floats2half2_rn(v.x * up - rounded.x, v.y * up - rounded.y);
              low[i] = *reinterpret_cast<const uint32_t*>(&rest);
            }
          }
          *at = make_uint4(high[0], high[1], high[2], high[3]);
          if (kWide) *low_at = make_uint4(low[0], low[1], low[2], low[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&bars->queries[which]);
      }
      // below open_high and from open_low on no row of the tile has a hidden key
      const int last = min(rows.count, (which + 1) * kRowTile) - 1;
      const int position0 = start + (rows.first + which * kRowTile) / p.group, position1 = start + (rows.first + last) / p.group;
      const int open_high = p.causal ? min(rows.length, position0 + 1) : rows.length;
      const int open_low = first_seen(p, position1);
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t sums = tmem + lanes + 256 + which * 128;
      for (int j = 0; ok && j < tiles; ++j) {
        const int own = kWide ? j & 1 : which;  // S, its barriers
        const uint32_t scores = tmem + lanes + own * 128;
        ok = mbar_wait_warp(&bars->scores[own], kWide ? j >> 1 & 1 : j & 1, abort_flag) &&
             mbar_wait_warp(&bars->meta[j % kMetaStages], j / kMetaStages & 1, abort_flag);
        if (!ok) break;
        __syncwarp();
        tc_fence_after_sync();
        const Meta& tile_meta = meta[j % kMetaStages];
        const int key0 = begin + j * kKeys;
        bool open = key0 + kKeys <= open_high && key0 >= open_low;
        if (open) {
#pragma unroll
          for (int g = 0; g < kGroups; ++g) open = open && tile_meta.present[g] != 0;
        }
        float* const keep_to = keep + j % kKeepStages * kRowTile + r;
        if (__all_sync(0xFFFFFFFFu, open)) {
          softmax_tile<DP, kUnit, kOpen, kWide>(scores, sums, tile_meta, row, key0, j == 0, &bars->halves[which], keep_to);
        } else {
          bool plain = true;
#pragma unroll 1
          for (int g = 0; g < kGroups; ++g) {
            const float2 scales = tile_meta.scales[g];
            const float factor = row.factor * scales.x;
            plain = plain && factor > 0.0f && factor < INFINITY && fabsf(scales.y) < INFINITY;
          }
          if (__all_sync(0xFFFFFFFFu, plain)) {
            softmax_tile<DP, kUnit, kHidden, kWide>(scores, sums, tile_meta, row, key0, j == 0, &bars->halves[which], keep_to);
          } else {
            softmax_tile<DP, kUnit, kSpecial, kWide>(scores, sums, tile_meta, row, key0, j == 0, &bars->halves[which], keep_to);
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->weights[own]);
        if (kWide && lane == 0) mbar_arrive(&bars->kept[j % kKeepStages]);
      }
      if (!kWide && ok && tiles > 0) ok = mbar_wait_warp(&bars->sums[which], 0, abort_flag);
      if (ok) {
        tc_fence_after_sync();
        const bool whole = splits_used(p, rows) == 1;
        // O stands against the maximum alone, the sum against that and the largest scale; what the sum carries is taken
        // from the partial results of O, as the kernel that joins them has it
        const float gain = row.sum == 0.0f ? 0.0f : whole ? row.largest / row.sum : row.largest * kCarriedInverse;
        const float maximum = row.sum == 0.0f ? -INFINITY : row.maximum - row.largest_log;
        const long long at = ((tile_index * p.splits + split) * kCtaRows + in_tile);
        if (kWide) {
          gains[r] = gain;
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->gain);
        } else {
          const long long to = whole ? row_at * p.out.token_stride + out_head * p.out.head_stride : at * p.dim;
          const bool staged = whole && p.out.type != QX_STORAGE_F32 && p.out.vector;  // (every product is done: so are the queries)
          uint8_t* const tile = smem + S::kQueries + which * S::kOperand;
#pragma unroll 1
          for (int c = 0; c < DP && c < p.dim; c += 32) {
            uint32_t o[32];
            if (tiles > 0) {
              tmem_ld_32x32(sums + c, o);
              tmem_ld_wait_for(o);
            }
            if (staged) stage_row<DP, false>(tile, p.out.type, o, gain, r, c);
            else if (real) write_row(p, o, gain, whole ? nullptr : p.partial, to, c);
          }
          if (staged) write_rows<DP, false>(p, tile, rows, head, which * kRowTile + (warp & 3) * 32);
        }
        if (real && !whole) *reinterpret_cast<float2*>(p.statistics + 2 * at) = make_float2(maximum, row.sum);
        if (real && whole && p.lse != nullptr) {
          p.lse[row_at * p.out.heads + out_head] =
              row.sum == 0.0f ? -INFINITY : (maximum + log2f(row.sum) - kPromptShift) * 0.69314718055994531f;
        }
      }
      if (!ok) {
        *abort_flag = 1;
        report_error(p.batch.error, 41);
      }
    }
  } else if (warp < 8 + kConvertWarps) {
    // ---- codes to operands ------------------------------------------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    const int w = warp - 8;
    const int32_t* const table = p.batch.table + s * p.batch.table_stride;
    constexpr int kHalves = DP / 64;     // 64 codes of a row: one swizzled row of f16
    constexpr int kLoads = 4 * kHalves;  // per thread and tile: 32 keys per warp, eight at a time
    uint4 codes[kLoads];  // of one operand: the next to be stored
    // ids of the blocks of this warp's two groups of 16 keys; -1: nothing there
    const auto ids_of = [&](int j, int (&id)[2]) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int key = begin + j * kKeys + 32 * w + 16 * g;
        id[g] = -1;
        if (j < tiles && key < end) {
          const int block = table[key >> p.block_shift];
          if (block >= 0 && block < p.batch.blocks) id[g] = block;
          else if (lane == 0) report_error(p.batch.error, kErrorBlock);
        }
      }
    };
    const auto load = [&](int j, const int (&id)[2], const int8_t* plane) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int slot = (begin + j * kKeys + 32 * w + 16 * g) & (p.block_tokens - 1);
        const int8_t* const from =
            plane + ((static_cast<long long>(max(id[g], 0)) * p.kv_heads + head) * p.block_tokens + slot) * p.dim;
#pragma unroll
        for (int i = 0; i < kLoads / 2; ++i) {
          const int r = i / kHalves * 8 + (lane >> 2), d = i % kHalves * 64 + (lane & 3) * 16;
          uint4 c = make_uint4(0, 0, 0, 0);  // (nothing there, or past the head: zeros)
          if (id[g] >= 0 && (DP == p.dim || d < p.dim)) c = __ldg(reinterpret_cast<const uint4*>(from + r * p.dim + d));
          codes[g * kLoads / 2 + i] = c;
        }
      }
    };
    const auto store = [&](uint8_t* operand) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int i = 0; i < kLoads / 2; ++i) {
          const int r = 32 * w + 16 * g + i / kHalves * 8 + (lane >> 2), c = (lane & 3) * 2;
          uint8_t* const row = operand + i % kHalves * (kKeys * 128) + r * 128;
          uint4 a, b;
          convert16(codes[g * kLoads / 2 + i], &a, &b);
          *reinterpret_cast<uint4*>(row + ((c ^ (r & 7)) << 4)) = a;
          *reinterpret_cast<uint4*>(row + (((c + 1) ^ (r & 7)) << 4)) = b;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    };
    float scales[2] = {0.0f, 0.0f};  // of lane 0, 1: its group's
    const auto load_scales = [&](const int (&id)[2]) {
      const int own = lane == 1 ? id[1] : id[0];
      if (lane < 2 && own >= 0) {
        const long long slice = static_cast<long long>(own) * p.kv_heads + head;
        scales[0] = p.k_scales[slice];
        scales[1] = p.v_scales[slice];
      }
    };
    int id[2], next[2];
    ids_of(0, id);
    load(0, id, p.k_codes);
    load_scales(id);
    ids_of(1, next);
    for (int j = 0; ok && j < tiles; ++j) {
      const int stage = j & 1;
      if (j >= 2) ok = mbar_wait_warp(&bars->key_empty[stage], ((j >> 1) - 1) & 1, abort_flag);
      if (!ok) break;
      if (lane < 2) {
        const float vs = scales[1];
        const float log = vs < kLeastScale ? kLeastLog : log2f(vs);  // (no number stays none)
        Meta& m = meta[j % kMetaStages];
        m.scales[2 * w + lane] = make_float2(scales[0], log);
        // (of the scale itself: so the rounding of its logarithm, 2^-19 of a scale of 2^-64, is the weight's as much as
        // the value's, and divided out; a whole number and the rest apart would keep it from the weights too, but take the
        // f32 kernel 41.6 in place of 40.8 us, two f32 prompts of up to 4096 760 in place of 737)
        m.value_inverse[2 * w + lane] = vs < kLeastScale ? exp2f(-kLeastLog) : 1.0f / vs;
        m.present[2 * w + lane] = (lane == 1 ? id[1] : id[0]) >= 0;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->meta[j % kMetaStages]);
      store(smem + S::kKeyRing + stage * S::kOperand);
      if (lane == 0) mbar_arrive(&bars->key_full[stage]);
      // (a scale of zero makes zeros of any codes; it has no logarithm, so the codes stand for it)
      const int value_id[2] = {__shfl_sync(0xFFFFFFFFu, scales[1], 0) < kLeastScale ? -1 : id[0],
                               __shfl_sync(0xFFFFFFFFu, scales[1], 1) < kLeastScale ? -1 : id[1]};
      load(j, value_id, p.v_codes);
      if (j + 1 < tiles) load_scales(next);
      if (j >= 2) ok = mbar_wait_warp(&bars->value_empty[stage], ((j >> 1) - 1) & 1, abort_flag);
      if (!ok) break;
      store(smem + S::kValueRing + stage * S::kOperand);
      if (lane == 0) mbar_arrive(&bars->value_full[stage]);
      if (j + 1 < tiles) load(j + 1, next, p.k_codes);
      id[0] = next[0];
      id[1] = next[1];
      ids_of(j + 2, next);
    }
    if (!ok) {
      *abort_flag = 1;
      report_error(p.batch.error, 42);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == 12 && elect_one()) {
    // ---- MMAs -------------------------------------------------------------------------------
    const uint32_t shape = (1u << 4) | (static_cast<uint32_t>(kRowTile >> 4) << 24);
    const uint32_t scores_desc = shape | (static_cast<uint32_t>(kKeys >> 3) << 17);
    const uint32_t sums_desc = shape | (static_cast<uint32_t>(DP >> 3) << 17) | (1u << 16);  // (B is N-major)
    const uint32_t base = smem_u32(smem);
    const auto scores_of = [&](int which, int stage) {
#pragma unroll
      for (int half = kWide ? 1 : 0; half >= 0; --half) {  // (the low halves first: what sums of theirs lose is nothing)
#pragma unroll
        for (int d = 0; d < DP; d += 16) {
          const uint32_t at = d / 64 * (kRowTile * 128) + d % 64 * 2;
          mma_f16_ss(tmem + (kWide ? stage : which) * 128, make_sw128_kmajor_desc(base + S::kQueries + (which + half) * S::kOperand + at),
                     make_sw128_kmajor_desc(base + S::kKeyRing + stage * S::kOperand + at), scores_desc, d > 0 || (kWide && half == 0));
        }
      }
      tc_commit(&bars->scores[kWide ? stage : which]);
    };
    for (int i = 0; ok && i < row_tiles; ++i) ok = mbar_wait(&bars->queries[i], 0, abort_flag);
    if (ok && tiles > 0) ok = mbar_wait(&bars->key_full[0], 0, abort_flag);
    tc_fence_after_sync();
    if (ok && tiles > 0) {
      for (int i = 0; i < row_tiles; ++i) scores_of(i, 0);
      tc_commit(&bars->key_empty[0]);
    }
    if (kWide && ok && tiles > 1) {  // S of a tile ahead
      ok = mbar_wait(&bars->key_full[1], 0, abort_flag);
      if (ok) {
        tc_fence_after_sync();
        scores_of(0, 1);
        tc_commit(&bars->key_empty[1]);
      }
    }
    for (int j = 0; ok && j < tiles; ++j) {
      const int stage = j & 1, after = (j + 1) & 1;
      for (int i = 0; ok && i < row_tiles; ++i) {
        if (i == 0) ok = mbar_wait(&bars->value_full[stage], j >> 1 & 1, abort_flag);
        if (kWide) {
          if (ok && j >= 2) ok = mbar_wait(&bars->taken[j & 1], (j >> 1) - 1 & 1, abort_flag);
          ok = ok && mbar_wait(&bars->weights[j & 1], j >> 1 & 1, abort_flag);
        } else {
          ok = ok && mbar_wait(&bars->halves[i], j & 1, abort_flag);
        }
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int half = kWide ? 1 : 0; half >= 0; --half) {
#pragma unroll
          for (int t = 0; t < kKeys; t += 16) {
            if (!kWide && t == kKeys / 2) {
              ok = mbar_wait(&bars->weights[i], j & 1, abort_flag);
              if (!ok) break;
              tc_fence_after_sync();
            }
            mma_f16_ts(tmem + 256 + (kWide ? j & 1 : i) * 128, tmem + (kWide ? j & 1 : i) * 128 + half * (kKeys / 2) + t / 2,
                       make_sw128_nmajor_desc(base + S::kValueRing + stage * S::kOperand + t * 128, kKeys * 128), sums_desc,
                       t > 0 || (kWide ? half == 0 : j > 0));
          }
        }
        if (!ok) break;
        if (kWide) {
          tc_commit(&bars->sums[j & 1]);
          continue;
        }
        if (j + 1 == tiles) {
          tc_commit(&bars->sums[i]);
          continue;
        }
        if (i == 0) ok = mbar_wait(&bars->key_full[after], (j + 1) >> 1 & 1, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        scores_of(i, after);
      }
      if (!ok) break;
      tc_commit(&bars->value_empty[stage]);
      if (kWide) {
        if (j + 2 >= tiles) continue;
        ok = mbar_wait(&bars->key_full[stage], (j + 2) >> 1 & 1, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        scores_of(0, stage);
        tc_commit(&bars->key_empty[stage]);
      } else if (j + 1 < tiles) {
        tc_commit(&bars->key_empty[after]);
      }
    }
    if (!ok) {
      *abort_flag = 1;
      report_error(p.batch.error, 43);
      tc_commit(&bars->drain);  // what is in flight ends before TMEM is freed
      const unsigned long long started = global_timer_ns();
      while (!mbar_try_wait(&bars->drain, 0) && global_timer_ns() - started < kWaitLimitNs) {
      }
    }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <int DP, int kUnit, bool kWide>
qx_status launch_prompt_of(const AttentionParams& p, long long grid, cudaStream_t stream) {
  static SmemOptIn opt_in;
  QX_TRY(opt_in.ensure(prompt_kernel<DP, kUnit, kWide>, TcShape<DP>::kBytes));
  return launch_behind(prompt_kernel<DP, kUnit, kWide>, grid, kTcThreads, TcShape<DP>::kBytes, stream, p);
}
template <bool kWide>
qx_status launch_prompt_sized(const AttentionParams& p, long long grid, cudaStream_t stream) {
  if (p.block_tokens < 32) {
    return p.dim <= 64 ? launch_prompt_of<64, 16, kWide>(p, grid, stream) : launch_prompt_of<128, 16, kWide>(p, grid, stream);
  }
  return p.dim <= 64 ? launch_prompt_of<64, 32, kWide>(p, grid, stream) : launch_prompt_of<128, 32, kWide>(p, grid, stream);
}

}  // namespace

qx_status launch_prompt(const AttentionParams& p, bool wide, long long grid, cudaStream_t stream) {
  return wide ? launch_prompt_sized<true>(p, grid, stream) : launch_prompt_sized<false>(p, grid, stream);
}

}  // namespace kv
}  // namespace qx
