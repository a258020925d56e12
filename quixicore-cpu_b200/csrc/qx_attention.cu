// Attention over the paged 8-bit cache, streamed: the kernel for single tokens, short runs of tokens, f32
// queries and every head size. (Long prompts of 16-bit queries: qx_attention_tc.cu.)
//
// softmax(scale q K^T) V with K = ks * codes, V = vs * codes, on warp-level MMAs with the cache as the operand
// of 16 rows, so that eight query rows (tokens x query heads of one kv head) fill the other side:
//   scores  [keys x rows]: the codes as they are (s8) against three balanced base-256 digits of the queries
//           (s8, 23 bits against the row's largest magnitude): exact whole-number sums. Those start at
//           1.5 * 2^23 as f32 bits, so that a subtraction makes f32 numbers of them;
//   output  [head elements x rows]: the codes as f16 (exact) against the weights as f16 (a rounding of 2^-11
//           relative, no further than the 16-bit outputs' own), as hi + lo pairs for f32 queries; f32 sums.
// The scales are applied to the sums: one multiplication per score (ks), one per 16 keys and output element (vs): a
// block of 16 keeps its own, however much larger its neighbour's is (blocks of 64 | 16 tokens, 32 sessions of up to 8192
// 64.6 | 67.2 us; one multiplication per 32 keys and the ratio of two blocks' scales in their weights, which loses those
// below 2^-26: 63.7 | 69.9, drafts 23.6 against 22.5).
//
// Split. A CTA takes 8 rows (16 where there are more) and a run of the keys; its four warps take tiles of 32
// keys in turn, each with a running maximum and sum of its own, and are joined at the end through shared
// memory. So one pass over the codes serves all heads of a group. Where every sequence is one tile of rows (tokens
// being decoded) the launch is balanced: the tiles of all sequences and kv heads form one line, which the resident
// CTAs cut into equal pieces, whatever the lengths; a CTA's first and last piece may be parts of an item (sequence,
// kv head), and the last CTA to finish a part of an item joins its parts, in their order. Otherwise keys are cut
// into chunks where there are few rows, joined by a second, small kernel.
//
// Data movement. Each warp has a ring of stages of its own (codes of 32 keys and values, their scales),
// filled by 16-byte asynchronous copies: tiles in flight while one is computed, nothing to wait for but the
// warp's own copies. The order of head elements inside a product, of keys inside P V and of output elements
// are free, so each lane takes the bytes that lie together (32 of a key row, 16 columns of four value rows):
// keys are MMA operands as they are read; values become f16 pairs of two keys by a byte permute and one
// logical operation (code ^ 0x6480 is 1152 + code). 16-byte pieces of a row are permuted among the eight bank
// groups so that these reads meet no conflicts for head sizes up to 128.
//
// Bound by HBM for long contexts: 2 * head_dim bytes per key and kv head, whatever the group. Measured (128 elements, 8
// kv heads): 32 sessions of up to 8192 tokens, 32 query heads, 64.5 us (314 MB, 4.9 TB/s, 0.74 of the copy bandwidth; 72
// where other calls' inputs have taken its own out of L2); one of 131072 tokens, 64 query heads, 54 us (5.0 TB/s; 61); one
// of 1000 tokens, f32, 7.5 us. What is above the bytes' time is a CTA's way in and out: about 9000 cycles before its first
// tile (cold instructions, length, table, queries) and 4000 behind its last. With 64 elements and 15 rows (drafts) the
// instructions bind: 32 sessions, windows of 4096, 55 us for 134 MB, issue slots 55 % taken.

#include <algorithm>
#include <cmath>

#include "qx_attention.cuh"

namespace qx {
namespace kv {
namespace {

// P is held times 2^12 where it is rounded to 16 bits, so that weights down to 2^-26 keep all their bits;
// sums of P carry the same factor, sums of P V do not (values near the end of f32's range stay in it).
constexpr float kShift = 12.0f;
constexpr float kCarried = 4096.0f, kCarriedInverse = 1.0f / kCarried;  // 2^kShift

constexpr int kWarps = 4, kThreads = 32 * kWarps, kTile = 32;
constexpr uint32_t kZeroSum = 0x4B400000u;  // 1.5 * 2^23: whole numbers below 2^22 added to the bits are exact

// Rows per sequence from which queries take the prompt kernel (f32 ones, of half as many rows per CTA and twice the
// products: later). Streamed | prompt kernel, us: f16, 4 sequences of 4096 keys, 32 rows 37 | 40, 48 rows 48 | 41, 192
// rows 101 | 54; one of 16384 keys, 48 rows 42 | 41; f32, 4 of 4096 keys, 64 rows 84 | 87, 100 rows 96 | 90; 16 whole
// texts of 64 tokens 25 | 29, of 100 tokens 40 | 32.
constexpr long long kPromptFrom = 48, kPromptFromWide = 96;

// CTAs per SM, as many as shared memory and 65536 registers hold.
constexpr int streamed_ctas(int dp, int row_tiles) { return dp == 64 ? (row_tiles == 1 ? 4 : 3) : dp == 128 ? (row_tiles == 1 ? 3 : 2) : 1; }

template <int DP, bool kWide, int kRowTiles>
struct Shape {
  static constexpr int kRows = 8 * kRowTiles;
  static constexpr int kChunks = DP / 16;                      // 16-byte pieces of a row
  static constexpr int kStageBytes = 2 * kTile * DP + 16;      // keys, values, scales
  static constexpr int kStages = DP == 64 ? 3 : 2;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kPitch = DP + 4;                        // floats per row when warps are joined
  static constexpr int kJoin = kWarps * kRows * (kPitch + 2) * 4;
  static constexpr int kQueries = 3 * kRows * DP;              // digits, as MMA operands
  static constexpr int kBytes = (kRing > kJoin ? kRing : kJoin) + kQueries + kRows * 4;
  static constexpr int kCtas = streamed_ctas(DP, kRowTiles);
};

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

// Codes are read once and leave L2 first: what every call needs again (its own instructions among it) stays.
__device__ __forceinline__ uint64_t evict_first() {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
template <int kLeft>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Byte `kByte` of a and of b, codes of two keys, as a pair of f16 codes.
template <int kByte>
__device__ __forceinline__ uint32_t codes_f16(uint32_t a, uint32_t b) {
  const uint32_t both = __byte_perm(a, b, 0x0400 + 0x0101 * kByte);
  const uint32_t raw = (both & 0x00FF00FFu) ^ 0x64806480u;  // 1024 + (code + 128)
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&raw), __half2half2(__ushort_as_half(0x6480)));  // 1152
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_s8(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first of a sum: from the bits of zero (1.5 * 2^23).
__device__ __forceinline__ void mma_s8_first(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kZeroSum));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit elements, a row's pairs in four lanes, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
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

// A balanced launch's line: per item, kItemCost units for what a CTA does before its first tile and behind its last, and
// one per tile (4 | 8 | 12 | 16 | 24 units, us: 32 sessions of up to 8192 66.4 | 65.0 | 64.5 | 64.7 | 67.2, 8 of five
// tokens in windows of 4096 29.0 | 26.7 | 26.2 | 26.2 | 27.0; later steps changed all alike).
constexpr int kItemCost = 12, kLeastPiece = 8, kBalancedSequences = 128;
struct Line {
  uint32_t begin[kBalancedSequences / 32];  // of sequence lane + 32 i
  uint32_t item[kBalancedSequences / 32];   // units per kv head
  uint32_t total, piece;                    // (the host has made sure that they fit)
};
template <int kRows>
__device__ __forceinline__ Line line_of(const AttentionParams& p) {
  const int lane = static_cast<int>(threadIdx.x & 31);
  Line line;
#pragma unroll
  for (int i = 0; i < kBalancedSequences / 32; ++i) {
    Rows rows;
    line.item[i] = 0;
    if (lane + 32 * i < p.batch.sequences && rows_of(p, lane + 32 * i, 0, kRows, &rows, true)) {
      line.item[i] = kItemCost + (rows.high - rows.low + kTile - 1) / kTile;
    }
  }
  line.total = 0;
#pragma unroll
  for (int i = 0; i < kBalancedSequences / 32; ++i) {
    line.begin[i] = line.total;
    if (32 * i >= p.batch.sequences) continue;
    const uint32_t cost = line.item[i] * p.kv_heads;
    uint32_t through = cost;
#pragma unroll
    for (int h = 1; h < 32; h <<= 1) {
      const uint32_t below = __shfl_up_sync(0xFFFFFFFFu, through, h);
      if (lane >= h) through += below;
    }
    line.begin[i] += through - cost;
    line.total += __shfl_sync(0xFFFFFFFFu, through, 31);
  }
  line.piece = max(static_cast<uint32_t>(kLeastPiece), (line.total + gridDim.x - 1) / gridDim.x);
  return line;
}
// The sequence at a place of the line, where it begins and its units per kv head.
__device__ __forceinline__ int sequence_at(const AttentionParams& p, const Line& line, uint32_t at, uint32_t* begin, uint32_t* item) {
  int found = 0;
#pragma unroll
  for (int i = 0; i < kBalancedSequences / 32; ++i) {
    if (32 * i >= p.batch.sequences) continue;
    const uint32_t lanes = __ballot_sync(0xFFFFFFFFu, at >= line.begin[i] && at - line.begin[i] < line.item[i] * p.kv_heads);
    if (lanes != 0) {
      const int lane = __ffs(lanes) - 1;
      found = lane + 32 * i;
      *begin = __shfl_sync(0xFFFFFFFFu, line.begin[i], lane);
      *item = __shfl_sync(0xFFFFFFFFu, line.item[i], lane);
    }
  }
  return found;
}

template <int DP, bool kWide, int kRowTiles, bool kBalanced>
__global__ void __launch_bounds__(kThreads, Shape<DP, kWide, kRowTiles>::kCtas)
    attention_kernel(const __grid_constant__ AttentionParams p) {
  using S = Shape<DP, kWide, kRowTiles>;
  constexpr int kRows = S::kRows, kStages = S::kStages, kSteps = DP / 32;  // steps of 32 head elements in a score
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  uint8_t* const queries = smem + (S::kRing > S::kJoin ? S::kRing : S::kJoin);
  float* const row_factor = reinterpret_cast<float*>(queries + S::kQueries);

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  __shared__ int last_part;
  Line line;
  uint32_t place = 0, place_end = 0;
  if (kBalanced) {
    line = line_of<kRows>(p);
    place_end = min((blockIdx.x + 1) * line.piece, line.total);
    place = min(blockIdx.x * line.piece, place_end);
  }
  for (bool once = true;; once = false) {
  int s, head, row_tile = 0, begin, end;
  long long part;           // where partial results go
  uint32_t first_part = 0;  // balanced: the first CTA that holds a part of the item
  uint32_t tile_index = 0;  // the item's number
  int parts = 1;
  Rows rows;
  if (kBalanced) {
    if (place >= place_end) return;
    uint32_t sequence_begin = 0, item = 1;
    s = sequence_at(p, line, place, &sequence_begin, &item);
    head = static_cast<int>((place - sequence_begin) / item);
    const uint32_t item_begin = sequence_begin + head * item, item_end = item_begin + item, stop = min(place_end, item_end);
    // (the item's first part is where its first tile is: a piece that ends before that leaves it to the next CTA)
    if (stop < item_end && stop - item_begin <= kItemCost) return;
    first_part = min(item_begin + kItemCost, item_end - 1) / line.piece;
    parts = static_cast<int>((item_end - 1) / line.piece - first_part) + 1;
    part = 2LL * blockIdx.x + (first_part == blockIdx.x ? 1 : 0);
    (void)rows_of(p, s, 0, kRows, &rows);
    tile_index = s * p.kv_heads + head;
    const int unit0 = max(0, static_cast<int>(place - item_begin) - kItemCost), unit1 = max(0, static_cast<int>(stop - item_begin) - kItemCost);
    begin = rows.low + unit0 * kTile;
    end = min(rows.high, rows.low + unit1 * kTile);
    place = stop;
  } else {
    if (!once) return;
    const uint32_t split = blockIdx.x % p.splits;
    tile_index = blockIdx.x / p.splits;
    const uint32_t index = tile_index / p.row_tiles;
    row_tile = static_cast<int>(tile_index - index * p.row_tiles);
    s = static_cast<int>(index / p.kv_heads);
    head = static_cast<int>(index - s * p.kv_heads);
    if (!rows_of(p, s, row_tile * kRows, kRows, &rows)) return;
    if (!chunk_of(p, rows, split, &begin, &end)) return;
    part = static_cast<long long>(blockIdx.x);
    parts = splits_used(p, rows);
  }
  const int32_t* const table = p.batch.table + s * p.batch.table_stride;
  const int tiles = (end - begin + kTile - 1) / kTile;  // (zero or less: the rows see nothing)

  // ---- copies -------------------------------------------------------------------------------
  const uint32_t ring = sm100::smem_u32(smem) + warp * (kStages * S::kStageBytes);
  uint8_t* const ring_bytes = smem + warp * (kStages * S::kStageBytes);
  const int pieces = p.dim / 16;
  const uint64_t policy = evict_first();
  // Ids of the two blocks that a tile's halves lie in (the same one from 32 tokens per block on); -1: nothing to see.
  const auto ids_of = [&](int tile, int (&id)[2]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int token = begin + tile * kTile + 16 * half;
      id[half] = -1;
      if (tile < tiles && token < end) {
        id[half] = table[token >> p.block_shift];
        if (static_cast<unsigned long long>(static_cast<long long>(id[half])) >= static_cast<unsigned long long>(p.batch.blocks)) {
          id[half] = -1;
          if (lane == 0) sm100::report_error(p.batch.error, kErrorBlock);
        }
      }
    }
  };
  // Of a tile's copies every lane has the same places in each stage: rows r of a half, 16-byte piece c.
  constexpr int kRowsAtOnce = 32 / S::kChunks > 0 ? 32 / S::kChunks : 1;
  const int own_row = lane / S::kChunks, own_piece = lane % S::kChunks;
  const auto issue = [&](int tile, int to_stage, const int (&id)[2]) {
    const uint32_t to = ring + to_stage * S::kStageBytes;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (id[half] < 0) continue;
      const int slot = (begin + tile * kTile + 16 * half) & (p.block_tokens - 1);
      const long long slice = static_cast<long long>(id[half]) * p.kv_heads + head;
      if (lane < 2) copy4(to + 2 * kTile * DP + 8 * lane + 4 * half, (lane == 0 ? p.k_scales : p.v_scales) + slice);
      const long long at = ((slice << p.block_shift) + slot) * p.dim;
      if (p.dim == DP) {  // (constant strides: the places are offsets in the instructions)
        const int8_t* const k = p.k_codes + at + own_row * DP + 16 * own_piece;
        const int8_t* const v = p.v_codes + at + own_row * DP + 16 * own_piece;
#pragma unroll
        for (int i = 0; i < 16 / kRowsAtOnce; ++i) {
          const int where = piece<DP>(16 * half + i * kRowsAtOnce + own_row, own_piece);
          copy16(to + where, k + i * kRowsAtOnce * DP, policy);
          copy16(to + kTile * DP + where, v + i * kRowsAtOnce * DP, policy);
        }
      } else {
        const long long from = at + own_row * p.dim + 16 * own_piece;
#pragma unroll
        for (int i = 0; i < 16 / kRowsAtOnce; ++i) {
          if (own_piece >= pieces) continue;
          const int where = piece<DP>(16 * half + i * kRowsAtOnce + own_row, own_piece);
          copy16(to + where, p.k_codes + from + i * kRowsAtOnce * p.dim, policy);
          copy16(to + kTile * DP + where, p.v_codes + from + i * kRowsAtOnce * p.dim, policy);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // Two bits for every tile in flight: which of its halves are there.
  uint32_t there = 0;
  const auto note = [&](const int (&id)[2]) { there = there << 2 | (id[0] >= 0 ? 1u : 0u) | (id[1] >= 0 ? 2u : 0u); };
  // (all loads that need no other's result before the first that does)
  int first_ids[kStages - 1][2], next_ids[2];
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) ids_of(warp + i * kWarps, first_ids[i]);
  ids_of(warp + (kStages - 1) * kWarps, next_ids);

  // ---- queries: whole numbers below 2^23 times a power of two per row, as three digits -----------------------
  // A lane takes four neighbouring elements (of 128 at a time; of two rows of 64), all of the warp's rows before any is
  // used.
  constexpr int kAtOnce = DP < 128 ? 128 / DP : 1, kRowLanes = 32 / kAtOnce;
  constexpr int kOwnRows = kRows / kWarps / kAtOnce, kOwnRuns = (DP + 127) / 128;
  const int own_lane = lane % kRowLanes;
  float v[kOwnRows][kOwnRuns][4];
#pragma unroll
  for (int own = 0; own < kOwnRows; ++own) {
    const int r = (own * kWarps + warp) * kAtOnce + lane / kRowLanes, token = (rows.first + r) / p.group;
    const long long base = (rows.row + token) * p.q.token_stride +
                           (static_cast<long long>(head) * p.group + (rows.first + r - token * p.group)) * p.q.head_stride;
#pragma unroll
    for (int i = 0; i < kOwnRuns; ++i) {
      const int d = i * 128 + own_lane * 4;
      v[own][i][0] = v[own][i][1] = v[own][i][2] = v[own][i][3] = 0.0f;
      if (r < rows.count && d < p.dim) load4(p.q.data, p.q.type, p.q.vector, base + d, v[own][i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    note(first_ids[i]);
    issue(warp + i * kWarps, i, first_ids[i]);
  }
#pragma unroll
  for (int own = 0; own < kOwnRows; ++own) {
    const int r = (own * kWarps + warp) * kAtOnce + lane / kRowLanes;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kOwnRuns; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[own][i][e]) & 0x7FFFFFFFu);
    }
    top = __reduce_max_sync(kAtOnce == 1 ? 0xFFFFFFFFu : lane < 16 ? 0xFFFFu : 0xFFFF0000u, top) >> 23;
    // the row's largest magnitude becomes 2^21 .. 2^22: three balanced digits reach 127 * (1 + 2^8 + 2^16)
    const int shift = min(126, max(-126, 148 - static_cast<int>(top)));
    const float factor = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
    if (own_lane == 0) {
      // (a row that holds a NaN or an infinity gives NaN)
      row_factor[r] = top >= 255 ? __uint_as_float(0x7FC00000u)
                                 : __uint_as_float(static_cast<uint32_t>(127 - shift) << 23) * p.scale_log2;
    }
#pragma unroll
    for (int i = 0; i < kOwnRuns; ++i) {
      const int d = i * 128 + own_lane * 4;
      uint32_t x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // digits + 128 are the bytes of x + 128 (1 + 2^8 + 2^16)
        const int whole = top >= 255 ? 0 : __float2int_rn(v[own][i][e] * factor);
        x[e] = static_cast<uint32_t>(whole + 0x808080) ^ 0x808080u;
      }
      // operand of step j: lane (row, t) holds elements 8 j .. 8 j + 7 of its share
      const int own_t = d / (DP / 4), rest = d % (DP / 4);
      const int at = ((r >> 3) * kSteps + rest / 8) * 256 + ((r & 7) * 4 + own_t) * 8 + rest % 8;
      if (d < DP) {
#pragma unroll
        for (int digit = 0; digit < 3; ++digit) {
          const uint32_t select = digit | (4 + digit) << 4;
          *reinterpret_cast<uint32_t*>(queries + digit * kRows * DP + at) =
              __byte_perm(__byte_perm(x[0], x[1], select), __byte_perm(x[2], x[3], select), 0x5410);
        }
      }
    }
  }
  __syncthreads();
  // (in registers where there is room for them, else read as they are needed)
  constexpr bool kResident = DP <= 64 && (kRowTiles == 1 || !kWide);
  constexpr int kOperands = 3 * kSteps * kRowTiles;
  uint2 resident[kResident ? kOperands : 1];
  if (kResident) {
#pragma unroll
    for (int i = 0; i < kOperands; ++i) resident[i] = reinterpret_cast<const uint2*>(queries)[i * 32 + lane];
  }
  const auto query = [&](int digit, int n, int j) {
    if (kResident) return resident[((digit * kRowTiles + n) * kSteps + j) % kOperands];
    return reinterpret_cast<const uint2*>(queries + digit * kRows * DP)[(n * kSteps + j) * 32 + lane];
  };

  // ---- this lane's rows: 2 t and 2 t + 1 of every tile of eight -----------------------------------------------
  const int start = rows.length - rows.n, position0 = start + rows.first / p.group;
  const int position1 = start + (rows.first + rows.count - 1) / p.group;
  const int open_high = p.causal ? min(rows.length, position0 + 1) : rows.length;  // below: no key is hidden
  const int open_low = first_seen(p, position1);
  float factor[kRowTiles][2];
  int low[kRowTiles][2], high[kRowTiles][2];  // keys [low, high) of the row
#pragma unroll
  for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * n + 2 * t + e;
      factor[n][e] = row_factor[r];
      low[n][e] = high[n][e] = 0;
      if (r < rows.count) {
        const int position = start + (rows.first + r) / p.group;
        high[n][e] = p.causal ? min(rows.length, position + 1) : rows.length;
        low[n][e] = first_seen(p, position);
      }
    }
  }

  float o[kRowTiles][DP / 16][4];
  float most[kRowTiles][2], sum[kRowTiles][2];
#pragma unroll
  for (int n = 0; n < kRowTiles; ++n) {
    most[n][0] = most[n][1] = -INFINITY;
    sum[n][0] = sum[n][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
  }

  int stage = 0;
  for (int tile = warp; tile < tiles; tile += kWarps) {
    const int ahead = tile + (kStages - 1) * kWarps;
    issue(ahead, stage == 0 ? kStages - 1 : stage - 1, next_ids);
    note(next_ids);
    ids_of(ahead + kWarps, next_ids);
    wait_copies<kStages - 1>();
    __syncwarp();
    const uint8_t* const keys = ring_bytes + stage * S::kStageBytes;
    const uint8_t* const values = keys + kTile * DP;
    const float* const meta = reinterpret_cast<const float*>(values + kTile * DP);
    const int token0 = begin + tile * kTile;
    const uint32_t present = there >> (2 * (kStages - 1)) & 3;
    const float4 scales = *reinterpret_cast<const float4*>(meta);
    // (of a half that is not there the stage holds anything)
    const float ks[2] = {scales.x, scales.y};
    const float vs[2] = {present & 1 ? scales.z * kCarriedInverse : 0.0f, present & 2 ? scales.w * kCarriedInverse : 0.0f};
    const bool open = token0 + kTile <= open_high && token0 >= open_low && present == 3;

    // ---- scores of 16 keys at a time: lane (g, t) gets keys g, g + 8 and rows 2 t, 2 t + 1 ----------------------
    float score[kRowTiles][2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t w[2][DP / 16];  // this lane's share of keys g and g + 8: DP / 4 codes
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < DP / 64; ++i) {
          const uint4 f = *reinterpret_cast<const uint4*>(keys + piece<DP>(16 * k + 8 * h + g, DP / 64 * t + i));
          w[h][4 * i] = f.x;
          w[h][4 * i + 1] = f.y;
          w[h][4 * i + 2] = f.z;
          w[h][4 * i + 3] = f.w;
        }
      }
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
        uint32_t digit[3][4];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            const uint2 b = query(i, n, j);
            if (j == 0) mma_s8_first(digit[i], w[0][0], w[1][0], w[0][1], w[1][1], b.x, b.y);
            else mma_s8(digit[i], w[0][2 * j], w[1][2 * j], w[0][2 * j + 1], w[1][2 * j + 1], b.x, b.y);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float zero = __uint_as_float(kZeroSum);
          const float d0 = __uint_as_float(digit[0][e]) - zero, d1 = __uint_as_float(digit[1][e]) - zero;
          const float d2 = __uint_as_float(digit[2][e]) - zero;
          score[n][k][e] = fmaf(d2, 65536.0f, fmaf(d1, 256.0f, d0)) * (factor[n][e & 1] * ks[k]);
        }
      }
    }

    // ---- softmax --------------------------------------------------------------------------
    // The scale of a half's values for a row: zero where the row sees none of them, so that a scale that is no number
    // meets weights of zero nowhere.
    float gain[kRowTiles][2][2];
#pragma unroll
    for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
      for (int k = 0; k < 2; ++k) gain[n][k][0] = gain[n][k][1] = vs[k];
    }
    if (!open) {
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int first = token0 + 16 * k;
            const bool sees = (present >> k & 1) && low[n][e] < first + 16 && high[n][e] > max(first, low[n][e]);
            if (!sees) gain[n][k][e] = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = first + 8 * h + g;
              if (!(present >> k & 1) || key < low[n][e] || key >= high[n][e]) score[n][k][2 * h + e] = -INFINITY;
            }
          }
        }
      }
      __syncwarp();  // (a branch, not predicates: most tiles skip this)
    }
    uint32_t weight[kRowTiles][4], low_weight[kRowTiles][4];  // of 8 keys each, as operands
    float keep[kRowTiles][2];
    bool moved = false;
#pragma unroll
    for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = fmaxf(fmaxf(score[n][0][e], score[n][0][2 + e]), fmaxf(score[n][1][e], score[n][1][2 + e]));
#pragma unroll
        for (int h = 4; h <= 16; h <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, h));
        top = fmaxf(top, most[n][e]);
        // (a row that has seen nothing yet: weights exp2(-inf) = 0 against any finite maximum)
        const float base = top == -INFINITY ? 0.0f : top, less = base - kShift;
        keep[n][e] = exp2_fast(most[n][e] - base);
        moved = moved || top != most[n][e];
        most[n][e] = top;
        float total = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& v = score[n][k][2 * h + e];
            v = exp2_fast(v - less);
            total += v;
          }
        }
        sum[n][e] = fmaf(sum[n][e], keep[n][e], total);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float a = score[n][k][2 * h], b = score[n][k][2 * h + 1];
          const uint32_t rounded = pair_f16(a, b);
          weight[n][2 * k + h] = transposed(rounded);
          if (kWide) low_weight[n][2 * k + h] = transposed(rest_f16(a, b, rounded));
        }
      }
    }
    if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          o[n][i][0] *= keep[n][0];
          o[n][i][1] *= keep[n][1];
          o[n][i][2] *= keep[n][0];
          o[n][i][3] *= keep[n][1];
        }
      }
    }

    // ---- values x weights: lane (g, t) gets head elements DP / 8 * g .. and rows 2 t, 2 t + 1 -------------------
    constexpr int kWords = 2;  // of a value row per lane and load
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
      uint32_t w[2][4][kWords];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 16 * k + 2 * t + (e & 1) + 8 * (e >> 1), at = DP / 64 * g + i;  // in pieces of 8 bytes
          const uint2 f = *reinterpret_cast<const uint2*>(values + piece<DP>(r, at >> 1) + 8 * (at & 1));
          w[k][e][0] = f.x;
          w[k][e][1] = f.y;
        }
      }
#pragma unroll
      for (int word = 0; word < kWords; ++word) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // two of the word's four head elements
          uint32_t a[2][4];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t(&u)[4][kWords] = w[k];
            a[k][0] = h == 0 ? codes_f16<0>(u[0][word], u[1][word]) : codes_f16<2>(u[0][word], u[1][word]);
            a[k][1] = h == 0 ? codes_f16<1>(u[0][word], u[1][word]) : codes_f16<3>(u[0][word], u[1][word]);
            a[k][2] = h == 0 ? codes_f16<0>(u[2][word], u[3][word]) : codes_f16<2>(u[2][word], u[3][word]);
            a[k][3] = h == 0 ? codes_f16<1>(u[2][word], u[3][word]) : codes_f16<3>(u[2][word], u[3][word]);
          }
#pragma unroll
          for (int n = 0; n < kRowTiles; ++n) {
            float (&out)[4] = o[n][4 * i + 2 * word + h];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float acc[4];
              mma_f16_first(acc, a[k], weight[n][2 * k], weight[n][2 * k + 1]);
              if (kWide) mma_f16(acc, a[k], low_weight[n][2 * k], low_weight[n][2 * k + 1]);
              out[0] = fmaf(acc[0], gain[n][k][0], out[0]);
              out[1] = fmaf(acc[1], gain[n][k][1], out[1]);
              out[2] = fmaf(acc[2], gain[n][k][0], out[2]);
              out[3] = fmaf(acc[3], gain[n][k][1], out[3]);
            }
          }
        }
      }
    }
    __syncwarp();  // the stage is free for the next copies
    if (++stage == kStages) stage = 0;
  }

  // ---- the four warps joined ---------------------------------------------------------------
  wait_copies<0>();
  __syncthreads();
  float* const joined = reinterpret_cast<float*>(smem);
  float* const stats = joined + kWarps * kRows * S::kPitch;  // [warp][row] {maximum, sum}
#pragma unroll
  for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int h = 4; h <= 16; h <<= 1) sum[n][e] += __shfl_xor_sync(0xFFFFFFFFu, sum[n][e], h);
      const int r = warp * kRows + 8 * n + 2 * t + e;
      float* const to = joined + r * S::kPitch + g * (DP / 8);
#pragma unroll
      for (int i = 0; i < DP / 16; i += 2) {
        *reinterpret_cast<float4*>(to + 2 * i) = make_float4(o[n][i][e], o[n][i][2 + e], o[n][i + 1][e], o[n][i + 1][2 + e]);
      }
      if (g == 0) *reinterpret_cast<float2*>(stats + 2 * r) = make_float2(most[n][e], sum[n][e]);
    }
  }
  __syncthreads();
  const bool whole = parts == 1;
  const int per_row = p.dim / 8;
  const auto place_of = [&](int r, long long* out_row, long long* out_head) {
    const int token = (rows.first + r) / p.group;
    *out_row = rows.row + token;
    *out_head = static_cast<long long>(head) * p.group + (rows.first + r - token * p.group);
  };
  for (int i = threadIdx.x; i < rows.count * per_row; i += kThreads) {
    const int r = i / per_row, d = (i - r * per_row) * 8;
    float top = -INFINITY, total = 0.0f, v[8], weight[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats[2 * (w * kRows + r)]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      weight[w] = exp2_fast(stats[2 * (w * kRows + r)] - base);
      total += stats[2 * (w * kRows + r) + 1] * weight[w];
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
      const long long at = part * kRows + r;
      float4* const to = reinterpret_cast<float4*>(p.partial + at * p.dim + d);
      to[0] = make_float4(v[0], v[1], v[2], v[3]);
      to[1] = make_float4(v[4], v[5], v[6], v[7]);
      if (d == 0) *reinterpret_cast<float2*>(p.statistics + 2 * at) = make_float2(top, total);
      continue;
    }
    long long out_row, out_head;
    place_of(r, &out_row, &out_head);
    const float inverse = total == 0.0f ? 0.0f : kCarried / total;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= inverse;
    store8(p.out.data, p.out.type, p.out.vector, out_row * p.out.token_stride + out_head * p.out.head_stride + d, v);
    if (p.lse != nullptr && d == 0) {
      p.lse[out_row * p.out.heads + out_head] =
          total == 0.0f ? -INFINITY : (top + log2f(total) - kShift) * 0.69314718055994531f;
    }
  }
  if (kBalanced || p.counters != nullptr) {
    if (!whole) {
      // The CTA that arrives last at the item's counter joins its parts, all of them from memory and in their order.
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        int* const counter = p.counters + tile_index;
        last_part = atomicAdd(counter, 1) == parts - 1;
        if (last_part) *counter = 0;
      }
      __syncthreads();
      if (last_part) {
        __threadfence();
        const int vectors = p.dim / 4;
        for (int i = threadIdx.x; i < rows.count * vectors; i += kThreads) {
          const int r = i / vectors, at = i - r * vectors;
          float top = -INFINITY, total = 0.0f;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          constexpr int kBatch = 8;  // loads under way
          for (int q0 = 0; q0 < parts; q0 += kBatch) {
            float2 stat[kBatch];
            float4 x[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              // (the item begins behind others in its first CTA, and at the start of the following ones)
              const long long from = (kBalanced ? 2LL * (first_part + q0 + b) + (q0 + b == 0 ? 1 : 0)
                                                : static_cast<long long>(tile_index) * p.splits + q0 + b) * kRows + r;
              stat[b] = make_float2(-INFINITY, 0.0f);
              x[b] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (q0 + b < parts) {
                stat[b] = __ldcg(reinterpret_cast<const float2*>(p.statistics) + from);
                x[b] = __ldcg(reinterpret_cast<const float4*>(p.partial + from * p.dim) + at);
              }
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              const float most = fmaxf(top, stat[b].x), base = most == -INFINITY ? 0.0f : most;
              const float keep = exp2_fast(top - base), weight = exp2_fast(stat[b].x - base);
              top = most;
              total = fmaf(total, keep, stat[b].y * weight);
              v.x = fmaf(v.x, keep, x[b].x * weight);
              v.y = fmaf(v.y, keep, x[b].y * weight);
              v.z = fmaf(v.z, keep, x[b].z * weight);
              v.w = fmaf(v.w, keep, x[b].w * weight);
            }
          }
          const float inverse = total == 0.0f ? 0.0f : kCarried / total;
          long long out_row, out_head;
          place_of(r, &out_row, &out_head);
          const long long to = out_row * p.out.token_stride + out_head * p.out.head_stride + 4 * at;
          store_one(p.out.data, p.out.type, to, v.x * inverse);
          store_one(p.out.data, p.out.type, to + 1, v.y * inverse);
          store_one(p.out.data, p.out.type, to + 2, v.z * inverse);
          store_one(p.out.data, p.out.type, to + 3, v.w * inverse);
          if (at == 0 && p.lse != nullptr) {
            p.lse[out_row * p.out.heads + out_head] =
                total == 0.0f ? -INFINITY : (top + log2f(total) - kShift) * 0.69314718055994531f;
          }
        }
      }
    }
    __syncthreads();  // shared memory is the next piece's
  }
  }
}

// Joins the chunks of one row, in an order that their number fixes: the threads are cut into parts, a thread of part i
// takes four head elements of chunks i, i + parts, ..., with several chunks' loads under way before it uses the first.
// Few chunks take 128 threads, many 512 (54 chunks of 64 rows: 14 us with 128 threads, one load after the other).
constexpr int kJoinThreads = 512, kJoinBatch = 4;
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
  if (!rows_of(p, s, row_tile * p.tile_rows, p.tile_rows, &rows) || r >= rows.count) return;
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

template <int DP, bool kWide, int kRowTiles, bool kBalanced>
qx_status launch_streamed(const AttentionParams& p, long long grid, cudaStream_t stream) {
  static SmemOptIn opt_in;
  constexpr int bytes = Shape<DP, kWide, kRowTiles>::kBytes;
  QX_TRY(opt_in.ensure(attention_kernel<DP, kWide, kRowTiles, kBalanced>, bytes));
  return launch_behind(attention_kernel<DP, kWide, kRowTiles, kBalanced>, grid, kThreads, bytes, stream, p);
}
template <int DP, bool kWide>
qx_status launch_rows(const AttentionParams& p, bool balanced, long long grid, cudaStream_t stream) {
  if (p.tile_rows == 8) {
    return balanced ? launch_streamed<DP, kWide, 1, true>(p, grid, stream) : launch_streamed<DP, kWide, 1, false>(p, grid, stream);
  }
  return balanced ? launch_streamed<DP, kWide, 2, true>(p, grid, stream) : launch_streamed<DP, kWide, 2, false>(p, grid, stream);
}
qx_status launch_sized(const AttentionParams& p, int dp, bool wide, bool balanced, long long grid, cudaStream_t stream) {
  if (dp == 64) return wide ? launch_rows<64, true>(p, balanced, grid, stream) : launch_rows<64, false>(p, balanced, grid, stream);
  if (dp == 128) return wide ? launch_rows<128, true>(p, balanced, grid, stream) : launch_rows<128, false>(p, balanced, grid, stream);
  return wide ? launch_rows<256, true>(p, balanced, grid, stream) : launch_rows<256, false>(p, balanced, grid, stream);
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
  while ((1 << p.block_shift) < p.block_tokens) ++p.block_shift;
  p.dim = cache->head_dim;
  p.q = device_heads(q);
  p.out = device_heads(out);
  p.lse = lse;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.causal = causal != 0;
  p.window = static_cast<int>(std::min<long long>(window, 0x7FFFFFFF));
  p.group = q->heads / cache->kv_heads;
  const long long most_rows = static_cast<long long>(batch->max_tokens) * p.group;
  const bool wide = q->type == QX_STORAGE_F32;
  const bool prompt = cache->head_dim <= 128 && most_rows >= (wide ? kPromptFromWide : kPromptFrom);
  p.tile_rows = prompt ? (wide ? kPromptRowsWide : kPromptRows) : most_rows <= 8 ? 8 : 16;
  p.shift = prompt ? kPromptShift : kShift;
  p.row_tiles = static_cast<int>((most_rows + p.tile_rows - 1) / p.tile_rows);
  const long long items = static_cast<long long>(batch->sequences) * cache->kv_heads * p.row_tiles;
  // Most keys that a tile can see.
  long long range = batch->max_length;
  if (p.window > 0 && p.causal) range = std::min<long long>(range, static_cast<long long>(p.window) + p.tile_rows);
  range += 31;  // (from a multiple of 32 on)
  // Chunks: one sequence fills the card with one round of equal chunks; several, of lengths that only the
  // device knows, get half as many again (measured with 1 | 1.5 | 3 | 6 rounds, us: 32 sessions of 1200 to 8192
  // 87 | 84 | 85 | 85, of up to 2000 31 | 34 | 38 | 38, 8 sessions of up to 20000 64 | 58 | 57 | 67). No chunk is
  // below a tile per warp (in the prompt kernel, four tiles): then the joining would cost more than the keys.
  const int dp = cache->head_dim <= 64 ? 64 : cache->head_dim <= 128 ? 128 : 256;
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
    return launch_sized(p, dp, wide, true, grid, stream);
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
  QX_TRY(prompt ? launch_prompt(p, wide, grid, stream) : launch_sized(p, dp, wide, false, grid, stream));
  return p.splits > 1 && p.counters == nullptr ? launch_behind(join_kernel, items * p.tile_rows, p.splits <= 16 ? 128 : kJoinThreads, 0, stream, p) : QX_STATUS_OK;
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
  return kv::launch_attention(cache, batch, q, out, lse_dev, scale, causal, window, ctx, workspace,
                              static_cast<cudaStream_t>(stream));
}
