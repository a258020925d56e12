// The paged key-value cache in 8 bits: append (rotation, scales, codes) and read.
//
// The unit of work is a (sequence, block that its new tokens reach, kv head) of the keys or of the values:
// one CTA owns the block's scale and codes, so nothing is atomic and the result does not depend on order.
// A code needs the block's final scale, so the new elements wait in registers for it (two units of 16 per thread
// at most; larger blocks are read twice, the second time out of the caches). Bound by HBM for prompts (element
// in, code out) and by the chain of loads length -> block -> scale for single tokens.
//
// Measured with the read behind it: 6570 f32 tokens of 8 heads of 128 elements, 49 us together (184 MB, 3.7 TB/s; the
// append 28 us by itself, under a profiler: waiting for its loads, issue slots half taken); 64 single bf16 tokens with
// 32 rotated query heads each, 14.7 us.

#include <algorithm>
#include <limits>

#include "qx_kv.cuh"

namespace qx {
namespace kv {
namespace {

constexpr int kThreads = 256;
// 2^-100: from here on every product and remainder below is a normal number, and so exact where it has to be.
constexpr float kSmallestScale = 7.8886090522101181e-31f;

struct AppendParams {
  Batch batch;
  int8_t* codes[2];    // keys, values
  float* scales[2];
  Heads x[2];
  Heads q, q_out;
  Rotation rotation;   // rotary 0: none
  const int64_t* positions;
  int kv_heads, block_tokens, dim;
  int blocks_per_sequence;  // that max_tokens tokens can reach
  int heads_per_cta, head_groups;
  int tokens_per_cta, query_ctas;  // of the queries: per CTA, CTAs per sequence
};

// Codes of x: the exact quotients x / scale rounded half to even. Added to 1.5 * 2^23 a quotient is rounded to a whole
// number, whose low byte is the code. That is off by one at most, and only where the remainder x - r * scale, exact in
// f32 (a multiple of half an ulp of the scale, no larger than the scale), reaches half a scale.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float scale, float inverse) {
  constexpr float kZero = 12582912.0f;
  const float half = 0.5f * scale;
  float m[8], furthest = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = fmaf(x[i], inverse, kZero);
    furthest = fmaxf(furthest, fabsf(fmaf(-(m[i] - kZero), scale, x[i])));
  }
  if (furthest >= half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float rest = fmaf(-(m[i] - kZero), scale, x[i]);
      const bool tie_to_odd = fabsf(rest) == half && (__float_as_uint(m[i]) & 1);
      if (fabsf(rest) > half || tie_to_odd) m[i] += copysignf(1.0f, rest);
    }
  }
  const auto word = [&](int i) {
    return __byte_perm(__byte_perm(__float_as_uint(m[i]), __float_as_uint(m[i + 1]), 0x40),
                       __byte_perm(__float_as_uint(m[i + 2]), __float_as_uint(m[i + 3]), 0x40), 0x5410);
  };
  return make_uint2(word(0), word(4));
}
// An older code on the grown scale: round half to even of code * before / scale. The products have at most
// 32 bits, so in 64-bit floats they and their difference are exact.
__device__ __forceinline__ int regrown(int code, double before, double scale, float ratio) {
  double r = rint(static_cast<double>(static_cast<float>(code) * ratio));
  const double rest = code * before - r * scale, half = 0.5 * scale;
  if (fabs(rest) > half || (fabs(rest) == half && (static_cast<int>(r) & 1))) r += copysign(1.0, rest);
  return static_cast<int>(r);
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (a & 255) | (b & 255) << 8 | (c & 255) << 16 | static_cast<uint32_t>(d) << 24;
}
__device__ __forceinline__ void rotate_queries(const AppendParams& p, long long item, float2* table) {
  const int s = static_cast<int>(item / p.query_ctas), chunk = static_cast<int>(item % p.query_ctas);
  Sequence q;
  if (!sequence_of(p.batch, s, true, &q)) return;
  const int token0 = chunk * p.tokens_per_cta, count = min(p.tokens_per_cta, q.n - token0);
  if (count <= 0) return;
  const int pairs = p.rotation.rotary / 2, units = p.dim / 16;
  for (int i = threadIdx.x; i < count * pairs; i += kThreads) {
    const int token = token0 + i / pairs;
    const long long position = p.positions != nullptr ? p.positions[q.row + token] : q.length - q.n + token;
    table[i] = turn(p.rotation, position, i % pairs);
  }
  __syncthreads();
  const int at_once = kThreads / units, first = threadIdx.x / units;
  if (first >= at_once) return;
  const Unit u = unit_of(static_cast<int>(threadIdx.x) - first * units, p.rotation.rotary, p.rotation.interleaved, p.dim);
  for (Walk walk(first, at_once, p.q.heads); walk.token < count; walk.advance()) {
    const long long from = (q.row + token0 + walk.token) * p.q.token_stride + walk.head * p.q.head_stride;
    const long long to = (q.row + token0 + walk.token) * p.q_out.token_stride + walk.head * p.q_out.head_stride;
    float a[8], b[8];
    load8(p.q.data, p.q.type, p.q.vector, from + u.first, a);
    load8(p.q.data, p.q.type, p.q.vector, from + u.second, b);
    rotate_unit(u, p.rotation.interleaved, table + walk.token * pairs, a, b);
    store8(p.q_out.data, p.q_out.type, p.q_out.vector, to + u.first, a);
    store8(p.q_out.data, p.q_out.type, p.q_out.vector, to + u.second, b);
  }
}

// kHeld: units of 16 elements that a thread holds in registers as they came, where the block has no more than that
// many per thread; the next head's are loaded while this one's are written. kType: their type, of keys and values.
// kHeld 0: any size, types and alignment, each element read twice.
template <int kHeld, int kType>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ __align__(16) float2 table[];
  __shared__ uint32_t warp_max[2][kThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const uint32_t per_kind = static_cast<uint32_t>(p.batch.sequences) * p.blocks_per_sequence * p.head_groups;
  uint32_t item = blockIdx.x;
  if (item >= 2 * per_kind) {
    rotate_queries(p, item - 2 * per_kind, table);
    return;
  }
  const int kind = item >= per_kind ? 1 : 0;
  item -= kind * per_kind;
  const uint32_t at = item / p.head_groups;
  const int group = static_cast<int>(item - at * p.head_groups);
  const int s = static_cast<int>(at / p.blocks_per_sequence), reached = static_cast<int>(at - s * p.blocks_per_sequence);
  Sequence q;
  if (!sequence_of(p.batch, s, true, &q) || q.n == 0) return;
  const int first = q.length - q.n;
  const int block_index = first / p.block_tokens + reached;
  const int begin = block_index * p.block_tokens;  // position of the block's slot 0
  if (begin >= q.length) return;
  const int from = max(first, begin), to = min(q.length, begin + p.block_tokens);
  const int kept = from - begin, count = to - from;  // older tokens of the block, new ones
  const long long row = q.row + (from - first);
  const Heads& x = p.x[kind];
  const bool rotated = kind == 0 && p.rotation.rotary > 0;
  const int pairs = p.rotation.rotary / 2, units = p.dim / 16, total = count * units;
  const int head0 = group * p.heads_per_cta, head1 = min(p.kv_heads, head0 + p.heads_per_cta);

  constexpr int kUnits = kHeld > 0 ? kHeld : 1, kWords = kType == QX_STORAGE_F32 ? 2 : 1;
  Unit unit[kUnits];
  int token[kUnits];
  long long source[kUnits];
  uint4 held[kUnits][2][kWords], next[kUnits][2][kWords];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const int i = threadIdx.x + k * kThreads;
    token[k] = i / units;
    unit[k] = unit_of(i - token[k] * units, rotated ? p.rotation.rotary : 0, p.rotation.interleaved, p.dim);
    source[k] = (row + token[k]) * x.token_stride + head0 * x.head_stride;
  }
  const auto load_held = [&]() {
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      if (threadIdx.x + k * kThreads < total) {
        load8_words<kType>(x.data, source[k] + unit[k].first, next[k][0]);
        load8_words<kType>(x.data, source[k] + unit[k].second, next[k][1]);
        source[k] += x.head_stride;
      }
    }
  };
  if (kHeld > 0) load_held();  // (needs no block)

  const long long block = p.batch.table[s * p.batch.table_stride + block_index];
  if (block < 0 || block >= p.batch.blocks) {
    if (threadIdx.x == 0) sm100::report_error(p.batch.error, kErrorBlock);
    return;
  }
  if (rotated) {
    for (int i = threadIdx.x; i < count * pairs; i += kThreads) {
      const int t = i / pairs;
      const long long position = p.positions != nullptr ? p.positions[row + t] : from + t;
      table[i] = turn(p.rotation, position, i - t * pairs);
    }
    __syncthreads();
  }
  for (int head = head0; head < head1; ++head) {
    // Magnitudes are compared as bit patterns: above those of all numbers come infinity and NaN.
    uint32_t top = 0;
    const auto measure = [&](const float (&a)[8], const float (&b)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = max(top, max(__float_as_uint(a[e]) & 0x7FFFFFFFu, __float_as_uint(b[e]) & 0x7FFFFFFFu));
      }
    };
    const auto held_unit = [&](int k, float (&a)[8], float (&b)[8]) {
      from_words<kType>(held[k][0], a);
      from_words<kType>(held[k][1], b);
      if (rotated) rotate_unit(unit[k], p.rotation.interleaved, table + token[k] * pairs, a, b);
    };
    const auto loaded_unit = [&](int i, Unit* u, float (&a)[8], float (&b)[8]) {
      const int t = i / units;
      *u = unit_of(i - t * units, rotated ? p.rotation.rotary : 0, p.rotation.interleaved, p.dim);
      const long long base = (row + t) * x.token_stride + head * x.head_stride;
      load8(x.data, x.type, x.vector, base + u->first, a);
      load8(x.data, x.type, x.vector, base + u->second, b);
      if (rotated) rotate_unit(*u, p.rotation.interleaved, table + t * pairs, a, b);
      return t;
    };
    float* const scale_at = p.scales[kind] + block * p.kv_heads + head;
    const float before = kept > 0 ? *scale_at : 0.0f;
    if (kHeld > 0) {
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          held[k][0][w] = next[k][0][w];
          held[k][1][w] = next[k][1][w];
        }
      }
      if (head + 1 < head1) load_held();
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        if (threadIdx.x + k * kThreads >= total) continue;
        if (kType != QX_STORAGE_F32 && !rotated) {
          // two 16-bit patterns at a time; the largest stands for its f32 value
          uint32_t pair = 0;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint4& w = held[k][r][0];
            pair = __vimax3_u16x2(pair, w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu);
            pair = __vimax3_u16x2(pair, w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu);
          }
          const uint32_t most = max(pair & 0xFFFFu, pair >> 16);
          const float value = kType == QX_STORAGE_F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(most)))
                                                      : __uint_as_float(most << 16);
          top = max(top, __float_as_uint(value));
        } else {
          float a[8], b[8];
          held_unit(k, a, b);
          measure(a, b);
        }
      }
    } else {
      for (int i = threadIdx.x; i < total; i += kThreads) {
        Unit u;
        float a[8], b[8];
        loaded_unit(i, &u, a, b);
        measure(a, b);
      }
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    // (two sets in turn: the one before is read until the next barrier)
    if ((threadIdx.x & 31) == 0) warp_max[head & 1][threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) top = max(top, warp_max[head & 1][w]);
    const bool number = top < 0x7F800000u && (__float_as_uint(before) & 0x7FFFFFFFu) < 0x7F800000u;
    float scale = fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), before);
    if (scale < kSmallestScale) scale = 0.0f;
    const float inverse = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    if (threadIdx.x == 0) *scale_at = number ? scale : __uint_as_float(0x7FC00000u);
    int8_t* const codes = p.codes[kind] + (block * p.kv_heads + head) * p.block_tokens * p.dim;
    if (number && scale > before) {  // (beside a scale of zero all codes stand for zeros, whatever they are)
      const float ratio = before * inverse;
      for (int i = threadIdx.x; i < kept * units; i += kThreads) {
        uint4* const words = reinterpret_cast<uint4*>(codes) + i;
        uint4 v = *words;
        uint32_t* const w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          int c[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            c[e] = before > 0.0f ? regrown(static_cast<int8_t>(w[k] >> (8 * e)), before, scale, ratio) : 0;
          }
          w[k] = pack4(c[0], c[1], c[2], c[3]);
        }
        *words = v;
      }
    }
    const auto write = [&](const Unit& u, int t, const float (&a)[8], const float (&b)[8]) {
      int8_t* const out = codes + (kept + t) * p.dim;
      uint2 first8 = make_uint2(0, 0), second8 = make_uint2(0, 0);
      if (number && scale > 0.0f) {
        first8 = codes8(a, scale, inverse);
        second8 = codes8(b, scale, inverse);
      }
      *reinterpret_cast<uint2*>(out + u.first) = first8;
      *reinterpret_cast<uint2*>(out + u.second) = second8;
    };
    if (kHeld > 0) {
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        if (threadIdx.x + k * kThreads >= total) continue;
        float a[8], b[8];
        held_unit(k, a, b);
        write(unit[k], token[k], a, b);
      }
    } else {
      for (int i = threadIdx.x; i < total; i += kThreads) {
        Unit u;
        float a[8], b[8];
        const int t = loaded_unit(i, &u, a, b);
        write(u, t, a, b);
      }
    }
  }
}

struct ReadParams {
  Batch batch;
  const int8_t* codes[2];
  const float* scales[2];
  Heads x[2];  // data NULL: not wanted
  int kv_heads, block_tokens, dim;
  int blocks_per_sequence, heads_per_cta, head_groups;
};

// A CTA takes the tokens that a sequence has in one block, of a few heads: their codes lie together. A thread takes
// as many codes as give 16 bytes of values (4 of f32, 8 of 16-bit ones), so that a warp's stores lie side by side, and
// four tokens' at a time.
template <bool kWide>
__device__ __forceinline__ void read_plane(const ReadParams& p, int kind, long long block, long long row, int slot, int count,
                                           int head0, int head1) {
  const Heads& x = p.x[kind];
  constexpr int kUnit = kWide ? 4 : 8, kBatch = 4;
  const int units = p.dim / kUnit, at_once = kThreads / units, first = threadIdx.x / units;
  if (first >= at_once) return;
  const int d = (static_cast<int>(threadIdx.x) - first * units) * kUnit;
  for (int head = head0; head < head1; ++head) {
    const long long slice = block * p.kv_heads + head;
    const float scale = __ldg(p.scales[kind] + slice);
    const int8_t* const codes = p.codes[kind] + (slice * p.block_tokens + slot) * p.dim + d;
    const long long to = row * x.token_stride + head * x.head_stride + d;
    for (int t0 = first; t0 < count; t0 += kBatch * at_once) {
      uint2 words[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int t = t0 + k * at_once;
        if (t >= count) continue;
        if (kWide) words[k].x = __ldg(reinterpret_cast<const uint32_t*>(codes + t * p.dim));
        else words[k] = __ldg(reinterpret_cast<const uint2*>(codes + t * p.dim));
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int t = t0 + k * at_once;
        if (t >= count) continue;
        const auto value = [&](uint32_t biased, int byte) {  // 2^23 + (code + 128) as f32 bits
          return (__uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7440 + byte)) - 8388736.0f) * scale;
        };
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = value(words[k].x ^ 0x80808080u, e);
        const long long out = to + t * x.token_stride;
        if (kWide) {
          float* const data = reinterpret_cast<float*>(x.data) + out;
          if (x.vector) {
            *reinterpret_cast<float4*>(data) = make_float4(v[0], v[1], v[2], v[3]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) data[e] = v[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 + e] = value(words[k].y ^ 0x80808080u, e);
          store8(x.data, x.type, x.vector, out, v);
        }
      }
    }
  }
}
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const uint32_t at = blockIdx.x / p.head_groups;
  const int group = static_cast<int>(blockIdx.x - at * p.head_groups);
  const int s = static_cast<int>(at / p.blocks_per_sequence), reached = static_cast<int>(at - s * p.blocks_per_sequence);
  Sequence q;
  if (!sequence_of(p.batch, s, true, &q) || q.n == 0) return;
  const int first = q.length - q.n, block_index = first / p.block_tokens + reached, begin = block_index * p.block_tokens;
  if (begin >= q.length) return;
  const int from = max(first, begin), count = min(q.length, begin + p.block_tokens) - from;
  const long long block = p.batch.table[s * p.batch.table_stride + block_index];
  if (block < 0 || block >= p.batch.blocks) {
    if (threadIdx.x == 0) sm100::report_error(p.batch.error, kErrorBlock);
    return;
  }
  const long long row = q.row + (from - first);
  const int head0 = group * p.heads_per_cta, head1 = min(p.kv_heads, head0 + p.heads_per_cta);
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    if (p.x[kind].data == nullptr) continue;
    if (p.x[kind].type == QX_STORAGE_F32) read_plane<true>(p, kind, block, row, from - begin, count, head0, head1);
    else read_plane<false>(p, kind, block, row, from - begin, count, head0, head1);
  }
}

int sm_count(DeviceContext* ctx) { return ctx->prop.multiProcessorCount; }

template <int kHeld, int kType>
qx_status launch_append_of(const AppendParams& p, long long grid, size_t smem, cudaStream_t stream) {
  static SmemOptIn opt_in;
  QX_TRY(opt_in.ensure(append_kernel<kHeld, kType>, 128 * 128 * sizeof(float2)));
  return launch_behind(append_kernel<kHeld, kType>, grid, kThreads, smem, stream, p);
}
template <int kType>
qx_status launch_append_held(const AppendParams& p, int units, long long grid, size_t smem, cudaStream_t stream) {
  if (units <= kThreads) return launch_append_of<1, kType>(p, grid, smem, stream);
  return launch_append_of<2, kType>(p, grid, smem, stream);
}

// Blocks that `most` tokens of one sequence can reach.
int blocks_reached(int most, int block_tokens) { return most <= 1 ? 1 : 1 + (most - 1 + block_tokens - 1) / block_tokens; }

}  // namespace

// ---- checks -------------------------------------------------------------------------------

qx_status check_heads(const qx_heads* view, long long rows, int dim, bool written) {
  if (view == nullptr) return QX_STATUS_INVALID_ARGUMENT;
  if (view->heads <= 0 || view->heads > (1 << 20) || view->token_stride < 0 || view->head_stride < 0) {
    return QX_STATUS_INVALID_SHAPE;
  }
  if (!known_type(view->type)) return QX_STATUS_UNSUPPORTED_FORMAT;
  if (rows <= 0) return QX_STATUS_OK;
  const __int128 by_token = static_cast<__int128>(rows - 1) * view->token_stride;
  const __int128 by_head = static_cast<__int128>(view->heads - 1) * view->head_stride;
  if ((by_token + by_head + dim) * 4 > std::numeric_limits<long long>::max()) return QX_STATUS_INVALID_SHAPE;
  if (written) {
    if (view->heads > 1 && view->head_stride < dim) return QX_STATUS_INVALID_SHAPE;
    if (rows > 1 && view->token_stride < dim) return QX_STATUS_INVALID_SHAPE;
    if (rows > 1 && view->heads > 1 && view->token_stride < by_head + dim && view->head_stride < by_token + dim) {
      return QX_STATUS_INVALID_SHAPE;
    }
  }
  if (view->data == nullptr || reinterpret_cast<uintptr_t>(view->data) % type_bytes(view->type) != 0) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  return QX_STATUS_OK;
}

qx_status check_cache(const qx_kv_cache* cache) {
  if (cache == nullptr) return QX_STATUS_INVALID_ARGUMENT;
  const int t = cache->block_tokens, d = cache->head_dim;
  if ((t != 16 && t != 32 && t != 64 && t != 128) || d < 16 || d > 256 || d % 16 != 0 || cache->kv_heads <= 0 ||
      cache->kv_heads > (1 << 20) || cache->blocks <= 0 || cache->blocks > (1LL << 31) ||
      !valid_product3(cache->blocks, cache->kv_heads, 1LL * t * d)) {
    return QX_STATUS_INVALID_SHAPE;
  }
  if (cache->k_codes == nullptr || cache->v_codes == nullptr || cache->k_scales == nullptr ||
      cache->v_scales == nullptr || reinterpret_cast<uintptr_t>(cache->k_codes) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(cache->v_codes) % 16 != 0 || reinterpret_cast<uintptr_t>(cache->k_scales) % 4 != 0 ||
      reinterpret_cast<uintptr_t>(cache->v_scales) % 4 != 0) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  return QX_STATUS_OK;
}

qx_status check_batch(const qx_kv_cache* cache, const qx_kv_batch* batch) {
  if (batch == nullptr) return QX_STATUS_INVALID_ARGUMENT;
  const long long reach = 0x7FFFFFFF - 4096;  // (positions and rows are 32-bit whole numbers, with room to round up)
  if (batch->sequences < 0 || batch->tokens < 0 || batch->max_tokens < 0 || batch->max_tokens > reach ||
      batch->max_length < 0 || batch->max_length > reach || batch->table_stride < 0 ||
      batch->table_stride < (batch->max_length + cache->block_tokens - 1LL) / cache->block_tokens) {
    return QX_STATUS_INVALID_SHAPE;
  }
  if (batch->sequences > 0 && batch->table_stride > std::numeric_limits<long long>::max() / 4 / batch->sequences) {
    return QX_STATUS_INVALID_SHAPE;
  }
  if (batch->token_begin == nullptr && batch->sequences > 0 &&
      static_cast<__int128>(batch->sequences) * batch->max_tokens > batch->tokens) {
    return QX_STATUS_INVALID_SHAPE;
  }
  if (batch->sequences > 0 && (batch->lengths == nullptr || (batch->max_length > 0 && batch->block_table == nullptr))) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  if (!on_boundary(batch->token_begin) || !on_boundary(batch->lengths) || !on_boundary(batch->block_table)) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  return QX_STATUS_OK;
}

Heads device_heads(const qx_heads* view) {
  Heads h{};
  if (view == nullptr) return h;
  h.data = static_cast<uint8_t*>(view->data);
  h.type = view->type;
  h.heads = view->heads;
  h.token_stride = view->token_stride;
  h.head_stride = view->head_stride;
  const size_t bytes = type_bytes(view->type);
  h.vector = reinterpret_cast<uintptr_t>(view->data) % 16 == 0 && view->token_stride * bytes % 16 == 0 &&
             view->head_stride * bytes % 16 == 0;
  return h;
}

Batch device_batch(const qx_kv_cache* cache, const qx_kv_batch* batch, int* error) {
  return Batch{batch->token_begin, batch->lengths, batch->block_table, batch->table_stride, batch->tokens,
               cache->blocks, batch->sequences, batch->max_tokens, batch->max_length, error};
}

qx_status check_append(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                       const qx_rope* rope, const int64_t* positions, const qx_heads* q, const qx_heads* q_out) {
  QX_TRY(check_cache(cache));
  QX_TRY(check_batch(cache, batch));
  QX_TRY(check_heads(k, batch->tokens, cache->head_dim, false));
  QX_TRY(check_heads(v, batch->tokens, cache->head_dim, false));
  if (k->heads != cache->kv_heads || v->heads != cache->kv_heads) return QX_STATUS_INVALID_SHAPE;
  if (rope != nullptr) {
    QX_TRY(check_rope(rope, cache->head_dim));
    if (rope->rotary_dim % 16 != 0) return QX_STATUS_INVALID_SHAPE;
  }
  if ((q == nullptr) != (q_out == nullptr) || (q != nullptr && rope == nullptr)) return QX_STATUS_INVALID_ARGUMENT;
  if (!on_boundary(positions)) return QX_STATUS_INVALID_ARGUMENT;
  if (q != nullptr) {
    QX_TRY(check_heads(q, batch->tokens, cache->head_dim, false));
    QX_TRY(check_heads(q_out, batch->tokens, cache->head_dim, true));
    if (q->heads != q_out->heads) return QX_STATUS_INVALID_SHAPE;
    if (q->type != q_out->type) return QX_STATUS_UNSUPPORTED_FORMAT;
    if (q->data == q_out->data && (q->token_stride != q_out->token_stride || q->head_stride != q_out->head_stride)) {
      return QX_STATUS_INVALID_ARGUMENT;
    }
  }
  return QX_STATUS_OK;
}

qx_status check_read(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v) {
  QX_TRY(check_cache(cache));
  QX_TRY(check_batch(cache, batch));
  for (const qx_heads* view : {k, v}) {
    if (view == nullptr) continue;
    QX_TRY(check_heads(view, batch->tokens, cache->head_dim, true));
    if (view->heads != cache->kv_heads) return QX_STATUS_INVALID_SHAPE;
  }
  return QX_STATUS_OK;
}

// ---- launches -----------------------------------------------------------------------------

qx_status launch_append(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                        const qx_rope* rope, const int64_t* positions, const qx_heads* q, const qx_heads* q_out,
                        DeviceContext* ctx, cudaStream_t stream) {
  if (batch->sequences == 0 || batch->max_tokens == 0 || batch->tokens == 0) return QX_STATUS_OK;
  AppendParams p{};
  p.batch = device_batch(cache, batch, ctx->error_dev);
  p.codes[0] = cache->k_codes;
  p.codes[1] = cache->v_codes;
  p.scales[0] = cache->k_scales;
  p.scales[1] = cache->v_scales;
  p.x[0] = device_heads(k);
  p.x[1] = device_heads(v);
  p.q = device_heads(q);
  p.q_out = device_heads(q_out);
  p.rotation = device_rotation(rope, false);
  p.positions = positions;
  p.kv_heads = cache->kv_heads;
  p.block_tokens = cache->block_tokens;
  p.dim = cache->head_dim;
  const int most = static_cast<int>(std::min<long long>(batch->max_tokens, batch->max_length));
  p.blocks_per_sequence = blocks_reached(most, cache->block_tokens);
  // The angles of a block's tokens are shared by the heads that a CTA takes, and the loads of one head run beside
  // the work on the one before: as many as leave a few CTAs for every SM (at least 4 | 12 | 36 CTAs, append and read of
  // 6570 f32 tokens, 8 heads, us: rotated with 32 query heads 108 | 116 | 144, not rotated 50 | 49 | 57).
  const long long blocks = static_cast<long long>(batch->sequences) * p.blocks_per_sequence;
  const long long spread = 4LL * sm_count(ctx);
  const long long heads = 2 * blocks * cache->kv_heads / (rope != nullptr ? spread : 3 * spread);
  p.heads_per_cta = static_cast<int>(std::min<long long>(std::max<long long>(heads, 1), cache->kv_heads));
  p.head_groups = (cache->kv_heads + p.heads_per_cta - 1) / p.heads_per_cta;
  long long grid = 2 * blocks * p.head_groups;
  const int pairs = p.rotation.rotary / 2;
  size_t smem = static_cast<size_t>(std::min(most, cache->block_tokens)) * pairs * sizeof(float2);
  const long long tokens = static_cast<long long>(batch->sequences) * most;
  if (q != nullptr && tokens > 3 * spread) {
    // many queries: a launch of their own, with the registers and shared memory that they need (beside the append | by
    // itself, append and read of bf16, 32 query heads, us: 1000 tokens 20.7 | 23.9, 2000 36.9 | 33.5, 6570 120 | 84)
    QX_TRY(launch_rope_batch(rope, q, q_out, positions, p.batch, most, cache->head_dim, ctx, stream));
  } else if (q != nullptr) {
    p.tokens_per_cta = 1;
    p.query_ctas = std::max(1, most);
    grid += static_cast<long long>(batch->sequences) * p.query_ctas;
    smem = std::max(smem, static_cast<size_t>(p.tokens_per_cta) * pairs * sizeof(float2));
  }
  // Elements held in registers | read twice, append and read, us: 6570 f32 tokens 49 | 57, bf16 42 | 60, 64 single
  // tokens 14.7 | 15.8.
  const int units = std::min(most, cache->block_tokens) * (cache->head_dim / 16);
  if (k->type != v->type || !p.x[0].vector || !p.x[1].vector || units > 2 * kThreads) {
    return launch_append_of<0, QX_STORAGE_F32>(p, grid, smem, stream);
  }
  if (k->type == QX_STORAGE_F32) return launch_append_held<QX_STORAGE_F32>(p, units, grid, smem, stream);
  if (k->type == QX_STORAGE_F16) return launch_append_held<QX_STORAGE_F16>(p, units, grid, smem, stream);
  return launch_append_held<QX_STORAGE_BF16>(p, units, grid, smem, stream);
}

qx_status launch_read(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                      DeviceContext* ctx, cudaStream_t stream) {
  if (batch->sequences == 0 || batch->max_tokens == 0 || batch->tokens == 0 || (k == nullptr && v == nullptr)) {
    return QX_STATUS_OK;
  }
  ReadParams p{};
  p.batch = device_batch(cache, batch, ctx->error_dev);
  p.codes[0] = cache->k_codes;
  p.codes[1] = cache->v_codes;
  p.scales[0] = cache->k_scales;
  p.scales[1] = cache->v_scales;
  p.x[0] = device_heads(k);
  p.x[1] = device_heads(v);
  p.kv_heads = cache->kv_heads;
  p.block_tokens = cache->block_tokens;
  p.dim = cache->head_dim;
  p.blocks_per_sequence = blocks_reached(static_cast<int>(std::min<long long>(batch->max_tokens, batch->max_length)), cache->block_tokens);
  // as many heads per CTA as leave a few CTAs for every SM
  const long long blocks = static_cast<long long>(batch->sequences) * p.blocks_per_sequence;
  const long long heads = blocks * cache->kv_heads / (12LL * sm_count(ctx));
  p.heads_per_cta = static_cast<int>(std::min<long long>(std::max<long long>(heads, 1), cache->kv_heads));
  p.head_groups = (cache->kv_heads + p.heads_per_cta - 1) / p.heads_per_cta;
  return launch_behind(read_kernel, blocks * p.head_groups, kThreads, 0, stream, p);
}

}  // namespace kv
}  // namespace qx

using namespace qx;

extern "C" {

qx_status qx_kv_append_dev(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                           const qx_rope* rope, const int64_t* positions_dev, const qx_heads* q, const qx_heads* q_out,
                           void* stream) {
  QX_TRY(kv::check_append(cache, batch, k, v, rope, positions_dev, q, q_out));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  return kv::launch_append(cache, batch, k, v, rope, positions_dev, q, q_out, ctx, static_cast<cudaStream_t>(stream));
}

qx_status qx_kv_read_dev(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                         void* stream) {
  QX_TRY(kv::check_read(cache, batch, k, v));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  return kv::launch_read(cache, batch, k, v, ctx, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
