// The paged key-value cache in 8 bits: append (rotation, scales, codes) and read.
//
// The unit of work is a (sequence, block that its new tokens reach, kv head) of the keys or of the values:
// one CTA owns the block's scale and codes, so nothing is atomic and the result does not depend on order.
// It reads the new elements twice, the second time out of the caches: once for their largest
// magnitude, once for the codes, because a code needs the block's final scale. Bound by HBM for prompts
// (element in, code out) and by the chain scale -> codes for single tokens.

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

// Code of x: the exact quotient x / scale rounded half to even, whatever the rounding of the product with
// the inverse did: that is off by one at most, and the remainder x - r * scale is exact in f32 (a
// multiple of half an ulp of the scale, no larger than the scale).
__device__ __forceinline__ int code_of(float x, float scale, float inverse) {
  float r = rintf(x * inverse);
  const float rest = fmaf(-r, scale, x), half = 0.5f * scale;
  const bool tie_to_odd = fabsf(rest) == half && (static_cast<int>(r) & 1);
  if (fabsf(rest) > half || tie_to_odd) r += copysignf(1.0f, rest);
  return static_cast<int>(fminf(127.0f, fmaxf(-127.0f, r)));
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
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float scale, float inverse) {
  int c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = code_of(v[i], scale, inverse);
  return make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
}

__device__ __forceinline__ void rotate_queries(const AppendParams& p, long long item, float2* table) {
  const int s = static_cast<int>(item / p.query_ctas), chunk = static_cast<int>(item % p.query_ctas);
  Sequence q;
  if (!sequence_of(p.batch, s, true, &q)) return;
  const int token0 = chunk * p.tokens_per_cta, count = min(p.tokens_per_cta, q.n - token0);
  if (count <= 0) return;
  const int pairs = p.rotation.rotary / 2, units = p.dim / 16, per_token = p.q.heads * units;
  for (int i = threadIdx.x; i < count * pairs; i += kThreads) {
    const int token = token0 + i / pairs;
    const long long position = p.positions != nullptr ? p.positions[q.row + token] : q.length - q.n + token;
    table[i] = turn(p.rotation, position, i % pairs);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * per_token; i += kThreads) {
    const int token = i / per_token, rest = i - token * per_token, head = rest / units;
    const Unit u = unit_of(rest - head * units, p.rotation.rotary, p.rotation.interleaved);
    const long long from = (q.row + token0 + token) * p.q.token_stride + head * p.q.head_stride;
    const long long to = (q.row + token0 + token) * p.q_out.token_stride + head * p.q_out.head_stride;
    float a[8], b[8];
    load8(p.q.data, p.q.type, p.q.vector, from + u.first, a);
    load8(p.q.data, p.q.type, p.q.vector, from + u.second, b);
    rotate_unit(u, p.rotation.interleaved, table + token * pairs, a, b);
    store8(p.q_out.data, p.q_out.type, p.q_out.vector, to + u.first, a);
    store8(p.q_out.data, p.q_out.type, p.q_out.vector, to + u.second, b);
  }
}

__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ float2 table[];
  __shared__ uint32_t warp_max[kThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const long long per_kind = static_cast<long long>(p.batch.sequences) * p.blocks_per_sequence * p.head_groups;
  long long item = blockIdx.x;
  if (item >= 2 * per_kind) {
    rotate_queries(p, item - 2 * per_kind, table);
    return;
  }
  const int kind = item >= per_kind ? 1 : 0;
  item -= kind * per_kind;
  const int group = static_cast<int>(item % p.head_groups);
  const long long at = item / p.head_groups;
  const int s = static_cast<int>(at / p.blocks_per_sequence), reached = static_cast<int>(at % p.blocks_per_sequence);
  Sequence q;
  if (!sequence_of(p.batch, s, true, &q) || q.n == 0) return;
  const int first = q.length - q.n;
  const int block_index = first / p.block_tokens + reached;
  const int begin = block_index * p.block_tokens;  // position of the block's slot 0
  if (begin >= q.length) return;
  const int from = max(first, begin), to = min(q.length, begin + p.block_tokens);
  const int kept = from - begin, count = to - from;  // older tokens of the block, new ones
  const long long row = q.row + (from - first);
  const long long block = p.batch.table[s * p.batch.table_stride + block_index];
  if (block < 0 || block >= p.batch.blocks) {
    if (threadIdx.x == 0) sm100::report_error(p.batch.error, kErrorBlock);
    return;
  }
  const Heads& x = p.x[kind];
  const bool rotated = kind == 0 && p.rotation.rotary > 0;
  const int pairs = p.rotation.rotary / 2, units = p.dim / 16;
  if (rotated) {
    for (int i = threadIdx.x; i < count * pairs; i += kThreads) {
      const int token = i / pairs;
      const long long position = p.positions != nullptr ? p.positions[row + token] : from + token;
      table[i] = turn(p.rotation, position, i % pairs);
    }
  }
  const int total = count * units;
  const int head0 = group * p.heads_per_cta, head1 = min(p.kv_heads, head0 + p.heads_per_cta);
  for (int head = head0; head < head1; ++head) {
    const auto load_unit = [&](int i, Unit* u, float (&a)[8], float (&b)[8]) {
      const int token = i / units;
      *u = unit_of(i - token * units, rotated ? p.rotation.rotary : 0, p.rotation.interleaved);
      const long long base = (row + token) * x.token_stride + head * x.head_stride;
      load8(x.data, x.type, x.vector, base + u->first, a);
      load8(x.data, x.type, x.vector, base + u->second, b);
      if (rotated) rotate_unit(*u, p.rotation.interleaved, table + token * pairs, a, b);
      return token;
    };
    // Magnitudes are compared as bit patterns: above those of all numbers come infinity and NaN.
    uint32_t top = 0;
    __syncthreads();  // the table is written; warp_max of the head before is read
    for (int i = threadIdx.x; i < total; i += kThreads) {
      Unit u;
      float a[8], b[8];
      load_unit(i, &u, a, b);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        top = max(top, max(__float_as_uint(a[k]) & 0x7FFFFFFFu, __float_as_uint(b[k]) & 0x7FFFFFFFu));
      }
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = top;
    float* const scale_at = p.scales[kind] + block * p.kv_heads + head;
    const float before = kept > 0 ? *scale_at : 0.0f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) top = max(top, warp_max[w]);
    const bool number = top < 0x7F800000u && (__float_as_uint(before) & 0x7FFFFFFFu) < 0x7F800000u;
    float scale = fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), before);
    if (scale < kSmallestScale) scale = 0.0f;
    const float inverse = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    if (threadIdx.x == 0) *scale_at = number ? scale : __uint_as_float(0x7FC00000u);
    int8_t* const codes = p.codes[kind] + (block * p.kv_heads + head) * p.block_tokens * p.dim;
    if (number && scale > before && before > 0.0f) {
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
            c[e] = regrown(static_cast<int8_t>(w[k] >> (8 * e)), before, scale, ratio);
          }
          w[k] = pack4(c[0], c[1], c[2], c[3]);
        }
        *words = v;
      }
    }
    for (int i = threadIdx.x; i < total; i += kThreads) {
      Unit u;
      float a[8], b[8];
      const int token = load_unit(i, &u, a, b);
      int8_t* const out = codes + (kept + token) * p.dim;
      uint2 first8 = make_uint2(0, 0), second8 = make_uint2(0, 0);
      if (number && scale > 0.0f) {
        first8 = codes8(a, scale, inverse);
        second8 = codes8(b, scale, inverse);
      }
      *reinterpret_cast<uint2*>(out + u.first) = first8;
      *reinterpret_cast<uint2*>(out + u.second) = second8;
    }
  }
}

struct ReadParams {
  Batch batch;
  const int8_t* codes[2];
  const float* scales[2];
  Heads x[2];  // data NULL: not wanted
  int kv_heads, block_tokens, dim;
  int tokens_per_cta, chunks;  // chunks of tokens per sequence
};

// A CTA takes a few tokens with all of their heads: 16 codes in, 16 values out per thread at a time.
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int s = static_cast<int>(blockIdx.x / p.chunks), chunk = static_cast<int>(blockIdx.x % p.chunks);
  Sequence q;
  if (!sequence_of(p.batch, s, true, &q)) return;
  const int token0 = chunk * p.tokens_per_cta, count = min(p.tokens_per_cta, q.n - token0);
  if (count <= 0) return;
  const int units = p.dim / 16, per_token = p.kv_heads * units;
  for (int i = threadIdx.x; i < 2 * count * per_token; i += kThreads) {
    const int kind = i >= count * per_token ? 1 : 0;
    const Heads& x = p.x[kind];
    if (x.data == nullptr) continue;
    const int rest0 = i - kind * count * per_token, token = rest0 / per_token, rest = rest0 - token * per_token;
    const int head = rest / units, unit = rest - head * units;
    const int position = q.length - q.n + token0 + token;
    const long long block = p.batch.table[s * p.batch.table_stride + position / p.block_tokens];
    if (block < 0 || block >= p.batch.blocks) {
      sm100::report_error(p.batch.error, kErrorBlock);
      continue;
    }
    const long long slice = block * p.kv_heads + head;
    const float scale = p.scales[kind][slice];
    const uint4 v = *reinterpret_cast<const uint4*>(
        p.codes[kind] + (slice * p.block_tokens + position % p.block_tokens) * p.dim + 16 * unit);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float a[8], b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = static_cast<float>(static_cast<int8_t>(w[e >> 2] >> (8 * (e & 3)))) * scale;
      b[e] = static_cast<float>(static_cast<int8_t>(w[2 + (e >> 2)] >> (8 * (e & 3)))) * scale;
    }
    const long long to = (q.row + token0 + token) * x.token_stride + head * x.head_stride + 16 * unit;
    store8(x.data, x.type, x.vector, to, a);
    store8(x.data, x.type, x.vector, to + 8, b);
  }
}

int sm_count(DeviceContext* ctx) { return ctx->prop.multiProcessorCount; }

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
                       const qx_rope* rope, const qx_heads* q, const qx_heads* q_out) {
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
  if (most == 0) p.blocks_per_sequence = 1;
  else p.blocks_per_sequence = 1 + (most - 1 + cache->block_tokens - 1) / cache->block_tokens;
  // The angles of a block's tokens are shared by the heads that a CTA takes: as many as leave a few CTAs for
  // every SM. Without a rotation there is nothing to share.
  const long long blocks = static_cast<long long>(batch->sequences) * p.blocks_per_sequence;
  const long long spread = 4LL * sm_count(ctx);
  long long heads = rope == nullptr ? 1 : blocks * cache->kv_heads / spread;
  p.heads_per_cta = static_cast<int>(std::min<long long>(std::max<long long>(heads, 1), cache->kv_heads));
  p.head_groups = (cache->kv_heads + p.heads_per_cta - 1) / p.heads_per_cta;
  long long grid = 2 * blocks * p.head_groups;
  const int pairs = p.rotation.rotary / 2;
  size_t smem = static_cast<size_t>(std::min(most, cache->block_tokens)) * pairs * sizeof(float2);
  if (q != nullptr) {
    const long long tokens = static_cast<long long>(batch->sequences) * most;
    p.tokens_per_cta = static_cast<int>(std::min<long long>(
        std::min<long long>(4, std::max<long long>(1, tokens / spread)), std::max(1, most)));
    p.query_ctas = (std::max(1, most) + p.tokens_per_cta - 1) / p.tokens_per_cta;
    grid += static_cast<long long>(batch->sequences) * p.query_ctas;
    smem = std::max(smem, static_cast<size_t>(p.tokens_per_cta) * pairs * sizeof(float2));
  }
  static SmemOptIn opt_in;
  QX_TRY(opt_in.ensure(append_kernel, 128 * 128 * sizeof(float2)));
  return launch_behind(append_kernel, grid, kThreads, smem, stream, p);
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
  // four rounds of the CTA's threads where that leaves a few CTAs for every SM
  const long long per_token = 2LL * cache->kv_heads * (cache->head_dim / 16);
  const long long tokens = static_cast<long long>(batch->sequences) * batch->max_tokens;
  long long t = std::min((4 * kThreads + per_token - 1) / per_token, tokens / (4 * sm_count(ctx)));
  p.tokens_per_cta = static_cast<int>(std::min<long long>(std::max<long long>(t, 1), batch->max_tokens));
  if (per_token * p.tokens_per_cta > (1 << 30)) return QX_STATUS_INVALID_SHAPE;
  p.chunks = (batch->max_tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  return launch_behind(read_kernel, static_cast<long long>(batch->sequences) * p.chunks, kThreads, 0, stream, p);
}

}  // namespace kv
}  // namespace qx

using namespace qx;

extern "C" {

qx_status qx_kv_append_dev(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                           const qx_rope* rope, const int64_t* positions_dev, const qx_heads* q, const qx_heads* q_out,
                           void* stream) {
  QX_TRY(kv::check_append(cache, batch, k, v, rope, q, q_out));
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
