// Rotary positions: frequencies (host) and the rotation of query and key heads.
//
// A CTA takes a few tokens with all of their heads: the {cos, sin} of a token's pairs are the same for
// every head, so they are computed once into shared memory (64-bit angle, see kv::turn) and the heads
// stream past them, 16 elements per thread at a time in 16-byte accesses. Each thread reads both halves
// of its pairs before it writes them, so x and y may be the same view. Bound by HBM: every element is
// read once and written once (8191 f16 tokens of 40 heads of 128 elements, 64 of them rotated: 168 MB in 30.7 us, 5.5 TB/s,
// 0.84 of the copy bandwidth; 32 tokens: 2.9 us).

#include <algorithm>
#include <cmath>

#include "qx_kv.cuh"

namespace qx {
namespace kv {
namespace {

struct RopeParams {
  Heads x, y;
  const int64_t* positions;
  long long tokens;
  int dim, tokens_per_cta, in_place;
  int chunks;  // of tokens per sequence of `batch`; 0: the tokens are no batch
  Batch batch;
  Rotation rotation;
};

// The rows of a CTA, and the position of the first where positions are places in a sequence.
struct Span {
  long long row;
  int count;
  long long position;
};
template <bool kBatch>
__device__ __forceinline__ Span span_of(const RopeParams& p) {
  if (!kBatch) {
    const long long row = static_cast<long long>(blockIdx.x) * p.tokens_per_cta;
    return {row, static_cast<int>(min(static_cast<long long>(p.tokens_per_cta), p.tokens - row)), 0};
  }
  const int s = static_cast<int>(blockIdx.x / p.chunks), first = static_cast<int>(blockIdx.x % p.chunks) * p.tokens_per_cta;
  Sequence q;
  if (!sequence_of(p.batch, s, true, &q)) return {0, 0, 0};
  return {q.row + first, min(p.tokens_per_cta, q.n - first), q.length - q.n + first};
}
template <bool kBatch>
__device__ __forceinline__ float2 turn_of(const RopeParams& p, const Span& span, int token, int pair) {
  return turn(p.rotation, !kBatch || p.positions != nullptr ? p.positions[span.row + token] : span.position + token, pair);
}

constexpr int kRopeThreads = 256;

// Whole units of 16 elements: head size and rotary part are multiples of 16, runs start on 16-byte boundaries, a head
// has no more units than the CTA threads.
template <int kType, bool kBatch>
__global__ void __launch_bounds__(kRopeThreads, 3) rope_units_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ __align__(16) float2 table[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int pairs = p.rotation.rotary / 2;
  const Span span = span_of<kBatch>(p);
  const int count = span.count;
  if (count <= 0) return;
  const int units = p.in_place ? p.rotation.rotary / 16 : p.dim / 16;  // (in place the rest is where it belongs)
  // a thread keeps its unit of the head and walks the (token, head) pairs; the first elements are under way while
  // the angles are taken
  const int at_once = kRopeThreads / units, first = threadIdx.x / units;
  const Unit unit = unit_of(static_cast<int>(threadIdx.x) - first * units, p.rotation.rotary, p.rotation.interleaved, p.dim);
  Walk walk(first, at_once, p.x.heads);
  if (first >= at_once) walk.token = count;  // (threads that are no whole row of units)
  constexpr int kWords = kType == QX_STORAGE_F32 ? 2 : 1;
  constexpr int kUnits = kType == QX_STORAGE_F32 ? 2 : 4;  // eight 16-byte loads in flight per thread
  uint4 a[kUnits][kWords], b[kUnits][kWords];
  int token[kUnits], head[kUnits];
  const auto load = [&]() {
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      token[k] = walk.token;
      head[k] = walk.head;
      walk.advance();
      if (token[k] >= count) continue;
      const long long from = (span.row + token[k]) * p.x.token_stride + head[k] * p.x.head_stride;
      load8_words<kType>(p.x.data, from + unit.first, a[k]);
      load8_words<kType>(p.x.data, from + unit.second, b[k]);
    }
  };
  load();
  for (int i = threadIdx.x; i < count * pairs; i += kRopeThreads) {
    table[i] = turn_of<kBatch>(p, span, i / pairs, i % pairs);
  }
  __syncthreads();
  while (token[0] < count) {
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      if (token[k] >= count) continue;
      if (unit.pair >= 0) {
        float x[8], y[8];
        from_words<kType>(a[k], x);
        from_words<kType>(b[k], y);
        rotate_unit(unit, p.rotation.interleaved, table + token[k] * pairs, x, y);
        to_words<kType>(x, a[k]);
        to_words<kType>(y, b[k]);
      }
      const long long to = (span.row + token[k]) * p.y.token_stride + head[k] * p.y.head_stride;
      store8_words<kType>(p.y.data, to + unit.first, a[k]);
      store8_words<kType>(p.y.data, to + unit.second, b[k]);
    }
    load();
  }
}

// Any head size and any even rotary part (heads of more than 4096 elements among them): one pair, or one element
// behind them, at a time.
template <bool kBatch>
__global__ void __launch_bounds__(kRopeThreads) rope_pairs_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ __align__(16) float2 table[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int rotary = p.rotation.rotary, pairs = rotary / 2;
  const Span span = span_of<kBatch>(p);
  const int count = span.count;
  if (count <= 0) return;
  const int per_head = pairs + (p.in_place ? 0 : p.dim - rotary);
  const int per_token = p.x.heads * per_head;
  for (int i = threadIdx.x; i < count * pairs; i += kRopeThreads) {
    table[i] = turn_of<kBatch>(p, span, i / pairs, i % pairs);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * per_token; i += kRopeThreads) {
    const int token = i / per_token, rest = i - token * per_token, head = rest / per_head, e = rest - head * per_head;
    const long long from = (span.row + token) * p.x.token_stride + head * p.x.head_stride;
    const long long to = (span.row + token) * p.y.token_stride + head * p.y.head_stride;
    if (e >= pairs) {
      store_one(p.y.data, p.y.type, to + rotary + (e - pairs), load_one(p.x.data, p.x.type, from + rotary + (e - pairs)));
      continue;
    }
    const int first = p.rotation.interleaved ? 2 * e : e, second = p.rotation.interleaved ? 2 * e + 1 : e + pairs;
    const float2 t = table[token * pairs + e];
    const float a = load_one(p.x.data, p.x.type, from + first), b = load_one(p.x.data, p.x.type, from + second);
    store_one(p.y.data, p.y.type, to + first, a * t.x - b * t.y);
    store_one(p.y.data, p.y.type, to + second, a * t.y + b * t.x);
  }
}

}  // namespace

qx_status check_rope(const qx_rope* rope, int dim) {
  if (rope == nullptr) return QX_STATUS_INVALID_ARGUMENT;
  if (rope->rotary_dim < 2 || rope->rotary_dim > 256 || rope->rotary_dim % 2 != 0 || rope->rotary_dim > dim) {
    return QX_STATUS_INVALID_SHAPE;
  }
  if (rope->style != QX_ROPE_HALVES && rope->style != QX_ROPE_INTERLEAVED) return QX_STATUS_UNSUPPORTED_FORMAT;
  if (!std::isfinite(rope->amplitude)) return QX_STATUS_INVALID_ARGUMENT;
  for (int i = 0; i < rope->rotary_dim / 2; ++i) {
    if (!std::isfinite(rope->frequency[i])) return QX_STATUS_INVALID_ARGUMENT;
  }
  return QX_STATUS_OK;
}

Rotation device_rotation(const qx_rope* rope, bool inverse) {
  Rotation r{};
  if (rope == nullptr) return r;
  r.rotary = rope->rotary_dim;
  r.interleaved = rope->style == QX_ROPE_INTERLEAVED;
  r.amplitude = static_cast<float>(rope->amplitude);
  r.sign = inverse ? -1.0f : 1.0f;
  for (int i = 0; i < r.rotary / 2; ++i) r.turns[i] = rope->frequency[i] * 0.15915494309189533577;  // 1 / (2 pi)
  return r;
}

qx_status check_rope_call(const qx_rope* rope, const qx_heads* x, const qx_heads* y, const int64_t* positions,
                          long long tokens, int dim) {
  if (tokens < 0 || dim <= 0 || dim > (1 << 20)) return QX_STATUS_INVALID_SHAPE;
  QX_TRY(check_rope(rope, dim));
  QX_TRY(check_heads(x, tokens, dim, false));
  QX_TRY(check_heads(y, tokens, dim, true));
  if (x->heads != y->heads) return QX_STATUS_INVALID_SHAPE;
  if (x->type != y->type) return QX_STATUS_UNSUPPORTED_FORMAT;
  if ((tokens > 0 && positions == nullptr) || !on_boundary(positions)) return QX_STATUS_INVALID_ARGUMENT;
  if (x->data == y->data && (x->token_stride != y->token_stride || x->head_stride != y->head_stride)) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  return QX_STATUS_OK;
}

namespace {

template <bool kBatch>
qx_status launch_sized(const RopeParams& p, bool whole, int type, long long grid, size_t smem, cudaStream_t stream) {
  if (!whole) return launch_behind(rope_pairs_kernel<kBatch>, grid, kRopeThreads, smem, stream, p);
  switch (type) {
    case QX_STORAGE_F32: return launch_behind(rope_units_kernel<QX_STORAGE_F32, kBatch>, grid, kRopeThreads, smem, stream, p);
    case QX_STORAGE_F16: return launch_behind(rope_units_kernel<QX_STORAGE_F16, kBatch>, grid, kRopeThreads, smem, stream, p);
    default: return launch_behind(rope_units_kernel<QX_STORAGE_BF16, kBatch>, grid, kRopeThreads, smem, stream, p);
  }
}

qx_status launch_rope(RopeParams& p, const qx_rope* rope, const qx_heads* x, const qx_heads* y, const int64_t* positions,
                      long long tokens, int dim, bool inverse, DeviceContext* ctx, cudaStream_t stream) {
  p.x = device_heads(x);
  p.y = device_heads(y);
  p.positions = positions;
  p.tokens = tokens;
  p.dim = dim;
  p.in_place = x->data == y->data;
  p.rotation = device_rotation(rope, inverse);
  // (a row of units takes a thread each; in place only the rotated ones, which are 16 at most)
  const bool whole = dim % 16 == 0 && rope->rotary_dim % 16 == 0 && p.x.vector && p.y.vector &&
                     (p.in_place || dim / 16 <= kRopeThreads);
  // Tokens per CTA: enough for four rounds of its threads where there are CTAs for every SM all the same,
  // and no more than 16 KB of {cos, sin}.
  const long long per_token = static_cast<long long>(x->heads) * (whole ? dim / 16 : dim);
  const int pairs = rope->rotary_dim / 2;
  long long t = (4 * kRopeThreads + per_token - 1) / per_token;
  t = std::min<long long>(t, 2048 / pairs);
  t = std::min<long long>(t, (tokens + 4 * ctx->prop.multiProcessorCount - 1) / (4 * ctx->prop.multiProcessorCount));
  p.tokens_per_cta = static_cast<int>(std::max<long long>(t, 1));
  if (per_token * p.tokens_per_cta > (1 << 28)) return QX_STATUS_INVALID_SHAPE;
  long long grid = (tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  if (p.chunks > 0) {  // (so far: the most tokens of a sequence)
    p.chunks = (p.chunks + p.tokens_per_cta - 1) / p.tokens_per_cta;
    grid = static_cast<long long>(p.batch.sequences) * p.chunks;
  }
  const size_t smem = static_cast<size_t>(p.tokens_per_cta) * pairs * sizeof(float2);
  if (p.chunks > 0) return launch_sized<true>(p, whole, x->type, grid, smem, stream);
  return launch_sized<false>(p, whole, x->type, grid, smem, stream);
}

}  // namespace

qx_status launch_rope_batch(const qx_rope* rope, const qx_heads* x, const qx_heads* y, const int64_t* positions,
                            const Batch& batch, int most, int dim, DeviceContext* ctx, cudaStream_t stream) {
  RopeParams p{};
  p.batch = batch;
  p.chunks = std::max(1, most);
  return launch_rope(p, rope, x, y, positions, static_cast<long long>(batch.sequences) * most, dim, false, ctx, stream);
}

}  // namespace kv
}  // namespace qx

using namespace qx;

extern "C" {

qx_status qx_rope_init(qx_rope* rope, int rotary_dim, int style, double base, const qx_rope_scaling* scaling) {
  if (rotary_dim < 2 || rotary_dim > 256 || rotary_dim % 2 != 0) return QX_STATUS_INVALID_SHAPE;
  if (style != QX_ROPE_HALVES && style != QX_ROPE_INTERLEAVED) return QX_STATUS_UNSUPPORTED_FORMAT;
  const int kind = scaling == nullptr ? QX_ROPE_PLAIN : scaling->kind;
  if (kind < QX_ROPE_PLAIN || kind > QX_ROPE_RAMP) return QX_STATUS_UNSUPPORTED_FORMAT;
  if (rope == nullptr || !std::isfinite(base) || base <= 1.0) return QX_STATUS_INVALID_ARGUMENT;
  if (kind != QX_ROPE_PLAIN && !(std::isfinite(scaling->factor) && scaling->factor > 0.0)) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  if (kind >= QX_ROPE_BANDS && !(std::isfinite(scaling->trained_length) && scaling->trained_length > 0.0 &&
                                 scaling->slow > 0.0 && scaling->slow < scaling->fast && std::isfinite(scaling->fast))) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  constexpr double kTwoPi = 6.283185307179586477;
  qx_rope out{};
  out.rotary_dim = rotary_dim;
  out.style = style;
  out.amplitude = kind == QX_ROPE_RAMP && scaling->factor > 1.0 ? 0.1 * std::log(scaling->factor) + 1.0 : 1.0;
  double low = 0.0, span = 1.0;
  if (kind == QX_ROPE_RAMP) {
    // the (fractional) index of the pair that turns r times over the trained length
    const auto index = [&](double r) {
      return rotary_dim * std::log(scaling->trained_length / (r * kTwoPi)) / (2.0 * std::log(base));
    };
    low = std::fmax(0.0, std::floor(index(scaling->fast)));
    const double high = std::fmin(rotary_dim - 1.0, std::ceil(index(scaling->slow)));
    span = high > low ? high - low : 0.001;
  }
  for (int i = 0; i < rotary_dim / 2; ++i) {
    const double f = std::pow(base, -2.0 * i / rotary_dim);
    double keep = 1.0;  // share of the frequency that is not divided
    if (kind == QX_ROPE_LINEAR) keep = 0.0;
    if (kind == QX_ROPE_BANDS) {
      const double turns = scaling->trained_length * f / kTwoPi;
      keep = std::fmin(1.0, std::fmax(0.0, (turns - scaling->slow) / (scaling->fast - scaling->slow)));
    }
    if (kind == QX_ROPE_RAMP) keep = 1.0 - std::fmin(1.0, std::fmax(0.0, (i - low) / span));
    out.frequency[i] = kind == QX_ROPE_PLAIN ? f : (1.0 - keep) * f / scaling->factor + keep * f;
  }
  *rope = out;
  return QX_STATUS_OK;
}

qx_status qx_rope_apply_dev(const qx_rope* rope, const qx_heads* x, const qx_heads* y, const int64_t* positions_dev,
                            long long tokens, int head_dim, int inverse, void* stream) {
  QX_TRY(kv::check_rope_call(rope, x, y, positions_dev, tokens, head_dim));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  if (tokens == 0) return QX_STATUS_OK;
  kv::RopeParams p{};
  return kv::launch_rope(p, rope, x, y, positions_dev, tokens, head_dim, inverse != 0, ctx, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
