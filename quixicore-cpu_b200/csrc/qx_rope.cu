// Rotary positions: frequencies (host) and the rotation of query and key heads.
//
// A CTA takes a few tokens with all of their heads: the {cos, sin} of a token's pairs are the same for
// every head, so they are computed once into shared memory (64-bit angle, see kv::turn) and the heads
// stream past them, 16 elements per thread at a time in 16-byte accesses. Each thread reads both halves
// of its pairs before it writes them, so x and y may be the same view. Bound by HBM: every element is
// read once and written once.

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
  Rotation rotation;
};

constexpr int kRopeThreads = 256;

// Whole units of 16 elements (head size and rotary part are multiples of 16), any alignment.
template <int kType>
__global__ void __launch_bounds__(kRopeThreads) rope_units_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ float2 table[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int pairs = p.rotation.rotary / 2;
  const long long token0 = static_cast<long long>(blockIdx.x) * p.tokens_per_cta;
  const int count = static_cast<int>(min(static_cast<long long>(p.tokens_per_cta), p.tokens - token0));
  const int per_head = p.dim / 16;
  const int units = p.in_place ? p.rotation.rotary / 16 : per_head;  // (in place the rest is where it belongs)
  const int per_token = p.x.heads * units;
  for (int i = threadIdx.x; i < count * pairs; i += kRopeThreads) {
    table[i] = turn(p.rotation, p.positions[token0 + i / pairs], i % pairs);
  }
  __syncthreads();
  // two units at a time: four 16-byte loads in flight per thread
  constexpr int kBatch = 2;
  const int total = count * per_token;
  for (int i = threadIdx.x; i < total; i += kBatch * kRopeThreads) {
    float a[kBatch][8], b[kBatch][8];
    Unit unit[kBatch];
    long long to[kBatch];
    int token[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int j = i + k * kRopeThreads;
      if (j >= total) break;
      token[k] = j / per_token;
      const int rest = j - token[k] * per_token, head = rest / units;
      unit[k] = unit_of(rest - head * units, p.rotation.rotary, p.rotation.interleaved);
      const long long from = (token0 + token[k]) * p.x.token_stride + head * p.x.head_stride;
      to[k] = (token0 + token[k]) * p.y.token_stride + head * p.y.head_stride;
      load8(p.x.data, kType, p.x.vector, from + unit[k].first, a[k]);
      load8(p.x.data, kType, p.x.vector, from + unit[k].second, b[k]);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (i + k * kRopeThreads >= total) break;
      rotate_unit(unit[k], p.rotation.interleaved, table + token[k] * pairs, a[k], b[k]);
      store8(p.y.data, kType, p.y.vector, to[k] + unit[k].first, a[k]);
      store8(p.y.data, kType, p.y.vector, to[k] + unit[k].second, b[k]);
    }
  }
}

// Any head size and any even rotary part: one pair, or one element behind them, at a time.
__global__ void __launch_bounds__(kRopeThreads) rope_pairs_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ float2 table[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int rotary = p.rotation.rotary, pairs = rotary / 2;
  const long long token0 = static_cast<long long>(blockIdx.x) * p.tokens_per_cta;
  const int count = static_cast<int>(min(static_cast<long long>(p.tokens_per_cta), p.tokens - token0));
  const int per_head = pairs + (p.in_place ? 0 : p.dim - rotary);
  const int per_token = p.x.heads * per_head;
  for (int i = threadIdx.x; i < count * pairs; i += kRopeThreads) {
    table[i] = turn(p.rotation, p.positions[token0 + i / pairs], i % pairs);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * per_token; i += kRopeThreads) {
    const int token = i / per_token, rest = i - token * per_token, head = rest / per_head, e = rest - head * per_head;
    const long long from = (token0 + token) * p.x.token_stride + head * p.x.head_stride;
    const long long to = (token0 + token) * p.y.token_stride + head * p.y.head_stride;
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
  if (tokens > 0 && positions == nullptr) return QX_STATUS_INVALID_ARGUMENT;
  if (x->data == y->data && (x->token_stride != y->token_stride || x->head_stride != y->head_stride)) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  return QX_STATUS_OK;
}

namespace {

qx_status launch_rope(const qx_rope* rope, const qx_heads* x, const qx_heads* y, const int64_t* positions,
                      long long tokens, int dim, bool inverse, DeviceContext* ctx, cudaStream_t stream) {
  RopeParams p{};
  p.x = device_heads(x);
  p.y = device_heads(y);
  p.positions = positions;
  p.tokens = tokens;
  p.dim = dim;
  p.in_place = x->data == y->data;
  p.rotation = device_rotation(rope, inverse);
  const bool whole = dim % 16 == 0 && rope->rotary_dim % 16 == 0;
  // Tokens per CTA: enough for four rounds of its threads where there are CTAs for every SM all the same,
  // and no more than 16 KB of {cos, sin}.
  const long long per_token = static_cast<long long>(x->heads) * (whole ? dim / 16 : dim);
  const int pairs = rope->rotary_dim / 2;
  long long t = (4 * kRopeThreads + per_token - 1) / per_token;
  t = std::min<long long>(t, 2048 / pairs);
  t = std::min<long long>(t, (tokens + 4 * ctx->prop.multiProcessorCount - 1) / (4 * ctx->prop.multiProcessorCount));
  p.tokens_per_cta = static_cast<int>(std::max<long long>(t, 1));
  if (per_token * p.tokens_per_cta > (1 << 28)) return QX_STATUS_INVALID_SHAPE;
  const long long grid = (tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  const size_t smem = static_cast<size_t>(p.tokens_per_cta) * pairs * sizeof(float2);
  if (!whole) return launch_behind(rope_pairs_kernel, grid, kRopeThreads, smem, stream, p);
  switch (x->type) {
    case QX_STORAGE_F32: return launch_behind(rope_units_kernel<QX_STORAGE_F32>, grid, kRopeThreads, smem, stream, p);
    case QX_STORAGE_F16: return launch_behind(rope_units_kernel<QX_STORAGE_F16>, grid, kRopeThreads, smem, stream, p);
    default: return launch_behind(rope_units_kernel<QX_STORAGE_BF16>, grid, kRopeThreads, smem, stream, p);
  }
}

}  // namespace
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
  return kv::launch_rope(rope, x, y, positions_dev, tokens, head_dim, inverse != 0, ctx, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
