// What lies between two blocks of a layer, in one pass: the norm behind a block, its gate and residual scale, the
// sum with the residual stream, the norm in front of the next block.
//
//   joined = residual + scale * gate * post(block),  normed = pre(joined)
//   rms(v) = v / sqrt(mean(v^2) + eps) * (weight + offset) + bias,  layer(v) = rms(v - mean(v))
//
// A row (token) is held in registers between its two norms, so everything is read once and written once whatever
// the number of norms; statistics are f32 (a layer norm's variance is that of the differences from the mean, taken
// in a second sum over the registers: no cancellation), and normed is taken from joined before its rounding. A row
// takes one CTA of up to 512 threads, or a part of one, each with vectors of eight elements; which depends on the
// row's length alone, so that a row has the same bits in every batch. Up to 8192 elements all loads of a row are under way
// before the first is used; longer rows hold registers enough for one operand at a time.
#include <cmath>
#include <limits>

#include "qx_host_arrays.cuh"

namespace qx {
namespace kv {
namespace {

constexpr int kNormThreads = 512, kMostVectors = 8;
constexpr int kMostDim = 8 * kNormThreads * kMostVectors;

struct View {
  uint8_t* data;  // NULL: there is none
  int type, vector;
  long long stride;
};
struct NormParams {
  View weight, bias;  // (of one row)
  int on, layer;
  float eps, offset;
};
struct JoinParams {
  View residual, block, gate, joined, normed;
  NormParams post, pre;
  float scale, inverse_dim;
  long long tokens;
  int dim;
};

// Eight neighbouring elements as they lie in memory; where they are no whole vector, each on its own as f32 bits.
struct Words {
  uint4 a[2];
  int type;
};
__device__ __forceinline__ Words load_words(const View& x, long long row, int d, int count) {
  Words w;
  const long long index = row * x.stride + d;
  w.type = x.type;
  w.a[1] = make_uint4(0, 0, 0, 0);
  if (x.vector && count == 8) {
    const uint4* const from = reinterpret_cast<const uint4*>(x.data + index * (x.type == QX_STORAGE_F32 ? 4 : 2));
    w.a[0] = from[0];
    if (x.type == QX_STORAGE_F32) w.a[1] = from[1];
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? load_one(x.data, x.type, index + i) : 0.0f;
    to_words<QX_STORAGE_F32>(v, w.a);
    w.type = QX_STORAGE_F32;
  }
  return w;
}
__device__ __forceinline__ void values_of(const Words& w, float (&v)[8]) {
  const uint4 narrow[1] = {w.a[0]};
  if (w.type == QX_STORAGE_F32) from_words<QX_STORAGE_F32>(w.a, v);
  else if (w.type == QX_STORAGE_F16) from_words<QX_STORAGE_F16>(narrow, v);
  else from_words<QX_STORAGE_BF16>(narrow, v);
}
__device__ __forceinline__ void store_values(const View& y, long long row, int d, int count, const float (&v)[8]) {
  const long long index = row * y.stride + d;
  if (count == 8) {
    store8(y.data, y.type, y.vector, index, v);
  } else {
    for (int i = 0; i < 8; ++i) {
      if (i < count) store_one(y.data, y.type, index + i, v[i]);
    }
  }
}

// The sum over the threads of a row, the same for each of them; `shared` is this sum's own.
__device__ __forceinline__ float row_sum(float v, float* shared) {
#pragma unroll
  for (int h = 16; h > 0; h >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, h);
  const int warps = blockDim.x / 32;
  if (warps == 1) return v;
  float* const own = shared + threadIdx.y * warps;
  if ((threadIdx.x & 31) == 0) own[threadIdx.x / 32] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  v = lane < warps ? own[lane] : 0.0f;
#pragma unroll
  for (int h = 8; h > 0; h >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, h);
  return __shfl_sync(0xFFFFFFFFu, v, 0);
}

constexpr int kSums = 4, kRowWarps = kNormThreads / 32;
constexpr int kEarly = 2;  // vectors a thread, up to which every operand is loaded ahead

// A thread's vectors lie blockDim.x vectors apart.
template <int kVectors>
__device__ __forceinline__ void normalise(const NormParams& n, float inverse_dim, int dim, float (&v)[kVectors][8],
                                          float (*shared)[kRowWarps]) {
  constexpr int kHeld = kVectors <= kEarly ? kVectors : 1;
  Words weight[kHeld], bias[kHeld];
  const auto place = [](int i) { return (static_cast<int>(threadIdx.x) + i * static_cast<int>(blockDim.x)) * 8; };
  const auto load = [&](int i, int held) {
    const int d = place(i), count = min(8, dim - d);
    if (n.weight.data != nullptr && count > 0) weight[held] = load_words(n.weight, 0, d, count);
    if (n.bias.data != nullptr && count > 0) bias[held] = load_words(n.bias, 0, d, count);
  };
  if (kVectors <= kEarly) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) load(i, i);
  }
  float mean = 0.0f;
  if (n.layer) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      sum += ((v[i][0] + v[i][1]) + (v[i][2] + v[i][3])) + ((v[i][4] + v[i][5]) + (v[i][6] + v[i][7]));
    }
    mean = row_sum(sum, shared[0]) * inverse_dim;
    // (places behind the row's end stay zeros, here and in the next norm)
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int count = dim - place(i);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] -= e < count ? mean : 0.0f;
    }
  }
  float squares = 0.0f;
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(v[i][e], v[i][e], s);
    squares += s;
  }
  const float factor = 1.0f / sqrtf(row_sum(squares, shared[1]) * inverse_dim + n.eps);
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    if (place(i) >= dim) continue;
    const int held = kVectors <= kEarly ? i : 0;
    if (kVectors > kEarly) load(i, held);
    float w[8], b[8];
    if (n.weight.data != nullptr) values_of(weight[held % kHeld], w);
    if (n.bias.data != nullptr) values_of(bias[held % kHeld], b);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = v[i][e] * factor;
      v[i][e] = n.weight.data != nullptr ? x * (w[e] + n.offset) : x;
      if (n.bias.data != nullptr) v[i][e] += b[e];
    }
  }
}

template <int kVectors>
__global__ void __launch_bounds__(kNormThreads) residual_norm_kernel(const __grid_constant__ JoinParams p) {
  __shared__ float sums[kSums][kRowWarps];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const long long row = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool there = row < p.tokens;  // (all threads reach the barriers)
  const auto place = [](int i) { return (static_cast<int>(threadIdx.x) + i * static_cast<int>(blockDim.x)) * 8; };
  constexpr int kHeld = kVectors <= kEarly ? kVectors : 1;
  Words block[kVectors], residual[kHeld], gate[kHeld];
  const auto load = [&](int i, int held) {
    const int d = place(i), count = min(8, p.dim - d);
    if (!there || count <= 0) return;
    if (p.residual.data != nullptr) residual[held] = load_words(p.residual, row, d, count);
    if (p.gate.data != nullptr) gate[held] = load_words(p.gate, row, d, count);
  };
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int d = place(i), count = min(8, p.dim - d);
    if (there && count > 0 && p.block.data != nullptr) block[i] = load_words(p.block, row, d, count);
    if (kVectors <= kEarly) load(i, i % kHeld);
  }
  float v[kVectors][8];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
    if (p.block.data != nullptr && there && place(i) < p.dim) values_of(block[i], v[i]);
  }
  if (p.post.on) normalise<kVectors>(p.post, p.inverse_dim, p.dim, v, sums);
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int d = place(i);
    if (!there || d >= p.dim) continue;
    const int held = kVectors <= kEarly ? i % kHeld : 0;
    if (kVectors > kEarly) load(i, held);
    if (p.gate.data != nullptr) {
      float g[8];
      values_of(gate[held], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= g[e];
    }
    if (p.residual.data != nullptr) {
      float r[8];
      values_of(residual[held], r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = p.block.data != nullptr ? fmaf(p.scale, v[i][e], r[e]) : r[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= p.scale;
    }
    if (p.joined.data != nullptr) store_values(p.joined, row, d, min(8, p.dim - d), v[i]);
  }
  if (!p.pre.on) return;
  normalise<kVectors>(p.pre, p.inverse_dim, p.dim, v, sums + 2);
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int d = place(i);
    if (there && d < p.dim) store_values(p.normed, row, d, min(8, p.dim - d), v[i]);
  }
}

bool aligned(const void* data, int type) { return reinterpret_cast<uintptr_t>(data) % type_bytes(type) == 0; }

qx_status check_rows(const qx_rows* view, long long tokens, long long dim, bool written) {
  if (view == nullptr) return QX_STATUS_OK;
  if (!known_type(view->type)) return QX_STATUS_UNSUPPORTED_FORMAT;
  if (view->stride < 0 || (written && tokens > 1 && view->stride < dim)) return QX_STATUS_INVALID_SHAPE;
  if (tokens <= 0) return QX_STATUS_OK;
  if ((static_cast<__int128>(tokens - 1) * view->stride + dim) * 4 > std::numeric_limits<long long>::max()) {
    return QX_STATUS_INVALID_SHAPE;
  }
  return view->data == nullptr || !aligned(view->data, view->type) ? QX_STATUS_INVALID_ARGUMENT : QX_STATUS_OK;
}
qx_status check_norm(const qx_norm* norm) {
  if (norm == nullptr) return QX_STATUS_OK;
  if (norm->kind != QX_NORM_RMS && norm->kind != QX_NORM_LAYER) return QX_STATUS_INVALID_ARGUMENT;
  if (norm->weight == nullptr && norm->bias == nullptr) {
    // (no type to look at)
  } else if (!known_type(norm->type)) {
    return QX_STATUS_UNSUPPORTED_FORMAT;
  } else if (!aligned(norm->weight, norm->type) || !aligned(norm->bias, norm->type)) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  return !std::isfinite(norm->eps) || norm->eps < 0 || !std::isfinite(norm->offset) ? QX_STATUS_INVALID_ARGUMENT
                                                                                    : QX_STATUS_OK;
}
// A written view is a read one itself, or lies elsewhere.
bool same_place(const qx_rows* read, const qx_rows* written) {
  return read != nullptr && written != nullptr && read->data == written->data;
}
bool same_view(const qx_rows* read, const qx_rows* written, long long tokens) {
  return read->type == written->type && (tokens <= 1 || read->stride == written->stride);
}

qx_status check_residual_norm(const qx_rows* residual, const qx_rows* block, const qx_norm* post, const qx_rows* gate,
                              float scale, const qx_rows* joined, const qx_norm* pre, const qx_rows* normed,
                              long long tokens, long long dim) {
  if (tokens < 0 || dim <= 0 || dim > kMostDim) return QX_STATUS_INVALID_SHAPE;
  if ((residual == nullptr && block == nullptr) || (joined == nullptr && normed == nullptr) ||
      (normed == nullptr) != (pre == nullptr) || (block == nullptr && (post != nullptr || gate != nullptr)) ||
      !std::isfinite(scale)) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  for (const qx_rows* view : {residual, block, gate}) QX_TRY(check_rows(view, tokens, dim, false));
  for (const qx_rows* view : {joined, normed}) QX_TRY(check_rows(view, tokens, dim, true));
  QX_TRY(check_norm(post));
  QX_TRY(check_norm(pre));
  if (tokens == 0) return QX_STATUS_OK;
  if (same_place(joined, normed)) return QX_STATUS_INVALID_ARGUMENT;
  for (const qx_rows* read : {residual, block, gate}) {
    for (const qx_rows* written : {joined, normed}) {
      if (same_place(read, written) && !same_view(read, written, tokens)) return QX_STATUS_INVALID_ARGUMENT;
    }
  }
  return QX_STATUS_OK;
}

bool whole_vectors(const void* data, int type, long long stride) {
  return reinterpret_cast<uintptr_t>(data) % 16 == 0 && stride * static_cast<long long>(type_bytes(type)) % 16 == 0;
}
View device_view(const qx_rows* view) {
  if (view == nullptr) return {};
  return {static_cast<uint8_t*>(view->data), view->type, whole_vectors(view->data, view->type, view->stride), view->stride};
}
View device_view(const void* row, int type) {
  if (row == nullptr) return {};
  return {static_cast<uint8_t*>(const_cast<void*>(row)), type, whole_vectors(row, type, 0), 0};
}
NormParams device_norm(const qx_norm* norm) {
  if (norm == nullptr) return {};
  return {device_view(norm->weight, norm->type), device_view(norm->bias, norm->type), 1, norm->kind == QX_NORM_LAYER,
          norm->eps, norm->offset};
}

template <int kVectors>
qx_status launch(const JoinParams& p, int threads, int rows, cudaStream_t stream) {
  const long long grid = (p.tokens + rows - 1) / rows;
  return launch_behind(residual_norm_kernel<kVectors>, grid, dim3(threads, rows), 0, stream, p);
}

qx_status launch_residual_norm(const qx_rows* residual, const qx_rows* block, const qx_norm* post, const qx_rows* gate,
                               float scale, const qx_rows* joined, const qx_norm* pre, const qx_rows* normed,
                               long long tokens, int dim, cudaStream_t stream) {
  if (tokens == 0) return QX_STATUS_OK;
  JoinParams p{};
  p.residual = device_view(residual);
  p.block = device_view(block);
  p.gate = device_view(gate);
  p.joined = device_view(joined);
  p.normed = device_view(normed);
  p.post = device_norm(post);
  p.pre = device_norm(pre);
  p.scale = scale;
  p.inverse_dim = 1.0f / dim;
  p.tokens = tokens;
  p.dim = dim;
  const int vectors = (dim + 7) / 8;
  int each = 1;
  while (each * kNormThreads < vectors) each *= 2;
  const int threads = ((vectors + each - 1) / each + 31) / 32 * 32;
  const int rows = std::max(1, 256 / threads);
  switch (each) {
    case 1: return launch<1>(p, threads, rows, stream);
    case 2: return launch<2>(p, threads, rows, stream);
    case 4: return launch<4>(p, threads, rows, stream);
    default: return launch<8>(p, threads, rows, stream);
  }
}

Runs runs_of(const qx_rows* view, long long tokens, long long dim) {
  const size_t size = type_bytes(view->type);
  return {tokens, 1, view->stride * size, 0, dim * size};
}

}  // namespace
}  // namespace kv
}  // namespace qx

using namespace qx;
using namespace qx::kv;

extern "C" {

qx_status qx_residual_norm_dev(const qx_rows* residual, const qx_rows* block, const qx_norm* post, const qx_rows* gate,
                               float scale, const qx_rows* joined, const qx_norm* pre, const qx_rows* normed,
                               long long tokens, long long dim, void* stream) {
  QX_TRY(check_residual_norm(residual, block, post, gate, scale, joined, pre, normed, tokens, dim));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  return launch_residual_norm(residual, block, post, gate, scale, joined, pre, normed, tokens, static_cast<int>(dim),
                              static_cast<cudaStream_t>(stream));
}

qx_status qx_residual_norm(const qx_rows* residual, const qx_rows* block, const qx_norm* post, const qx_rows* gate,
                           float scale, const qx_rows* joined, const qx_norm* pre, const qx_rows* normed,
                           long long tokens, long long dim) {
  QX_TRY(check_residual_norm(residual, block, post, gate, scale, joined, pre, normed, tokens, dim));
  return guarded([&]() -> qx_status {
    DeviceContext* ctx = nullptr;
    QX_TRY(current_context(&ctx));
    if (tokens == 0) return QX_STATUS_OK;
    std::lock_guard<std::mutex> lock(ctx->mutex);
    Arrays a;
    const qx_rows* const views[5] = {residual, block, gate, joined, normed};  // (two that are written behind three that are read)
    qx_rows on_device[5];
    int number[5];
    for (int i = 0; i < 5; ++i) {
      number[i] = -1;
      if (views[i] == nullptr) continue;
      on_device[i] = *views[i];
      // a written view that is a read one's place goes back from there
      for (int j = 0; i >= 3 && j < 3; ++j) {
        if (same_place(views[j], views[i])) number[i] = number[j];
      }
      const bool out = i >= 3 || same_place(views[i], joined) || same_place(views[i], normed);
      if (number[i] < 0) number[i] = a.add(views[i]->data, runs_of(views[i], tokens, dim), out);
    }
    const qx_norm* const norms[2] = {post, pre};
    qx_norm norms_on_device[2];
    int weights[2] = {-1, -1}, biases[2] = {-1, -1};
    for (int i = 0; i < 2; ++i) {
      if (norms[i] == nullptr) continue;
      norms_on_device[i] = *norms[i];
      const size_t bytes = dim * type_bytes(norms[i]->type);
      if (norms[i]->weight != nullptr) weights[i] = a.add(norms[i]->weight, bytes, false);
      if (norms[i]->bias != nullptr) biases[i] = a.add(norms[i]->bias, bytes, false);
    }
    QX_TRY(a.to_device(ctx));
    const qx_rows* v[5];
    for (int i = 0; i < 5; ++i) {
      v[i] = number[i] < 0 ? nullptr : &on_device[i];
      if (number[i] >= 0) on_device[i].data = a.device<void>(number[i]);
    }
    const qx_norm* n[2];
    for (int i = 0; i < 2; ++i) {
      n[i] = norms[i] == nullptr ? nullptr : &norms_on_device[i];
      norms_on_device[i].weight = a.device<void>(weights[i]);
      norms_on_device[i].bias = a.device<void>(biases[i]);
    }
    QX_TRY(launch_residual_norm(v[0], v[1], n[0], v[2], scale, v[3], n[1], v[4], tokens, static_cast<int>(dim),
                                ctx->stream));
    return a.from_device();
  });
}

}  // extern "C"
