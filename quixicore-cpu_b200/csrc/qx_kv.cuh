// Shared by the kernels between the qkv projection and the output projection: views of heads, the
// batch of packed sequences, typed loads and stores, rotation constants.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qx_common.cuh"
#include "qx_sm100.cuh"

namespace qx {
namespace kv {

// Codes of the error word (qx_check_device_errors) for device arrays that contradict the call.
constexpr int kErrorSequence = sm100::kErrorFirstBatch;   // a sequence's rows or length do not fit the bounds
constexpr int kErrorBlock = sm100::kErrorFirstBatch + 1;  // a block id outside the cache

// On a boundary of its elements; NULL is.
template <class T>
bool on_boundary(const T* data) {
  return reinterpret_cast<uintptr_t>(data) % sizeof(T) == 0;
}

struct Heads {
  uint8_t* data;
  int type;
  int heads;
  long long token_stride, head_stride;
  int vector;  // 1: data and strides keep every 8th element on a 16-byte boundary
};

struct Batch {
  const int32_t* begin;
  const int32_t* lengths;
  const int32_t* table;
  long long table_stride, tokens, blocks;
  int sequences, max_tokens, max_length;
  int* error;
};

// Turns per position (frequency / 2 pi) instead of radians: the angle modulo a turn is then one
// rounding away, and the half-turn functions take it from there.
struct Rotation {
  int rotary, interleaved;
  float amplitude, sign;  // sign -1: the other way
  double turns[128];
};

struct Sequence {
  long long row;  // first row in the packed views
  int n, length;
};

// False (and a report) where the sequence's numbers do not fit: nothing of it is touched then. `each`: every thread
// asks for a sequence of its own.
__device__ __forceinline__ bool sequence_of(const Batch& b, int s, bool rows_are_cached, Sequence* out, bool each = false) {
  const long long row = b.begin != nullptr ? b.begin[s] : static_cast<long long>(s) * b.max_tokens;
  const long long n = b.begin != nullptr ? b.begin[s + 1] - row : b.max_tokens;
  const int length = b.lengths[s];
  out->row = row;
  out->n = static_cast<int>(n);
  out->length = length;
  const bool fits = row >= 0 && n >= 0 && n <= b.max_tokens && row + n <= b.tokens && length >= 0 &&
                    length <= b.max_length && (!rows_are_cached || n <= length);
  if (!fits && (each || threadIdx.x == 0)) sm100::report_error(b.error, kErrorSequence);
  return fits;
}

__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ float load_one(const uint8_t* data, int type, long long index) {
  if (type == QX_STORAGE_F32) return reinterpret_cast<const float*>(data)[index];
  const uint16_t bits = reinterpret_cast<const uint16_t*>(data)[index];
  if (type == QX_STORAGE_F16) return __half2float(__ushort_as_half(bits));
  return __uint_as_float(static_cast<uint32_t>(bits) << 16);
}
__device__ __forceinline__ void store_one(uint8_t* data, int type, long long index, float v) {
  if (type == QX_STORAGE_F32) {
    reinterpret_cast<float*>(data)[index] = v;
  } else if (type == QX_STORAGE_F16) {
    reinterpret_cast<__half*>(data)[index] = __float2half_rn(v);
  } else {
    reinterpret_cast<__nv_bfloat16*>(data)[index] = __float2bfloat16_rn(v);
  }
}

// Four neighbouring elements, as below.
__device__ __forceinline__ void load4(const uint8_t* data, int type, int vector, long long index, float (&v)[4]) {
  if (!vector) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = load_one(data, type, index + i);
  } else if (type == QX_STORAGE_F32) {
    const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(data) + index);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
    const uint2 a = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(data) + index);
    if (type == QX_STORAGE_F16) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a.x));
      const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&a.y));
      v[0] = x.x; v[1] = x.y; v[2] = y.x; v[3] = y.y;
    } else {
      v[0] = bf16_low(a.x); v[1] = bf16_high(a.x); v[2] = bf16_low(a.y); v[3] = bf16_high(a.y);
    }
  }
}
// Eight neighbouring elements as they lie in memory (one 16-byte word of 16-bit ones, two of f32), and as f32.
template <int kType>
__device__ __forceinline__ void load8_words(const uint8_t* data, long long index, uint4 (&w)[kType == QX_STORAGE_F32 ? 2 : 1]) {
  const uint4* const from = reinterpret_cast<const uint4*>(data + index * (kType == QX_STORAGE_F32 ? 4 : 2));
  w[0] = from[0];
  if (kType == QX_STORAGE_F32) w[kType == QX_STORAGE_F32 ? 1 : 0] = from[1];
}
template <int kType>
__device__ __forceinline__ void store8_words(uint8_t* data, long long index, const uint4 (&w)[kType == QX_STORAGE_F32 ? 2 : 1]) {
  uint4* const to = reinterpret_cast<uint4*>(data + index * (kType == QX_STORAGE_F32 ? 4 : 2));
  to[0] = w[0];
  if (kType == QX_STORAGE_F32) to[1] = w[kType == QX_STORAGE_F32 ? 1 : 0];
}
template <int kType>
__device__ __forceinline__ void from_words(const uint4 (&words)[kType == QX_STORAGE_F32 ? 2 : 1], float (&v)[8]) {
  const uint32_t w[4] = {words[0].x, words[0].y, words[0].z, words[0].w};
  if constexpr (kType == QX_STORAGE_F32) {
    const uint4& high = words[kType == QX_STORAGE_F32 ? 1 : 0];
    const uint32_t h[4] = {high.x, high.y, high.z, high.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __uint_as_float(w[i]);
      v[4 + i] = __uint_as_float(h[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (kType == QX_STORAGE_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = bf16_low(w[i]);
        v[2 * i + 1] = bf16_high(w[i]);
      }
    }
  }
}
template <int kType>
__device__ __forceinline__ void to_words(const float (&v)[8], uint4 (&words)[kType == QX_STORAGE_F32 ? 2 : 1]) {
  if constexpr (kType == QX_STORAGE_F32) {
    words[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    words[kType == QX_STORAGE_F32 ? 1 : 0] =
        make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (kType == QX_STORAGE_F16) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    words[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// The same for a type that only the launch knows. `vector`: the first of them is on a 16-byte boundary.
template <int kType>
__device__ __forceinline__ void load8_typed(const uint8_t* data, long long index, float (&v)[8]) {
  uint4 w[kType == QX_STORAGE_F32 ? 2 : 1];
  load8_words<kType>(data, index, w);
  from_words<kType>(w, v);
}
__device__ __forceinline__ void load8(const uint8_t* data, int type, int vector, long long index, float (&v)[8]) {
  if (!vector) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = load_one(data, type, index + i);
  } else if (type == QX_STORAGE_F32) {
    load8_typed<QX_STORAGE_F32>(data, index, v);
  } else if (type == QX_STORAGE_F16) {
    load8_typed<QX_STORAGE_F16>(data, index, v);
  } else {
    load8_typed<QX_STORAGE_BF16>(data, index, v);
  }
}
template <int kType>
__device__ __forceinline__ void store8_typed(uint8_t* data, long long index, const float (&v)[8]) {
  uint4 w[kType == QX_STORAGE_F32 ? 2 : 1];
  to_words<kType>(v, w);
  store8_words<kType>(data, index, w);
}
__device__ __forceinline__ void store8(uint8_t* data, int type, int vector, long long index, const float (&v)[8]) {
  if (!vector) {
#pragma unroll
    for (int i = 0; i < 8; ++i) store_one(data, type, index + i, v[i]);
  } else if (type == QX_STORAGE_F32) {
    store8_typed<QX_STORAGE_F32>(data, index, v);
  } else if (type == QX_STORAGE_F16) {
    store8_typed<QX_STORAGE_F16>(data, index, v);
  } else {
    store8_typed<QX_STORAGE_BF16>(data, index, v);
  }
}

// A head is cut into units of 16 elements, two runs of eight that lie half of the rotated (or of the other) part
// apart, so that the runs of neighbouring units, neighbouring threads, lie side by side. The runs hold eight whole
// pairs where the unit is rotated.
struct Unit {
  int first, second;
  int pair, second_pair;  // of the first pairs of the runs (QX_ROPE_HALVES: of both), -1: not rotated
};
__device__ __forceinline__ Unit unit_of(int u, int rotary, int interleaved, int dim) {
  if (16 * u >= rotary) {
    const int first = rotary + 8 * (u - rotary / 16);
    return {first, first + (dim - rotary) / 2, -1, -1};
  }
  if (interleaved) return {8 * u, 8 * u + rotary / 2, 4 * u, 4 * u + rotary / 4};
  return {8 * u, 8 * u + rotary / 2, 8 * u, 8 * u + 4};
}
// `table`: {cos, sin} of the token's pairs, times the amplitude; two of them are read at a time.
__device__ __forceinline__ void rotate_unit(const Unit& u, int interleaved, const float2* table, float (&a)[8],
                                            float (&b)[8]) {
  if (u.pair < 0) return;
  float4 s[2], t[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s[i] = reinterpret_cast<const float4*>(table + u.pair)[i];
    t[i] = reinterpret_cast<const float4*>(table + u.second_pair)[i];
  }
  const auto turn_pair = [](float& x, float& y, float c, float s) {
    const float p = x, q = y;
    x = p * c - q * s;
    y = p * s + q * c;
  };
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      turn_pair(a[4 * i], a[4 * i + 1], s[i].x, s[i].y);
      turn_pair(a[4 * i + 2], a[4 * i + 3], s[i].z, s[i].w);
      turn_pair(b[4 * i], b[4 * i + 1], t[i].x, t[i].y);
      turn_pair(b[4 * i + 2], b[4 * i + 3], t[i].z, t[i].w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      turn_pair(a[2 * i], b[2 * i], s[i].x, s[i].y);
      turn_pair(a[2 * i + 1], b[2 * i + 1], s[i].z, s[i].w);
      turn_pair(a[4 + 2 * i], b[4 + 2 * i], t[i].x, t[i].y);
      turn_pair(a[5 + 2 * i], b[5 + 2 * i], t[i].z, t[i].w);
    }
  }
}
// A thread's way through the (token, head) pairs of a few tokens, `step` pairs at a time, without divisions.
struct Walk {
  int token, head, tokens_on, heads_on, heads;
  __device__ __forceinline__ Walk(int at, int step, int heads_) : heads(heads_) {
    token = at / heads;
    head = at - token * heads;
    tokens_on = step / heads;
    heads_on = step - tokens_on * heads;
  }
  __device__ __forceinline__ void advance() {
    token += tokens_on;
    head += heads_on;
    if (head >= heads) {
      head -= heads;
      ++token;
    }
  }
};
// {cos, sin} of position * turns[pair], times the amplitude. The product is taken in 64 bits and brought to
// within half a turn there: in 32 bits a position of a million has lost the angle.
__device__ __forceinline__ float2 turn(const Rotation& r, long long position, int pair) {
  const double t = static_cast<double>(position) * r.turns[pair];
  float s, c;
  sincospif(2.0f * static_cast<float>(t - rint(t)), &s, &c);
  return make_float2(c * r.amplitude, s * r.amplitude * r.sign);
}

// ---- host side -----------------------------------------------------------------------------
inline bool known_type(int type) { return type >= QX_STORAGE_F32 && type <= QX_STORAGE_BF16; }
inline size_t type_bytes(int type) { return type == QX_STORAGE_F32 ? 4 : 2; }
// Shape, type and pointer of a view; `rows` tokens of `dim` elements, written to or only read.
qx_status check_heads(const qx_heads* view, long long rows, int dim, bool written);
qx_status check_cache(const qx_kv_cache* cache);
// The same of rows of `dim` elements; NULL is fine.
qx_status check_rows(const qx_rows* view, long long tokens, long long dim, bool written);
qx_status check_batch(const qx_kv_cache* cache, const qx_kv_batch* batch);
qx_status check_rope(const qx_rope* rope, int dim);
// The queries of a batch, at positions[row] or, with positions NULL, at their places in their sequences.
qx_status launch_rope_batch(const qx_rope* rope, const qx_heads* x, const qx_heads* y, const int64_t* positions,
                            const Batch& batch, int most, int dim, DeviceContext* ctx, cudaStream_t stream);
qx_status check_rope_call(const qx_rope* rope, const qx_heads* x, const qx_heads* y, const int64_t* positions,
                          long long tokens, int dim);
Heads device_heads(const qx_heads* view);
Batch device_batch(const qx_kv_cache* cache, const qx_kv_batch* batch, int* error);
Rotation device_rotation(const qx_rope* rope, bool inverse);

// A launch that may start while the kernel in front of it on the stream still runs: the kernel waits for it
// itself (griddepcontrol.wait) before it touches memory.
template <class Kernel, class Params>
qx_status launch_behind(Kernel kernel, long long grid, dim3 threads, size_t smem, cudaStream_t stream, const Params& p) {
  if (grid > 0x7FFFFFFFLL) {
    set_last_error_text("the call needs more thread blocks than one launch has");
    return QX_STATUS_INVALID_SHAPE;
  }
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(grid));
  config.blockDim = threads;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  QX_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, p));
  count_launch();
  return QX_STATUS_OK;
}

}  // namespace kv

// Waits for the context's stream and reports what its kernels reported (qx_api.cu).
qx_status finish_host_call(DeviceContext* ctx);

}  // namespace qx
