// A mixture-of-experts layer for few tokens, in two kernels: the router, and the experts' products.
//
//   l = x Wr^T, s = softmax(l) or sigmoid(l); the `top` experts of the largest l (or s + bias); weights s, normalised
//   y = sum over the chosen e of w_e down_e (act(gate_e x) * (up_e x)), and over the shared experts with weight 1
//
// What bounds it is the reading of the touched experts' blocks, once: 18 or 34 bytes per 32 weights. Everything else is
// arranged around keeping those loads under way from the first to the last.
//
// Router (moe_router_kernel). Both operands are cut into bf16 terms that add up to them (one for bf16, two for f16, three for
// f32), so that every product on bf16 MMAs is exact; sums over 32 columns are the MMAs', f32, in 2 .. 18 steps, those over the rest
// 64-bit: a logit is off by no more than 36 * 2^-24 of the sum of |x w|, and two experts closer than that may change places
// at the border of the choice. A CTA takes 16 experts and eight tokens, its
// 16 warps 32 columns each in turn; the CTAs of eight tokens are a cluster, whose first gets all their logits in shared
// memory and chooses the experts, a warp per token. Beside them, other CTAs turn the activations into digits. What it costs
// is latency, a good part of it that of instructions which are fetched once, so loops stay loops here.
//
// Experts (moe_experts_kernel). Every CTA sorts the (token, expert) pairs by expert, in shared memory: a microsecond, which a
// kernel of its own or the router's last CTA would add to the launch as well. Work is cut into units that CTAs draw as tickets, in this order:
//   up       64 rows (32 of gate, the same 32 of up) of one expert, for up to eight tokens of it (f32: four)
//   down     64 rows of the down projection of one expert, once all of its up units are done
//   combine  1024 elements of one token's output, once all down units are done
// A ticket only waits for smaller ones, which their CTAs have begun: no CTA has to be resident for another to go on. Eight
// warps multiply what two others bring into a ring of stages: one the weights, across units as far ahead as the ring reaches,
// one the activations, which it waits for where a unit depends on others.
//
// Products. Whole-number MMAs (16 x 8 x 32, s8) with the weights as the operand of 16 rows: codes as they are (q8_0), or
// nibbles, laid out as the signed n - 8, as 16 times that in the upper halves of bytes (q4_0), against the activations as
// balanced base-256 digits under a power of two per 32 columns: two digits for 16-bit inputs (2^-15 of a block's largest), three
// for f32 ones (2^-23). An MMA takes a block and gives exact sums. A token's digits are neighbouring columns: a lane joins two
// of them, exactly (up to 2^28), rounds that to f32 and multiplies with the block's d and the activations' scale. Four tokens
// (f32: two) cost no more than one.
// (As f16 pairs on f16 MMAs the conversion of the codes took three quarters of the instructions, and the layer twice the
// time; sums that start at the bits of 1.5 * 2^23, to be f32 numbers after a subtraction, cost four moves an MMA.) The
// products of gate and up get digits in the same way.
//
// A row's bits do not depend on the other tokens: columns are independent, and every sum has a fixed order.
//
// Measured, whole calls on weights that have left L2: 64 bf16 tokens, 8 of 128 q4_0 experts (4096 x 1536): 265 us, under lasting
// load 296 (the clock falls), 5.0 to 4.5 TB/s, 0.77 to 0.69 of the copy bandwidth (63 % of the issue slots: most of it block sums
// made f32 and scaled); 8 f16 tokens, 6 of 64 and 2 shared q8_0 experts (2048 x 1408): 66 us, 0.78; one bf16 token, 8 of 64 q4_0
// experts (2048 x 1024): 19.5 us, of which 4.4 are its bytes: router 5.5, sorting 0.5, up 6.6, down 3.5, combining 1.5, a chain; 5
// f32 tokens, 2 of 8 and 1 shared q8_0 experts (1120 x 2016): 26 to 27.
//
// Every wait is bounded (two seconds); one that runs out raises the CTA's abort flag, is reported, and the copies in flight are
// waited for (bounded).

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "qx_host_arrays.cuh"
#include "qx_moe.cuh"
#include "qx_moe_units.h"
#include "qx_scaled_gemm.cuh"
#include "qx_tile_pipe.cuh"

namespace qx {
namespace moe {
namespace {

using namespace sm100;

// ---- preparation -----------------------------------------------------------------------------
// One warp per record.
template <int kFormat>
__global__ void __launch_bounds__(256) moe_relayout_kernel(const uint8_t* __restrict__ first, const uint8_t* __restrict__ second,
                                                           uint8_t* __restrict__ to, long long tiles, int tiles_each, int blocks) {
  constexpr int kBlock = kFormat == QX_FORMAT_Q4_0 ? 18 : 34, kRecord = record_bytes(kFormat);
  const long long record = blockIdx.x * 8LL + threadIdx.x / 32;
  if (record >= tiles * blocks) return;
  const long long expert = record / (static_cast<long long>(tiles_each) * blocks);
  const long long in_expert = record - expert * tiles_each * blocks;
  const int unit = static_cast<int>(in_expert / (kUnitTiles * blocks)), in_unit = static_cast<int>(in_expert - static_cast<long long>(unit) * kUnitTiles * blocks);
  const int in_block = min(kUnitTiles, tiles_each - unit * kUnitTiles), block = in_unit / in_block;
  const long long tile = expert * tiles_each + unit * kUnitTiles + in_unit % in_block;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* const out = to + record * kRecord;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // interleaved: rows g of both matrices; else rows g and g + 8 of one
    const uint8_t* const matrix = h == 0 || second == nullptr ? first : second;
    const long long row = second == nullptr ? tile * 16 + 8 * h + g : tile * 8 + g;
    const uint8_t* const from = matrix + (row * blocks + block) * kBlock;
    if (kFormat == QX_FORMAT_Q4_0) {
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // elements 8 t + i and 8 t + 4 + i share byte i
        const int e = 8 * t + i;
        const uint32_t byte = from[2 + (e & 15)], nibble = e < 16 ? byte & 15 : byte >> 4;
        word |= (nibble ^ 8) << (8 * (i & 3) + 4 * (i >> 2));
      }
      reinterpret_cast<uint32_t*>(out)[2 * lane + h] = word;
    } else {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) word |= static_cast<uint32_t>(from[2 + 8 * t + 4 * w + i]) << (8 * i);
        reinterpret_cast<uint32_t*>(out)[4 * lane + 2 * w + h] = word;
      }
    }
    if (t == 0) {
      reinterpret_cast<uint16_t*>(out + kRecord - 32)[2 * g + h] = static_cast<uint16_t>(from[0] | from[1] << 8);
    }
  }
}

// ---- router ------------------------------------------------------------------------------------
constexpr int kRouterTokens = 8, kRouterExperts = 16, kRouterWarps = 16, kRouterThreads = 32 * kRouterWarps, kRouterCluster = 8;

// Eight neighbouring elements as they lie in memory; off 16-byte boundaries as f32.
struct Words {
  uint4 w[2];
  __device__ __forceinline__ void load(const uint8_t* data, int type, int vector, long long index) {
    if (!vector) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = kv::load_one(data, type, index + i);
      kv::to_words<QX_STORAGE_F32>(v, w);
    } else {
      const uint4* const from = reinterpret_cast<const uint4*>(data + index * (type == QX_STORAGE_F32 ? 4 : 2));
      w[0] = from[0];
      if (type == QX_STORAGE_F32) w[1] = from[1];
    }
  }
  __device__ __forceinline__ void values(int type, int vector, float (&v)[8]) const {
    const uint4 narrow[1] = {w[0]};
    if (!vector || type == QX_STORAGE_F32) kv::from_words<QX_STORAGE_F32>(w, v);
    else if (type == QX_STORAGE_F16) kv::from_words<QX_STORAGE_F16>(narrow, v);
    else kv::from_words<QX_STORAGE_BF16>(narrow, v);
  }
};

// The power of two that brings a block whose largest magnitude is `top` (as f32 bits) to what two or three balanced digits
// hold (127 * 257, 127 * 65793), and its inverse; NaN for a block that holds a NaN or an infinity. No digit stands for less than
// 2^-102: times the smallest d of a block that is still a normal number.
struct Factor {
  float up, down;
};
__device__ __forceinline__ Factor block_factor(uint32_t top, int digits) {
  const int bits = digits == 2 ? 14 : 22, exponent = max(25 + bits, static_cast<int>((top + 0x10200u) >> 23));
  return {__uint_as_float(static_cast<uint32_t>(bits + 254 - exponent) << 23),
          top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(static_cast<uint32_t>(exponent - bits) << 23)};
}
// The digits of a value under its block's factor: signed bytes, the lowest first.
__device__ __forceinline__ uint32_t digits_of(float v, const Factor& f, int digits) {
  const int whole = f.down != f.down ? 0 : __float2int_rn(v * f.up);
  const uint32_t half = digits == 2 ? 0x8080u : 0x808080u;
  return (static_cast<uint32_t>(whole) + half) ^ half;
}

// A warp turns 128 columns of a token into digits.
__device__ __forceinline__ void convert_columns(const Params& p, int token, int part) {
  const int lane = threadIdx.x & 31, d = part * 128 + lane * 4;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (d < p.dim) kv::load4(p.x, p.x_type, p.x_vector, token * p.x_stride + d, v);
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
#pragma unroll
  for (int h = 1; h < 8; h <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, h));
  const Factor factor = block_factor(top, p.digits);
  uint32_t x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = digits_of(v[e], factor, p.digits);
  for (int digit = 0; digit < p.digits; ++digit) {
    const uint32_t select = digit | (4 + digit) << 4;
    const uint32_t word = __byte_perm(__byte_perm(x[0], x[1], select), __byte_perm(x[2], x[3], select), 0x5410);
    if (d < p.dim) *reinterpret_cast<uint32_t*>(p.x_digits + (static_cast<long long>(token) * p.digits + digit) * p.dim + d) = word;
  }
  if (d < p.dim && (lane & 7) == 0) p.x_scales[static_cast<long long>(token) * scales_of(p.dim) + d / 32] = factor.down;
}

constexpr float kLeastScore = 7.8886090522101181e-31f;  // 2^-100: from here on f32 holds scores and their quotients

// Order-preserving whole number of a double, and back; NaN is above everything.
__device__ __forceinline__ unsigned long long ordered(double v) {
  const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(v));
  if (v != v) return ~0ull;
  return bits >> 63 ? ~bits : bits | 1ull << 63;
}
__device__ __forceinline__ double from_ordered(unsigned long long key) {
  return __longlong_as_double(static_cast<long long>(key >> 63 ? key & ~(1ull << 63) : ~key));
}
template <class T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int h = 16; h > 0; h >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, h);
  return v;
}

// The weight of a lane's expert where scores run out of f32 (sigmoids, or logits far below the largest):
// quotients by logarithms, in 64 bits, where no score is too small. `most`, `all`: of a softmax, the largest of all logits and the
// sum of all e^(l - most). (Rare, so not inline: what every token runs stays together.)
__device__ __noinline__ float far_weight(double logit, bool sigmoid, double most, double all, bool takes, bool normalise, float scale) {
  double power = sigmoid ? fmin(logit, 0.0) - log1p(exp(-fabs(logit))) : logit - most - log(all), sum = 1.0;
  if (normalise) {
    double top = takes ? power : -INFINITY;
#pragma unroll
    for (int h = 16; h > 0; h >>= 1) top = fmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, h));
    power -= top;
    sum = warp_sum(takes ? exp(power) : 0.0);
  }
  return static_cast<float>(exp(power) / sum * scale);
}

// A warp chooses a token's experts by their keys: logits, or scores and biases (`scores`, `logits`: without the biases).
__device__ __forceinline__ void choose(const Params& p, unsigned long long* keys, double* logits, float* scores, int token) {
  const int lane = threadIdx.x & 31, places = p.top + p.shared, each = (p.experts + 31) / 32;
  double most = -INFINITY, all = 1.0;  // softmax: the largest of all logits, the sum of all e^(l - most) where the weights need it
  if (p.bias != nullptr && p.score == QX_MOE_SOFTMAX) {  // (scores need all logits)
    for (int e = lane; e < p.experts; e += 32) {
      logits[e] = from_ordered(keys[e]);
      most = fmax(most, logits[e]);
    }
#pragma unroll
    for (int h = 16; h > 0; h >>= 1) most = fmax(most, __shfl_xor_sync(0xFFFFFFFFu, most, h));
    all = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
      for (int e = lane; e < p.experts; e += 32) {
        const double score = exp(logits[e] - most);
        if (pass == 0) {
          all += score;
        } else {
          scores[e] = static_cast<float>(score / all);
          keys[e] = ordered(score / all + static_cast<double>(p.bias[e]));
        }
      }
      if (pass == 0) all = warp_sum(all);
    }
    __syncwarp();
  }
  uint32_t left = 0;
  for (int i = 0; i < each; ++i) left |= lane + 32 * i < p.experts ? 1u << i : 0u;
  unsigned long long mine = 0;  // of the place that is this lane's
  int expert = 0;
  for (int place = 0; place < p.top; ++place) {
    // the largest key left, of the lowest expert where it is there twice
    unsigned long long best = 0;
    int at = -1;
    for (int i = 0; i < each; ++i) {
      if (!(left >> i & 1)) continue;
      const unsigned long long key = keys[lane + 32 * i];
      if (at < 0 || key > best) {
        best = key;
        at = i;
      }
    }
    const uint32_t high = __reduce_max_sync(0xFFFFFFFFu, at < 0 ? 0 : static_cast<uint32_t>(best >> 32));
    const bool still = at >= 0 && static_cast<uint32_t>(best >> 32) == high;
    const uint32_t low = __reduce_max_sync(0xFFFFFFFFu, still ? static_cast<uint32_t>(best) : 0);
    const bool is = still && static_cast<uint32_t>(best) == low;
    const uint32_t chosen = __reduce_min_sync(0xFFFFFFFFu, is ? static_cast<uint32_t>(lane + 32 * at) : 0x7FFFFFFFu);
    if (static_cast<uint32_t>(lane) == (chosen & 31)) left &= ~(1u << (chosen >> 5));
    if (lane == place) {
      mine = static_cast<unsigned long long>(high) << 32 | low;
      expert = static_cast<int>(chosen);
    }
  }
  // Scores: differences of logits from the largest are exact enough in 32 bits.
  const bool takes = lane < p.top;
  const double key = from_ordered(mine), largest = __shfl_sync(0xFFFFFFFFu, key, 0);
  float score = 0.0f, total = 1.0f;
  if (p.bias != nullptr) {
    if (takes) score = scores[expert];
  } else if (p.score == QX_MOE_SIGMOID) {
    if (takes) score = 1.0f / (1.0f + expf(static_cast<float>(-key)));
  } else {
    if (takes) score = expf(static_cast<float>(key - largest));
    if (!p.normalise) {
      total = 0.0f;
      for (int e = lane; e < p.experts; e += 32) total += expf(static_cast<float>(from_ordered(keys[e]) - largest));
      total = warp_sum(total);
      all = total;
    }
    most = largest;
  }
  if (p.normalise) total = warp_sum(score);
  if (takes) {
    const float weight = score / total * p.scale;
    p.picks[token * places + lane] = expert;
    p.weights[token * places + lane] = weight;
    if (p.chosen != nullptr) p.chosen[static_cast<long long>(token) * p.top + lane] = expert;
    if (p.chosen_weights != nullptr) p.chosen_weights[static_cast<long long>(token) * p.top + lane] = weight;
  }
  if (lane < p.shared) {
    p.picks[token * places + p.top + lane] = p.experts + lane;
    p.weights[token * places + p.top + lane] = 1.0f;
  }
  // Once more where scores ran out of f32. (Behind all else, which costs the others 0.1 us; as a choice of the weight in front of the
  // stores 0.3.)
  if (__any_sync(0xFFFFFFFFu, takes && score < kLeastScore)) {
    const double logit = p.bias != nullptr && takes ? logits[expert] : key;
    const float weight = far_weight(logit, p.score == QX_MOE_SIGMOID, most, all, takes, p.normalise != 0, p.scale);
    if (takes) {
      p.weights[token * places + lane] = weight;
      if (p.chosen_weights != nullptr) p.chosen_weights[static_cast<long long>(token) * p.top + lane] = weight;
    }
  }
}

// Eight elements as bf16 terms, pairs of them as MMA operands.
template <int kType>
struct Terms {
  static constexpr int kCount = kType == QX_STORAGE_BF16 ? 1 : kType == QX_STORAGE_F16 ? 2 : 3;
  uint32_t w[kCount][4];
  __device__ __forceinline__ Terms(const Words& words, int vector) {
    if (kType == QX_STORAGE_BF16 && vector) {
      w[0][0] = words.w[0].x;
      w[0][1] = words.w[0].y;
      w[0][2] = words.w[0].z;
      w[0][3] = words.w[0].w;
      return;
    }
    float v[8];
    words.values(kType, vector, v);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // (cut off, not rounded: what is left is exact and has eight bits less)
        const uint32_t a = __float_as_uint(v[2 * j]), b = __float_as_uint(v[2 * j + 1]);
        w[i][j] = __byte_perm(a, b, 0x7632);
        v[2 * j] -= __uint_as_float(a & 0xFFFF0000u);
        v[2 * j + 1] -= __uint_as_float(b & 0xFFFF0000u);
      }
    }
  }
};
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A warp's part of the logits of 16 experts and eight tokens: lane (g, t) has experts g, g + 8 and tokens 2 t, 2 t + 1. Lane
// (g, t) reads columns 8 t .. 8 t + 7 of a run of 32: any order of columns does that is both operands'.
template <int kX, int kW>
__device__ __forceinline__ void sum_logits(const Params& p, int token0, int expert0, double (&sum)[4]) {
  constexpr int kBatch = kX == QX_STORAGE_F32 || kW == QX_STORAGE_F32 ? 2 : 4;  // runs under way
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long x_row = min(token0 + g, p.tokens - 1) * p.x_stride;
  const long long rows[2] = {static_cast<long long>(min(expert0 + g, p.experts - 1)) * p.dim,
                             static_cast<long long>(min(expert0 + g + 8, p.experts - 1)) * p.dim};
  for (int k0 = static_cast<int>(threadIdx.x) / 32 * 32 + t * 8; k0 < p.dim; k0 += kBatch * kRouterWarps * 32) {
    Words x[kBatch], w[kBatch][2];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int k = k0 + i * kRouterWarps * 32;
      if (k >= p.dim) continue;
      x[i].load(p.x, kX, p.x_vector, x_row + k);
      w[i][0].load(p.router, kW, p.router_vector, rows[0] + k);
      w[i][1].load(p.router, kW, p.router_vector, rows[1] + k);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (k0 + i * kRouterWarps * 32 >= p.dim) continue;
      const Terms<kX> b(x[i], p.x_vector);
      const Terms<kW> a0(w[i][0], p.router_vector), a1(w[i][1], p.router_vector);
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      // (the smallest products first)
#pragma unroll
      for (int u = Terms<kW>::kCount - 1; u >= 0; --u) {
#pragma unroll
        for (int v = Terms<kX>::kCount - 1; v >= 0; --v) {
          mma_bf16(part, a0.w[u][0], a1.w[u][0], a0.w[u][1], a1.w[u][1], b.w[v][0], b.w[v][1]);
          mma_bf16(part, a0.w[u][2], a1.w[u][2], a0.w[u][3], a1.w[u][3], b.w[v][2], b.w[v][3]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += static_cast<double>(part[e]);
    }
  }
}
// Shared memory: a cluster's first CTA holds the keys of eight tokens, with a bias their logits and scores too, behind the
// parts of sums.
constexpr int kPartBytes = kRouterWarps * kRouterExperts * kRouterTokens * 8;
constexpr int key_bytes(bool biased) { return biased ? 8 + 8 + 4 : 8; }

// Grid: a cluster for every eight tokens, then those that convert activations. kX, kW: types of activations and router.
template <int kX, int kW>
__global__ void __launch_bounds__(kRouterThreads, 1) moe_router_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  auto& parts = *reinterpret_cast<double(*)[kRouterWarps][kRouterExperts][kRouterTokens]>(smem);
  unsigned long long* const keys = reinterpret_cast<unsigned long long*>(smem + kPartBytes);  // [token][expert]
  double* const logits = reinterpret_cast<double*>(keys + kRouterTokens * p.experts);
  float* const scores = reinterpret_cast<float*>(logits + kRouterTokens * p.experts);
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("barrier.cluster.arrive.relaxed.aligned;");  // (its CTAs run: their shared memory may be written)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;");
  uint32_t rank, size;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int token_groups = (p.tokens + kRouterTokens - 1) / kRouterTokens;
  const int expert_groups = (p.experts + kRouterExperts - 1) / kRouterExperts;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, token_group = static_cast<int>(blockIdx.x / size);
  if (token_group >= token_groups) {
    const int each = (p.dim + 127) / 128, item = (static_cast<int>(blockIdx.x) - token_groups * static_cast<int>(size)) * kRouterWarps + warp;
    if (item < p.tokens * each) convert_columns(p, item / each, item % each);
    return;
  }
  if (blockIdx.x == 0) {
    const int most = p.tokens * (p.top + p.shared);
    for (int i = threadIdx.x; i < most; i += kRouterThreads) p.up_done[i] = 0;
    if (threadIdx.x == 0) *p.progress = {0, 0};
  }
  const int token0 = token_group * kRouterTokens;
  for (int expert_group = static_cast<int>(rank); expert_group < expert_groups; expert_group += static_cast<int>(size)) {
    const int expert0 = expert_group * kRouterExperts;
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    sum_logits<kX, kW>(p, token0, expert0, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) parts[warp][(lane >> 2) + 8 * (e >> 1)][2 * (lane & 3) + (e & 1)] = sum[e];
    __syncthreads();
    const int e = threadIdx.x / kRouterTokens, t = threadIdx.x % kRouterTokens;
    if (threadIdx.x < kRouterExperts * kRouterTokens && expert0 + e < p.experts) {
      double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int i = 0; i < kRouterWarps; ++i) v[i & 3] += parts[i][e][t];
      double key = (v[0] + v[1]) + (v[2] + v[3]);
      uint32_t to;
      if (p.bias != nullptr && p.score == QX_MOE_SIGMOID) {
        const double score = 1.0 / (1.0 + exp(-key));
        asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(logits + t * p.experts + expert0 + e)));
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(key) : "memory");
        key = score + static_cast<double>(p.bias[expert0 + e]);
        asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(scores + t * p.experts + expert0 + e)));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(static_cast<float>(score)) : "memory");
      }
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(keys + t * p.experts + expert0 + e)));
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(ordered(key)) : "memory");
    }
    __syncthreads();
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0 && warp < kRouterTokens && token0 + warp < p.tokens) {
    choose(p, keys + warp * p.experts, logits + warp * p.experts, scores + warp * p.experts, token0 + warp);
  }
}

// ---- experts -----------------------------------------------------------------------------------
constexpr int kMathWarps = 8, kExpertThreads = 32 * (kMathWarps + 2);
constexpr int kWeightWarp = kMathWarps, kColumnWarp = kMathWarps + 1;
constexpr int kUnitRows = kUnitTiles * kTileRows;
constexpr int kMostTokens = 8;
static_assert(kUpWidth == kUnitRows / 2 && kDownWidth == kUnitRows && kCombineWidth == 4 * 32 * kMathWarps, "what the kernel cuts");
constexpr int kReduceTile = 64 + 1, kReduceWarp = kUnitTiles * kReduceTile;  // floats: [row g, g + 8][lane]
enum { kUp = 0, kDown = 1, kCombine = 2, kExit = 3 };

// What a unit is, beside its first stage.
struct UnitInfo {
  int kind, blocks, tiles, unit;
  int group, count, unused[2];
  uint16_t entries[8];
};
// The pairs of a pass by expert, and how each expert's are cut into groups.
struct Group {
  uint32_t expert : 10, first : 11, count : 4;  // entries list[first .. first + count - 1]
};
constexpr int kAllExperts = kMostExperts + kMostShared, kMostGroups = kAllExperts + kPassEntries / 4;
struct Plan {
  int groups;
  uint16_t list[kPassEntries];  // entries, by expert, ascending
  Group group[kMostGroups];
};
constexpr int kMaskWords = kPassTokens / 32;
struct SortSpace {
  uint32_t tokens[kAllExperts][kMaskWords];  // of each expert
  uint16_t first[kAllExperts];
  int sums[2][kExpertThreads / 32];
};

template <int kFormat>
struct ExpertShape {
  static constexpr int kRecord = record_bytes(kFormat);
  static constexpr int kBlocks = kFormat == QX_FORMAT_Q4_0 ? 16 : 8;  // of a stage
  static constexpr int kStages = kFormat == QX_FORMAT_Q4_0 ? 3 : 4;
  // Between columns, and tokens' scales: lanes of an 8-byte load, four columns at a time, and of a 4-byte one meet no conflicts.
  static constexpr int kColumnBytes = kBlocks * 32 + 32, kScaleBytes = kBlocks * 4 + 16;
  static constexpr int kWeights = kBlocks * kUnitTiles * kRecord;
  static constexpr int kScales = kWeights + kColumns * kColumnBytes;
  static constexpr int kStage = kScales + kMostTokens * kScaleBytes;
  static constexpr int kReduce = kStages * kStage;
  static constexpr int kInfo = kReduce + (2 * kMathWarps * kReduceWarp * 4 + 15) / 16 * 16;
  static constexpr int kBars = kInfo + kStages * static_cast<int>(sizeof(UnitInfo));
  static constexpr int kPlan = kBars + 3 * kStages * 8 + 16;
  static constexpr int kBytes = kPlan + static_cast<int>(sizeof(Plan));
  static_assert(sizeof(SortSpace) <= kStages * kStage, "sorting takes the ring's place");
};

// All threads of the CTA sort the pairs, into groups of `most` tokens.
__device__ __forceinline__ void sort_pairs(const Params& p, int most, SortSpace& s, Plan& plan) {
  const int experts = p.experts + p.shared, places = p.top + p.shared, entries = p.tokens * places;
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  if (p.tokens == 1) {  // a group for every pick
    if (threadIdx.x < entries) {
      plan.list[threadIdx.x] = static_cast<uint16_t>(threadIdx.x);
      Group& to = plan.group[threadIdx.x];
      to.expert = static_cast<uint32_t>(__ldcg(p.picks + threadIdx.x));
      to.first = threadIdx.x;
      to.count = 1;
    }
    if (threadIdx.x == 0) plan.groups = entries;
    __syncthreads();
    return;
  }
  constexpr int kEach = (kPassEntries + kExpertThreads - 1) / kExpertThreads;
  int pick[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = threadIdx.x + j * kExpertThreads;
    if (i < entries) pick[j] = __ldcg(p.picks + i);
  }
  for (int i = threadIdx.x; i < experts * kMaskWords; i += kExpertThreads) s.tokens[i / kMaskWords][i % kMaskWords] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = threadIdx.x + j * kExpertThreads, token = i / places;
    if (i < entries) atomicOr(&s.tokens[pick[j]][token / 32], 1u << (token & 31));
  }
  __syncthreads();
  // Running numbers of entries and groups in front of each expert, a thread per expert at a time.
  int entries_before = 0, groups_before = 0;
  for (int e0 = 0; e0 < experts; e0 += kExpertThreads) {
    const int e = e0 + static_cast<int>(threadIdx.x);
    int count = 0;
    if (e < experts) {
#pragma unroll
      for (int w = 0; w < kMaskWords; ++w) count += __popc(s.tokens[e][w]);
    }
    const int cuts = (count + most - 1) / most;
    int through = count, cuts_through = cuts;
#pragma unroll
    for (int h = 1; h < 32; h <<= 1) {
      const int a = __shfl_up_sync(0xFFFFFFFFu, through, h), b = __shfl_up_sync(0xFFFFFFFFu, cuts_through, h);
      if (lane >= h) {
        through += a;
        cuts_through += b;
      }
    }
    if (lane == 31) {
      s.sums[0][warp] = through;
      s.sums[1][warp] = cuts_through;
    }
    __syncthreads();
    int first = entries_before + through - count, group = groups_before + cuts_through - cuts;
#pragma unroll
    for (int w = 0; w < kExpertThreads / 32; ++w) {
      const int a = s.sums[0][w], b = s.sums[1][w];
      first += w < warp ? a : 0;
      group += w < warp ? b : 0;
      entries_before += a;
      groups_before += b;
    }
    if (e < experts) {
      s.first[e] = static_cast<uint16_t>(first);
      for (int i = 0; i < cuts; ++i) {
        Group& to = plan.group[group + i];
        to.expert = static_cast<uint32_t>(e);
        to.first = static_cast<uint32_t>(first + i * most);
        to.count = static_cast<uint32_t>(min(most, count - i * most));
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = threadIdx.x + j * kExpertThreads;
    if (i >= entries) continue;
    const int token = i / places;
    int rank = __popc(s.tokens[pick[j]][token / 32] & ((1u << (token & 31)) - 1));
#pragma unroll
    for (int w = 0; w < kMaskWords; ++w) rank += w < token / 32 ? __popc(s.tokens[pick[j]][w]) : 0;
    plan.list[s.first[pick[j]] + rank] = static_cast<uint16_t>(i);
  }
  if (threadIdx.x == 0) plan.groups = groups_before;
  __syncthreads();
}

// A block's sums.
__device__ __forceinline__ void mma_block(int (&d)[4], const uint32_t (&a)[4], uint2 b) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(0));
}
// The codes (q4_0: 16 times) of a lane's columns 8 t .. 8 t + 7 of rows g and g + 8: operands of the block's MMA.
template <int kFormat>
__device__ __forceinline__ void load_codes(const uint8_t* record, int lane, uint32_t (&a)[4]) {
  if (kFormat == QX_FORMAT_Q4_0) {
    const uint2 w = *reinterpret_cast<const uint2*>(record + lane * 8);
    a[0] = w.x << 4 & 0xF0F0F0F0u;
    a[1] = w.y << 4 & 0xF0F0F0F0u;
    a[2] = w.x & 0xF0F0F0F0u;
    a[3] = w.y & 0xF0F0F0F0u;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(record + lane * 16);
    a[0] = w.x;
    a[1] = w.y;
    a[2] = w.z;
    a[3] = w.w;
  }
}

// A warp's blocks of a stage, every eighth: 64 rows x 8 kN columns, sums in `total` [tile][column tile][row g, row g + 8] of
// the lane's pair of digits; `join`: how many of the lower digit one of the higher is. The pointers are at the warp's first
// block (scales: of the lane's token); `blocks` is what the stage has from there on. kWhole: all of four tiles.
template <int kFormat, int kN, int kTokens, bool kWhole>
__device__ __forceinline__ void multiply(const uint8_t* records, int tiles_there, const uint8_t* columns, const uint8_t* scales, int blocks,
                                         int join, float (&total)[kUnitTiles][2][2]) {
  using S = ExpertShape<kFormat>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tiles = kWhole ? kUnitTiles : tiles_there;
#pragma unroll
  for (int b = 0; b < S::kBlocks / kMathWarps; ++b) {
    if (!kWhole && b * kMathWarps >= blocks) continue;
    uint2 x[kN];
    float scale[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      x[n] = *reinterpret_cast<const uint2*>(columns + (8 * n + g) * S::kColumnBytes + b * kMathWarps * 32 + t * 8);
      scale[n] = *reinterpret_cast<const float*>(scales + n * kTokens * S::kScaleBytes + b * kMathWarps * 4);
    }
#pragma unroll
    for (int i = 0; i < kUnitTiles; ++i) {
      if (!kWhole && i >= tiles) continue;
      const uint8_t* const record = records + (b * kMathWarps * tiles + i) * S::kRecord;
      uint32_t a[4];
      load_codes<kFormat>(record, lane, a);
      const float2 d = __half22float2(reinterpret_cast<const __half2*>(record + S::kRecord - 32)[g]);
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        int sum[4];
        mma_block(sum, a, x[n]);
        // (below 2^28: rounded once, to f32)
        total[i][n][0] = fmaf(static_cast<float>(sum[1] * join + sum[0]), scale[n] * d.x, total[i][n][0]);
        total[i][n][1] = fmaf(static_cast<float>(sum[3] * join + sum[2]), scale[n] * d.y, total[i][n][1]);
      }
    }
  }
}

// The math warps meet: barrier 1.
__device__ __forceinline__ void math_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kMathWarps) : "memory"); }

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// This thread's arrival at a barrier, once its copies so far have landed.
__device__ __forceinline__ void arrive_behind_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ int load_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// The copying warps' bounded wait: they run ahead, and polls would take issue slots from the products.
__device__ __forceinline__ bool wait_asleep(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  bool done = mbar_try_wait(bar, parity);
  if (!done) {
    const unsigned long long start = global_timer_ns();
    for (uint32_t spin = 1; !done; ++spin) {
      __nanosleep(32);
      done = mbar_try_wait(bar, parity);
      if ((spin & 63u) == 0u && (*abort_flag != 0 || global_timer_ns() - start > kWaitLimitNs)) break;
    }
  }
  return __all_sync(0xFFFFFFFFu, done);
}
// Until *counter >= target; false where the time runs out or the CTA gives up.
__device__ __forceinline__ bool wait_for_count(const int* counter, int target, volatile int* abort_flag) {
  if (load_acquire(counter) >= target) return true;
  const unsigned long long start = global_timer_ns();
  for (uint32_t spin = 1;; ++spin) {
    if (load_acquire(counter) >= target) return true;
    __nanosleep(32);
    if ((spin & 63u) == 0u && (*abort_flag != 0 || global_timer_ns() - start > kWaitLimitNs)) return false;
  }
}

template <int kFormat, int kDigits>
__global__ void __launch_bounds__(kExpertThreads, 2) moe_experts_kernel(const __grid_constant__ Params p) {
  using S = ExpertShape<kFormat>;
  constexpr int kStages = S::kStages, kSpan = columns_of(kDigits), kTokens = 8 / kSpan;
  extern __shared__ __align__(128) uint8_t smem[];
  float* const reduce = reinterpret_cast<float*>(smem + S::kReduce);
  UnitInfo* const infos = reinterpret_cast<UnitInfo*>(smem + S::kInfo);
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* const empty = full + kStages;
  uint64_t* const begun = empty + kStages;
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(begun + kStages);
  Plan& plan = *reinterpret_cast<Plan*>(smem + S::kPlan);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, 1 + 32);  // (the weights, and each lane's copies of activations)
      mbar_init(empty + i, kMathWarps);
      mbar_init(begun + i, 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int next = 0;
  if (threadIdx.x == 32 * kWeightWarp) next = atomicAdd(&p.progress->ticket, 1);
  sort_pairs(p, 2 * kTokens, *reinterpret_cast<SortSpace*>(smem), plan);

  const int up_blocks = p.dim / 32, down_blocks = p.inner / 32;
  const int up_units = p.inner / 32, down_tiles = p.dim / kTileRows, down_units = (down_tiles + kUnitTiles - 1) / kUnitTiles;

  if (warp == kWeightWarp) {
    // ---- weights, as far ahead as the ring reaches ---------------------------------------------
    const int combine_chunks = (p.dim + kCombineWidth - 1) / kCombineWidth;
    const int ups = plan.groups * up_units, downs = plan.groups * down_units, all = ups + downs + p.tokens * combine_chunks;
    tile::Ring ring;
    int issued = 0;  // stages, as far as the ring's size
    bool ok = true;
    asm volatile("fence.proxy.async;" ::: "memory");  // (the ring's place was the sorting's)
    for (bool more = true; ok && more;) {
      const int ticket = __shfl_sync(0xFFFFFFFFu, next, 0);
      if (lane == 0 && ticket < all) next = atomicAdd(&p.progress->ticket, 1);  // (needed a unit later)
      UnitInfo unit;
      unit.kind = ticket < ups ? kUp : ticket < ups + downs ? kDown : ticket < all ? kCombine : kExit;
      unit.blocks = unit.tiles = unit.count = unit.group = unit.unit = 0;
      more = unit.kind != kExit;
      int entry = 0, stages = 1;
      const uint8_t* weights = nullptr;
      if (unit.kind == kUp || unit.kind == kDown) {
        const bool up = unit.kind == kUp;
        const int units = up ? up_units : down_units, at = up ? ticket : ticket - ups;
        unit.group = at / units;
        unit.unit = at - unit.group * units;
        const Group work = plan.group[unit.group];
        unit.count = work.count;
        unit.blocks = up ? up_blocks : down_blocks;
        unit.tiles = up ? kUnitTiles : min(kUnitTiles, down_tiles - unit.unit * kUnitTiles);
        stages = (unit.blocks + S::kBlocks - 1) / S::kBlocks;
        const long long tile0 = static_cast<long long>(work.expert) * (up ? p.inner / 8 : down_tiles) + unit.unit * kUnitTiles;
        weights = (up ? p.up : p.down) + tile0 * unit.blocks * S::kRecord;
        if (lane < unit.count) entry = plan.list[work.first + lane];
      } else if (unit.kind == kCombine) {
        unit.group = (ticket - ups - downs) / combine_chunks;  // (the token)
        unit.unit = ticket - ups - downs - unit.group * combine_chunks;
      }
      for (int stage = 0; stage < stages; ++stage) {
        ok = issued < kStages || wait_asleep(empty + ring.slot, ring.phase ^ 1u, abort_flag);
        if (!ok) break;
        issued = min(issued + 1, kStages);
        if (stage == 0) {
          UnitInfo& info = infos[ring.slot];
          if (lane == 0) {
            info.kind = unit.kind;
            info.blocks = unit.blocks;
            info.tiles = unit.tiles;
            info.unit = unit.unit;
            info.group = unit.group;
            info.count = unit.count;
          }
          if (lane < unit.count) info.entries[lane] = static_cast<uint16_t>(entry);
          __syncwarp();
        }
        if (lane == 0) {
          mbar_arrive(begun + ring.slot);
          const uint32_t bytes = min(S::kBlocks, unit.blocks - stage * S::kBlocks) * unit.tiles * S::kRecord;
          mbar_arrive_expect_tx(full + ring.slot, bytes);
          if (bytes > 0) {
            tile::bulk_load(smem + ring.slot * S::kStage, weights + static_cast<long long>(stage) * S::kBlocks * unit.tiles * S::kRecord,
                            bytes, full + ring.slot);
          }
        }
        ring.advance(kStages);
      }
    }
    if (!ok) {
      if (lane == 0 && *abort_flag == 0) report_error(p.error, 52);
      *abort_flag = 1;
      // what is in flight has to land before the CTA's memory is another's: the last use of each stage, or half a
      // second where its activations never come
      __syncwarp();
      const unsigned long long start = global_timer_ns();
      for (int slot = 0; slot < issued; ++slot) {
        const uint32_t phase = slot < static_cast<int>(ring.slot) ? ring.phase : ring.phase ^ 1u;
        while (!mbar_try_wait(full + slot, phase) && global_timer_ns() - start < kWaitLimitNs / 4) {
        }
      }
    }
    return;
  }

  if (warp == kColumnWarp) {
    // ---- activations, once they are there --------------------------------------------------------
    const int downs = plan.groups * down_units;
    tile::Ring ring;
    bool ok = true;
    for (;;) {
      ok = wait_asleep(begun + ring.slot, ring.phase, abort_flag);
      if (!ok) break;
      const UnitInfo& info = infos[ring.slot];
      const int kind = info.kind, blocks = info.blocks, count = info.count, group = info.group;
      const int width = kind == kUp ? p.dim : p.inner;
      const int8_t* const digits = kind == kUp ? p.x_digits : p.inner_digits;
      const float* const scales = kind == kUp ? p.x_scales : p.inner_scales;
      // Lane c < 16 looks after column c, a digit of a token: its row.
      const int place = lane / kSpan;
      int token = -1, row = -1;
      if (lane < kColumns && place < count) {
        token = kind == kUp ? info.entries[place] / (p.top + p.shared) : info.entries[place];
        if (lane % kSpan < kDigits) row = token * kDigits + lane % kSpan;
      }
      // 16 bytes a lane: a column takes 2 * kBlocks lanes, a token's scales kBlocks / 4.
      constexpr int kLanes = 2 * S::kBlocks, kScaleLanes = S::kBlocks / 4, kTurns = kColumns * kLanes / 32;
      int from[kTurns];
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int r = __shfl_sync(0xFFFFFFFFu, row, i * (32 / kLanes) + lane / kLanes);
        from[i] = r < 0 ? -1 : r * width + lane % kLanes * 16;
      }
      static_assert(kMostTokens * kScaleLanes <= 32, "the scales of all tokens are one turn");
      const int scale_token = __shfl_sync(0xFFFFFFFFu, token, lane / kScaleLanes * kSpan);
      const int scales_from = scale_token < 0 || lane / kScaleLanes >= count ? -1 : scale_token * scales_of(width) + lane % kScaleLanes * 4;
      if (kind == kDown) ok = wait_for_count(p.up_done + group, up_units, abort_flag);
      if (kind == kCombine) ok = wait_for_count(&p.progress->down_done, downs, abort_flag);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      for (int first = 0;;) {
        const int in_stage = min(S::kBlocks, blocks - first);
        const uint32_t to = smem_u32(smem + ring.slot * S::kStage);
        const bool value = lane % kLanes < in_stage * 2;
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
          if (value && from[i] >= 0) {
            copy16(to + S::kWeights + (i * (32 / kLanes) + lane / kLanes) * S::kColumnBytes + lane % kLanes * 16, digits + from[i] + first * 32);
          }
        }
        if (scales_from >= 0 && lane % kScaleLanes * 4 < in_stage) {
          copy16(to + S::kScales + lane / kScaleLanes * S::kScaleBytes + lane % kScaleLanes * 16, scales + scales_from + first);
        }
        if (kind == kCombine) mbar_arrive(full + ring.slot);  // (no copies: hands on what the wait has seen)
        else arrive_behind_copies(full + ring.slot);
        ring.advance(kStages);
        first += S::kBlocks;
        if (first >= blocks) break;
        ok = wait_asleep(begun + ring.slot, ring.phase, abort_flag);
        if (!ok) break;
      }
      if (!ok || kind == kExit) break;
    }
    if (!ok) {
      if (lane == 0 && *abort_flag == 0) report_error(p.error, 51);
      *abort_flag = 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  // ---- products ------------------------------------------------------------------------------
  const int places = p.top + p.shared;
  const int join = kSpan == 4 && (lane & 1) ? 0 : 256;  // (a third digit stands alone)
  tile::Ring ring;
  float total[kUnitTiles][2][2] = {};
  const auto wait_for_stage = [&]() {
    if (mbar_wait_warp(full + ring.slot, ring.phase, abort_flag)) return true;
    if (threadIdx.x == 0 && *abort_flag == 0) report_error(p.error, 53);
    *abort_flag = 1;
    return false;  // (the other math warps see the flag, or run into the same wait)
  };
  const auto free_stage = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + ring.slot);
    ring.advance(kStages);
  };
  for (;;) {
    if (!wait_for_stage()) return;
    const UnitInfo& info = infos[ring.slot];
    const int kind = info.kind, unit = info.unit, group = info.group, count = info.count, tiles = info.tiles, blocks = info.blocks;
    if (kind == kExit) return;
    const int entry = lane < count ? info.entries[lane] : 0;
    if (kind == kCombine) free_stage();
    if (kind == kCombine) {
      const int d = unit * kCombineWidth + static_cast<int>(threadIdx.x) * 4;
      if (d < p.dim) {
        const float* const from = p.products + static_cast<long long>(group) * places * p.dim + d;
        const float* const weight = p.weights + group * places;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i0 = 0; i0 < places; i0 += 8) {
          float4 v[8];
          float w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i0 + i >= places) continue;
            v[i] = __ldcg(reinterpret_cast<const float4*>(from + static_cast<long long>(i0 + i) * p.dim));
            w[i] = __ldcg(weight + i0 + i);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i0 + i >= places) continue;
            sum.x = fmaf(w[i], v[i].x, sum.x);
            sum.y = fmaf(w[i], v[i].y, sum.y);
            sum.z = fmaf(w[i], v[i].z, sum.z);
            sum.w = fmaf(w[i], v[i].w, sum.w);
          }
        }
        const long long to = group * p.out_stride + d;
        kv::store_one(p.out, p.out_type, to, sum.x);
        kv::store_one(p.out, p.out_type, to + 1, sum.y);
        kv::store_one(p.out, p.out_type, to + 2, sum.z);
        kv::store_one(p.out, p.out_type, to + 3, sum.w);
      }
      continue;
    }
    bool ok = true;
    const auto multiply_unit = [&](auto column_tiles) {
      constexpr int kN = decltype(column_tiles)::value;
      for (int left = blocks;;) {
        const uint8_t* const stage = smem + ring.slot * S::kStage;
        const uint8_t* const records = stage + warp * tiles * S::kRecord;
        const uint8_t* const columns = stage + S::kWeights + warp * 32;
        const uint8_t* const scales = stage + S::kScales + (lane & 3) * 2 / kSpan * S::kScaleBytes + warp * 4;
        if (left >= S::kBlocks && tiles == kUnitTiles) multiply<kFormat, kN, kTokens, true>(records, tiles, columns, scales, S::kBlocks, join, total);
        else multiply<kFormat, kN, kTokens, false>(records, tiles, columns, scales, min(left, S::kBlocks) - warp, join, total);
        free_stage();
        left -= S::kBlocks;
        if (left <= 0) return;
        ok = wait_for_stage();
        if (!ok) return;
      }
    };
    if (count <= kTokens) multiply_unit(std::integral_constant<int, 1>());
    else multiply_unit(std::integral_constant<int, 2>());
    if (!ok) return;

    // ---- the unit's sums: every warp has a part of each ------------------------------------------
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (n * kTokens >= count) continue;
#pragma unroll
      for (int i = 0; i < kUnitTiles; ++i) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          reduce[(n * kMathWarps + warp) * kReduceWarp + i * kReduceTile + r * 32 + lane] = total[i][n][r];
          total[i][n][r] = 0.0f;
        }
      }
    }
    // Row g (or g + 8) of a tile for a token: its pairs of digits, from all warps.
    const auto sum_of = [&](int tile_at, int row, int token) {
      const float* const at = reduce + token / kTokens * kMathWarps * kReduceWarp + tile_at * kReduceTile + (row >> 3) * 32 + (row & 7) * 4 +
                              token % kTokens * (kSpan / 2);
      float v[kSpan / 2];
#pragma unroll
      for (int pair = 0; pair < kSpan / 2; ++pair) {
        float part[kMathWarps];
#pragma unroll
        for (int w = 0; w < kMathWarps; ++w) part[w] = at[w * kReduceWarp + pair];
        v[pair] = ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
      }
      const float sum = kSpan == 2 ? v[0] : fmaf(v[kSpan / 2 - 1], 65536.0f, v[0]);
      return kFormat == QX_FORMAT_Q4_0 ? sum * 0.0625f : sum;
    };
    math_barrier();
    if (kind == kUp) {
      // a warp takes a token, a lane a column of the inner activations: a block of 32
      static_assert(2 * kTokens <= kMathWarps, "a warp for every token");
      if (warp < count) {
        const float gate = sum_of(lane >> 3, lane & 7, warp), up = sum_of(lane >> 3, 8 + (lane & 7), warp);
        const float a = projection_activation(gate, p.activation) * up;
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(a) & 0x7FFFFFFFu);
        const Factor factor = block_factor(top, kDigits);
        const uint32_t x = digits_of(a, factor, kDigits);
        const int at = __shfl_sync(0xFFFFFFFFu, entry, warp);
#pragma unroll
        for (int digit = 0; digit < kDigits; ++digit) {
          p.inner_digits[(static_cast<long long>(at) * kDigits + digit) * p.inner + unit * 32 + lane] = static_cast<int8_t>(x >> (8 * digit));
        }
        if (lane == 0) p.inner_scales[static_cast<long long>(at) * scales_of(p.inner) + unit] = factor.down;
      }
    } else {
      const int r = threadIdx.x & (kUnitRows - 1), row = unit * kUnitRows + r;
#pragma unroll
      for (int c0 = 0; c0 < 2 * kTokens; c0 += 32 * kMathWarps / kUnitRows) {
        const int c = c0 + static_cast<int>(threadIdx.x) / kUnitRows, at = __shfl_sync(0xFFFFFFFFu, entry, c);
        if (c < count && row < p.dim) p.products[static_cast<long long>(at) * p.dim + row] = sum_of(r >> 4, r & 15, c);
      }
    }
    math_barrier();
    if (static_cast<int>(threadIdx.x) == (unit & (kMathWarps - 1)) * 32) {  // (not always the same warp's time)
      __threadfence();
      atomicAdd(kind == kUp ? p.up_done + group : &p.progress->down_done, 1);
    }
  }
}

// ---- host side ------------------------------------------------------------------------------------

qx_status check_prepare(int format, const void* gate, const void* up, const void* down, int experts, int shared, long long dim,
                        long long inner, qx_moe** out) {
  if (out == nullptr) return QX_STATUS_INVALID_ARGUMENT;
  *out = nullptr;
  if (gate == nullptr || up == nullptr || down == nullptr) return QX_STATUS_INVALID_ARGUMENT;
  size_t block_bytes = 0;
  if (!format_info(format, &block_bytes)) return QX_STATUS_UNSUPPORTED_FORMAT;
  if (experts < 1 || experts > kMostExperts || shared < 0 || shared > kMostShared || dim <= 0 || inner <= 0 || dim % kBlockK != 0 ||
      inner % kBlockK != 0 || dim > kMostWidth || inner > kMostWidth) {
    return QX_STATUS_INVALID_SHAPE;
  }
  return QX_STATUS_OK;
}

// `count` experts of `rows` rows.
qx_status relayout(int format, const uint8_t* first, const uint8_t* second, uint8_t* to, int count, int rows, int columns,
                   cudaStream_t stream) {
  const int each = (second == nullptr ? rows : 2 * rows) / kTileRows;
  const long long tiles = static_cast<long long>(count) * each, records = tiles * (columns / 32);
  const long long grid = (records + 7) / 8;
  if (grid > 0x7FFFFFFFLL) return QX_STATUS_INVALID_SHAPE;
  if (format == QX_FORMAT_Q4_0) {
    moe_relayout_kernel<QX_FORMAT_Q4_0><<<static_cast<unsigned>(grid), 256, 0, stream>>>(first, second, to, tiles, each, columns / 32);
  } else {
    moe_relayout_kernel<QX_FORMAT_Q8_0><<<static_cast<unsigned>(grid), 256, 0, stream>>>(first, second, to, tiles, each, columns / 32);
  }
  QX_CUDA_TRY(cudaGetLastError());
  count_launch();
  return QX_STATUS_OK;
}

qx_status prepare(int format, const uint8_t* gate, const uint8_t* up, const uint8_t* down, int experts, int shared, int dim,
                  int inner, bool host, DeviceContext* ctx, cudaStream_t stream, qx_moe** out) {
  auto* m = new (std::nothrow) qx_moe();
  if (m == nullptr) return QX_STATUS_OUT_OF_MEMORY;
  m->device = ctx->device;
  m->format = format;
  m->experts = experts;
  m->shared = shared;
  m->dim = dim;
  m->inner = inner;
  const int count = experts + shared;
  const size_t matrix = static_cast<size_t>(inner) * (dim / 32);  // blocks
  const size_t block = format == QX_FORMAT_Q4_0 ? 18 : 34, bytes = matrix * block;
  m->up_bytes = 2 * bytes * count;
  m->down_bytes = bytes * count;
  void* temp = nullptr;
  const auto fill = [&]() -> qx_status {
    QX_CUDA_TRY(cudaMalloc(reinterpret_cast<void**>(&m->up), m->up_bytes));
    QX_CUDA_TRY(cudaMalloc(reinterpret_cast<void**>(&m->down), m->down_bytes));
    if (!host) {
      QX_TRY(relayout(format, gate, up, m->up, count, inner, dim, stream));
      return relayout(format, down, nullptr, m->down, count, dim, inner, stream);
    }
    QX_CUDA_TRY(cudaMalloc(&temp, 3 * bytes));  // (one expert at a time)
    uint8_t* const to = static_cast<uint8_t*>(temp);
    for (int e = 0; e < count; ++e) {
      QX_CUDA_TRY(cudaMemcpyAsync(to, gate + e * bytes, bytes, cudaMemcpyHostToDevice, stream));
      QX_CUDA_TRY(cudaMemcpyAsync(to + bytes, up + e * bytes, bytes, cudaMemcpyHostToDevice, stream));
      QX_CUDA_TRY(cudaMemcpyAsync(to + 2 * bytes, down + e * bytes, bytes, cudaMemcpyHostToDevice, stream));
      QX_TRY(relayout(format, to, to + bytes, m->up + 2 * bytes * e, 1, inner, dim, stream));
      QX_TRY(relayout(format, to + 2 * bytes, nullptr, m->down + bytes * e, 1, dim, inner, stream));
    }
    QX_CUDA_TRY(cudaStreamSynchronize(stream));
    return QX_STATUS_OK;
  };
  const qx_status status = fill();
  if (temp != nullptr) (void)cudaFree(temp);
  if (status != QX_STATUS_OK) {
    qx_moe_destroy(m);
    return status;
  }
  *out = m;
  return QX_STATUS_OK;
}

qx_status check_apply(const qx_moe* m, const qx_moe_router* router, const qx_rows* x, const qx_rows* out, long long tokens,
                      int activation, const int32_t* chosen, const float* weights) {
  if (m == nullptr || router == nullptr || x == nullptr || out == nullptr || tokens < 0) return QX_STATUS_INVALID_ARGUMENT;
  if (!kv::known_type(router->type)) return QX_STATUS_UNSUPPORTED_FORMAT;
  if (router->top < 1 || router->top > std::min(kMostTop, m->experts)) return QX_STATUS_INVALID_SHAPE;
  if (router->weights == nullptr || reinterpret_cast<uintptr_t>(router->weights) % kv::type_bytes(router->type) != 0 || !kv::on_boundary(router->bias) ||
      (router->score != QX_MOE_SOFTMAX && router->score != QX_MOE_SIGMOID) || !std::isfinite(router->scale) ||
      activation < QX_ACTIVATION_NONE || activation > QX_ACTIVATION_RELU2 || !kv::on_boundary(chosen) || !kv::on_boundary(weights)) {
    return QX_STATUS_INVALID_ARGUMENT;
  }
  QX_TRY(kv::check_rows(x, tokens, m->dim, false));
  QX_TRY(kv::check_rows(out, tokens, m->dim, true));
  if (tokens > 0 && x->data == out->data && (x->type != out->type || (tokens > 1 && x->stride != out->stride))) {
    return QX_STATUS_INVALID_ARGUMENT;  // (the inputs' place, but another view)
  }
  return QX_STATUS_OK;
}

// Scratch behind the workspace's arrival counters.
struct Layout {
  size_t total = kWorkspaceCounterBytes;
  size_t take(size_t bytes) {
    const size_t at = total;
    total = align_up(total + bytes, 256);
    return at;
  }
};

template <int kX, int kW>
qx_status launch_router(const Params& p, cudaStream_t stream) {
  static SmemOptIn opt_in;
  QX_TRY(opt_in.ensure(moe_router_kernel<kX, kW>, kPartBytes + kRouterTokens * kMostExperts * key_bytes(true)));
  int size = 1;
  while (size < kRouterCluster && size * kRouterExperts < p.experts) size *= 2;
  const int convert = (p.tokens * ((p.dim + 127) / 128) + kRouterWarps - 1) / kRouterWarps;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(((p.tokens + kRouterTokens - 1) / kRouterTokens + (convert + size - 1) / size) * size);
  config.blockDim = dim3(kRouterThreads);
  config.dynamicSmemBytes = kPartBytes + static_cast<size_t>(kRouterTokens) * p.experts * key_bytes(p.bias != nullptr);
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = size;
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  config.attrs = attributes;
  config.numAttrs = 2;
  QX_CUDA_TRY(cudaLaunchKernelEx(&config, moe_router_kernel<kX, kW>, p));
  count_launch();
  return QX_STATUS_OK;
}

template <int kX>
qx_status launch_router(const Params& p, cudaStream_t stream) {
  switch (p.router_type) {
    case QX_STORAGE_F32: return launch_router<kX, QX_STORAGE_F32>(p, stream);
    case QX_STORAGE_F16: return launch_router<kX, QX_STORAGE_F16>(p, stream);
    default: return launch_router<kX, QX_STORAGE_BF16>(p, stream);
  }
}

template <int kFormat, int kDigits>
qx_status launch_experts(const Params& p, long long grid, cudaStream_t stream) {
  static SmemOptIn opt_in;
  constexpr int bytes = ExpertShape<kFormat>::kBytes;
  static_assert(2 * (bytes + 1024) <= 228 * 1024, "two CTAs share an SM");
  QX_TRY(opt_in.ensure(moe_experts_kernel<kFormat, kDigits>, bytes));
  return kv::launch_behind(moe_experts_kernel<kFormat, kDigits>, grid, kExpertThreads, bytes, stream, p);
}

qx_status launch_apply(const qx_moe* m, const qx_moe_router* router, const qx_rows* x, const qx_rows* out, long long tokens,
                       int activation, int32_t* chosen, float* weights, DeviceContext* ctx, qx_workspace* workspace,
                       cudaStream_t stream) {
  if (tokens == 0) return QX_STATUS_OK;
  const size_t x_size = kv::type_bytes(x->type), out_size = kv::type_bytes(out->type);
  const auto whole = [](const void* data, size_t row_bytes) { return reinterpret_cast<uintptr_t>(data) % 16 == 0 && row_bytes % 16 == 0; };
  Params p{};
  p.up = m->up;
  p.down = m->down;
  p.experts = m->experts;
  p.shared = m->shared;
  p.dim = m->dim;
  p.inner = m->inner;
  p.router = static_cast<const uint8_t*>(router->weights);
  p.router_type = router->type;
  p.router_vector = whole(router->weights, 0);
  p.bias = router->bias;
  p.top = router->top;
  p.score = router->score;
  p.normalise = router->normalise != 0;
  p.scale = router->scale;
  p.x_type = x->type;
  p.x_vector = whole(x->data, x->stride * x_size);
  p.x_stride = x->stride;
  p.out_type = out->type;
  p.out_stride = out->stride;
  p.activation = activation;
  p.digits = x->type == QX_STORAGE_F32 ? 3 : 2;
  p.error = ctx->error_dev;

  const long long pass = std::min<long long>(tokens, std::min(kPassTokens, kPassEntries / (p.top + p.shared)));
  const size_t entries = static_cast<size_t>(pass) * (p.top + p.shared);
  Layout l;
  const size_t at_x = l.take(pass * p.digits * p.dim), at_x_scales = l.take(pass * scales_of(p.dim) * sizeof(float));
  const size_t at_picks = l.take(entries * sizeof(int)), at_weights = l.take(entries * sizeof(float));
  const size_t at_progress = l.take(sizeof(Progress)), at_done = l.take(entries * sizeof(int));
  const size_t at_inner = l.take(entries * p.digits * p.inner);
  const size_t at_inner_scales = l.take(entries * scales_of(p.inner) * sizeof(float));
  const size_t at_products = l.take(entries * p.dim * sizeof(float));
  QX_TRY(workspace->reserve(l.total));
  uint8_t* const base = static_cast<uint8_t*>(workspace->base);
  p.x_digits = reinterpret_cast<int8_t*>(base + at_x);
  p.x_scales = reinterpret_cast<float*>(base + at_x_scales);
  p.picks = reinterpret_cast<int*>(base + at_picks);
  p.weights = reinterpret_cast<float*>(base + at_weights);
  p.progress = reinterpret_cast<Progress*>(base + at_progress);
  p.up_done = reinterpret_cast<int*>(base + at_done);
  p.inner_digits = reinterpret_cast<int8_t*>(base + at_inner);
  p.inner_scales = reinterpret_cast<float*>(base + at_inner_scales);
  p.products = reinterpret_cast<float*>(base + at_products);

  for (long long t0 = 0; t0 < tokens; t0 += pass) {
    p.tokens = static_cast<int>(std::min(pass, tokens - t0));
    p.x = static_cast<const uint8_t*>(x->data) + t0 * x->stride * x_size;
    p.out = static_cast<uint8_t*>(out->data) + t0 * out->stride * out_size;
    p.chosen = chosen == nullptr ? nullptr : chosen + t0 * p.top;
    p.chosen_weights = weights == nullptr ? nullptr : weights + t0 * p.top;
    QX_TRY(p.x_type == QX_STORAGE_F32   ? launch_router<QX_STORAGE_F32>(p, stream)
           : p.x_type == QX_STORAGE_F16 ? launch_router<QX_STORAGE_F16>(p, stream)
                                        : launch_router<QX_STORAGE_BF16>(p, stream));
    const long long grid = std::min(2LL * ctx->prop.multiProcessorCount, pass_blocks(p.tokens, p.top + p.shared, p.dim, p.inner));
    if (m->format == QX_FORMAT_Q4_0) {
      QX_TRY(p.digits == 2 ? (launch_experts<QX_FORMAT_Q4_0, 2>(p, grid, stream)) : (launch_experts<QX_FORMAT_Q4_0, 3>(p, grid, stream)));
    } else {
      QX_TRY(p.digits == 2 ? (launch_experts<QX_FORMAT_Q8_0, 2>(p, grid, stream)) : (launch_experts<QX_FORMAT_Q8_0, 3>(p, grid, stream)));
    }
  }
  return QX_STATUS_OK;
}

}  // namespace
}  // namespace moe
}  // namespace qx

using namespace qx;

extern "C" {

qx_status qx_moe_prepare(int format, const void* gate, const void* up, const void* down, int experts, int shared, long long dim,
                         long long inner, qx_moe** out) {
  QX_TRY(moe::check_prepare(format, gate, up, down, experts, shared, dim, inner, out));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  std::lock_guard<std::mutex> lock(ctx->mutex);
  return moe::prepare(format, static_cast<const uint8_t*>(gate), static_cast<const uint8_t*>(up), static_cast<const uint8_t*>(down),
                      experts, shared, static_cast<int>(dim), static_cast<int>(inner), true, ctx, ctx->stream, out);
}

qx_status qx_moe_prepare_dev(int format, const void* gate_dev, const void* up_dev, const void* down_dev, int experts, int shared,
                             long long dim, long long inner, void* stream, qx_moe** out) {
  QX_TRY(moe::check_prepare(format, gate_dev, up_dev, down_dev, experts, shared, dim, inner, out));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  return moe::prepare(format, static_cast<const uint8_t*>(gate_dev), static_cast<const uint8_t*>(up_dev),
                      static_cast<const uint8_t*>(down_dev), experts, shared, static_cast<int>(dim), static_cast<int>(inner), false,
                      ctx, static_cast<cudaStream_t>(stream), out);
}

void qx_moe_destroy(qx_moe* moe) {
  if (moe == nullptr) return;
  if (moe->up != nullptr) (void)cudaFree(moe->up);
  if (moe->down != nullptr) (void)cudaFree(moe->down);
  delete moe;
}

qx_status qx_moe_apply_dev(const qx_moe* moe, const qx_moe_router* router, const qx_rows* x, const qx_rows* out, long long tokens,
                           int activation, int32_t* chosen_dev, float* weights_dev, qx_workspace* workspace, void* stream) {
  QX_TRY(moe::check_apply(moe, router, x, out, tokens, activation, chosen_dev, weights_dev));
  DeviceContext* ctx = nullptr;
  QX_TRY(current_context(&ctx));
  if (workspace == nullptr) workspace = &ctx->workspace;
  if (workspace->device != ctx->device || moe->device != ctx->device) return QX_STATUS_INVALID_ARGUMENT;
  return moe::launch_apply(moe, router, x, out, tokens, activation, chosen_dev, weights_dev, ctx, workspace,
                           static_cast<cudaStream_t>(stream));
}

qx_status qx_moe_apply(const qx_moe* moe, const qx_moe_router* router, const qx_rows* x, const qx_rows* out, long long tokens,
                       int activation, int32_t* chosen, float* weights) {
  QX_TRY(moe::check_apply(moe, router, x, out, tokens, activation, chosen, weights));
  return kv::guarded([&]() -> qx_status {
    DeviceContext* ctx = nullptr;
    QX_TRY(current_context(&ctx));
    if (moe->device != ctx->device) return QX_STATUS_INVALID_ARGUMENT;
    if (tokens == 0) return QX_STATUS_OK;
    std::lock_guard<std::mutex> lock(ctx->mutex);
    kv::Arrays a;
    const int from = a.add(x->data, kv::runs_of(x, tokens, moe->dim), x->data == out->data);
    const int to = x->data == out->data ? from : a.add(out->data, kv::runs_of(out, tokens, moe->dim), true);
    const int rows = a.add(router->weights, static_cast<size_t>(moe->experts) * moe->dim * kv::type_bytes(router->type), false);
    const int bias = router->bias == nullptr ? -1 : a.add(router->bias, moe->experts * sizeof(float), false);
    const size_t picks = static_cast<size_t>(tokens) * router->top;
    const int ids = chosen == nullptr ? -1 : a.add(chosen, picks * sizeof(int32_t), true);
    const int shares = weights == nullptr ? -1 : a.add(weights, picks * sizeof(float), true);
    QX_TRY(a.to_device(ctx));
    qx_rows dx = *x, dout = *out;
    qx_moe_router r = *router;
    dx.data = a.device<void>(from);
    dout.data = a.device<void>(to);
    r.weights = a.device<void>(rows);
    r.bias = a.device<float>(bias);
    QX_TRY(moe::launch_apply(moe, &r, &dx, &dout, tokens, activation, a.device<int32_t>(ids), a.device<float>(shares), ctx,
                             &ctx->workspace, ctx->stream));
    return a.from_device();
  });
}

}  // extern "C"
