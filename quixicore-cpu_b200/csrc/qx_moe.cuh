// The mixture-of-experts layer: prepared experts, and what its kernels hand each other.
#pragma once

#include "qx_kv.cuh"

struct qx_moe {
  int device = -1;
  int format = 0, experts = 0, shared = 0;
  int dim = 0, inner = 0;
  uint8_t* up = nullptr;    // gate and up projections, interleaved
  uint8_t* down = nullptr;
  size_t up_bytes = 0, down_bytes = 0;
};

namespace qx {
namespace moe {

// Limits of a layer, and of one pass over it: tokens, and (token, expert) pairs.
constexpr int kMostExperts = 512, kMostShared = 32, kMostTop = 32, kMostWidth = 65536;
constexpr int kPassTokens = 128, kPassEntries = 1024;

// Weights lie as records of a tile of 16 rows and a block of 32 columns: the codes as a warp's lanes take them (lane
// (g, t): columns 8 t .. 8 t + 7 of rows g and g + 8, as they are operands of an MMA), then {d of row g, d of row g + 8} as f16 pairs. Four tiles of an expert
// (a unit of work; the last may have two) lie together, block by block, so that a stage of any number of blocks is one
// run of bytes. A tile of the first matrix is 8 rows of the gate and the same 8 of the up projection.
constexpr int kTileRows = 16, kUnitTiles = 4;
constexpr int record_bytes(int format) { return (format == QX_FORMAT_Q4_0 ? 256 : 512) + 32; }

// Activations lie as rows of 8-bit digits, a row per token and digit (the lowest first), and beside them, a row per token,
// an f32 scale per 32 of them. Rows of scales are whole 16-byte pieces.
inline __host__ __device__ int scales_of(int columns) { return (columns / 32 + 3) / 4 * 4; }
// Columns of an MMA that a token takes: two digits, or three and one to spare.
constexpr int columns_of(int digits) { return digits == 2 ? 2 : 4; }

// A unit of work takes 16 columns: eight tokens, or four.
constexpr int kColumns = 16;

// How far the units of a pass have come.
struct Progress {
  int ticket, down_done;
};

struct Params {
  // the layer
  const uint8_t* up;
  const uint8_t* down;
  int experts, shared, dim, inner;
  // the router
  const uint8_t* router;
  int router_type, router_vector;
  const float* bias;
  int top, score, normalise;
  float scale;
  // the tokens
  const uint8_t* x;
  int x_type, x_vector;
  long long x_stride;
  uint8_t* out;
  int out_type;
  long long out_stride;
  int tokens, activation, digits;
  int32_t* chosen;       // [token][top], may be NULL
  float* chosen_weights;
  // scratch
  int8_t* x_digits;      // [token][digit][dim]
  float* x_scales;
  int* picks;            // [token][top + shared] experts
  float* weights;        // [token][top + shared]
  Progress* progress;
  int* up_done;          // [group] units
  int8_t* inner_digits;  // [entry][digit][inner], entry = token * (top + shared) + place
  float* inner_scales;
  float* products;       // [entry][dim]
  int* error;
};

}  // namespace moe
}  // namespace qx
