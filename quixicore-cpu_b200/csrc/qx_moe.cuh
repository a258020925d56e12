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

// Limits of a layer, and of one pass over it.
constexpr int kMostExperts = 512, kMostShared = 32, kMostTop = 32, kMostWidth = 65536;
constexpr int kPassTokens = 128;

// Weights lie as tiles of 16 rows; a tile is a row of records, one per 32 columns: the codes as a warp's lanes take
// them (lane (g, t): columns 8 t .. 8 t + 7 of rows g and g + 8), then {d of row g, d of row g + 8} as f16 pairs. A tile
// of the first matrix is 8 rows of the gate and the same 8 of the up projection.
constexpr int kTileRows = 16;
constexpr int record_bytes(int format) { return (format == QX_FORMAT_Q4_0 ? 256 : 512) + 32; }

// Activations lie as slabs of four blocks of 32 columns: 4 x 32 f16 values, then their four f32 scales.
constexpr int kSlabBlocks = 4, kSlabBytes = kSlabBlocks * (64 + 4);
inline __host__ __device__ int slabs_of(int columns) { return (columns / 32 + kSlabBlocks - 1) / kSlabBlocks; }

// Columns of a product (tokens of one expert, times the terms of an activation) that one unit of work takes.
constexpr int kColumns = 16;

struct Group {
  int expert, first, count;  // entries list[first .. first + count - 1]
};
// What the router leaves for the experts' kernel: `groups`, and how often each place has been counted.
struct Plan {
  int groups, ticket, down_done, unused;
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
  int out_type, out_vector;
  long long out_stride;
  int tokens, activation, terms;
  int32_t* chosen;       // [token][top], may be NULL
  float* chosen_weights;
  // scratch
  int* arrivals;         // zero between calls: one per eight tokens, one for all
  uint8_t* x_terms;      // [token][term][slab]
  double* logits;        // [token][expert]
  int* picks;            // [token][top + shared] experts
  float* weights;        // [token][top + shared]
  Plan* plan;
  int* up_done;          // [group]
  Group* groups;
  int* list;             // entries (token * (top + shared) + place), by expert, ascending
  uint8_t* inner_terms;  // [entry][term][slab]
  float* products;       // [entry][dim]
  int* error;
};

}  // namespace moe
}  // namespace qx
