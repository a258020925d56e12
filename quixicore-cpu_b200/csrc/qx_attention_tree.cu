// The streamed attention kernel for trees of drafts: rows whose masks say which drafts they see. A file of its own, which
// compiles beside the other.

#include "qx_attention_streamed.cuh"

namespace qx {
namespace kv {

qx_status launch_tree_streamed(const AttentionParams& p, int dp, bool wide, bool balanced, long long grid, cudaStream_t stream) {
  return launch_sized<true>(p, dp, wide, balanced, grid, stream);
}

}  // namespace kv
}  // namespace qx
