// Host-pointer forms of the rotary, cache and attention entry points: everything is checked on the host
// (the contents of the batch too, which the device forms can only report), the blocks that the batch
// names travel to the device packed together, the kernels are those of the device forms.

#include <algorithm>
#include <limits>
#include <vector>

#include "qx_attention.cuh"
#include "qx_host_arrays.cuh"

namespace qx {
namespace kv {

qx_status check_append(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                       const qx_rope* rope, const int64_t* positions, const qx_heads* q, const qx_heads* q_out);
qx_status check_read(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v);
qx_status check_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                          const float* lse, float scale, long long window);
qx_status launch_append(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                        const qx_rope* rope, const int64_t* positions, const qx_heads* q, const qx_heads* q_out,
                        DeviceContext* ctx, cudaStream_t stream);
qx_status launch_read(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                      DeviceContext* ctx, cudaStream_t stream);
qx_status launch_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                           float* lse, float scale, int causal, long long window, const uint64_t* tree, DeviceContext* ctx,
                           qx_workspace* workspace, cudaStream_t stream);
qx_status check_tree_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                               const float* lse, float scale, long long window, const uint64_t* seen);

namespace {

Runs runs_of(const qx_heads* view, long long rows, int dim) {
  const size_t size = type_bytes(view->type);
  return {rows, view->heads, view->token_stride * size, view->head_stride * size, dim * size};
}

int add_view(Arrays* a, const qx_heads* view, long long rows, int dim, bool out) {
  return view == nullptr ? -1 : a->add(view->data, runs_of(view, rows, dim), out);
}
qx_heads on_device(const Arrays& a, const qx_heads* view, int number) {
  qx_heads v = *view;
  v.data = a.device<void>(number);
  return v;
}

// The batch as the device gets it: the blocks that its sequences use, numbered in the order of their first
// use, and tables of those numbers.
struct Packed {
  std::vector<int32_t> begin, lengths, table, blocks;
  std::vector<int8_t> k_codes, v_codes;
  std::vector<float> k_scales, v_scales;
  long long width = 0;
  size_t block_codes = 0;
};

// Checks what the arrays say. `append`: blocks that new tokens reach belong to one sequence, and once.
qx_status pack(const qx_kv_cache* cache, const qx_kv_batch* batch, bool rows_are_cached, bool append, Packed* out) {
  const int size = cache->block_tokens;
  const size_t heads = cache->kv_heads;
  std::vector<int32_t> number(static_cast<size_t>(cache->blocks), -1);
  std::vector<int32_t> users(append ? static_cast<size_t>(cache->blocks) : 0, 0);
  std::vector<uint8_t> written(append ? static_cast<size_t>(cache->blocks) : 0, 0);
  for (int s = 0; s < batch->sequences; ++s) {
    const int length = batch->lengths[s];
    if (length < 0 || length > batch->max_length) return QX_STATUS_INVALID_ARGUMENT;
    out->width = std::max<long long>(out->width, (length + size - 1LL) / size);
  }
  long long before = 0;
  for (int s = 0; s < batch->sequences; ++s) {
    const long long row = batch->token_begin != nullptr ? batch->token_begin[s] : 1LL * s * batch->max_tokens;
    const long long next = batch->token_begin != nullptr ? batch->token_begin[s + 1] : row + batch->max_tokens;
    const long long n = next - row;
    const int length = batch->lengths[s];
    if (row < before || n < 0 || n > batch->max_tokens || next > batch->tokens || (rows_are_cached && n > length)) {
      return QX_STATUS_INVALID_ARGUMENT;
    }
    if (next > std::numeric_limits<int32_t>::max()) return QX_STATUS_INVALID_SHAPE;  // (the packed batch counts in 32 bits)
    before = next;
    out->begin.push_back(static_cast<int32_t>(row));
    out->lengths.push_back(length);
    for (long long i = 0; i < out->width; ++i) {
      int32_t local = 0;
      if (i * size < length) {
        const int32_t block = batch->block_table[s * batch->table_stride + i];
        if (block < 0 || block >= cache->blocks) return QX_STATUS_INVALID_ARGUMENT;
        if (number[block] < 0) {
          number[block] = static_cast<int32_t>(out->blocks.size());
          out->blocks.push_back(block);
        }
        local = number[block];
        if (append) {
          ++users[block];
          if (n > 0 && (i + 1) * size > length - n) written[block] = 1;
        }
      }
      out->table.push_back(local);
    }
  }
  out->begin.push_back(static_cast<int32_t>(before));
  for (size_t b = 0; b < written.size(); ++b) {
    if (written[b] && users[b] > 1) return QX_STATUS_INVALID_ARGUMENT;
  }
  out->block_codes = heads * size * cache->head_dim;
  const size_t count = out->blocks.size();
  out->k_codes.resize(count * out->block_codes);
  out->v_codes.resize(count * out->block_codes);
  out->k_scales.resize(count * heads);
  out->v_scales.resize(count * heads);
  for (size_t i = 0; i < count; ++i) {
    const size_t b = static_cast<size_t>(out->blocks[i]);
    std::copy_n(cache->k_codes + b * out->block_codes, out->block_codes, out->k_codes.begin() + i * out->block_codes);
    std::copy_n(cache->v_codes + b * out->block_codes, out->block_codes, out->v_codes.begin() + i * out->block_codes);
    std::copy_n(cache->k_scales + b * heads, heads, out->k_scales.begin() + i * heads);
    std::copy_n(cache->v_scales + b * heads, heads, out->v_scales.begin() + i * heads);
  }
  return QX_STATUS_OK;
}
void unpack(const qx_kv_cache* cache, const Packed& in) {
  const size_t heads = cache->kv_heads;
  for (size_t i = 0; i < in.blocks.size(); ++i) {
    const size_t b = static_cast<size_t>(in.blocks[i]);
    std::copy_n(in.k_codes.begin() + i * in.block_codes, in.block_codes, cache->k_codes + b * in.block_codes);
    std::copy_n(in.v_codes.begin() + i * in.block_codes, in.block_codes, cache->v_codes + b * in.block_codes);
    std::copy_n(in.k_scales.begin() + i * heads, heads, cache->k_scales + b * heads);
    std::copy_n(in.v_scales.begin() + i * heads, heads, cache->v_scales + b * heads);
  }
}

struct PackedArrays {
  int begin, lengths, table, k_codes, v_codes, k_scales, v_scales;
  void add(Arrays* a, const Packed& p, bool written) {
    begin = a->add(p.begin.data(), p.begin.size() * 4, false);
    lengths = a->add(p.lengths.data(), p.lengths.size() * 4, false);
    table = a->add(p.table.data(), p.table.size() * 4, false);
    k_codes = a->add(p.k_codes.data(), p.k_codes.size(), written);
    v_codes = a->add(p.v_codes.data(), p.v_codes.size(), written);
    k_scales = a->add(p.k_scales.data(), p.k_scales.size() * 4, written);
    v_scales = a->add(p.v_scales.data(), p.v_scales.size() * 4, written);
  }
  qx_kv_cache cache(const Arrays& a, const qx_kv_cache* host, const Packed& p) const {
    qx_kv_cache c = *host;
    c.k_codes = a.device<int8_t>(k_codes);
    c.v_codes = a.device<int8_t>(v_codes);
    c.k_scales = a.device<float>(k_scales);
    c.v_scales = a.device<float>(v_scales);
    c.blocks = std::max<long long>(1, static_cast<long long>(p.blocks.size()));
    return c;
  }
  qx_kv_batch batch(const Arrays& a, const qx_kv_batch* host, const Packed& p) const {
    qx_kv_batch b = *host;
    b.token_begin = a.device<int32_t>(begin);
    b.lengths = a.device<int32_t>(lengths);
    b.block_table = a.device<int32_t>(table);
    b.table_stride = p.width;
    int longest = 0;
    for (int32_t v : p.lengths) longest = std::max(longest, v);
    b.max_length = longest;
    return b;
  }
};

}  // namespace
}  // namespace kv
}  // namespace qx

using namespace qx;
using namespace qx::kv;

// `seen`: masks of drafts, or NULL.
static qx_status attention_of(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out, float* lse,
                              float scale, int causal, long long window, const uint64_t* seen) {
  return guarded([&]() -> qx_status {
    Packed p;
    QX_TRY(pack(cache, batch, false, false, &p));
    DeviceContext* ctx = nullptr;
    QX_TRY(current_context(&ctx));
    std::lock_guard<std::mutex> lock(ctx->mutex);
    Arrays a;
    PackedArrays pa;
    pa.add(&a, p, false);
    const int aq = add_view(&a, q, batch->tokens, cache->head_dim, false);
    const int ao = add_view(&a, out, batch->tokens, cache->head_dim, true);
    const int al = lse == nullptr ? -1 : a.add(lse, static_cast<size_t>(batch->tokens) * q->heads * 4, true);
    const int at = seen == nullptr ? -1 : a.add(seen, static_cast<size_t>(batch->tokens) * sizeof(uint64_t), false);
    QX_TRY(a.to_device(ctx));
    const qx_kv_cache dc = pa.cache(a, cache, p);
    const qx_kv_batch db = pa.batch(a, batch, p);
    const qx_heads dq = on_device(a, q, aq), dout = on_device(a, out, ao);
    QX_TRY(launch_attention(&dc, &db, &dq, &dout, a.device<float>(al), scale, causal, window, a.device<uint64_t>(at), ctx,
                            &ctx->workspace, ctx->stream));
    return a.from_device();
  });
}

extern "C" {

qx_status qx_rope_apply(const qx_rope* rope, const qx_heads* x, const qx_heads* y, const int64_t* positions,
                        long long tokens, int head_dim, int inverse) {
  QX_TRY(check_rope_call(rope, x, y, positions, tokens, head_dim));
  return guarded([&]() -> qx_status {
    DeviceContext* ctx = nullptr;
    QX_TRY(current_context(&ctx));
    if (tokens == 0) return QX_STATUS_OK;
    std::lock_guard<std::mutex> lock(ctx->mutex);
    Arrays a;
    const int from = add_view(&a, x, tokens, head_dim, x->data == y->data);
    const int to = x->data == y->data ? from : add_view(&a, y, tokens, head_dim, true);
    const int at = a.add(positions, static_cast<size_t>(tokens) * 8, false);
    QX_TRY(a.to_device(ctx));
    const qx_heads dx = on_device(a, x, from), dy = on_device(a, y, to);
    QX_TRY(qx_rope_apply_dev(rope, &dx, &dy, a.device<int64_t>(at), tokens, head_dim, inverse, ctx->stream));
    return a.from_device();
  });
}

qx_status qx_kv_append(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v,
                       const qx_rope* rope, const int64_t* positions, const qx_heads* q, const qx_heads* q_out) {
  QX_TRY(check_append(cache, batch, k, v, rope, positions, q, q_out));
  return guarded([&]() -> qx_status {
    Packed p;
    QX_TRY(pack(cache, batch, true, true, &p));
    DeviceContext* ctx = nullptr;
    QX_TRY(current_context(&ctx));
    std::lock_guard<std::mutex> lock(ctx->mutex);
    const int dim = cache->head_dim;
    Arrays a;
    PackedArrays pa;
    pa.add(&a, p, true);
    const int ak = add_view(&a, k, batch->tokens, dim, false), av = add_view(&a, v, batch->tokens, dim, false);
    const bool in_place = q != nullptr && q->data == q_out->data;
    const int aq = add_view(&a, q, batch->tokens, dim, in_place);
    const int ao = in_place ? aq : add_view(&a, q_out, batch->tokens, dim, true);
    const int at = positions == nullptr ? -1 : a.add(positions, static_cast<size_t>(batch->tokens) * 8, false);
    QX_TRY(a.to_device(ctx));
    const qx_kv_cache dc = pa.cache(a, cache, p);
    const qx_kv_batch db = pa.batch(a, batch, p);
    const qx_heads dk = on_device(a, k, ak), dv = on_device(a, v, av);
    qx_heads dq{}, dout{};
    if (q != nullptr) {
      dq = on_device(a, q, aq);
      dout = on_device(a, q_out, ao);
    }
    QX_TRY(launch_append(&dc, &db, &dk, &dv, rope, a.device<int64_t>(at), q == nullptr ? nullptr : &dq,
                         q == nullptr ? nullptr : &dout, ctx, ctx->stream));
    QX_TRY(a.from_device());
    unpack(cache, p);
    return QX_STATUS_OK;
  });
}

qx_status qx_kv_read(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* k, const qx_heads* v) {
  QX_TRY(check_read(cache, batch, k, v));
  return guarded([&]() -> qx_status {
    Packed p;
    QX_TRY(pack(cache, batch, true, false, &p));
    DeviceContext* ctx = nullptr;
    QX_TRY(current_context(&ctx));
    std::lock_guard<std::mutex> lock(ctx->mutex);
    Arrays a;
    PackedArrays pa;
    pa.add(&a, p, false);
    const int ak = add_view(&a, k, batch->tokens, cache->head_dim, true);
    const int av = add_view(&a, v, batch->tokens, cache->head_dim, true);
    QX_TRY(a.to_device(ctx));
    const qx_kv_cache dc = pa.cache(a, cache, p);
    const qx_kv_batch db = pa.batch(a, batch, p);
    qx_heads dk{}, dv{};
    if (k != nullptr) dk = on_device(a, k, ak);
    if (v != nullptr) dv = on_device(a, v, av);
    QX_TRY(launch_read(&dc, &db, k == nullptr ? nullptr : &dk, v == nullptr ? nullptr : &dv, ctx, ctx->stream));
    return a.from_device();
  });
}

qx_status qx_kv_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                          float* lse, float scale, int causal, long long window) {
  QX_TRY(check_attention(cache, batch, q, out, lse, scale, window));
  return attention_of(cache, batch, q, out, lse, scale, causal, window, nullptr);
}

qx_status qx_kv_tree_attention(const qx_kv_cache* cache, const qx_kv_batch* batch, const qx_heads* q, const qx_heads* out,
                               float* lse, float scale, long long window, const uint64_t* seen) {
  QX_TRY(check_tree_attention(cache, batch, q, out, lse, scale, window, seen));
  return attention_of(cache, batch, q, out, lse, scale, 1, window, seen);
}

}  // extern "C"
