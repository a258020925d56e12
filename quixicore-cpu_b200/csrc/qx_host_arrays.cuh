// What the host-pointer entry points share: host arrays on their way to the device and back, and the end of
// exceptions.
#pragma once

#include <algorithm>
#include <cstring>
#include <new>
#include <stdexcept>
#include <vector>

#include "qx_kv.cuh"

namespace qx {
namespace kv {

// Where the elements of a view lie in memory: `rows` x `heads` runs of `bytes`, strides in bytes.
struct Runs {
  long long rows, heads;
  size_t row_stride, head_stride, bytes;
  size_t extent() const {
    return rows <= 0 ? 0 : (rows - 1) * row_stride + (heads - 1) * head_stride + bytes;
  }
  bool gapless() const { return extent() == static_cast<size_t>(rows) * heads * bytes; }
};
inline Runs runs_of(const qx_rows* view, long long tokens, long long dim) {
  const size_t size = type_bytes(view->type);
  return {tokens, 1, view->stride * size, 0, dim * size};
}
// Host arrays that a call uses, laid out one behind the other in the context's staging memory. What comes back is
// the elements of the views that are written, run by run: between them may lie another view's, or what is none of
// the call's business.
class Arrays {
 public:
  // Returns the array's number. `out`: it is copied back.
  int add(const void* host, size_t bytes, bool out) { return add(host, Runs{1, 1, 0, 0, bytes}, out); }
  int add(const void* host, const Runs& runs, bool out) {
    items_.push_back({const_cast<void*>(host), runs, runs.extent(), total_, out, {}});
    total_ += align_up(std::max<size_t>(items_.back().bytes, 1), 256);
    return static_cast<int>(items_.size()) - 1;
  }
  qx_status to_device(DeviceContext* ctx) {
    ctx_ = ctx;
    QX_TRY(ctx->ensure_staging(total_));
    for (const Item& i : items_) {
      if (i.bytes == 0) continue;
      QX_CUDA_TRY(cudaMemcpyAsync(at(i), i.host, i.bytes, cudaMemcpyHostToDevice, ctx->stream));
    }
    return QX_STATUS_OK;
  }
  // Waits for the stream, and for what the kernels reported.
  qx_status from_device() {
    for (Item& i : items_) {
      if (!i.out || i.bytes == 0) continue;
      void* to = i.host;
      if (!i.runs.gapless()) {
        i.back.resize(i.bytes);
        to = i.back.data();
      }
      QX_CUDA_TRY(cudaMemcpyAsync(to, at(i), i.bytes, cudaMemcpyDeviceToHost, ctx_->stream));
    }
    QX_TRY(finish_host_call(ctx_));
    for (const Item& i : items_) {
      if (i.back.empty()) continue;
      for (long long r = 0; r < i.runs.rows; ++r) {
        for (long long h = 0; h < i.runs.heads; ++h) {
          const size_t offset = r * i.runs.row_stride + h * i.runs.head_stride;
          std::memcpy(static_cast<uint8_t*>(i.host) + offset, i.back.data() + offset, i.runs.bytes);
        }
      }
    }
    return QX_STATUS_OK;
  }
  template <class T>
  T* device(int number) const {
    return number < 0 ? nullptr : reinterpret_cast<T*>(at(items_[number]));
  }

 private:
  struct Item {
    void* host;
    Runs runs;
    size_t bytes, offset;
    bool out;
    std::vector<uint8_t> back;
  };
  uint8_t* at(const Item& i) const { return static_cast<uint8_t*>(ctx_->staging) + i.offset; }
  std::vector<Item> items_;
  size_t total_ = 0;
  DeviceContext* ctx_ = nullptr;
};

// No exception leaves an entry point.
template <class Call>
qx_status guarded(Call call) {
  try {
    return call();
  } catch (const std::bad_alloc&) {
    return QX_STATUS_OUT_OF_MEMORY;
  } catch (const std::length_error&) {
    return QX_STATUS_OUT_OF_MEMORY;
  }
}

}  // namespace kv
}  // namespace qx
