// pages.hpp -- the paged KV cache as its kernels see it, and the checks its
// entry points share (pages.hip, pages_attn.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <initializer_list>
#include <string>
#include <utility>

#include "common.hpp"
#include "errors.hpp"

namespace ferry_amd {

constexpr int kPageTokens = 16;
constexpr int kPageDim = 128;
constexpr int kMaxLanes = 65536;
constexpr int kMaxLanePages = 1 << 20;

// Caller-owned buffers of one cache (ferry_pages), passed to kernels by value.
struct PageView {
  int L, H, n_pages, n_lanes, max_pages;
  uint32_t bb;  // bytes of one record (K and V)
  uint8_t* pool;
  float* scales;
  uint32_t* table;
  int32_t* len;
  uint32_t* refs;
  int* error;
  __host__ __device__ uint64_t record(int layer, uint32_t page, int head) const {
    return ((uint64_t)layer * n_pages + page) * H + head;
  }
};

// The calling thread's GPU is `device` for one entry point and its own again
// afterwards.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    if (hipGetDevice(&prev_) != hipSuccess) prev_ = -1;
    ok_ = prev_ == device || hipSetDevice(device) == hipSuccess;
    moved_ = ok_ && prev_ >= 0 && prev_ != device;
  }
  ~OnDevice() {
    if (moved_) (void)hipSetDevice(prev_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
  bool ok() const { return ok_; }

 private:
  int prev_ = -1;
  bool ok_ = false, moved_ = false;
};

// An entry point's body; nothing it throws reaches C.
template <class Body>
int entry(Body&& body) noexcept {
  try {
    return body();
  } catch (...) {
    return FERRY_ENOMEM;
  }
}

// A buffer a kernel reads or writes: memory HIP knows, and device memory of the
// cache's own GPU.
inline int check_on(const void* p, const char* name, int device) {
  if (!p) return report(FERRY_EINVAL, std::string("null ") + name);
  hipPointerAttribute_t a{};
  if (hipPointerGetAttributes(&a, p) != hipSuccess || a.type == hipMemoryTypeUnregistered) {
    (void)hipGetLastError();
    return report(FERRY_EINVAL, std::string(name) +
                                    " is not device-accessible memory (device, managed or pinned host)");
  }
  if (a.type == hipMemoryTypeDevice && a.device != device)
    return report(FERRY_EINVAL, std::string(name) + " is on GPU " + std::to_string(a.device) +
                                    ", the cache on " + std::to_string(device));
  return FERRY_OK;
}
inline int check_all(std::initializer_list<std::pair<const void*, const char*>> bufs, int device) {
  for (const auto& b : bufs)
    if (int rc = check_on(b.first, b.second, device)) return rc;
  return FERRY_OK;
}

inline int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return FERRY_OK;
  return report(FERRY_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}

// Geometry of a cache (no device call).
int page_geometry(const ferry_pages* p, PageView* out);
// ... and its buffers: pool, scales, table, len and error; refs where `manage`.
int page_buffers(const ferry_pages* p, bool manage);
// CUs of a GPU (read once per GPU).
int gpu_cus(int device);

}  // namespace ferry_amd
