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
constexpr int kTreeWords = 64;  // 64-bit words of a row of drafts

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

// Scratch of the managing calls: a header, then arrays sized by the cache.
struct Plan {
  int ok;         // the call is made
  uint32_t need;  // pages taken (reserve)
  uint32_t copies;  // pages copied (reserve) or moved (compact)
  int handed;     // tables, lengths and refs hold the pages taken (reserve)
};
struct Work {
  Plan* plan;
  uint32_t* free_ids;  // [n_pages] pages taken, in order (reserve); new id of each page (compact)
  uint32_t* uses;      // [n_pages] listed lanes whose last page this is (reserve)
  uint32_t* last;      // [n_pages] the last of them
  uint32_t* base;      // [n_lanes] first of a listed lane's places in free_ids
  uint32_t* had;       // [n_lanes] its tokens before the call
  uint32_t* grown;     // [n_lanes] and after it
  uint32_t* copy_lane;  // [n_lanes] list places whose last page is copied
  uint32_t* copy_from;  // [n_lanes] ... and that page
  uint32_t* from;      // [n_pages] pages moved (compact)
};

inline uint64_t up16(uint64_t x) { return (x + 15) & ~15ull; }

inline Work split_work(void* w, int n_pages, int n_lanes) {
  uint8_t* p = static_cast<uint8_t*>(w);
  const uint64_t pg = up16((uint64_t)n_pages * 4), ln = up16((uint64_t)n_lanes * 4);
  Work r;
  r.plan = reinterpret_cast<Plan*>(p), p += 64;
  r.free_ids = reinterpret_cast<uint32_t*>(p), p += pg;
  r.uses = reinterpret_cast<uint32_t*>(p), p += pg;
  r.last = reinterpret_cast<uint32_t*>(p), p += pg;
  r.from = r.uses;
  r.base = reinterpret_cast<uint32_t*>(p), p += ln;
  r.had = reinterpret_cast<uint32_t*>(p), p += ln;
  r.grown = reinterpret_cast<uint32_t*>(p), p += ln;
  r.copy_lane = reinterpret_cast<uint32_t*>(p), p += ln;
  r.copy_from = reinterpret_cast<uint32_t*>(p);
  return r;
}

__device__ inline int pages_of(int tokens) { return (tokens + kPageTokens - 1) / kPageTokens; }

// Names each lane of the list in an LDS bitmap (n_lanes bits); false where one
// is out of range or named twice.  The caller clears the bitmap first.
__device__ inline bool name_lane(uint32_t* bits, int lane, int n_lanes) {
  if (lane < 0 || lane >= n_lanes) return false;
  return !(atomicOr(&bits[lane >> 5], 1u << (lane & 31)) >> (lane & 31) & 1u);
}

// A workgroup takes the pages behind `kept` of its `held` tokens from a lane.
__device__ inline void drop_pages(const PageView& v, int lane, int held, int kept) {
  uint32_t* row = v.table + (uint64_t)lane * v.max_pages;
  for (int e = pages_of(kept) + threadIdx.x; e < pages_of(held); e += blockDim.x) {
    const uint32_t id = row[e];
    row[e] = kNone;
    if (id >= (uint32_t)v.n_pages) {
      set_error(v.error, FERRY_ESTATE);
    } else if ((int)atomicSub(&v.refs[id], 1u) <= 0) {  // counted as free: it stays so
      atomicAdd(&v.refs[id], 1u);
      set_error(v.error, FERRY_ESTATE);
    }
  }
}

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
// The common start of the managing calls.
int manage(const ferry_pages* p, int n, PageView* v, Work* w);
// A list of n values that a managing call reads (or writes): device memory apart from what
// the call changes, since its workgroups read the list while others already change that.
// of_len: the call has read the list before it changes len.
int check_list(const ferry_pages* p, const void* list, const char* name, int n, bool of_len = false);
// CUs of a GPU (read once per GPU).
int gpu_cus(int device);

}  // namespace ferry_amd
