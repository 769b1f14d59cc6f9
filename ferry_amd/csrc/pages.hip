// pages.hip -- the paged KV cache: managing pages (reserve, fork, trim,
// compact), rotary positions and the write of new tokens into pages.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <mutex>
#include <type_traits>

#include "attn_common.hpp"
#include "pages.hpp"

using namespace ferry_amd;

namespace ferry_amd {

int page_geometry(const ferry_pages* p, PageView* v) {
  if (!p) return report(FERRY_EINVAL, "null pages");
  if (p->dtype < FERRY_F32 || p->dtype > FERRY_FP8_E4M3)
    return report(FERRY_EINVAL, "unknown dtype");
  if (p->head_dim != kPageDim || p->block_tokens != kPageTokens)
    return report(FERRY_EINVAL, "head_dim must be 128 and block_tokens 16");
  if (p->n_layers < 1 || p->kv_heads < 1 || p->n_pages < 1 || p->n_lanes < 1 || p->max_pages < 1)
    return report(FERRY_EINVAL, "layers, kv heads, pages, lanes and pages per lane must be positive");
  if (p->n_lanes > kMaxLanes || p->max_pages > kMaxLanePages)
    return report(FERRY_EINVAL, "at most 65536 lanes of 2^20 pages");
  if (p->kv_heads > 4096 || p->n_layers > 65536) return report(FERRY_EINVAL, "at most 4096 kv heads, 65536 layers");
  const uint32_t es = p->dtype == FERRY_F32 ? 4 : p->dtype == FERRY_FP8_E4M3 ? 1 : 2;
  *v = PageView{p->n_layers, p->kv_heads, p->n_pages, p->n_lanes, p->max_pages,
                2u * kPageTokens * kPageDim * es,
                static_cast<uint8_t*>(p->pool), p->scales, p->table, p->len, p->refs, p->error};
  return FERRY_OK;
}

int page_buffers(const ferry_pages* p, bool manage) {
  if (int rc = check_all({{p->pool, "pool"}, {p->table, "table"}, {p->len, "len"}, {p->error, "error"}},
                         p->device))
    return rc;
  if (reinterpret_cast<uintptr_t>(p->pool) % 16)
    return report(FERRY_EINVAL, "pool must be 16-byte aligned");
  if (p->dtype == FERRY_FP8_E4M3) {
    if (int rc = check_on(p->scales, "scales", p->device)) return rc;
    if (reinterpret_cast<uintptr_t>(p->scales) % 8)
      return report(FERRY_EINVAL, "scales must be 8-byte aligned");
  } else if (p->scales) {
    return report(FERRY_EINVAL, "scales go with fp8 pages only");
  }
  if (manage) {
    if (int rc = check_all({{p->refs, "refs"}, {p->work, "work"}}, p->device)) return rc;
    uint64_t need = 0;
    if (int rc = ferry_pages_work_bytes(p, &need)) return rc;
    if (p->work_bytes < need) return report(FERRY_EINVAL, "work is smaller than ferry_pages_work_bytes");
    if (reinterpret_cast<uintptr_t>(p->work) % 16)
      return report(FERRY_EINVAL, "work must be 16-byte aligned");
  } else if (p->refs) {
    if (int rc = check_on(p->refs, "refs", p->device)) return rc;
  }
  return FERRY_OK;
}

int gpu_cus(int device) {
  static std::mutex mu;
  static int cus[64] = {};
  if (device < 0 || device >= 64) return 256;
  std::lock_guard<std::mutex> lk(mu);
  if (!cus[device]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n < 1) {
      (void)hipGetLastError();
      return 256;
    }
    cus[device] = n;
  }
  return cus[device];
}

}  // namespace ferry_amd

namespace {

constexpr int kPlan = 1024;  // threads of the one-workgroup kernels that plan a call
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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

uint64_t up16(uint64_t x) { return (x + 15) & ~15ull; }

Work split_work(void* w, int n_pages, int n_lanes) {
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

uint64_t work_bytes(int n_pages, int n_lanes) {
  return 64 + 3 * up16((uint64_t)n_pages * 4) + 5 * up16((uint64_t)n_lanes * 4);
}

__device__ inline int pages_of(int tokens) { return (tokens + kPageTokens - 1) / kPageTokens; }

// Exclusive prefix sum of x over the workgroup of kPlan threads; *total gets the sum.
__device__ inline uint64_t block_scan(uint64_t x, uint64_t* total) {
  __shared__ uint64_t part[kPlan / 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  uint64_t s = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t y = __shfl_up(s, d);
    if (lane >= d) s += y;
  }
  if (lane == 63) part[w] = s;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kPlan / 64; ++i) {
    if (i < w) before += part[i];
    all += part[i];
  }
  __syncthreads();
  *total = all;
  return before + s - x;
}

// Names each lane of the list in an LDS bitmap (n_lanes bits); false where one
// is out of range or named twice.  The caller clears the bitmap first.
__device__ inline bool name_lane(uint32_t* bits, int lane, int n_lanes) {
  if (lane < 0 || lane >= n_lanes) return false;
  return !(atomicOr(&bits[lane >> 5], 1u << (lane & 31)) >> (lane & 31) & 1u);
}

// ---- reserve -------------------------------------------------------------------
constexpr int kIdsInLds = 4096;  // pages that the plan hands out by itself
constexpr int kOwnPages = 64;    // ... of one lane

// The lowest `need` free ids (refs 0) into w.free_ids and the first of them into ids;
// returns how many there are.  first: refs of pages 4 tid .. 4 tid + 3.
__device__ inline uint64_t find_free(const PageView& v, const Work& w, uint64_t need, uint32_t* ids,
                                     const uint32_t (&first)[4]) {
  uint64_t got = 0;
  auto take = [&](int64_t p0, auto count, auto&& refs) {
    constexpr int N = decltype(count)::value;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += refs(i) == 0;
    uint64_t all, at = got + block_scan(n, &all);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (refs(i) == 0) {
        if (at < need) {
          w.free_ids[at] = (uint32_t)(p0 + i);
          if (at < kIdsInLds) ids[at] = (uint32_t)(p0 + i);
        }
        ++at;
      }
    got += all;
  };
  take(4ll * threadIdx.x, std::integral_constant<int, 4>{}, [&](int i) { return first[i]; });
  // the rest 16 to a thread, all of them on their way at once
  for (int64_t c = 4 * kPlan; c < v.n_pages && got < need; c += 16 * kPlan) {
    const int64_t p0 = c + 16ll * threadIdx.x;
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = p0 + i < v.n_pages ? v.refs[p0 + i] : 1u;
    take(p0, std::integral_constant<int, 16>{}, [&](int i) { return r[i]; });
  }
  return got;
}

// One workgroup decides the whole call: which last pages are copied, how many
// pages each listed lane takes, and which (the lowest free ids).  It is a chain of
// dependent reads: a lane's length, its last page, that page's refs, while the first
// refs are on their way.  SMALL: a thread per listed lane; the lanes of a shared
// page are then counted in LDS, else by atomics in the scratch.
template <bool SMALL>
__global__ __launch_bounds__(kPlan) void k_reserve_plan(PageView v, Work w, const int32_t* __restrict__ lanes,
                                                        const int32_t* tokens, int n) {
  __shared__ uint32_t bits[kMaxLanes / 32];
  __shared__ uint32_t ids[kIdsInLds];
  __shared__ uint32_t last_page[SMALL ? kPlan : 1];
  __shared__ int bad, longest;
  const int tid = threadIdx.x;
  uint32_t first[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) first[i] = 4 * tid + i < v.n_pages ? v.refs[4 * tid + i] : 1u;
  for (int i = tid; i < (v.n_lanes + 31) / 32; i += kPlan) bits[i] = 0;
  if (tid == 0) bad = longest = 0;
  __syncthreads();
  int my_lane = 0, my_had = 0, my_tokens = 0;  // SMALL: the thread's lane
  uint32_t my_page = kNone, my_refs = 0;
  for (int i = tid; i < n; i += kPlan) {
    const int lane = lanes[i], t = tokens[i];
    if (!name_lane(bits, lane, v.n_lanes) || t < 0) {
      atomicMin(&bad, FERRY_EINVAL);
    } else {
      const int had = v.len[lane];
      w.had[i] = had, w.grown[i] = (uint32_t)had + (uint32_t)t;
      my_lane = lane, my_had = had, my_tokens = t;
      if (had < 0 || (int64_t)had + t > (int64_t)v.max_pages * kPageTokens) {
        atomicMin(&bad, FERRY_ECAPACITY);
      } else if (had % kPageTokens) {
        const uint32_t page = v.table[(uint64_t)lane * v.max_pages + had / kPageTokens];
        if (page >= (uint32_t)v.n_pages) {
          atomicMin(&bad, FERRY_ESTATE);
        } else if constexpr (SMALL) {
          my_page = page, my_refs = v.refs[page];
        } else {
          atomicExch(&w.uses[page], 0u);
          atomicExch(&w.last[page], 0u);
        }
      }
    }
  }
  if constexpr (SMALL) last_page[tid] = my_page;
  __syncthreads();
  if (bad) {
    if (tid == 0) w.plan->ok = 0, set_error(v.error, bad);
    return;
  }
  if constexpr (!SMALL) {
    for (int i = tid; i < n; i += kPlan) {
      const int had = (int)w.had[i];
      if (had % kPageTokens) {
        const uint32_t page = v.table[(uint64_t)lanes[i] * v.max_pages + had / kPageTokens];
        atomicAdd(&w.uses[page], 1u);
        atomicMax(&w.last[page], (uint32_t)i);
      }
    }
    __syncthreads();
  }
  // what each lane takes, in the order of the list (copies in the high half of a sum)
  uint64_t need = 0;
  uint32_t copies = 0, my_base = 0, my_fresh = 0;
  bool my_copy = false;
  for (int i0 = 0; i0 < n; i0 += kPlan) {
    const int i = i0 + tid;
    uint32_t fresh = 0, page = my_page;
    bool copy = false;
    if (i < n) {
      const int had = SMALL ? my_had : (int)w.had[i], t = SMALL ? my_tokens : tokens[i];
      if (had % kPageTokens) {
        // of the listed lanes that share the page, with no others, the last one keeps it
        if constexpr (SMALL) {
          if (my_refs > 1) {
            uint32_t uses = 0;
            int last = 0;
            for (int j = 0; j < n; ++j)
              if (last_page[j] == my_page) ++uses, last = j;
            copy = uses < my_refs || last != i;
          }
        } else {
          page = v.table[(uint64_t)lanes[i] * v.max_pages + had / kPageTokens];
          copy = aload(&w.uses[page]) < v.refs[page] || aload(&w.last[page]) != (uint32_t)i;
        }
      }
      fresh = (uint32_t)(pages_of(had + t) - pages_of(had));
    }
    uint64_t all;
    const uint64_t at = block_scan((uint64_t)copy << 40 | (copy + fresh), &all), mask = (1ull << 40) - 1;
    if (i < n) {
      w.base[i] = my_base = (uint32_t)(need + (at & mask));
      my_copy = copy, my_fresh = fresh;
      const uint32_t c = copies + (uint32_t)(at >> 40);
      if (copy) w.copy_lane[c] = i, w.copy_from[c] = page;
      if (SMALL && copy + fresh > kOwnPages) longest = 1;
    }
    need += all & mask;
    copies += (uint32_t)(all >> 40);
  }
  const uint64_t got = need <= (uint64_t)v.n_pages ? find_free(v, w, need, ids, first) : 0;
  __syncthreads();
  // the plan hands out few pages by itself
  const bool own = SMALL && need <= kIdsInLds && !longest, ok = need <= got;
  if (own && ok && tid < n) {
    v.len[my_lane] = my_had + my_tokens;
    uint32_t* row = v.table + (uint64_t)my_lane * v.max_pages + pages_of(my_had) - (my_copy ? 1 : 0);
    for (uint32_t e = 0; e < my_copy + my_fresh; ++e) {
      const uint32_t id = ids[my_base + e];
      row[e] = id;
      v.refs[id] = 1;
    }
  }
  if (tid == 0) {
    w.plan->ok = ok;
    w.plan->need = (uint32_t)need;
    w.plan->handed = own;
    w.plan->copies = copies;
    if (!ok) set_error(v.error, FERRY_ECAPACITY);
  }
}

// One page of one layer, all kv heads, by one workgroup.  KEEP: the copy is soon read
// (a lane's last page); else it streams past the caches: 5.0 against 4.7 TB/s (1.66 GB moved).
template <bool KEEP>
__device__ inline void copy_page(const PageView& v, int layer, uint32_t from, uint32_t to) {
  constexpr int kEach = 4;  // words of a thread on their way at once
  const uint32_t words = (uint32_t)v.H * (v.bb / 16);
  const u32x4* s = reinterpret_cast<const u32x4*>(v.pool) + ((uint64_t)layer * v.n_pages + from) * words;
  u32x4* d = reinterpret_cast<u32x4*>(v.pool) + ((uint64_t)layer * v.n_pages + to) * words;
  for (uint32_t i0 = threadIdx.x; i0 < words; i0 += kEach * blockDim.x) {
    u32x4 x[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (i0 + j * blockDim.x < words) x[j] = load_kv<!KEEP>(s + i0 + j * blockDim.x);
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (i0 + j * blockDim.x < words) {
        if constexpr (KEEP) d[i0 + j * blockDim.x] = x[j];
        else __builtin_nontemporal_store(x[j], d + i0 + j * blockDim.x);
      }
  }
  if (v.scales) {
    const float* a = v.scales + ((uint64_t)layer * v.n_pages + from) * v.H * 2;
    float* b = v.scales + ((uint64_t)layer * v.n_pages + to) * v.H * 2;
    for (int i = threadIdx.x; i < v.H * 2; i += blockDim.x) b[i] = a[i];
  }
}

__global__ __launch_bounds__(256) void k_reserve(PageView v, Work w, const int32_t* __restrict__ lanes, int n) {
  if (!w.plan->ok) return;
  const uint32_t need = w.plan->handed ? 0 : w.plan->need, copies = w.plan->copies;
  const uint32_t step = gridDim.x * blockDim.x, at = blockIdx.x * blockDim.x + threadIdx.x;
  if (!w.plan->handed)
    for (uint32_t i = at; i < (uint32_t)n; i += step) v.len[lanes[i]] = (int)w.grown[i];
  // taken page r belongs to the last list place whose base is at most r
  for (uint32_t r = at; r < need; r += step) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (w.base[mid] <= r) lo = mid; else hi = mid - 1;
    }
    const int had = (int)w.had[lo];
    const uint32_t taken = (lo + 1 < n ? w.base[lo + 1] : need) - w.base[lo];
    const int fresh = pages_of((int)w.grown[lo]) - pages_of(had);
    const bool copy = taken > (uint32_t)fresh;
    const int col = pages_of(had) - (copy ? 1 : 0) + (int)(r - w.base[lo]);
    const uint32_t id = w.free_ids[r];
    v.table[(uint64_t)lanes[lo] * v.max_pages + col] = id;
    v.refs[id] = 1;
  }
  for (uint64_t c = blockIdx.x; c < (uint64_t)copies * v.L; c += gridDim.x) {
    const uint32_t k = (uint32_t)(c / v.L), from = w.copy_from[k];
    if (c % v.L == 0 && threadIdx.x == 0) atomicSub(&v.refs[from], 1u);
    copy_page<true>(v, (int)(c % v.L), from, w.free_ids[w.base[w.copy_lane[k]]]);
  }
}

// ---- fork and trim ----------------------------------------------------------------
// Checks a list of lanes (fork: src and dst); every thread of the workgroup gets the
// error, 0 if it is fine.  fine(i): whether entry i's counts are, once its lanes are.
template <class Fine>
__device__ inline int check_lanes(const PageView& v, const int32_t* __restrict__ src,
                                  const int32_t* __restrict__ lanes, int n, Fine&& fine) {
  __shared__ uint32_t bits[kMaxLanes / 32];
  __shared__ int bad;
  const int tid = threadIdx.x, threads = blockDim.x;
  for (int i = tid; i < (v.n_lanes + 31) / 32; i += threads) bits[i] = 0;
  if (tid == 0) bad = 0;
  __syncthreads();
  for (int i = tid; i < n; i += threads)
    if (!name_lane(bits, lanes[i], v.n_lanes)) bad = FERRY_EINVAL;
  __syncthreads();
  for (int i = tid; i < n; i += threads) {
    const int lane = lanes[i], from = src ? src[i] : lane;
    bool ok = lane >= 0 && lane < v.n_lanes && from >= 0 && from < v.n_lanes;
    if (ok && src) ok = !(bits[from >> 5] >> (from & 31) & 1u);
    if (!ok || !fine(i, from, lane)) bad = FERRY_EINVAL;
  }
  __syncthreads();
  return bad;
}

// Tokens that entry i of a fork or trim keeps of what lane `from` holds; false: not so many.
__device__ inline bool kept_tokens(const PageView& v, const int32_t* keep, int i, int from, int otherwise,
                                   int* kept) {
  const int held = v.len[from];
  *kept = keep ? keep[i] : otherwise < 0 ? held : otherwise;
  return *kept >= 0 && *kept <= held && held <= v.max_pages * kPageTokens;
}

// One workgroup checks a fork's list; w.had gets the tokens each dst will hold.
__device__ inline bool fork_plan(const PageView& v, const Work& w, const int32_t* src, const int32_t* dst,
                                 const int32_t* keep, int n) {
  const int bad = check_lanes(v, src, dst, n, [&](int i, int from, int lane) {
    int kept;
    const bool ok = kept_tokens(v, keep, i, from, -1, &kept) && v.len[lane] == 0;
    w.had[i] = kept;
    return ok;
  });
  if (bad && threadIdx.x == 0) set_error(v.error, bad);
  return bad == 0;
}
// Entry e of a forked row.
__device__ inline void fork_entry(const PageView& v, int src, int dst, int e) {
  const uint32_t id = v.table[(uint64_t)src * v.max_pages + e];
  v.table[(uint64_t)dst * v.max_pages + e] = id;
  if (id < (uint32_t)v.n_pages) atomicAdd(&v.refs[id], 1u);
  else set_error(v.error, FERRY_ESTATE);
}

// A short list of short tables: the one workgroup that checks it copies the rows too,
// a wavefront each.
__global__ __launch_bounds__(kPlan) void k_fork_small(PageView v, Work w, const int32_t* __restrict__ src,
                                                      const int32_t* __restrict__ dst,
                                                      const int32_t* __restrict__ keep, int n) {
  if (!fork_plan(v, w, src, dst, keep, n)) return;
  for (int i = threadIdx.x >> 6; i < n; i += kPlan / 64) {
    const int kept = (int)w.had[i], from = src[i], to = dst[i];
    for (int e = threadIdx.x & 63; e < pages_of(kept); e += 64) fork_entry(v, from, to, e);
    if ((threadIdx.x & 63) == 0) v.len[to] = kept;
  }
}

__global__ __launch_bounds__(kPlan) void k_fork_plan(PageView v, Work w, const int32_t* __restrict__ src,
                                                     const int32_t* __restrict__ dst,
                                                     const int32_t* __restrict__ keep, int n) {
  const bool ok = fork_plan(v, w, src, dst, keep, n);
  if (threadIdx.x == 0) w.plan->ok = ok;
}
__global__ __launch_bounds__(256) void k_fork(PageView v, Work w, const int32_t* __restrict__ src,
                                              const int32_t* __restrict__ dst, int n) {
  if (!w.plan->ok) return;
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int kept = (int)w.had[i], from = src[i], to = dst[i];
    for (int e = threadIdx.x; e < pages_of(kept); e += blockDim.x) fork_entry(v, from, to, e);
    if (threadIdx.x == 0) v.len[to] = kept;
  }
}

// Every workgroup checks the list for itself and trims its own lanes of it.  What
// another one has done by then does not change the answer: a lane's length only
// becomes what it keeps, and a list that is not fine is left alone by all.
__global__ __launch_bounds__(256) void k_trim(PageView v, const int32_t* __restrict__ lanes,
                                              const int32_t* __restrict__ keep, int n) {
  const int bad = check_lanes(v, nullptr, lanes, n, [&](int i, int from, int) {
    int kept;
    return kept_tokens(v, keep, i, from, 0, &kept);
  });
  if (bad) {
    if (threadIdx.x == 0 && blockIdx.x == 0) set_error(v.error, bad);
    return;
  }
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int lane = lanes[i], kept = keep ? keep[i] : 0, held = v.len[lane];
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
    __syncthreads();  // all have read the length
    if (threadIdx.x == 0) v.len[lane] = kept;
  }
}

// ---- compact ----------------------------------------------------------------------
// One workgroup pairs the pages in use at or behind `live` with the free ids
// before it, both in ascending order: the two lists do not meet, so the moves
// need no order among themselves.  free_ids becomes the new id of every page.
// EACH pages of a thread are on their way at once; where that covers the pool (ONE)
// they are read once.
template <int EACH, bool ONE>
__global__ __launch_bounds__(kPlan) void k_compact_plan(PageView v, Work w, int32_t* live_out) {
  const int tid = threadIdx.x;
  auto read = [&](int64_t p0, uint32_t (&r)[EACH]) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) r[i] = p0 + i < v.n_pages ? v.refs[p0 + i] : 0u;
  };
  uint32_t mine = 0, r[EACH];
  for (int64_t c = 0; c < v.n_pages; c += EACH * kPlan) {
    read(c + (int64_t)EACH * tid, r);
#pragma unroll
    for (int i = 0; i < EACH; ++i) mine += r[i] != 0;
  }
  uint64_t all;
  (void)block_scan(mine, &all);
  const int64_t live = (int64_t)all;
  uint32_t gaps = 0, moves = 0;
  for (int64_t c = 0; c < v.n_pages; c += EACH * kPlan) {
    const int64_t p0 = c + (int64_t)EACH * tid;
    if (!ONE) read(p0, r);
    uint64_t n = 0;  // gaps below, moves in the high half
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (p0 + i < live) n += r[i] == 0;
      else n += (uint64_t)(r[i] != 0) << 32;
    }
    const uint64_t at = block_scan(n, &all);
    uint32_t g = gaps + (uint32_t)at, m = moves + (uint32_t)(at >> 32);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (p0 + i >= v.n_pages) break;
      w.free_ids[p0 + i] = (uint32_t)(p0 + i);
      if (p0 + i < live) {
        if (r[i] == 0) w.last[g++] = (uint32_t)(p0 + i);
      } else if (r[i] != 0) {
        w.from[m++] = (uint32_t)(p0 + i);
      }
    }
    gaps += (uint32_t)all;
    moves += (uint32_t)(all >> 32);
  }
  __syncthreads();
  for (uint32_t m = tid; m < moves; m += kPlan) {
    const uint32_t from = w.from[m], to = w.last[m];
    w.free_ids[from] = to;
    v.refs[to] = v.refs[from];
    v.refs[from] = 0;
  }
  if (tid == 0) {
    w.plan->copies = moves;
    if (live_out) *live_out = (int32_t)live;
  }
}

__global__ __launch_bounds__(256) void k_compact(PageView v, Work w) {
  const uint32_t moves = w.plan->copies;
  if (!moves) return;
  for (uint64_t c = blockIdx.x; c < (uint64_t)moves * v.L; c += gridDim.x) {
    const uint32_t m = (uint32_t)(c / v.L);
    copy_page<false>(v, (int)(c % v.L), w.from[m], w.last[m]);
  }
  for (int i = blockIdx.x; i < v.n_lanes; i += gridDim.x) {
    uint32_t* row = v.table + (uint64_t)i * v.max_pages;
    const int held = v.len[i];
    const int pages = held <= 0 ? 0 : min(pages_of(held), v.max_pages);
    for (int e = threadIdx.x; e < pages; e += blockDim.x) {
      const uint32_t id = row[e];
      if (id < (uint32_t)v.n_pages) row[e] = w.free_ids[id];
      else set_error(v.error, FERRY_ESTATE);
    }
  }
}

// ---- append -------------------------------------------------------------------------
struct AppendArgs {
  int n, Hq, rot, pairs, out_type;
  int heads;  // heads (of q, k and v, in this order) per workgroup
  float factor;
  const int32_t* lane;
  const int32_t* pos;
  const double* inv_freq;
  const float* kv_scale;
  const void *q, *k, *v;
  void* q_out;
  int64_t qs[2], ks[2], vs[2], os[2];
};

// cos and sin of 2 pi t in fp32.  The part of a turn is taken in 64 bits (positions of
// 2^24 leave 2^-30 of a turn), down to the eighth of a turn next to a quarter, so that
// fp32 rounds only a small angle.
__device__ inline void turn(double t, float* c, float* s) {
  const double quarters = rint(4.0 * (t - rint(t)));
  const float r = (float)((t - rint(t)) - 0.25 * quarters);
  float sn, cs;
  sincospif(2.0f * r, &sn, &cs);
  const int k = (int)quarters & 3;
  const float x = k & 1 ? sn : cs, y = k & 1 ? cs : sn;
  *c = k == 1 || k == 2 ? -x : x;
  *s = k >= 2 ? -y : y;
}

template <int DT>
__device__ inline float load_elem(const void* p, int64_t i) {
  if constexpr (DT == FERRY_F32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == FERRY_F16) return (float)static_cast<const _Float16*>(p)[i];
  else return bits_f32((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}
template <int DT>
__device__ inline void store_elem(void* p, int64_t i, float x) {
  if constexpr (DT == FERRY_F32) static_cast<float*>(p)[i] = x;
  else if constexpr (DT == FERRY_F16) static_cast<_Float16*>(p)[i] = (_Float16)x;
  else if constexpr (DT == FERRY_BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(x);
  else static_cast<uint8_t*>(p)[i] = f32_to_e4m3(x);
}
// ... 8 of them, 16-byte aligned (8 for E4M3)
template <int DT>
__device__ inline void load8(const u32x4 (&w)[DT == FERRY_F32 ? 2 : 1], float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == FERRY_F32) x[i] = bits_f32(w[i >> 2][i & 3]);
    else if constexpr (DT == FERRY_BF16) x[i] = bits_f32(i & 1 ? w[0][i >> 1] & 0xFFFF0000u : w[0][i >> 1] << 16);
    else {
      typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
      x[i] = (float)__builtin_bit_cast(f16x2, (uint32_t)w[0][i >> 1])[i & 1];
    }
  }
}
template <int DT>
__device__ inline void store8(void* p, int64_t at, const float (&x)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == FERRY_F32) {
    u32x4* to = reinterpret_cast<u32x4*>(static_cast<float*>(p) + at);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      to[i] = u32x4{f32_bits(x[4 * i]), f32_bits(x[4 * i + 1]), f32_bits(x[4 * i + 2]), f32_bits(x[4 * i + 3])};
  } else if constexpr (DT == FERRY_FP8_E4M3) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i] == x[i] ? __builtin_amdgcn_fmed3f(x[i], -448.0f, 448.0f) : x[i];
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
      w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], lo, true);
    }
    *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(p) + at) = w;
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 y = {x[2 * i], x[2 * i + 1]};
      if constexpr (DT == FERRY_BF16) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, bf16x2));
      else w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, f16x2));
    }
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at) = w;
  }
}
// x / s, correctly rounded, from inv = 1 / s, where x * inv is finite; else by the
// division itself (infinities, quotients that overflow, an s whose inverse does)
__device__ inline float divide(float x, float s, float inv) {
  const float q = x * inv;
  if (!(fabsf(q) < INFINITY)) return x / s;
  return __builtin_fmaf(__builtin_fmaf(-q, s, x), inv, q);
}

// The page of token t, or -1 where it is padding or has no place (reported once per
// token).
__device__ inline int64_t append_page(const PageView& v, const AppendArgs& a, int t, int pos) {
  const int lane = a.lane ? a.lane[t] : 0;
  if (a.lane && lane < 0) return -1;
  if (!a.k) return 0;
  int bad = 0;
  uint32_t page = 0;
  if (lane >= v.n_lanes || pos < 0 || pos >= v.len[lane] || pos / kPageTokens >= v.max_pages) {
    bad = FERRY_ERANGE;
  } else {
    page = v.table[(uint64_t)lane * v.max_pages + pos / kPageTokens];
    if (page >= (uint32_t)v.n_pages) bad = FERRY_ERANGE;
    else if (v.refs && v.refs[page] > 1) bad = FERRY_ESTATE;
  }
  if (!bad) return page;
  if (threadIdx.x == 0 && blockIdx.y == 0) set_error(v.error, bad);
  return -1;
}

// A workgroup per token and `heads` of its heads, 16 lanes per head with 8 values each:
// one read of q, k and v, one write.  The angles are computed once for the heads, while
// the values are on their way.  In the halves layout a lane reads its pair's other
// eight too (the head's line is in the L1 cache) and all lanes of a head read before
// one writes, which makes q_out = q safe.  Bound by memory: 18,000 tokens of 48 heads
// (466 MB) in 87 us, 5.3 TB/s read and written (a torch copy: 4.6).
template <int XT, int PT>
__global__ __launch_bounds__(256) void k_append(PageView v, int layer, AppendArgs a) {
  constexpr int W = XT == FERRY_F32 ? 2 : 1;  // 16-byte words of 8 values
  constexpr int kAhead = 3;                   // heads of a lane on their way
  __shared__ __attribute__((aligned(16))) float cs[64], sn[64];
  const int t = blockIdx.x, tid = threadIdx.x, d = (tid & 15) * 8;
  const int pos = a.pos[t];
  const int64_t page = append_page(v, a, t, pos);
  if (page < 0) return;
  const int all = a.Hq + (a.k ? 2 * v.H : 0);
  const int h0 = blockIdx.y * a.heads, h1 = min(all, h0 + a.heads);
  const int half = a.rot / 2, mate = d < half ? d + half : d - half;
  bool first = true;
  for (int g = h0; g < h1; g += 16 * kAhead) {
    u32x4 own[kAhead][W], other[kAhead][W];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int h = g + 16 * j + (tid >> 4);
      if (h >= h1) continue;
      const char* p = static_cast<const char*>(h < a.Hq ? a.q : h < a.Hq + v.H ? a.k : a.v);
      const int64_t at = h < a.Hq           ? t * a.qs[0] + h * a.qs[1]
                         : h < a.Hq + v.H ? t * a.ks[0] + (h - a.Hq) * a.ks[1]
                                            : t * a.vs[0] + (h - a.Hq - v.H) * a.vs[1];
      const u32x4* x = reinterpret_cast<const u32x4*>(p + (at + d) * (XT == FERRY_F32 ? 4 : 2));
      const u32x4* y = reinterpret_cast<const u32x4*>(p + (at + mate) * (XT == FERRY_F32 ? 4 : 2));
#pragma unroll
      for (int w = 0; w < W; ++w) {
        own[j][w] = x[w];
        if (!a.pairs && d < a.rot && h < a.Hq + v.H) other[j][w] = y[w];
      }
    }
    if (first) {
      first = false;
      if (tid < half) {
        float c, s;
        turn((double)pos * (a.inv_freq[tid] * 0.15915494309189535), &c, &s);
        cs[tid] = c * a.factor, sn[tid] = s * a.factor;
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int h = g + 16 * j + (tid >> 4);
      if (h >= h1) continue;
      float x[8], y[8];
      load8<XT>(own[j], x);
      if (d < a.rot && h < a.Hq + v.H) {
        if (a.pairs) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float c = cs[d / 2 + i], s = sn[d / 2 + i], p = x[2 * i], q = x[2 * i + 1];
            x[2 * i] = p * c - q * s, x[2 * i + 1] = q * c + p * s;
          }
        } else {
          load8<XT>(other[j], y);
          const int i0 = d < half ? d : mate;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float s = d < half ? -sn[i0 + i] : sn[i0 + i];
            x[i] = x[i] * cs[i0 + i] + y[i] * s;
          }
        }
      }
      if (h < a.Hq) {
        const int64_t at = t * a.os[0] + h * a.os[1] + d;
        if (a.out_type == FERRY_F32) store8<FERRY_F32>(a.q_out, at, x);
        else if (a.out_type == FERRY_F16) store8<FERRY_F16>(a.q_out, at, x);
        else store8<FERRY_BF16>(a.q_out, at, x);
      } else {
        const int value = h >= a.Hq + v.H, kv = h - a.Hq - (value ? v.H : 0);
        const uint64_t rec = v.record(layer, (uint32_t)page, kv);
        if constexpr (PT == FERRY_FP8_E4M3) {
          const float s = a.kv_scale[2 * kv + value], inv = 1.0f / s;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = divide(x[i], s, inv);
          if (d == 0) v.scales[2 * rec + value] = s;
        }
        store8<PT>(v.pool + rec * v.bb, (value * kPageTokens + pos % kPageTokens) * kPageDim + d, x);
      }
    }
  }
}

// The same for tensors that are not 16-byte aligned and for rotated parts that do not
// end between eights: a value per thread.
template <int XT, int PT>
__global__ __launch_bounds__(256) void k_append_any(PageView v, int layer, AppendArgs a) {
  __shared__ float cs[64], sn[64];
  const int t = blockIdx.x, tid = threadIdx.x, half = a.rot / 2;
  const int pos = a.pos[t];
  const int64_t page = append_page(v, a, t, pos);
  if (page < 0) return;
  if (tid < half) {
    float c, s;
    turn((double)pos * (a.inv_freq[tid] * 0.15915494309189535), &c, &s);
    cs[tid] = c * a.factor, sn[tid] = s * a.factor;
  }
  __syncthreads();
  auto turned = [&](const void* x, int64_t base, int d) {
    const float self = load_elem<XT>(x, base + d);
    if (d >= a.rot) return self;
    const int i = a.pairs ? d / 2 : d % half;
    const bool second = a.pairs ? d & 1 : d >= half;
    const float other = load_elem<XT>(x, base + (a.pairs ? d ^ 1 : second ? d - half : d + half));
    return second ? self * cs[i] + other * sn[i] : self * cs[i] - other * sn[i];
  };
  for (int e0 = 0; e0 < a.Hq * kPageDim; e0 += 256) {
    const int e = e0 + tid, h = e / kPageDim, d = e % kPageDim;
    float y = 0.0f;
    if (e < a.Hq * kPageDim) y = turned(a.q, t * a.qs[0] + h * a.qs[1], d);
    __syncthreads();  // q_out may be q: a pair is read before it is written
    const int64_t at = t * a.os[0] + h * a.os[1] + d;
    if (e < a.Hq * kPageDim) {
      if (a.out_type == FERRY_F32) store_elem<FERRY_F32>(a.q_out, at, y);
      else if (a.out_type == FERRY_F16) store_elem<FERRY_F16>(a.q_out, at, y);
      else store_elem<FERRY_BF16>(a.q_out, at, y);
    }
  }
  if (!a.k) return;
  for (int e = tid; e < v.H * kPageDim; e += 256) {
    const int h = e / kPageDim, d = e % kPageDim;
    const uint64_t rec = v.record(layer, (uint32_t)page, h);
    float k = turned(a.k, t * a.ks[0] + h * a.ks[1], d);
    float x = load_elem<XT>(a.v, t * a.vs[0] + h * a.vs[1] + d);
    if constexpr (PT == FERRY_FP8_E4M3) {
      const float sk = a.kv_scale[2 * h], sv = a.kv_scale[2 * h + 1];
      k = divide(k, sk, 1.0f / sk), x = divide(x, sv, 1.0f / sv);
      if (d == 0) v.scales[2 * rec] = sk, v.scales[2 * rec + 1] = sv;
    }
    uint8_t* to = v.pool + rec * v.bb;
    store_elem<PT>(to, (pos % kPageTokens) * kPageDim + d, k);
    store_elem<PT>(to, (kPageTokens + pos % kPageTokens) * kPageDim + d, x);
  }
}

template <int XT, int PT>
void launch_append(const PageView& v, int layer, AppendArgs a, int cus, hipStream_t s) {
  const int es = XT == FERRY_F32 ? 4 : 2, os = a.out_type == FERRY_F32 ? 4 : 2;
  uint64_t low = 0;
  auto aligned = [&](const void* p, const int64_t (&stride)[2], int size) {
    if (p) low |= reinterpret_cast<uintptr_t>(p) | (uint64_t)(stride[0] * size) | (uint64_t)(stride[1] * size);
  };
  aligned(a.q, a.qs, es), aligned(a.k, a.ks, es), aligned(a.v, a.vs, es), aligned(a.q ? a.q_out : nullptr, a.os, os);
  if (low % 16 == 0 && a.rot % (a.pairs ? 8 : 16) == 0) {
    // All heads of a token in a workgroup, which computes its angles once, where that
    // fills the GPU (18,000 tokens of 48 heads: 87 us, 95 with 16 heads each), else 16
    // (64 tokens: 3.6 us, 5.2 with all 48).
    const int all = a.Hq + (a.k ? 2 * v.H : 0);
    a.heads = a.n >= 4 * cus ? all : 16;
    k_append<XT, PT><<<dim3(a.n, (all + a.heads - 1) / a.heads), 256, 0, s>>>(v, layer, a);
  } else {
    k_append_any<XT, PT><<<a.n, 256, 0, s>>>(v, layer, a);
  }
}
template <int XT>
void launch_append(const PageView& v, int layer, const AppendArgs& a, int pt, int cus, hipStream_t s) {
  if (pt == FERRY_F32) launch_append<XT, FERRY_F32>(v, layer, a, cus, s);
  else if (pt == FERRY_F16) launch_append<XT, FERRY_F16>(v, layer, a, cus, s);
  else if (pt == FERRY_BF16) launch_append<XT, FERRY_BF16>(v, layer, a, cus, s);
  else launch_append<XT, FERRY_FP8_E4M3>(v, layer, a, cus, s);
}

// Tokens [t, t + kLaunchTokens) of a call: a launch has a workgroup per token, and fewer
// than 2^32 threads.
constexpr int kLaunchTokens = 1 << 23;
AppendArgs tokens_from(AppendArgs a, int t, int x_size, int out_size) {
  a.n = std::min(a.n - t, kLaunchTokens);
  if (a.lane) a.lane += t;
  a.pos += t;
  auto at = [&](const void* x, int64_t stride, int size) -> const void* {
    return x ? static_cast<const uint8_t*>(x) + t * stride * size : nullptr;
  };
  a.q = at(a.q, a.qs[0], x_size), a.k = at(a.k, a.ks[0], x_size), a.v = at(a.v, a.vs[0], x_size);
  a.q_out = const_cast<void*>(at(a.q_out, a.os[0], out_size));
  return a;
}

// The common start of the managing calls.
int manage(const ferry_pages* p, int n, PageView* v, Work* w) {
  if (int rc = page_geometry(p, v)) return rc;
  if (n < 0 || n > p->n_lanes) return report(FERRY_EINVAL, "n must be in [0, n_lanes]");
  if (int rc = page_buffers(p, true)) return rc;
  *w = split_work(p->work, p->n_pages, p->n_lanes);
  return FERRY_OK;
}

// A list of n values that a managing call reads (or writes): device memory apart from what
// the call changes, since its workgroups read the list while others already change that.
// of_len: the call has read the list before it changes len.
int check_list(const ferry_pages* p, const void* list, const char* name, int n, bool of_len = false) {
  if (int rc = check_on(list, name, p->device)) return rc;
  const uintptr_t from = reinterpret_cast<uintptr_t>(list), to = from + (uintptr_t)n * 4;
  auto meets = [&](const void* buf, uint64_t entries) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(buf);
    return from < at + entries * 4 && at < to;
  };
  if ((!of_len && meets(p->len, p->n_lanes)) || meets(p->refs, p->n_pages) || meets(p->table, (uint64_t)p->n_lanes * p->max_pages))
    return report(FERRY_EINVAL, std::string(name) + " is a part of the cache's own table, len or refs");
  return FERRY_OK;
}

}  // namespace

extern "C" {

int ferry_pages_work_bytes(const ferry_pages* p, uint64_t* bytes) {
  return entry([&]() -> int {
    PageView v;
    if (int rc = page_geometry(p, &v)) return rc;
    if (!bytes) return report(FERRY_EINVAL, "null bytes");
    *bytes = work_bytes(p->n_pages, p->n_lanes);
    return FERRY_OK;
  });
}

int ferry_pages_reserve(const ferry_pages* p, const int32_t* lanes, const int32_t* tokens, int32_t n,
                        void* stream) {
  return entry([&]() -> int {
    PageView v;
    Work w;
    if (int rc = manage(p, n, &v, &w)) return rc;
    if (n == 0) return FERRY_OK;
    if (int rc = check_list(p, lanes, "lanes", n)) return rc;
    if (int rc = check_list(p, tokens, "tokens", n, true)) return rc;
    OnDevice on(p->device);
    if (!on.ok()) return report(FERRY_EHIP, "cannot use the cache's GPU");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n <= kPlan) k_reserve_plan<true><<<1, kPlan, 0, s>>>(v, w, lanes, tokens, n);
    else k_reserve_plan<false><<<1, kPlan, 0, s>>>(v, w, lanes, tokens, n);
    const int64_t most = std::min<int64_t>((int64_t)n * v.L + 64, 8l * gpu_cus(p->device));
    k_reserve<<<(unsigned)most, 256, 0, s>>>(v, w, lanes, n);
    return launched("ferry_pages_reserve");
  });
}

int ferry_pages_fork(const ferry_pages* p, const int32_t* src, const int32_t* dst, const int32_t* keep,
                     int32_t n, void* stream) {
  return entry([&]() -> int {
    PageView v;
    Work w;
    if (int rc = manage(p, n, &v, &w)) return rc;
    if (n == 0) return FERRY_OK;
    if (int rc = check_list(p, src, "src", n)) return rc;
    if (int rc = check_list(p, dst, "dst", n)) return rc;
    if (keep)
      if (int rc = check_list(p, keep, "keep", n, true)) return rc;
    OnDevice on(p->device);
    if (!on.ok()) return report(FERRY_EHIP, "cannot use the cache's GPU");
    hipStream_t s = static_cast<hipStream_t>(stream);
    // One launch where each of its 16 wavefronts has at most four times 64 entries of a row
    // (24 lanes of 58 pages: 4.0 us, 5.7 in two launches); else what the workgroup does alone
    // takes longer than a launch (128 lanes of 64 pages: 8.2 and 5.9; 1,000 of 8: 70 and 11;
    // one of 8,192: 41 and 15).
    const int64_t rounds = (int64_t)((n + 15) / 16) * ((p->max_pages + 63) / 64);
    if (rounds <= 4) {
      k_fork_small<<<1, kPlan, 0, s>>>(v, w, src, dst, keep, n);
    } else {
      k_fork_plan<<<1, kPlan, 0, s>>>(v, w, src, dst, keep, n);
      k_fork<<<n, 256, 0, s>>>(v, w, src, dst, n);
    }
    return launched("ferry_pages_fork");
  });
}

int ferry_pages_trim(const ferry_pages* p, const int32_t* lanes, const int32_t* keep, int32_t n, void* stream) {
  return entry([&]() -> int {
    PageView v;
    Work w;
    if (int rc = manage(p, n, &v, &w)) return rc;
    if (n == 0) return FERRY_OK;
    if (int rc = check_list(p, lanes, "lanes", n)) return rc;
    if (keep)
      if (int rc = check_list(p, keep, "keep", n)) return rc;
    OnDevice on(p->device);
    if (!on.ok()) return report(FERRY_EHIP, "cannot use the cache's GPU");
    hipStream_t s = static_cast<hipStream_t>(stream);
    // each workgroup reads the whole list: a long one goes to fewer of them
    k_trim<<<n <= 1024 ? n : 256, 256, 0, s>>>(v, lanes, keep, n);
    return launched("ferry_pages_trim");
  });
}

int ferry_pages_compact(const ferry_pages* p, int32_t* live, void* stream) {
  return entry([&]() -> int {
    PageView v;
    Work w;
    if (int rc = manage(p, 0, &v, &w)) return rc;
    if (live)
      if (int rc = check_list(p, live, "live", 1)) return rc;
    OnDevice on(p->device);
    if (!on.ok()) return report(FERRY_EHIP, "cannot use the cache's GPU");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (v.n_pages <= 4 * kPlan) k_compact_plan<4, true><<<1, kPlan, 0, s>>>(v, w, live);
    else k_compact_plan<16, false><<<1, kPlan, 0, s>>>(v, w, live);
    k_compact<<<(unsigned)std::min<int64_t>((int64_t)v.n_pages * v.L, 8l * gpu_cus(p->device)), 256, 0, s>>>(v, w);
    return launched("ferry_pages_compact");
  });
}

int ferry_pages_append(const ferry_pages* p, int32_t layer, const ferry_append* a, void* stream) {
  return entry([&]() -> int {
    PageView v;
    if (int rc = page_geometry(p, &v)) return rc;
    if (!a) return report(FERRY_EINVAL, "null args");
    if (layer < 0 || layer >= p->n_layers) return report(FERRY_EINVAL, "layer out of range");
    if (a->n_tokens < 0) return report(FERRY_EINVAL, "n_tokens must not be negative");
    if (a->x_dtype < FERRY_F32 || a->x_dtype > FERRY_BF16)
      return report(FERRY_EINVAL, "x_dtype must be F32, F16 or BF16");
    if (a->rot_dim < 2 || a->rot_dim > kPageDim || a->rot_dim % 2)
      return report(FERRY_EINVAL, "rot_dim must be even, 2..128");
    if (a->n_tokens == 0) return FERRY_OK;
    if (!a->q && !a->k) return report(FERRY_EINVAL, "neither q nor k");
    if (!a->k != !a->v) return report(FERRY_EINVAL, "k and v go together");
    if (a->q && (a->q_out_dtype < FERRY_F32 || a->q_out_dtype > FERRY_BF16))
      return report(FERRY_EINVAL, "q_out_dtype must be F32, F16 or BF16");
    if (a->q && (a->q_heads < 1 || a->q_heads > 65536)) return report(FERRY_EINVAL, "q_heads out of range");
    if (int rc = page_buffers(p, false)) return rc;
    if (int rc = check_all({{a->pos, "pos"}, {a->inv_freq, "inv_freq"}}, p->device)) return rc;
    if (a->k || a->lane)
      if (int rc = check_on(a->lane, "lane", p->device)) return rc;
    if (a->q)
      if (int rc = check_all({{a->q, "q"}, {a->q_out, "q_out"}}, p->device)) return rc;
    if (a->k)
      if (int rc = check_all({{a->k, "k"}, {a->v, "v"}}, p->device)) return rc;
    if (a->k && p->dtype == FERRY_FP8_E4M3)
      if (int rc = check_on(a->kv_scale, "kv_scale", p->device)) return rc;
    if (a->q && a->q_out == a->q &&
        (a->q_out_dtype != a->x_dtype || a->q_stride[0] != a->q_out_stride[0] || a->q_stride[1] != a->q_out_stride[1]))
      return report(FERRY_EINVAL, "q_out is q with another type or other strides");
    OnDevice on(p->device);
    if (!on.ok()) return report(FERRY_EHIP, "cannot use the cache's GPU");
    const int ot = a->q ? a->q_out_dtype : a->x_dtype;
    AppendArgs d{a->n_tokens, a->q ? a->q_heads : 0, a->rot_dim, a->pairs != 0, ot, 0, a->factor, a->lane, a->pos,
                 a->inv_freq, a->kv_scale, a->q, a->k, a->v, a->q_out,
                 {a->q_stride[0], a->q_stride[1]}, {a->k_stride[0], a->k_stride[1]},
                 {a->v_stride[0], a->v_stride[1]}, {a->q_out_stride[0], a->q_out_stride[1]}};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int cus = gpu_cus(p->device);
    for (int t = 0; t < a->n_tokens; t += kLaunchTokens) {
      const AppendArgs part = tokens_from(d, t, a->x_dtype == FERRY_F32 ? 4 : 2, ot == FERRY_F32 ? 4 : 2);
      if (a->x_dtype == FERRY_F32) launch_append<FERRY_F32>(v, layer, part, p->dtype, cus, s);
      else if (a->x_dtype == FERRY_F16) launch_append<FERRY_F16>(v, layer, part, p->dtype, cus, s);
      else launch_append<FERRY_BF16>(v, layer, part, p->dtype, cus, s);
      if (int rc = launched("ferry_pages_append")) return rc;
      if (a->n_tokens - t <= kLaunchTokens) break;
    }
    return FERRY_OK;
  });
}

int ferry_rope_freqs(int kind, int32_t rot_dim, double base, double stretch, double trained_ctx, double slow,
                     double fast, double* out) {
  return entry([&]() -> int {
    if (!out) return report(FERRY_EINVAL, "null out");
    if (rot_dim < 2 || rot_dim > kPageDim || rot_dim % 2) return report(FERRY_EINVAL, "rot_dim must be even, 2..128");
    if (kind < FERRY_ROPE_PLAIN || kind > FERRY_ROPE_PARTS) return report(FERRY_EINVAL, "unknown kind");
    if (!(base > 0.0) || !(stretch > 0.0) || !std::isfinite(base) || !std::isfinite(stretch))
      return report(FERRY_EINVAL, "base and stretch must be positive");
    if (kind == FERRY_ROPE_BASE && rot_dim < 4) return report(FERRY_EINVAL, "FERRY_ROPE_BASE needs rot_dim of 4 or more");
    if (kind == FERRY_ROPE_PARTS && !(trained_ctx > 0.0 && fast > slow && std::isfinite(trained_ctx + fast - slow)))
      return report(FERRY_EINVAL, "FERRY_ROPE_PARTS needs trained_ctx > 0 and fast > slow, all finite");
    if (kind == FERRY_ROPE_BASE) base *= std::pow(stretch, (double)rot_dim / (rot_dim - 2));
    for (int i = 0; i < rot_dim / 2; ++i) {
      const double f = std::pow(base, -2.0 * i / rot_dim);
      double x = f;
      if (kind == FERRY_ROPE_LINEAR) x = f / stretch;
      if (kind == FERRY_ROPE_PARTS) {
        const double turns = trained_ctx * f / (2.0 * M_PI);
        const double keep = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
        x = f * keep + f / stretch * (1.0 - keep);
      }
      out[i] = x;
    }
    return FERRY_OK;
  });
}

}  // extern "C"
