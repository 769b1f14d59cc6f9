// pages_drafts.hip -- drafted tokens in the paged KV cache: their ancestors and
// positions from their parents (ferry_pages_tree), and what the model agrees with
// moved up behind the context (ferry_pages_accept).
#include <algorithm>

#include "pages.hpp"

using namespace ferry_amd;

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ inline int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// ---- tree ------------------------------------------------------------------------
struct TreeArgs {
  int n_req, n_tokens, words;
  const int32_t* lanes;
  const int32_t* q_start;
  const int32_t* parent;
  uint64_t* tree;
  int32_t* at;
  int32_t* place;
  int32_t* lane;
};

__device__ inline void tree_row(const TreeArgs& a, int64_t t, int at, int place, int lane) {
  if (a.at) a.at[t] = at;
  if (a.place) a.place[t] = place;
  if (a.lane) a.lane[t] = lane;
}

__device__ inline void no_row(const TreeArgs& a, int64_t t) {
  tree_row(a, t, 0, -1, -1);
  for (int w = 0; w < a.words; ++w) a.tree[t * a.words + w] = 0;
}

// A workgroup per request, a token per thread (`blockDim.x` of them at a time).  Parents come
// before their children, so of a token's ancestors those in its own 64 are found by its
// wavefront in six rounds (each takes over what the ancestor reached so far has, and its
// reach); the topmost of these has its parent among earlier tokens, and what that one found
// is the next word that is not 0.  So all words of all tokens are made at once, in as many
// steps as there are words, from LDS; only tokens behind the first blockDim.x read back
// rows that are written.  Bound by latency: the offsets, the lane, its length and the parents
// are dependent reads; 256 requests of 150 to 300 tokens write 3 MB in 5.3 us (8.0 with a
// wavefront per request that goes on 64 by 64).  The last of the rounds pads the tokens of
// no request.
constexpr int kTreeThreads = 1024, kTreeGroups = 1 << 16;
__global__ __launch_bounds__(kTreeThreads) void k_tree(PageView v, TreeArgs a) {
  __shared__ uint64_t found[kTreeThreads];  // of a token's own 64
  __shared__ int before[kTreeThreads];      // the parent of the topmost of these, -1: none
  const int tid = threadIdx.x, l = tid & 63, threads = blockDim.x;
  auto token_of = [&](int r) { return a.q_start ? clampi(a.q_start[r], 0, a.n_tokens) : min(r, a.n_tokens); };
  for (int64_t r64 = blockIdx.x; r64 <= a.n_req; r64 += gridDim.x) {
    const int r = (int)r64;
    if (r == a.n_req) {
      const int first = token_of(0), end = max(first, token_of(a.n_req));
      for (int64_t i = tid; i < (int64_t)first + a.n_tokens - end; i += threads) no_row(a, i < first ? i : i - first + end);
      break;
    }
    const int t0 = token_of(r), n = max(0, token_of(r + 1) - t0), lane = a.lanes[r];
    const int len = lane >= 0 && lane < v.n_lanes ? v.len[lane] : 0;
    const bool held = len >= n && len <= v.max_pages * kPageTokens;
    const bool fine = lane >= 0 && lane < v.n_lanes && held;
    bool bad = lane != -1 && !fine;
    if (a.q_start) bad |= a.q_start[r] < 0 || a.q_start[r] > a.q_start[r + 1] || a.q_start[r + 1] > a.n_tokens;
    if (n > 64 * a.words) bad = true;
    for (int b0 = 0; b0 < n; b0 += threads) {
      const int c = b0 + tid, c0 = c & ~63;  // (blocks are whole 64s)
      const int64_t t = (int64_t)t0 + c;
      if (!fine) {
        if (c < n) no_row(a, t);
        continue;
      }
      int p = c < n ? a.parent[t] : -1;
      if (p < -1 || p >= c) {
        bad |= c < n;
        p = -1;
      }
      uint64_t mine = 1ull << l;
      int up = p >= c0 ? p - c0 : l;  // the ancestor reached, itself at the end
#pragma unroll
      for (int i = 0; i < 6; ++i) {
        mine |= __shfl(mine, up);
        up = __shfl(up, up);
      }
      int e = __shfl(p, up);
      __threadfence_block();
      __syncthreads();  // rows of the blocks before are written, what they found is read
      found[tid] = mine, before[tid] = e;
      __syncthreads();
      if (c >= n) continue;
      int deep = 0;
      uint64_t* row = a.tree + t * a.words;
      for (int w = c >> 6; w >= 0; --w) {  // words above are 0
        uint64_t x = mine;
        if (w != c >> 6) {
          x = 0;
          if (e >= b0 && e >> 6 == w) x = found[e - b0], e = before[e - b0];
          else if (e >= 0 && e < b0 && w < a.words) x = a.tree[((int64_t)t0 + e) * a.words + w];
        }
        deep += __popcll(x);
        if (w < a.words) row[w] = x;
      }
      for (int w = (c >> 6) + 1; w < a.words; ++w) row[w] = 0;
      tree_row(a, t, len - n + deep - 1, len - n + c, lane);
    }
    if (__builtin_amdgcn_ballot_w64(bad) && l == 0) set_error(v.error, FERRY_ERANGE);
    __syncthreads();  // the next request's tokens take the places
  }
}

// ---- accept ----------------------------------------------------------------------
struct AcceptArgs {
  int n_req, n_tokens;
  const int32_t* lanes;
  const int32_t* q_start;
  const int32_t* parent;
  const int32_t* draft;
  const int32_t* chosen;
  int32_t* path;
  int32_t* kept;
  int32_t* next;
};
constexpr int kThreads = 256;
constexpr int kMoves = 512;  // tokens moved at once
constexpr int kAhead = 4;    // ... of a thread on their way

// Whether a call can be made; every thread of the workgroup gets the answer.
__device__ inline bool accept_fine(const PageView& v, const AcceptArgs& a) {
  __shared__ uint32_t bits[kMaxLanes / 32];
  __shared__ int bad;
  for (int i = threadIdx.x; i < (v.n_lanes + 31) / 32; i += kThreads) bits[i] = 0;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  for (int r = threadIdx.x; r < a.n_req; r += kThreads) {
    const int lane = a.lanes[r], t0 = a.q_start ? a.q_start[r] : r, t1 = a.q_start ? a.q_start[r + 1] : r + 1;
    bool ok = t0 >= 0 && t0 <= t1 && t1 <= a.n_tokens;
    if (lane != -1) {
      ok = ok && name_lane(bits, lane, v.n_lanes);
      if (ok) {
        const int len = v.len[lane];
        ok = len >= t1 - t0 && len <= v.max_pages * kPageTokens;
      }
    }
    if (!ok) bad = 1;
  }
  __syncthreads();
  return !bad;
}

// A request's tokens that stay, one after the other: a token's child comes behind it,
// so its wavefront goes over the tokens once, 64 in its lanes' registers.
struct Walk {
  int n, now, c0;
  int parent, draft, chosen;  // of token c0 + lane
  __device__ void load(const AcceptArgs& a, int64_t t0) {
    const int c = c0 + (int)threadIdx.x;
    parent = -2, draft = chosen = 0;
    if (c < n) {
      parent = a.parent ? a.parent[t0 + c] : c - 1;
      draft = a.draft[t0 + c], chosen = a.chosen[t0 + c];
    }
  }
  __device__ int choice() const { return __builtin_amdgcn_readlane(chosen, now - c0); }  // after `now`
};

// 16 codes of scale `from` as codes of scale `to`.
__device__ inline u32x4 rescaled(u32x4 x, float from, float to) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int c = (int)x[w];
    float y[4] = {__builtin_amdgcn_cvt_f32_fp8(c, 0), __builtin_amdgcn_cvt_f32_fp8(c, 1),
                  __builtin_amdgcn_cvt_f32_fp8(c, 2), __builtin_amdgcn_cvt_f32_fp8(c, 3)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float z = y[i] * from / to;
      y[i] = z == z ? __builtin_amdgcn_fmed3f(z, -448.0f, 448.0f) : z;
    }
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    x[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  }
  return x;
}

// Workgroups (x: requests, y: parts of the layers' heads).  Each checks the call and walks
// its request by itself; the first of a request writes the results.  A thread
// then moves 16 bytes of each kept token's K or V, in their order: a token only moves
// towards the lane's start and past no later one, so what is read ahead is not yet written
// over.  Bound by latency in ordinary calls: the check, the walk, the table and the move
// are dependent reads.
template <bool F8>
__global__ __launch_bounds__(kThreads) void k_accept(PageView v, Work w, AcceptArgs a) {
  __shared__ int node[kMoves];  // the request's kept tokens from the `from`-th on
  __shared__ uint32_t src[kMoves], dst[kMoves];  // their pages, kNone: not moved
  __shared__ int count, over, following;
  const int tid = threadIdx.x;
  const bool fine = accept_fine(v, a);
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) {
    w.plan->ok = fine;
    if (!fine) set_error(v.error, FERRY_EINVAL);
  }
  if (!fine) return;
  const int words = (int)(v.bb / 32);           // 16-byte words of a record's K
  const int per = words / kPageTokens * 2;      // ... of a token's K and V: a thread each
  const int sets = kThreads / per, part = tid % per, value = part / (per / 2), piece = part % (per / 2);
  for (int r = blockIdx.x; r < a.n_req; r += gridDim.x) {
    const int lane = a.lanes[r], t0 = a.q_start ? a.q_start[r] : r, n = (a.q_start ? a.q_start[r + 1] : r + 1) - t0;
    const bool writes = blockIdx.y == 0;
    if (lane < 0 || n == 0) {
      if (writes) {
        for (int i = tid; i < n; i += kThreads) a.path[(int64_t)t0 + i] = -1;
        if (tid == 0) a.kept[r] = 0, a.next[r] = -1, w.had[r] = lane < 0 ? 0u : (uint32_t)v.len[lane];
      }
      continue;
    }
    const int base = v.len[lane] - n;
    const uint32_t* row = v.table + (uint64_t)lane * v.max_pages;
    Walk k{n, 0, 0, 0, 0, 0};
    if (tid < 64) k.load(a, t0);
    for (int from = 0;;) {
      __syncthreads();  // the last moves are made
      if (tid < 64) {
        int m = 0;
        if (from == 0) {
          if (tid == 0) node[0] = 0;
          m = 1;
        }
        int want = k.choice();
        while (m < kMoves && k.c0 < n) {
          const int c = k.c0 + tid;
          const uint64_t hit = __builtin_amdgcn_ballot_w64(c > k.now && k.parent == k.now && k.draft == want);
          if (hit) {
            k.now = k.c0 + __builtin_ctzll(hit);
            want = k.choice();
            if (tid == 0) node[m] = k.now;
            ++m;
          } else {
            k.c0 += 64;
            k.load(a, t0);
          }
        }
        if (tid == 0) count = m, over = k.c0 >= n, following = want;
      }
      __syncthreads();
      const int m = count;
      for (int i = tid; i < m; i += kThreads) {
        const int c = node[i], to = base + from + i, at = base + c;
        src[i] = dst[i] = kNone;
        if (writes) a.path[(int64_t)t0 + from + i] = t0 + c;
        if (c == from + i) continue;
        const uint32_t s = row[at / kPageTokens], d = row[to / kPageTokens];
        if (s >= (uint32_t)v.n_pages || d >= (uint32_t)v.n_pages || v.refs[d] > 1) {
          if (writes) set_error(v.error, FERRY_ESTATE);
        } else {
          src[i] = s, dst[i] = d;
        }
      }
      __syncthreads();
      const int records = v.L * v.H;
      for (int g = blockIdx.y * sets + tid / per; g < records; g += gridDim.y * sets) {
        const int layer = g / v.H, head = g - layer * v.H;
        for (int i0 = 0; i0 < m; i0 += kAhead) {
          u32x4 x[kAhead];
          u32x4* to[kAhead];
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            const int i = i0 + j;
            to[j] = nullptr;
            if (i >= m || dst[i] == kNone) continue;
            const uint64_t s = v.record(layer, src[i], head), d = v.record(layer, dst[i], head);
            auto place = [&](uint64_t record, int tok) {
              return reinterpret_cast<u32x4*>(v.pool + record * v.bb) + value * words +
                     tok % kPageTokens * (per / 2) + piece;
            };
            to[j] = place(d, base + from + i);
            x[j] = *place(s, base + node[i]);
            if constexpr (F8) {
              const float f = v.scales[2 * s + value], e = v.scales[2 * d + value];
              if (__builtin_bit_cast(uint32_t, f) != __builtin_bit_cast(uint32_t, e)) x[j] = rescaled(x[j], f, e);
            }
          }
#pragma unroll
          for (int j = 0; j < kAhead; ++j)
            if (to[j]) *to[j] = x[j];
        }
      }
      from += m;
      if (over) {
        if (writes) {
          for (int i = from + tid; i < n; i += kThreads) a.path[(int64_t)t0 + i] = -1;
          if (tid == 0) a.kept[r] = from, a.next[r] = following, w.had[r] = (uint32_t)(base + from);
        }
        break;
      }
    }
    __syncthreads();  // `over` and `following` are the next request's
  }
}

// The lanes get their new lengths, once all workgroups have read the old ones and the
// pages behind them.
__global__ __launch_bounds__(kThreads) void k_accept_trim(PageView v, Work w, const int32_t* __restrict__ lanes, int n) {
  if (!w.plan->ok) return;
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int lane = lanes[i];
    if (lane < 0) continue;
    const int held = v.len[lane], left = (int)w.had[i];
    drop_pages(v, lane, held, left);
    __syncthreads();  // all have read the length
    if (threadIdx.x == 0) v.len[lane] = left;
  }
}

bool meet(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + b_bytes && y < x + a_bytes;
}

}  // namespace

extern "C" {

int ferry_pages_tree(const ferry_pages* p, const ferry_tree* a, void* stream) {
  return entry([&]() -> int {
    PageView v;
    if (int rc = page_geometry(p, &v)) return rc;
    if (!a) return report(FERRY_EINVAL, "null args");
    if (a->n_req < 0 || a->n_tokens < 0) return report(FERRY_EINVAL, "n_req and n_tokens must not be negative");
    if (a->tree_words < 1 || a->tree_words > kTreeWords) return report(FERRY_EINVAL, "tree_words must be 1..64");
    if (!a->q_start && a->n_tokens != a->n_req)
      return report(FERRY_EINVAL, "without q_start a request has one token");
    if (a->n_tokens == 0) return FERRY_OK;
    if (int rc = page_buffers(p, false)) return rc;
    const uint64_t rows = (uint64_t)a->n_tokens * 4;
    struct Buffer {
      const void* p;
      uint64_t bytes;
      const char* name;
    };
    const Buffer in[] = {{a->lanes, (uint64_t)a->n_req * 4, "lanes"}, {a->q_start, (uint64_t)a->n_req * 4 + 4, "q_start"},
                         {a->parent, rows, "parent"}, {p->len, (uint64_t)p->n_lanes * 4, "len"}};
    const Buffer out[] = {{a->tree, 2 * rows * a->tree_words, "tree"}, {a->at, rows, "at"}, {a->place, rows, "place"},
                          {a->lane, rows, "lane"}};
    if (a->n_req)
      if (int rc = check_on(a->lanes, "lanes", p->device)) return rc;
    if (int rc = check_all({{a->parent, "parent"}, {a->tree, "tree"}}, p->device)) return rc;
    if (reinterpret_cast<uintptr_t>(a->tree) % 8) return report(FERRY_EINVAL, "tree must be 8-byte aligned");
    if (a->q_start)
      if (int rc = check_on(a->q_start, "q_start", p->device)) return rc;
    for (const Buffer& o : out) {
      if (!o.p) continue;
      if (int rc = check_on(o.p, o.name, p->device)) return rc;
      for (const Buffer& i : in)
        if (meet(o.p, o.bytes, i.p, i.bytes)) return report(FERRY_EINVAL, std::string(o.name) + " overlaps " + i.name);
      for (const Buffer& q : out)
        if (&q != &o && meet(o.p, o.bytes, q.p, q.bytes))
          return report(FERRY_EINVAL, std::string(o.name) + " overlaps " + q.name);
    }
    OnDevice on(p->device);
    if (!on.ok()) return report(FERRY_EHIP, "cannot use the cache's GPU");
    const TreeArgs d{a->n_req, a->n_tokens, a->tree_words, a->lanes, a->q_start, a->parent,
                     a->tree, a->at, a->place, a->lane};
    const int groups = (int)std::min<int64_t>((int64_t)a->n_req + 1, kTreeGroups);
    k_tree<<<groups, std::min(64 * a->tree_words, kTreeThreads), 0, static_cast<hipStream_t>(stream)>>>(v, d);
    return launched("ferry_pages_tree");
  });
}

int ferry_pages_accept(const ferry_pages* p, const ferry_accept* a, void* stream) {
  return entry([&]() -> int {
    PageView v;
    Work w;
    if (int rc = page_geometry(p, &v)) return rc;
    if (!a) return report(FERRY_EINVAL, "null args");
    if (a->n_tokens < 0) return report(FERRY_EINVAL, "n_tokens must not be negative");
    if (!a->q_start && a->n_tokens != a->n_req)
      return report(FERRY_EINVAL, "without q_start a request has one token");
    if (int rc = manage(p, a->n_req, &v, &w)) return rc;
    if (a->n_req == 0) return FERRY_OK;
    struct Buffer {
      const void* p;
      uint64_t entries;
      const char* name;
    };
    const uint64_t rows = a->n_tokens, reqs = a->n_req;
    const Buffer in[] = {{a->lanes, reqs, "lanes"}, {a->q_start, reqs + 1, "q_start"}, {a->parent, rows, "parent"},
                         {a->draft, rows, "draft"}, {a->chosen, rows, "chosen"}};
    const Buffer out[] = {{a->path, rows, "path"}, {a->kept, reqs, "kept"}, {a->next, reqs, "next"}};
    for (const Buffer& b : in) {
      const bool may_lack = b.p == nullptr && (&b == &in[1] || &b == &in[2] || b.entries == 0);
      if (!may_lack)
        if (int rc = check_list(p, b.p, b.name, (int)b.entries)) return rc;
    }
    for (const Buffer& o : out) {
      if (!o.p && o.entries == 0) continue;
      if (int rc = check_list(p, o.p, o.name, (int)o.entries)) return rc;
      for (const Buffer& i : in)
        if (meet(o.p, 4 * o.entries, i.p, 4 * i.entries))
          return report(FERRY_EINVAL, std::string(o.name) + " overlaps " + i.name);
      for (const Buffer& q : out)
        if (&q != &o && meet(o.p, 4 * o.entries, q.p, 4 * q.entries))
          return report(FERRY_EINVAL, std::string(o.name) + " overlaps " + q.name);
    }
    OnDevice on(p->device);
    if (!on.ok()) return report(FERRY_EHIP, "cannot use the cache's GPU");
    const AcceptArgs d{a->n_req, a->n_tokens, a->lanes, a->q_start, a->parent, a->draft, a->chosen,
                       a->path, a->kept, a->next};
    hipStream_t s = static_cast<hipStream_t>(stream);
    // 8 workgroups a CU, and of a request no more than it has records for
    const int sets = kThreads / (int)(v.bb / 16 / kPageTokens);
    const int64_t groups = ((int64_t)v.L * v.H + sets - 1) / sets, most = 8l * gpu_cus(p->device);
    const int x = (int)std::min<int64_t>(a->n_req, most);
    const int y = (int)std::max<int64_t>(1, std::min(groups, most / x));
    if (p->dtype == FERRY_FP8_E4M3) k_accept<true><<<dim3(x, y), kThreads, 0, s>>>(v, w, d);
    else k_accept<false><<<dim3(x, y), kThreads, 0, s>>>(v, w, d);
    k_accept_trim<<<x, kThreads, 0, s>>>(v, w, a->lanes, a->n_req);
    return launched("ferry_pages_accept");
  });
}

}  // extern "C"
