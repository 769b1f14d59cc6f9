// pages_attn.hip -- attention of new query tokens over the pages of their lanes
// (ferry_pages_attend), with pages that a group of requests shares read once.
//
// Rows and segments.  A row is one query token and one query head; the G =
// q_heads / kv_heads heads of a kv head attend to the same K and V, so the rows of
// consecutive tokens, [token][G], are consecutive columns of the same products.
// A segment is a run of rows and the pages they all attend to: the shared pages of
// a group with the rows of all its members, or the remaining pages of one request
// with its own rows.  A row's output joins its (at most two) segments.
//
// Schedule.  A segment's rows are cut into tiles (16, 32 or 128 rows), its pages into
// steps of four; a unit of work is one step of one tile of one kv head.  All units
// of the call, in the order (segment, kv head, tile, step), are cut into equal runs,
// one per workgroup of a grid that fills the GPU once: ragged lengths balance, and
// a long axis is split where there are few rows.  Every workgroup finds its run from
// the lengths by itself (a prefix sum over the segments), so nothing is planned on
// the host and a captured call follows the lengths of its replay.  A tile that one
// workgroup finishes alone, of a row with one segment, is written out; otherwise its
// (max, sum, output) in fp32 go to scratch, and k_attend_join adds them up in order.
// The result depends on the lengths and on the number of CUs, not on timing.
//
// Softmax.  One pass with a reference m and the sum of the weights 2^(score - m) of each
// row, in base 2.  m is raised only when a score exceeds it by kMost, and then so that this
// one's weight is 2^kTop: weights are at most 2^kMost and the accumulator is rarely
// rescaled.  Scores, references, sums and the accumulator are fp32; weights are rounded to
// the operand type for the second product.  That is half a step relative (2^-8 of a
// weight in bf16, 2^-11 in fp16), as large as the rounding of the output, where the type
// holds them as normal numbers: bf16 has fp32's range, but fp16 ends at 2^-14, so there
// kTop is 7 and the row's largest weight is 2^7 .. 2^15.  A weight below 2^-21 of the largest
// is then rounded to a multiple of 2^-31 of it, which for n tokens moves the output by
// n 2^-32 of their values at most: as much as its own rounding from 2^21 tokens on.
// A second product with what the rounding took would keep 16 bits of bf16 weights.  In
// tiles of 128 rows, bound by the matrix instructions, it costs 13 to 31 % (samples 100 us
// for 89, chunks 640 for 487); in tiles of 16, bound by bytes, nothing (long 153), but
// there the rest, which may be 0 or negative, would meet an infinite value and make NaN of
// it.  So weights are as exact as the output that they make, in every form.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_common.hpp"
#include "pages.hpp"

using namespace ferry_amd;

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kStep = 4;           // pages per step
constexpr int kWide = 128;         // rows of the widest tile
constexpr int kGroupsInLds = 512;  // groups whose offsets are looked up in LDS
constexpr int kPad = 132;          // floats per row of the merge buffer
constexpr int kPerCu = 2;          // workgroups per CU

struct AttendArgs {
  int n_req, n_tokens, n_groups, Hq, G;
  float scale;
  const int32_t* lanes;
  const int32_t* q_start;
  const int32_t* group_start;
  const int32_t* shared;
  const void* q;
  void* out;
  float* lse;
  int64_t qs[2], os[2];
  int aligned;  // q and out rows are 16-byte aligned
  uint32_t g_mul;  // row / G = row * g_mul >> g_shift, for rows below 2^30
  int g_shift;
};

// Where a row's parts of one segment are (per kv head).
struct Where {
  int first;  // first workgroup of its tile
  int count;  // workgroups that share the tile; 1: the row's own place; 0: written out
  int row;    // row within the tile
  int has;    // own pages only: bit 0: the row has shared pages too, bit 1: it sees a token
};

// Scratch.  rows = n_tokens * G.
struct Scratch {
  Where* where;    // [2 (shared, own)][H][rows]
  float* part_ml;  // [2 * grid][tile rows][2]: the first and the last tile of each workgroup
  float* part_o;   // [2 * grid][tile rows][128]
  float* row_ml;   // [2][H][rows][2]: whole tiles of rows with two segments
  float* row_o;    // [2][H][rows][128]
  int tile_rows;   // rows per part
};

// ---- element types -------------------------------------------------------------
template <int DT>
struct Kv {
  static constexpr bool F8 = DT == FERRY_FP8_E4M3, F32 = DT == FERRY_F32;
  static constexpr bool BF = DT == FERRY_BF16 || F8;  // operand type of the products
  static constexpr int ES = F32 ? 4 : F8 ? 1 : 2;
  static constexpr int ROW = kPageDim * ES;          // bytes of a token's K or V
  static constexpr int HALF = kPageTokens * ROW;     // bytes of a record's K
  static constexpr int NK = ROW / 64;                // 16-byte K words per lane and page
  static constexpr int VW = 2 * ES;                  // dwords of V per token and lane
  // log2 of the largest weight, and of the largest when the reference is raised
  static constexpr float kMost = DT == FERRY_F16 ? 15.0f : 8.0f, kTop = DT == FERRY_F16 ? 7.0f : 0.0f;
};

template <bool BF>
__device__ inline uint32_t pack2(float a, float b) {
  const f32x2 x = {a, b};
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
}

// 4 E4M3 codes -> 4 exact bf16 values
__device__ inline u32x2 e4m3x4_to_bf16(uint32_t w) {
  const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
  const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
  return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

template <bool BF>
__device__ inline f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {  // 16 x 16 x 32
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool BF>
__device__ inline f32x4 mma16h(u32x2 a, u32x2 b, f32x4 c) {  // 16 x 16 x 16
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, a),
                                                     __builtin_bit_cast(i16x4, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                                 __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}
template <bool BF>
__device__ inline f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {  // 32 x 32 x 16
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// What weights are taken against: the reference m, or 0 while no score was finite.
__device__ inline float against(float m) { return m == -INFINITY ? 0.0f : m; }

// One K or V element of a record as fp32 (fp8: the code's value), one of q.
template <int DT>
__device__ inline float k_elem(const uint8_t* p, int tok, int d) {
  const int i = tok * kPageDim + d;
  if constexpr (DT == FERRY_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (DT == FERRY_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  else if constexpr (DT == FERRY_BF16) return bits_f32((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
  else return bits_f32(e4m3x4_to_bf16(p[i])[0] << 16);
}
template <int DT>
__device__ inline float v_elem(const uint8_t* rec, int tok, int d) {
  return k_elem<DT>(rec + Kv<DT>::HALF, tok, d);
}
template <int DT>
__device__ inline float q_elem(const void* q, int64_t i) {
  if constexpr (DT == FERRY_F32) return static_cast<const float*>(q)[i];
  else if constexpr (DT == FERRY_F16) return (float)static_cast<const _Float16*>(q)[i];
  else return bits_f32((uint32_t)static_cast<const uint16_t*>(q)[i] << 16);
}
__device__ inline bool finite(float x) { return (f32_bits(x) & 0x7F800000u) != 0x7F800000u; }

// Whether a dword of two 16-bit operand values (or one fp32) holds what is not finite.
template <int DT>
__device__ inline bool not_finite(uint32_t w) {
  if constexpr (Kv<DT>::F32) return (w & 0x7F800000u) == 0x7F800000u;
  constexpr uint32_t e = Kv<DT>::BF ? 0x7F80u : 0x7C00u;
  return (w & e) == e || (w >> 16 & e) == e;
}

__device__ inline int token_of_row(const AttendArgs& a, int row) {
  return (int)((uint64_t)(uint32_t)row * a.g_mul >> a.g_shift);
}

// ---- segments -------------------------------------------------------------------
struct Seg {
  int own;        // 1: one request's own pages, 0: a group's shared pages
  int row0, rows;  // its rows
  int tile, tiles;  // rows per tile, tiles
  int p0, p1;     // pages [p0, p1) of the lane's table
  int base, len;  // own: the first row's token sees `base` tokens; tokens of the lane
  int lane;       // whose table is read; -1: no pages
  int req;        // request, or group
  int tok0;       // first row's token
  int group;      // own: the group that the request belongs to, -1: none
};

// Rows per tile: what each wavefront can hold where there are few rows (the tile is then
// bound by its pages' bytes and the wavefronts share out the pages), else the 128 rows
// of four wavefronts that share pages in LDS.  16 agents of 4 rows on 517 shared pages:
// 134 us in the 128-row form, 189 in a 64-row form of the first kind; 8 agents: 181 us
// with 32 rows, 227 in the 128-row form.  fp32 pages have the 16-row form only.
template <int DT>
__device__ inline int tile_rows(int rows) {
  if (Kv<DT>::F32 || rows <= 16) return 16;
  return rows <= 32 ? 32 : kWide;
}

__device__ inline int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
__device__ inline int pages_of(int tokens) { return (tokens + kPageTokens - 1) / kPageTokens; }

// First row's token of request r (r = n_req: the end), made to stay in the batch.
__device__ inline int token_of(const AttendArgs& a, int r) {
  return a.q_start ? clampi(a.q_start[r], 0, a.n_tokens) : r;
}
__device__ inline int lane_of(const PageView& v, const AttendArgs& a, int r) {
  const int lane = a.lanes[r];
  return lane >= 0 && lane < v.n_lanes ? lane : -1;
}
__device__ inline int len_of(const PageView& v, int lane) {
  return lane < 0 ? 0 : clampi(v.len[lane], 0, v.max_pages * kPageTokens);
}

// Pages that the requests [b, e) of a group attend to together: none where they have
// a widest tile's rows each, and would read the pages once per tile in any case.  Alone,
// their rows have one segment and need no join.
template <int DT>
__device__ inline int group_pages(const PageView& v, const AttendArgs& a, int b, int e, int shared) {
  constexpr int kRows = Kv<DT>::F32 ? 16 : kWide;
  const int64_t rows = (int64_t)(token_of(a, e) - token_of(a, b)) * a.G;
  return rows >= (int64_t)kRows * (e - b) ? 0 : clampi(shared, 0, v.max_pages);
}

// Shared pages of request r: those of the last group that starts at or before it,
// if that has not ended.
template <int DT>
__device__ inline int shared_of(const PageView& v, const AttendArgs& a, const int* gs, const int* gp, int r,
                                int* group) {
  *group = -1;
  if (a.n_groups == 0 || gs[0] > r) return 0;
  int lo = 0, hi = a.n_groups - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (gs[mid] <= r) lo = mid; else hi = mid - 1;
  }
  const int b = clampi(gs[lo], 0, a.n_req), e = clampi(gs[lo + 1], b, a.n_req);
  if (r >= e) return 0;
  *group = lo;
  return group_pages<DT>(v, a, b, e, gp[lo]);
}

// Segment s: groups first, then requests.  gs, gp: the groups' offsets and pages.
template <int DT>
__device__ inline Seg segment(const PageView& v, const AttendArgs& a, const int* gs, const int* gp, int s) {
  Seg g;
  if (s < a.n_groups) {
    const int b = clampi(gs[s], 0, a.n_req), e = clampi(gs[s + 1], b, a.n_req);
    g.own = 0, g.req = s, g.p0 = 0, g.p1 = group_pages<DT>(v, a, b, e, gp[s]);
    g.lane = -1, g.base = g.len = 0;
    for (int r = b; r < e && g.lane < 0; ++r) g.lane = lane_of(v, a, r);
    const int t0 = token_of(a, b), t1 = max(t0, token_of(a, e));
    g.tok0 = t0, g.row0 = t0 * a.G, g.group = s;
    g.rows = g.p1 > 0 && g.lane >= 0 ? (t1 - t0) * a.G : 0;
  } else {
    const int r = s - a.n_groups, t0 = token_of(a, r), t1 = max(t0, token_of(a, r + 1));
    g.own = 1, g.req = r, g.lane = lane_of(v, a, r), g.len = len_of(v, g.lane);
    g.tok0 = t0, g.row0 = t0 * a.G, g.rows = (t1 - t0) * a.G;
    g.base = g.len - (t1 - t0) + 1;
    const int shared = shared_of<DT>(v, a, gs, gp, r, &g.group);
    g.p0 = g.lane < 0 ? 0 : shared;
    g.p1 = max(g.p0, pages_of(g.len));
  }
  g.tile = tile_rows<DT>(g.rows);
  g.tiles = (g.rows + g.tile - 1) / g.tile;
  return g;
}

// Steps of tile j: up to the last token its last row sees, and at least one, so
// that every tile has a workgroup that writes its rows.
__device__ inline int tile_steps(const AttendArgs& a, const Seg& g, int j) {
  int p1 = g.p1;
  if (g.own) {
    const int last = clampi(g.base + token_of_row(a, min((j + 1) * g.tile, g.rows) - 1), 0, g.len);
    p1 = min(p1, pages_of(last));
  }
  return max(1, (p1 - g.p0 + kStep - 1) / kStep);
}
// Units of work: step_units() for a step, tile_units() for a tile's beginning and end.
// Step i of a tile belongs to the workgroup whose run holds the first of its units.
// A unit is a fifth of a microsecond of a workgroup, measured in batches of all forms
// (samples of one prompt, agents in groups, prompts in chunks) on a full GPU.
template <int DT>
__device__ constexpr int step_units(int tile) {
  constexpr bool F8 = Kv<DT>::F8;
  return Kv<DT>::F32 ? 16 : tile == 16 ? (F8 ? 4 : 8) : tile == 32 ? (F8 ? 7 : 11) : (F8 ? 11 : 9);
}
template <int DT>
__device__ constexpr int tile_units(int tile) { return tile == 16 ? 26 : tile == 32 ? 35 : 65; }
template <int DT>
__device__ inline int tile_work(const AttendArgs& a, const Seg& g, int j) {
  return tile_steps(a, g, j) * step_units<DT>(g.tile) + tile_units<DT>(g.tile);
}
// ... of all tiles of a segment, per kv head
template <int DT>
__device__ inline uint64_t seg_work(const AttendArgs& a, const Seg& g) {
  if (!g.own) return (uint64_t)g.tiles * tile_work<DT>(a, g, 0);
  uint64_t n = 0;
  for (int j = 0; j < g.tiles; ++j) n += tile_work<DT>(a, g, j);
  return n;
}

// The thread's number, anew: what a tile's code derives from it is then computed for
// each tile.  Otherwise the compiler computes all lane addresses of all tile forms
// once, before the loop over the tiles, and keeps them in spilled registers.
__device__ inline int this_thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// What is `at` bytes behind a scalar address in global memory.
template <class T>
__device__ inline T global_at(const void* base, uint32_t at) {
  typedef __attribute__((address_space(1))) const uint8_t* Bytes;
  return *(__attribute__((address_space(1))) const T*)((Bytes)base + at);
}
template <class T>
__device__ inline T stream_at(const void* base, uint32_t at) {  // not kept in the caches
  typedef __attribute__((address_space(1))) const uint8_t* Bytes;
  return __builtin_nontemporal_load((__attribute__((address_space(1))) const T*)((Bytes)base + at));
}

// ---- one tile --------------------------------------------------------------------
// What a tile's products need, the same for all threads.
struct Tile {
  const uint32_t* table;  // the lane's pages
  const uint8_t* base;    // page 0's record of this layer and kv head
  const float* scales;    // ... and its scales (fp8)
  uint32_t page_bytes;    // from one page's record to the next one's
  int row0, rows;  // first row, rows (<= the tile's width)
  int h;           // kv head
  int p0, p1;      // pages of this workgroup's steps of it
  int lim_lo, lim_hi;  // tokens that its least and its most seeing row see
};

// A record that is the same for all lanes, in scalar registers.
template <class T>
__device__ inline T uniform(const T& x) {
  static_assert(sizeof(T) % 4 == 0, "whole words");
  int w[sizeof(T) / 4];
  __builtin_memcpy(w, &x, sizeof(T));
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); ++i) w[i] = first_lane_i(w[i]);
  T y;
  __builtin_memcpy(&y, w, sizeof(T));
  return y;
}

// A segment in the order of all units.
struct SegAt {
  Seg g;
  uint64_t at, work;  // its first unit; units of all its tiles (per kv head)
};
constexpr int kListed = 32;

// FORMS: 1: 16-row tiles only, 2: 32-row tiles too, 3: 128-row tiles too.
template <int FORMS>
struct Shared {
  struct Kv {
    uint8_t k[2][kStep * 4096], v[2][kStep * 4096];
  };
  struct None {};
  union {
    float merge[4 * (FORMS == 1 ? 16 : 32) * kPad];  // [wavefront][row][dim]: accumulators to be joined
    std::conditional_t<FORMS == 3, Kv, None> kv;     // two steps' tokens, chunks swizzled
  };
  float ml[4][32][2];
  int lim[kWide];  // tokens that each row sees
  int lim_lo, lim_hi;
  int odd[3];      // a step's V holds what is not finite (step s: place s % 3)
  int left_out;    // the tile has pages that were left out for that
  int gs[kGroupsInLds + 1], gp[kGroupsInLds];
  uint64_t sums[kThreads / 64];
  int seg;          // first segment of this workgroup's run
  int gl[kGroupsInLds];  // least number of tokens that a row of a group sees
  SegAt list[kListed];  // consecutive segments of the run
};

// 8 query values of a row as two 16-bit values per dword, times the sign of the
// scale (scores are then compared before they are scaled).
__device__ inline u32x4 load_q8(const uint16_t* p, bool aligned, uint32_t sign) {
  u32x4 x;
  if (aligned) {
    x = *reinterpret_cast<const u32x4*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] ^= sign;
  return x;
}

// Element offset of row `row`'s query (or output) in a tensor of strides s.
__device__ inline int64_t row_at(const AttendArgs& a, const int64_t (&s)[2], int row, int h) {
  const int t = token_of_row(a, row);
  return t * s[0] + (int64_t)(h * a.G + (row - t * a.G)) * s[1];
}

__device__ inline uint32_t checked_page(const PageView& v, uint32_t id) {
  if (id < (uint32_t)v.n_pages) return id;
  set_error(v.error, FERRY_ERANGE);
  return 0;
}

// The K and V words of one page that a lane holds for the 16-column products.
template <int DT>
struct PageRegs {
  u32x4 k[Kv<DT>::NK];
  uint32_t v[4][Kv<DT>::VW];
  float ks, vs;
};

// The address is a scalar and a lane's 32-bit offset.
template <int DT>
__device__ inline void load_page(const Tile& t, int kv_heads, uint32_t page, int l, PageRegs<DT>& r) {
  using K = Kv<DT>;
  const uint32_t n = l & 15, grp = l >> 4;
  const uint8_t* kp = t.base + (uint64_t)page * t.page_bytes;
  const uint8_t* vp = kp + K::HALF;
  const uint32_t k_at = n * K::ROW + grp * 16, v_at = 4 * grp * K::ROW + n * (8 * K::ES);
#pragma unroll
  for (int w = 0; w < K::NK; ++w) r.k[w] = stream_at<u32x4>(kp, k_at + 64 * w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (K::F8) {
      const u32x2 x = stream_at<u32x2>(vp, v_at + i * K::ROW);
      r.v[i][0] = x[0], r.v[i][1] = x[1];
    } else {
#pragma unroll
      for (int w = 0; w < K::VW / 4; ++w) {
        const u32x4 x = stream_at<u32x4>(vp, v_at + i * K::ROW + 16 * w);
#pragma unroll
        for (int j = 0; j < 4; ++j) r.v[i][4 * w + j] = x[j];
      }
    }
  }
  if constexpr (K::F8) {
    int z;  // a vector load: it is counted in order with the others
    asm("v_mov_b32 %0, 0" : "=v"(z));
    const f32x2 s = global_at<f32x2>(t.scales + (uint64_t)page * (2u * kv_heads), z);
    r.ks = s[0], r.vs = s[1];
  } else {
    r.ks = r.vs = 1.0f;
  }
}

// A tile of few rows.  Columns of 16 x 16 products are rows: each wavefront holds all
// NT tiles of 16, and the four share out the pages, straight from memory into
// registers, a page ahead.  Lane l of a wavefront: column n = l % 16, quarter
// grp = l / 16.
//   S^T[16 tokens][16 rows] = K Q^T: lane holds tokens 4 grp + i of row n,
//   O^T[128 dims][16 rows] += V^T P^T: that is just the P^T operand of the next
//   product, and V^T's is V[4 grp + i][8 n .. 8 n + 7] as loaded, so that the
//   accumulator holds dims 32 grp + 8 i + nb of row n (o[nb][i]).
// Bound by the pages' bytes: 32 rows take 192 matrix cycles a page and wavefront,
// 8 KiB a page, which 256 CUs could read at 100 TB/s.  221,000 tokens of 8 kv heads
// (906 MB), bf16: 149 us, 6.1 TB/s.
template <int DT, int NT>
struct Narrow {
  using K = Kv<DT>;
  u32x4 q[NT][K::F32 ? 8 : 4];
  f32x4 o[NT][8];
  float m[NT], sum[NT];
  int lim[NT];

  // One page.  MASKED: some row may not see all of its tokens; false: left out, as one
  // does not and V or its scale holds what is not finite among those that one sees.
  template <bool MASKED>
  __device__ __forceinline__ bool consume(const PageRegs<DT>& r, int l, int t0, int lim_lo, int lim_hi, float scale) {
    const int grp = l >> 4;
    // V rows as operand values: 8 dims of 4 tokens
    constexpr int VD = K::F32 ? 8 : 4;
    uint32_t vv[4][VD];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if constexpr (K::F8) {
        const u32x2 a = e4m3x4_to_bf16(r.v[t][0]), b = e4m3x4_to_bf16(r.v[t][1]);
        vv[t][0] = a[0], vv[t][1] = a[1], vv[t][2] = b[0], vv[t][3] = b[1];
      } else {
#pragma unroll
        for (int i = 0; i < VD; ++i) vv[t][i] = r.v[t][i];
      }
    }
    float vs = r.vs;
    if constexpr (MASKED) {
      if (t0 >= lim_hi) vs = 0.0f;  // no row sees the page
      bool odd = K::F8 && !finite(vs);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bool seen = t < lim_hi - t0 - 4 * grp;
#pragma unroll
        for (int i = 0; i < VD; ++i) {
          odd |= seen && not_finite<DT>(vv[t][i]);
          vv[t][i] = seen ? vv[t][i] : 0u;
        }
      }
      if (t0 + kPageTokens > lim_lo && __builtin_amdgcn_ballot_w64(odd)) return false;
    }
    u32x4 k16[4];
    if constexpr (K::F8) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const u32x2 a = e4m3x4_to_bf16(r.k[w][0]), b = e4m3x4_to_bf16(r.k[w][1]);
        const u32x2 c = e4m3x4_to_bf16(r.k[w][2]), d = e4m3x4_to_bf16(r.k[w][3]);
        k16[2 * w] = u32x4{a[0], a[1], b[0], b[1]};
        k16[2 * w + 1] = u32x4{c[0], c[1], d[0], d[1]};
      }
    } else if constexpr (!K::F32) {
#pragma unroll
      for (int w = 0; w < 4; ++w) k16[w] = r.k[w];
    }
    u32x2 vop[8];
    if constexpr (!K::F32) {
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) {
        const uint32_t sel = (nb & 1) ? 0x07060302u : 0x05040100u;
        vop[nb] = u32x2{__builtin_amdgcn_perm(vv[1][nb >> 1], vv[0][nb >> 1], sel),
                        __builtin_amdgcn_perm(vv[3][nb >> 1], vv[2][nb >> 1], sel)};
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (K::F32) {
#pragma unroll
        for (int w = 0; w < 8; ++w)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f32(r.k[w][e]), bits_f32(q[nt][w][e]), s, 0, 0, 0);
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) s = mma16<K::BF>(k16[w], q[nt][w], s);
      }
      const float c = K::F8 ? scale * r.ks : scale;
      float x[4], top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        x[t] = s[t] * c;
        if (MASKED && t >= lim[nt] - t0 - 4 * grp) x[t] = -INFINITY;
        top = fmaxf(top, x[t]);
      }
      top = max_over_groups(top);
      const bool raise = top > m[nt] + K::kMost;
      if (__builtin_amdgcn_ballot_w64(raise)) {
        const float to = raise ? top - K::kTop : m[nt], f = raise ? exp2_fast(m[nt] - to) : 1.0f;
        m[nt] = to;
        sum[nt] *= f;
#pragma unroll
        for (int nb = 0; nb < 8; ++nb) o[nt][nb] *= f;
      }
      const float ref = against(m[nt]);
      float p[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) p[t] = exp2_fast(x[t] - ref);
      sum[nt] += (p[0] + p[1]) + (p[2] + p[3]);
      if constexpr (K::F8) {
#pragma unroll
        for (int t = 0; t < 4; ++t) p[t] *= vs;
      }
      if constexpr (K::F32) {
#pragma unroll
        for (int nb = 0; nb < 8; ++nb)
#pragma unroll
          for (int t = 0; t < 4; ++t)
            o[nt][nb] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f32(vv[t][nb]), p[t], o[nt][nb], 0, 0, 0);
      } else {
        const u32x2 pop = {pack2<K::BF>(p[0], p[1]), pack2<K::BF>(p[2], p[3])};
#pragma unroll
        for (int nb = 0; nb < 8; ++nb) o[nt][nb] = mma16h<K::BF>(vop[nb], pop, o[nt][nb]);
      }
    }
    return true;
  }

  // The tile's steps; then sh.merge and sh.ml hold each wavefront's rows.
  template <class Sh>
  __device__ __forceinline__ void run(const PageView& v, const AttendArgs& a, const Tile& t, Sh& sh) {
    const int tid = this_thread(), l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = l & 15, grp = l >> 4;
    const float scale = a.scale * 1.4426950408889634f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = nt * 16 + n;
      lim[nt] = row < t.rows ? sh.lim[row] : 0;
      m[nt] = -INFINITY, sum[nt] = 0.0f;
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) o[nt][nb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      const int64_t at = row < t.rows ? row_at(a, a.qs, t.row0 + row, t.h) : 0;
#pragma unroll
      for (int w = 0; w < (K::F32 ? 8 : 4); ++w) {
        u32x4 x = {0u, 0u, 0u, 0u};
        if (row < t.rows) {
          if constexpr (K::F32) {
            const float* p = static_cast<const float*>(a.q) + at + 4 * (4 * w + grp);
            if (a.aligned) x = *reinterpret_cast<const u32x4*>(p);
            else x = u32x4{f32_bits(p[0]), f32_bits(p[1]), f32_bits(p[2]), f32_bits(p[3])};
          } else {
            const int d = K::F8 ? 16 * (4 * (w >> 1) + grp) + 8 * (w & 1) : 8 * (4 * w + grp);
            x = load_q8(static_cast<const uint16_t*>(a.q) + at + d, a.aligned, 0u);
          }
        }
        q[nt][w] = x;
      }
    }
    // page i of this wavefront: one of each of the steps of kStep pages in [p0, p1)
    static_assert(kStep == kThreads / 64, "a page per wavefront and step");
    const int count = (t.p1 - t.p0 + kStep - 1) / kStep;
    auto page_no = [&](int i) { return t.p0 + kStep * i + wave; };
    uint32_t ids = 0;  // lane j: the table's entry for page 64 k + j
    auto fill_ids = [&](int i0) {
      const int p = page_no(i0 + l);
      ids = p < t.p1 && i0 + l < count ? checked_page(v, global_at<uint32_t>(t.table, 4 * p)) : 0u;
    };
    auto id_of = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane((int)ids, i & 63); };
    if (t.p0 < t.p1) {
      fill_ids(0);
      PageRegs<DT> r[2];
      auto fetch = [&](int i, int b) __attribute__((always_inline)) {  // past the last page its entry is 0: a page that is not used
        if ((i & 63) == 0 && i) fill_ids(i);
        load_page<DT>(t, v.H, id_of(i), l, r[b]);
      };
      // pages that every row sees whole, two at a time, then the others (the last of an odd
      // number of whole ones among them, which is never left out)
      const int seen = t.lim_lo / kPageTokens - t.p0;  // such pages of all teams
      const int mine = clampi(seen / kStep + (seen % kStep > wave ? 1 : 0), 0, count);
      fetch(0, 0);
      int i = 0;
      for (; i + 1 < mine; i += 2) {
        fetch(i + 1, 1);
        consume<false>(r[0], l, 0, 0, 0, scale);
        fetch(i + 2, 0);
        consume<false>(r[1], l, 0, 0, 0, scale);
      }
      for (; page_no(i) < t.p1; ++i) {
        if (!consume<true>(r[0], l, page_no(i) * kPageTokens, t.lim_lo, t.lim_hi, scale)) sh.left_out = 1;
        fetch(i + 1, 0);
      }
    }
    // hand over: [wavefront][row][dim]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      sum[nt] = sum_over_groups(sum[nt]);
      float* to = sh.merge + (wave * 16 * NT + nt * 16 + n) * kPad + 32 * grp;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int nb = 0; nb < 8; nb += 4)
          *reinterpret_cast<f32x4*>(to + 8 * i + nb) =
              f32x4{o[nt][nb][i], o[nt][nb + 1][i], o[nt][nb + 2][i], o[nt][nb + 3][i]};
      if (grp == 0) sh.ml[wave][nt * 16 + n][0] = m[nt], sh.ml[wave][nt * 16 + n][1] = sum[nt];
    }
  }
};

// Writes a row's 8 output dims from d on (x: the sum of weighted values, inv: 1 / sum).
template <int DT>
__device__ inline void write_out(const AttendArgs& a, int64_t at, int d, const float (&x)[8], float inv) {
  if constexpr (DT == FERRY_F32) {
    float* p = static_cast<float*>(a.out) + at + d;
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i] * inv;
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2<Kv<DT>::BF>(x[2 * i] * inv, x[2 * i + 1] * inv);
    uint16_t* p = static_cast<uint16_t*>(a.out) + at + d;
    if (a.aligned) {
      *reinterpret_cast<u32x4*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// Joins the teams of a Narrow tile and writes its rows: to the output where they are
// finished (`to_o` null), else as a part.
template <int DT, int NT, class Sh>
__device__ __forceinline__ void narrow_write(const AttendArgs& a, const Tile& t, Sh& sh, float* to_ml, float* to_o) {
  const int tid = this_thread();
#pragma unroll
  for (int r0 = 0; r0 < 16 * NT; r0 += 16) {
    const int row = r0 + tid / 16, d = tid % 16 * 8;
    if (row >= t.rows) continue;
    float m = -INFINITY, sum = 0.0f, x[8] = {};
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, sh.ml[w][row][0]);
    const float ref = against(m);
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      const float f = exp2_fast(sh.ml[w][row][0] - ref);
      sum += f * sh.ml[w][row][1];
      const float* o = sh.merge + (w * 16 * NT + row) * kPad + d;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] += f * o[i];
    }
    if (!to_o) {
      const bool none = sh.lim[row] <= 0;
      write_out<DT>(a, row_at(a, a.os, t.row0 + row, t.h), d, x, none ? 0.0f : 1.0f / sum);
      if (a.lse && d == 0) {
        const int tok = token_of_row(a, t.row0 + row), g = t.row0 + row - tok * a.G;
        a.lse[(int64_t)tok * a.Hq + t.h * a.G + g] = none ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += 4)
        *reinterpret_cast<f32x4*>(to_o + (int64_t)row * kPageDim + d + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
      if (d == 0) to_ml[2 * row] = m, to_ml[2 * row + 1] = sum;
    }
  }
}

// A tile of up to 128 rows: four wavefronts of 32, which share each step's 64 tokens
// in LDS as 16-bit values.  Columns of 32 x 32 x 16 products are rows; lane l: column
// l % 32, half h = l / 32.
//   S^T[64 tokens][32 rows]: register i of token tile tt is token 32 tt + 8 (i / 4) +
//   4 h + i % 4, so registers 8 j .. 8 j + 7 are the P^T operand of the product over
//   tokens 16 j .. 16 j + 15 in the order (4 h + 0..3, 8 + 4 h + 0..3), and the V^T
//   operand in that order is two transposing LDS reads.
// A token's sixteen 16-byte chunks are stored at chunk ^ swizzle(token): the reads of
// K (one chunk of 32 tokens) and of V (four chunks of 8 tokens) then spread over all
// banks.
// K is a step ahead of V: while one step's weights are computed the next one's scores
// are, and the loads of V of the next and K of the one after it are on their way,
// straight into LDS (fp8: through registers, widened on the way).  A step is 1,024
// matrix cycles a wavefront, and as many of vector instructions next to them.  3,600
// rows of 32 heads over 6,700 tokens (377 GFLOP), fp16: 458 us, 815 TFLOP/s; 564 us
// with products, weights and loads one after the other.  The GPU's clock falls to 1.5
// GHz meanwhile (a library product of 8192^3 reaches 1,137 TFLOP/s).
// An LDS address as a number, and what is there: 16 bytes, or 4 values of a column
// (the 16 lanes of a group name 4 tokens of 16 dims, 4 dims each).
__device__ inline uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p;
}
template <class T>
__device__ inline T lds(uint32_t at) {
  return *(__attribute__((address_space(3))) const T*)(uintptr_t)at;
}
__device__ inline u32x2 lds_turned(uint32_t at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) i16x4*)(uintptr_t)at));
}

// 16 bytes per lane from memory straight into LDS, lane after lane from `to` on.  The
// wait is the caller's: the compiler does not know of them.  m0 is a reserved register,
// which the compiler does not let an asm name; it has no use of its own for it in these
// kernels, and sets it before each use where it has.
__device__ inline void load_lds(uint32_t to, const void* base, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(first_lane_i((int)to)), "v"(at), "s"(uniform(base)) : "memory");
}

__device__ inline int swizzle(int tok) { return (tok & 3) << 2 | (tok >> 2 & 3); }

template <int DT>
struct Wide {
  using K = Kv<DT>;
  typedef std::conditional_t<K::F8, u32x2, u32x4> Word;  // 8 values
  u32x4 q[8];
  f32x16 o[4];
  float m, sum;
  int lim;

  // The largest of a lane's scores of step s.  fp8: they get their pages' scales; MASKED:
  // what the row does not see becomes -inf.
  template <bool MASKED>
  struct Largest {
    float c[kStep], scale;  // factor on a page's scores
    int mine;               // of the lane's tokens, in steps of 4 and gaps of 4
    __device__ __forceinline__ Largest(const Wide& w, const Tile& t, int s, int steps, int h, float scale, float scales)
        : scale(scale), mine(s < steps ? w.lim - (t.p0 + kStep * s) * kPageTokens - 4 * h : 0) {
#pragma unroll
      for (int i = 0; i < kStep; ++i) c[i] = K::F8 ? scale * scale_of(scales, s, i) : scale;
    }
    __device__ __forceinline__ void among(f32x16 (&x)[2], int from, int n, float& top) const {
#pragma unroll
      for (int i = from; i < from + n; ++i) {
        float y = x[i >> 4][i & 15];
        if (K::F8) y *= c[i >> 3];
        if (MASKED && 8 * (i >> 2) + (i & 3) >= mine) y = -INFINITY;
        x[i >> 4][i & 15] = y;
        top = fmaxf(top, y);
      }
    }
    __device__ __forceinline__ float of_row(float top) const {  // scaled
      const mx_u32x2 two = pair_values<32>(top);
      top = fmaxf(bits_f32(two[0]), bits_f32(two[1]));
      return K::F8 ? top : top * scale;
    }
  };

  // fp8: of the scales of a window's pages that of page i of step s
  static __device__ __forceinline__ float scale_of(float scales, int s, int i) {
    return bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(scales), (kStep * s + i) & 63));
  }

  template <class Sh>
  __device__ __forceinline__ void run(const PageView& v, const AttendArgs& a, const Tile& t, Sh& sh) {
    const int tid = this_thread(), l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = l & 31, h = l >> 5, row = wave * 32 + col;
    const float scale = fabsf(a.scale) * 1.4426950408889634f;
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
    const bool busy = wave * 32 < t.rows;  // the others only help to load
    lim = row < t.rows ? sh.lim[row] : 0;
    m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    const int64_t at = row < t.rows ? row_at(a, a.qs, t.row0 + row, t.h) : 0;
#pragma unroll
    for (int s = 0; s < 8; ++s)
      q[s] = row < t.rows ? load_q8(static_cast<const uint16_t*>(a.q) + at + 16 * s + 8 * h, a.aligned, sign)
                          : u32x4{0u, 0u, 0u, 0u};
    const int steps = (t.p1 - t.p0 + kStep - 1) / kStep;
    // Page ids: lane j holds page 64 w + j of window w; the next window is read ahead.
    auto read_ids = [&](int w) __attribute__((always_inline)) {
      const int p = t.p0 + 64 * w + l;
      return p < t.p1 ? global_at<uint32_t>(t.table, 4 * p) : 0u;
    };
    uint32_t ids = checked_page(v, read_ids(0)), ids_next = 0;
    uint32_t pages[kStep];  // of the step whose K was loaded last
    // The thread's 16 bytes of a page in LDS: token tid / 16, chunk tid % 16 ^ swizzle.
    const int tok = tid >> 4;
    const uint32_t at_word = tok * K::ROW + ((tid & 15) ^ swizzle(tok)) * (uint32_t)sizeof(Word);
    const uint32_t k_base = lds_at(sh.kv.k[0]) + wave * 1024, v_base = lds_at(sh.kv.v[0]) + wave * 1024;
    Word kr[K::F8 ? kStep : 1], vr[K::F8 ? kStep : 1];  // fp8: on their way
    // fp8: the scales of the windows' pages, of K where step s + 1 is, of V where s is
    f32x2 scales = {};
    float k_scales = 0.0f, v_scales = 0.0f;
    // Pages that no row sees, those behind p1 among them, count as 0: their weights are 0
    // and must not meet a scale that is not finite.
    auto read_scales = [&](int w) __attribute__((always_inline)) {
      if constexpr (K::F8) {
        scales = *reinterpret_cast<const f32x2*>(t.scales + (uint64_t)ids * (2u * v.H));
        const int p = t.p0 + 64 * w + l;
        if (p >= t.p1 || p * kPageTokens >= t.lim_hi) scales[1] = 0.0f;
      }
    };
    // Page i of the step whose K or V is loaded next.  Pages from p1 on are page 0: they
    // are loaded for nothing.
    auto window = [&](int s) __attribute__((always_inline)) {  // before K of step s > 1
      if ((s - 1 & 15) == 0) k_scales = scales[0];
      if ((s - 2 & 15) == 0) v_scales = scales[1];
      if ((s & 15) == 0) ids = checked_page(v, ids_next), read_scales(s / 16);
      if ((s & 15) == 8) ids_next = read_ids(s / 16 + 1);
    };
    auto begin_k = [&](int i, int s, Word& to) __attribute__((always_inline)) {
      pages[i] = (uint32_t)__builtin_amdgcn_readlane((int)ids, (kStep * s + i) & 63);
      const uint8_t* p = t.base + (uint64_t)pages[i] * t.page_bytes;
      if constexpr (K::F8) to = global_at<Word>(uniform(p), at_word);
      else load_lds(k_base + ((s & 1) << 14) + (i << 12), p, at_word);
    };
    auto begin_v = [&](int i, int s) __attribute__((always_inline)) {  // the step of the last begin_k
      const uint8_t* p = t.base + (uint64_t)pages[i] * t.page_bytes + K::HALF;
      if constexpr (K::F8) vr[i] = global_at<Word>(uniform(p), at_word);
      else load_lds(v_base + ((s & 1) << 14) + (i << 12), p, at_word);
    };
    auto widen = [&](const Word& w) -> u32x4 {
      if constexpr (K::F8) {
        const u32x2 x = e4m3x4_to_bf16(w[0]), y = e4m3x4_to_bf16(w[1]);
        return u32x4{x[0], x[1], y[0], y[1]};
      } else {
        return w;
      }
    };
    // fp8: stores what was loaded, with room in LDS for 16-bit values.
    auto store_k = [&](const Word (&w)[K::F8 ? kStep : 1], int s) __attribute__((always_inline)) {
      if constexpr (K::F8) {
#pragma unroll
        for (int i = 0; i < kStep; ++i) *reinterpret_cast<u32x4*>(sh.kv.k[s & 1] + 4096 * i + tid * 16) = widen(w[i]);
      }
    };
    // Ends the loads of V of step s: what no row sees of it becomes zero.
    auto land = [&](int s) __attribute__((always_inline)) {
      const uint32_t to = tid * 16;
      if constexpr (K::F8) {
#pragma unroll
        for (int i = 0; i < kStep; ++i) *reinterpret_cast<u32x4*>(sh.kv.v[s & 1] + 4096 * i + to) = widen(vr[i]);
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      const int t0 = (t.p0 + kStep * s) * kPageTokens;
      if (s < steps && t0 + kStep * kPageTokens > t.lim_lo) {
        bool bad = false;
        if constexpr (K::F8) {  // the lanes that hold the step's V scales
          bad = l >> 2 == (s & 15) && !finite((s & 15) == 0 ? scales[1] : v_scales);
        }
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
          u32x4* at = reinterpret_cast<u32x4*>(sh.kv.v[s & 1] + 4096 * i + to);
          u32x4 x = *at;
          const bool seen = t0 + kPageTokens * i + tok < t.lim_hi && t.p0 + kStep * s + i < t.p1;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            bad |= seen && not_finite<DT>(x[w]);
            x[w] = seen ? x[w] : 0u;
          }
          *at = x;
        }
        if (bad) sh.odd[s % 3] = 1;
      }
      __syncthreads();
    };
    // K: token col, chunk h; V: token 4 h + (l % 16) / 4, dims 16 (l / 16 % 2) + 4 (l % 4)
    const uint32_t k_lane = lds_at(sh.kv.k[0]) + (col << 8) + ((h ^ swizzle(col)) << 4);
    const int vt = 4 * h + (l >> 2 & 3), vd = 16 * (l >> 4 & 1) + 4 * (l & 3);
    const uint32_t v_lane = lds_at(sh.kv.v[0]) + (vt << 8) + (((vd >> 3) ^ swizzle(vt)) << 4) + (vd & 4) * 2;
    // S^T of step s
    auto products = [&](f32x16 (&x)[2], int s) __attribute__((always_inline)) {
      // The lane's place in this step's K; the others follow by flipping address bits.
      // Opaque, so that they are not all kept in registers over the loop.
      uint32_t at = k_lane + ((s & 1) << 14);
      asm("" : "+v"(at));
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[tt][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c)  // chunk 2 c + h of token 32 tt + col
          x[tt] = mma32<K::BF>(lds<u32x4>((at ^ c << 5) + 8192 * tt), q[c], x[tt]);
      }
    };
    auto raise_to = [&](float top, bool raise) __attribute__((always_inline)) {
      if (__builtin_amdgcn_ballot_w64(raise)) {
        const float to = raise ? top - K::kTop : m, f = raise ? exp2_fast(m - to) : 1.0f;
        m = to;
        sum *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= f;
      }
    };
    // weights of scores y0, y1, the lane's i-th and next of step s
    auto weights2 = [&](float y0, float y1, float ref, int s, int i) __attribute__((always_inline)) {
      float p0 = exp2_fast(K::F8 ? y0 - ref : __builtin_fmaf(y0, scale, -ref));
      float p1 = exp2_fast(K::F8 ? y1 - ref : __builtin_fmaf(y1, scale, -ref));
      sum += p0 + p1;
      if constexpr (K::F8) {
        const float f = scale_of(v_scales, s, i >> 3);
        p0 *= f, p1 *= f;
      }
      return pack2<K::BF>(p0, p1);
    };
    auto begin_step = [&](int s) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        begin_v(i, s);
        begin_k(i, s + 1, kr[K::F8 ? i : 0]);
      }
    };
    // the steps that every row sees whole
    const int whole = clampi((t.lim_lo - t.p0 * kPageTokens) / (kStep * kPageTokens), 0, steps);
    f32x16 x[2], y[2];
    {
      Word k0[K::F8 ? kStep : 1];
#pragma unroll
      for (int i = 0; i < kStep; ++i) begin_k(i, 0, k0[K::F8 ? i : 0]);
      read_scales(0);
      begin_step(0);
      k_scales = scales[0], v_scales = scales[1];
      store_k(k0, 0);
      store_k(kr, 1);
      land(0);
      if (busy) {
        products(x, 0);
        const Largest<true> see(*this, t, 0, steps, h, scale, k_scales);
        float top = -INFINITY;
        see.among(x, 0, 32, top);
        top = see.of_row(top);
        raise_to(top, top > m + K::kMost);
      }
      __syncthreads();  // all have read K of step 0: the first step loads over it
    }
    // Step s, whose scores are in x, while those of step s + 1 come into y (MASKED: some row
    // may not see them all): next to each product a part of the weights, then of the
    // maximum, is computed and a load begun, and operands are read three products ahead.
    auto step = [&](auto masked_, f32x16 (&x)[2], f32x16 (&y)[2], int s) __attribute__((always_inline)) {
      constexpr bool MASKED = decltype(masked_)::value;
      window(s + 2);
      if (MASKED) {
        if (tid == 0) sh.odd[(s + 2) % 3] = 0;
        if (first_lane_i(sh.odd[s % 3])) {  // left out, as V holds what is not finite
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i >> 4][i & 15] = -INFINITY;
#pragma unroll
          for (int i = 0; i < kStep; ++i) *reinterpret_cast<u32x4*>(sh.kv.v[s & 1] + 4096 * i + tid * 16) = u32x4{0u, 0u, 0u, 0u};
          if (K::F8 && l >> 2 == (s & 15)) v_scales = 0.0f;  // of its pages
          if (tid == 0) sh.left_out = 1;
          __syncthreads();
        }
      }
      if (busy) {
        uint32_t k_at = k_lane + ((s + 1 & 1) << 14), v_at = v_lane + ((s & 1) << 14), pop[16];
        asm("" : "+v"(k_at), "+v"(v_at));
        auto read_k = [&](int i) __attribute__((always_inline)) {
          return lds<u32x4>((k_at ^ (i >> 1) << 5) + 8192 * (i & 1));
        };
        auto read_v = [&](int i) __attribute__((always_inline)) {
          // tokens 16 j + 4 h .. + 3 and those 8 behind, whose swizzle flips chunk bit 1
          const u32x2 lo = lds_turned((v_at ^ (i & 3) << 6) + 4096 * (i >> 2));
          const u32x2 hi = lds_turned((v_at ^ (i & 3) << 6 ^ 32) + 4096 * (i >> 2) + 2048);
          return u32x4{lo[0], lo[1], hi[0], hi[1]};
        };
        auto begin = [&](int i) __attribute__((always_inline)) {
          if (i >= 2 * kStep) return;
          if (i & 1) begin_k(i >> 1, s + 2, kr[K::F8 ? i >> 1 : 0]);
          else begin_v(i >> 1, s + 1);
        };
        u32x4 a[4];
#pragma unroll
        for (int i = 0; i < 3; ++i) a[i] = read_k(i);
#pragma unroll
        for (int i = 0; i < 16; ++i) y[0][i] = y[1][i] = 0.0f;
        const float ref = against(m);
        // The half with the weights goes before another wavefront's half without: 458 us
        // instead of 474 (chunks).
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          a[i + 3 & 3] = i + 3 < 16 ? read_k(i + 3) : read_v(i - 13);
          y[i & 1] = mma32<K::BF>(a[i & 3], q[i >> 1], y[i & 1]);
          if (!K::F8) begin(i);
          pop[i] = weights2(x[i >> 3][2 * i & 15], x[i >> 3][(2 * i & 15) + 1], ref, s, 2 * i);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        const Largest<MASKED> see(*this, t, s + 1, steps, h, scale, k_scales);
        float top = -INFINITY;
        bool raise = false;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (i + 3 < 16) a[i + 3 & 3] = read_v(i + 3);
          o[i & 3] = mma32<K::BF>(a[i & 3], u32x4{pop[i & 12], pop[(i & 12) + 1], pop[(i & 12) + 2], pop[(i & 12) + 3]},
                                  o[i & 3]);
          if (K::F8) begin(i);  // into the registers that x has left
          if (i >= 2 && i < 10) see.among(y, 4 * (i - 2), 4, top);
          if (i == 11) top = see.of_row(top);
          if (i == 12) raise = top > m + K::kMost;
          __builtin_amdgcn_sched_barrier(0);
        }
        raise_to(top, raise);
      } else {
        begin_step(s + 1);
      }
      store_k(kr, s + 2);
      land(s + 1);
    };
    int s = 0;
    if constexpr (K::F8) {
      for (; s + 1 < whole; ++s) {
        step(std::false_type{}, x, y, s);
        x[0] = y[0], x[1] = y[1];
      }
    } else {  // two at a time need no copies, but registers that fp8 does not have
      for (; s + 2 < whole; s += 2) step(std::false_type{}, x, y, s), step(std::false_type{}, y, x, s + 1);
    }
    for (; s < steps; ++s) {
      step(std::true_type{}, x, y, s);
      x[0] = y[0], x[1] = y[1];
    }
    {
      const mx_u32x2 two = pair_values<32>(sum);
      sum = bits_f32(two[0]) + bits_f32(two[1]);
    }
  }

  __device__ __forceinline__ void write(const AttendArgs& a, const Tile& t, float* to_ml, float* to_o) {
    const int tid = this_thread(), l = tid & 63, h = l >> 5, row = (tid >> 6) * 32 + (l & 31);
    if (row >= t.rows) return;
    if (to_o) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<f32x4*>(to_o + (int64_t)row * kPageDim + 32 * dt + 2 * e + 4 * h) =
              f32x4{o[dt][e], o[dt][e + 1], o[dt][e + 2], o[dt][e + 3]};
      if (h == 0) to_ml[2 * row] = m, to_ml[2 * row + 1] = sum;
      return;
    }
    const float inv = lim <= 0 ? 0.0f : 1.0f / sum;
    uint16_t* p = static_cast<uint16_t*>(a.out) + row_at(a, a.os, t.row0 + row, t.h) + 4 * h;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const u32x2 w = {pack2<K::BF>(o[dt][e] * inv, o[dt][e + 1] * inv),
                         pack2<K::BF>(o[dt][e + 2] * inv, o[dt][e + 3] * inv)};
        uint16_t* to = p + 32 * dt + 2 * e;
        if (a.aligned) {
          *reinterpret_cast<u32x2*>(to) = w;
        } else {
          to[0] = (uint16_t)w[0], to[1] = (uint16_t)(w[0] >> 16), to[2] = (uint16_t)w[1], to[3] = (uint16_t)(w[1] >> 16);
        }
      }
    if (a.lse && h == 0) {
      const int tok = token_of_row(a, t.row0 + row), g = t.row0 + row - tok * a.G;
      a.lse[(int64_t)tok * a.Hq + t.h * a.G + g] = lim <= 0 ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
    }
  }
};

// The last value of a row: two dims a lane (x, y: the sums of weighted values).
template <int DT>
__device__ __forceinline__ void finish_row(const AttendArgs& a, int row, int h, float m, float sum, float x, float y,
                                  bool none) {
  const int l = threadIdx.x & 63;
  const float inv = none ? 0.0f : 1.0f / sum;
  const int64_t at = row_at(a, a.os, row, h) + 2 * l;
  if constexpr (Kv<DT>::F32) {
    float* p = static_cast<float*>(a.out) + at;
    p[0] = x * inv, p[1] = y * inv;
  } else {
    const uint32_t w = pack2<Kv<DT>::BF>(x * inv, y * inv);
    uint16_t* p = static_cast<uint16_t*>(a.out) + at;
    p[0] = (uint16_t)w, p[1] = (uint16_t)(w >> 16);
  }
  if (a.lse && l == 0)
    a.lse[(int64_t)token_of_row(a, row) * a.Hq + h * a.G + row - token_of_row(a, row) * a.G] = none ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}

// The pages that a tile's products left out, which are among those that not every row
// sees whole: a value that is not finite must not meet the zero weight of a row that
// does not see it, so here each row takes only the tokens it sees, one at a time, two
// dims a lane.  ml, o: the tile's rows as a
// part, which this adds to.  unit: pages that are left out together.
template <int DT>
__device__ __forceinline__ void add_left_out(const PageView& v, const AttendArgs& a, const Tile& t, int unit,
                                                             const int* lims, float* ml, float* o) {
  using K = Kv<DT>;
  const int tid = this_thread(), l = tid & 63, wave = tid >> 6;
  const float scale = a.scale * 1.4426950408889634f;
  const int whole = max(0, t.lim_lo / kPageTokens - t.p0) / unit * unit;
  for (int p = t.p0 + whole; p < t.p1; p += unit) {
    bool odd = false;
    for (int i = 0; i < unit && p + i < t.p1; ++i) {
      const uint64_t page = checked_page(v, t.table[p + i]);
      const uint8_t* rec = t.base + page * t.page_bytes;
      for (int e = l; e < kPageTokens * kPageDim; e += 64)
        odd |= (p + i) * kPageTokens + e / kPageDim < t.lim_hi && !finite(v_elem<DT>(rec, e / kPageDim, e % kPageDim));
      if (K::F8) odd |= (p + i) * kPageTokens < t.lim_hi && !finite(t.scales[page * (2u * v.H) + 1]);
    }
    if (!__builtin_amdgcn_ballot_w64(odd)) continue;
    for (int row = wave; row < t.rows; row += kThreads / 64) {
      const int lim = lims[row];
      const int64_t at = row_at(a, a.qs, t.row0 + row, t.h) + 2 * l;
      const float q0 = q_elem<DT>(a.q, at), q1 = q_elem<DT>(a.q, at + 1);
      float m = ml[2 * row], sum = ml[2 * row + 1];
      float x = o[(int64_t)row * kPageDim + 2 * l], y = o[(int64_t)row * kPageDim + 2 * l + 1];
      for (int tok = p * kPageTokens; tok < min(lim, min(p + unit, t.p1) * kPageTokens); ++tok) {
        const uint64_t page = checked_page(v, t.table[tok / kPageTokens]);
        const uint8_t* rec = t.base + page * t.page_bytes;
        const float* sc = t.scales + page * (2u * v.H);
        const int i = tok % kPageTokens;
        float s = q0 * k_elem<DT>(rec, i, 2 * l) + q1 * k_elem<DT>(rec, i, 2 * l + 1);
        for (int d = 32; d; d /= 2) s += __shfl_xor(s, d);
        s *= K::F8 ? scale * sc[0] : scale;
        const float top = fmaxf(m, s), f = exp2_fast(m - against(top)), w = exp2_fast(s - against(top));
        const float wv = K::F8 ? w * sc[1] : w;
        m = top;
        sum = sum * f + w;
        x = x * f + wv * v_elem<DT>(rec, i, 2 * l);
        y = y * f + wv * v_elem<DT>(rec, i, 2 * l + 1);
      }
      o[(int64_t)row * kPageDim + 2 * l] = x, o[(int64_t)row * kPageDim + 2 * l + 1] = y;
      if (l == 0) ml[2 * row] = m, ml[2 * row + 1] = sum;
    }
  }
}

// ---- the call -------------------------------------------------------------------
template <int DT, int FORMS>
__global__ __launch_bounds__(kThreads, kPerCu) void k_attend(PageView v, int layer, AttendArgs a, Scratch ws) {
  __shared__ __attribute__((aligned(1024))) Shared<FORMS> sh;
  const int tid = threadIdx.x, grid = gridDim.x;
  // consecutive runs of work on one XCD (workgroups go to the 8 XCDs in turn), so
  // that tiles of the same pages meet in its L2
  const int wg = grid % 8 ? (int)blockIdx.x : (int)(blockIdx.x % 8) * (grid / 8) + (int)blockIdx.x / 8;
  const int nseg = a.n_groups + a.n_req;
  const int *gs = a.group_start, *gp = a.shared;
  if (a.n_groups && a.n_groups <= kGroupsInLds) {
    for (int i = tid; i <= a.n_groups; i += kThreads) {
      sh.gs[i] = a.group_start[i];
      if (i < a.n_groups) sh.gp[i] = a.shared[i], sh.gl[i] = 0x7FFFFFFF;
    }
    gs = sh.gs, gp = sh.gp;
    __syncthreads();
  }
  // units of this thread's segments, and their sum over all threads before it
  const int per_thread = (nseg + kThreads - 1) / kThreads, s0 = min(tid * per_thread, nseg),
            s1 = min(s0 + per_thread, nseg);
  uint64_t mine = 0;
  Seg kept;  // the thread's only segment, where it has one
  uint64_t kept_work = 0;
  for (int s = s0; s < s1; ++s) {
    kept = segment<DT>(v, a, gs, gp, s);
    kept_work = seg_work<DT>(a, kept);
    mine += kept_work * v.H;
    if (kept.own && kept.group >= 0 && kept.rows > 0 && gs == sh.gs) atomicMin(&sh.gl[kept.group], max(0, kept.base));
    if (wg == 0) {  // what is out of range, once
      bool bad = false;
      if (kept.own) {
        const int lane = a.lanes[kept.req];
        bad = lane < -1 || lane >= v.n_lanes || (kept.lane >= 0 && v.len[kept.lane] != kept.len);
        if (a.q_start)
          bad |= a.q_start[kept.req] < 0 || a.q_start[kept.req] > a.q_start[kept.req + 1] ||
                 a.q_start[kept.req + 1] > a.n_tokens;
      } else {
        bad = gs[s] < 0 || gs[s] > gs[s + 1] || gs[s + 1] > a.n_req || gp[s] < 0 || gp[s] > v.max_pages;
      }
      if (bad) set_error(v.error, FERRY_ERANGE);
    }
  }
  uint64_t before = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t y = __shfl_up(before, d);
    if ((tid & 63) >= d) before += y;
  }
  if ((tid & 63) == 63) sh.sums[tid >> 6] = before;
  __syncthreads();
  uint64_t total = 0;
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < tid >> 6) before += sh.sums[i];
    total += sh.sums[i];
  }
  before -= mine;
  total = first_lane_u64(total);
  // no run is shorter than a step, so that each one within a tile begins one
  constexpr int kMost = FORMS == 1 ? step_units<DT>(16) : 11;
  static_assert(FORMS == 1 || (step_units<DT>(16) <= kMost && step_units<DT>(32) <= kMost && step_units<DT>(kWide) <= kMost));
  const uint64_t per = max((uint64_t)kMost, first_lane_u64((total + grid - 1) / grid));
  const uint64_t u0 = per * wg, u1 = min(total, u0 + per);
  if (u0 >= u1) return;
  const uint32_t per32 = (uint32_t)min(per, (uint64_t)0x7FFFFFFF);
  // Each thread lists those of its segments that are among the kListed from `from` on.
  auto list = [&](int from, auto first) __attribute__((always_inline)) {
    const int s0 = min(this_thread() * per_thread, nseg), s1 = min(s0 + per_thread, nseg);
    uint64_t at = before;
    for (int s = s0; s < s1; ++s) {
      SegAt x;
      const bool have = decltype(first)::value && per_thread == 1;
      x.g = have ? kept : segment<DT>(v, a, gs, gp, s);
      x.work = have ? kept_work : seg_work<DT>(a, x.g);
      x.at = at;
      if (s >= from && s < from + kListed) sh.list[s - from] = x;
      at += x.work * v.H;
    }
    __syncthreads();
  };
  if (u0 >= before && u0 < before + mine) {  // one thread: it has the run's first segment
    uint64_t at = before;
    int s = s0;
    if (per_thread > 1)
      for (;; ++s) {
        at += seg_work<DT>(a, segment<DT>(v, a, gs, gp, s)) * v.H;
        if (u0 < at) break;
      }
    sh.seg = s;
  }
  __syncthreads();

  int s = first_lane_i(sh.seg), from = s;
  list(from, std::true_type{});
  uint64_t u = u0, tile_at = 0;
  int h = -1, j = 0;
  SegAt x;
  auto listed = [&](int i) { x = uniform(sh.list[i]); };
  listed(0);
  while (u < u1) {
    const int tid = this_thread();
    if (u >= x.at + x.work * v.H) {  // the next segment
      if (++s == from + kListed) {
        __syncthreads();
        from = s;
        list(from, std::false_type{});
      }
      listed(s - from);
      h = -1;
      continue;
    }
    const Seg& g = x.g;
    if (h < 0) {
      h = u == x.at ? 0 : (int)((u - x.at) / x.work);
      tile_at = x.at + h * x.work;  // unit of the tile's first step
      j = 0;
    }
    int work = tile_work<DT>(a, g, j);
    while (u >= tile_at + work) {
      tile_at += work;
      if (++j == g.tiles) j = 0, ++h;
      work = tile_work<DT>(a, g, j);
    }
    // this workgroup's steps [k0, k1) of the tile's `len`
    const int per_step = step_units<DT>(g.tile), len = first_lane_i(tile_steps(a, g, j));
    auto steps_in = [&](int units) {  // begun within so many units
      const int n = units + per_step - 1;
      return first_lane_i(g.tile == 16 ? n / step_units<DT>(16) : g.tile == 32 ? n / step_units<DT>(32) : n / step_units<DT>(kWide));
    };
    const int k0 = steps_in((int)(u - tile_at)), k1 = min(len, steps_in((int)min((uint64_t)work, u1 - tile_at)));
    u = tile_at + work;
    if (k0 >= k1) continue;  // the workgroup before has done them all
    Tile t;
    t.row0 = g.row0 + j * g.tile, t.rows = min(g.tile, g.rows - j * g.tile), t.h = h;
    t.p0 = g.p0 + kStep * k0, t.p1 = min(g.p1, g.p0 + kStep * k1);
    if (t.p1 < t.p0) t.p1 = t.p0;
    t.table = v.table + (uint64_t)(g.lane < 0 ? 0 : g.lane) * v.max_pages;
    t.page_bytes = (uint32_t)v.H * (2u * Kv<DT>::HALF);
    t.base = v.pool + (uint64_t)layer * v.n_pages * t.page_bytes + (uint32_t)h * (2u * Kv<DT>::HALF);
    t.scales = v.scales + ((uint64_t)layer * v.n_pages * v.H + h) * 2;
    // the workgroups that share the tile
    const int first = tile_at >= u0 ? wg : wg - (int)(((uint32_t)(u0 - tile_at) + per32 - 1) / per32);
    const uint64_t end = tile_at + (uint32_t)(len - 1) * per_step;  // the last step's unit
    const int last = end < u1 ? wg : wg + (int)((uint32_t)(end - u0) / per32);
    const int count = last - first + 1;
    const bool two = g.own ? a.n_groups && g.p0 > 0 : true;
    __syncthreads();  // the last tile's rows are written
    const bool all_seen = !g.own && gs == sh.gs && first_lane_i(sh.gl[g.req]) >= g.p1 * kPageTokens;
    const int tok0 = token_of_row(a, t.row0), tok1 = token_of_row(a, t.row0 + t.rows - 1);
    if (g.own) {
      t.lim_lo = clampi(g.base + tok0 - g.tok0, 0, g.len);
      t.lim_hi = clampi(g.base + tok1 - g.tok0, 0, g.len);
    } else {
      t.lim_lo = t.lim_hi = g.p1 * kPageTokens;
      if (!all_seen) {
        if (tid == 0) sh.lim_lo = 0x7FFFFFFF, sh.lim_hi = 0;
        __syncthreads();
      }
    }
    if (tid < 3) sh.odd[tid] = 0;
    if (tid == 0) sh.left_out = 0;
    if (tid < t.rows) {
      const int row = t.row0 + tid, tok = token_of_row(a, row);
      int lim = t.lim_lo;
      if (g.own) {
        lim = clampi(g.base + (tok - g.tok0), 0, g.len);
      } else if (!all_seen) {
        int lo = tok;
        if (a.q_start) {  // the request of this token
          lo = clampi(gs[g.req], 0, a.n_req);
          int hi = clampi(gs[g.req + 1], lo, a.n_req) - 1;
          while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (token_of(a, mid) <= tok) lo = mid; else hi = mid - 1;
          }
        }
        const int n = len_of(v, lane_of(v, a, lo));
        lim = min(clampi(n - token_of(a, lo + 1) + tok + 1, 0, n), g.p1 * kPageTokens);
        atomicMin(&sh.lim_lo, lim);
        atomicMax(&sh.lim_hi, lim);
      }
      sh.lim[tid] = lim;
      if (k0 == 0)
        ws.where[((uint64_t)g.own * v.H + h) * a.n_tokens * a.G + row] =
            Where{first, !two && count == 1 ? 0 : count, tid, (two ? 1 : 0) | (lim > 0 ? 2 : 0)};
    }
    __syncthreads();
    if (!g.own && !all_seen) t.lim_lo = first_lane_i(sh.lim_lo), t.lim_hi = first_lane_i(sh.lim_hi);
    t = uniform(t);
    float *to_ml = nullptr, *to_o = nullptr;
    if (count > 1) {
      const uint64_t part = 2 * (uint64_t)wg + (wg == first ? 1 : 0);
      to_ml = ws.part_ml + part * ws.tile_rows * 2;
      to_o = ws.part_o + part * ws.tile_rows * kPageDim;
    } else if (two) {
      const uint64_t r = ((uint64_t)g.own * v.H + h) * a.n_tokens * a.G + t.row0;
      to_ml = ws.row_ml + r * 2;
      to_o = ws.row_o + r * kPageDim;
    }
    // Writes the rows by `write`; with pages left out, as a part first, in any case.
    auto finish = [&](int unit, auto&& write) __attribute__((always_inline)) {
      __syncthreads();
      if (!sh.left_out) {
        write(to_ml, to_o);
        return;
      }
      // a tile that is written out ends here: the last part's place is free
      float* ml = to_o ? to_ml : ws.part_ml + (2 * (uint64_t)wg + 1) * ws.tile_rows * 2;
      float* o = to_o ? to_o : ws.part_o + (2 * (uint64_t)wg + 1) * ws.tile_rows * kPageDim;
      write(ml, o);
      __threadfence_block();
      __syncthreads();
      add_left_out<DT>(v, a, t, unit, sh.lim, ml, o);
      if (to_o) return;
      __threadfence_block();
      __syncthreads();
      for (int row = tid >> 6; row < t.rows; row += kThreads / 64) {
        const float* r = o + (int64_t)row * kPageDim + 2 * (tid & 63);
        finish_row<DT>(a, t.row0 + row, t.h, ml[2 * row], ml[2 * row + 1], r[0], r[1], sh.lim[row] <= 0);
      }
    };
    auto narrow = [&](auto nt) __attribute__((always_inline)) {
      constexpr int NT = decltype(nt)::value;
      Narrow<DT, NT> x;
      x.run(v, a, t, sh);
      finish(1, [&](float* ml, float* o) __attribute__((always_inline)) { narrow_write<DT, NT>(a, t, sh, ml, o); });
    };
    std::integral_constant<int, 1> one;
    std::integral_constant<int, 2> pair;
    if constexpr (FORMS == 1) {
      narrow(one);
    } else {
      if (g.tile == 16) narrow(one);
      else if (FORMS == 2 || g.tile == 32) narrow(pair);
      else if constexpr (FORMS == 3) {
        Wide<DT> x;
        x.run(v, a, t, sh);
        finish(kStep, [&](float* ml, float* o) __attribute__((always_inline)) { x.write(a, t, ml, o); });
      }
    }
  }
}

// Joins the parts of the rows that have some, in the order of their pages, the shared
// ones first.  16 lanes take a row, 8 dims each; SPLIT such teams share out a row's
// parts (16, a workgroup, where the rows are few and their parts may be many, else 1).
// Bound by the latency of three dependent reads (where, part, write), so many rows are
// in flight and four parts of each.  r0: the launch's first row.
template <int DT, int SPLIT>
__global__ __launch_bounds__(kThreads) void k_attend_join(PageView v, AttendArgs a, Scratch ws, int grid, uint64_t r0) {
  constexpr int kTeams = kThreads / 16, kAhead = 4;
  __shared__ float got[SPLIT > 1 ? kTeams : 1][kPad];
  const int team = threadIdx.x >> 4, d = (threadIdx.x & 15) * 8;
  const uint32_t rows = (uint32_t)a.n_tokens * a.G;
  const uint64_t all = (uint64_t)rows * v.H;
  const uint64_t r = SPLIT > 1 ? blockIdx.x : r0 + (uint64_t)blockIdx.x * kTeams + team;
  if (r >= all) return;
  const uint32_t h = (uint32_t)(r / rows), row = (uint32_t)(r % rows);
  const int tok = token_of_row(a, (int)row);
  if (tok < token_of(a, 0) || tok >= token_of(a, a.n_req)) return;
  const Where own = ws.where[all + r];
  if (own.count == 0) return;
  Where part[2] = {Where{0, 0, 0, 0}, own};
  if (own.has & 1) part[0] = ws.where[r];
  int n[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // stay in the scratch, whatever the offsets were
    part[k].first = clampi(part[k].first, 0, grid - 1);
    part[k].row = clampi(part[k].row, 0, ws.tile_rows - 1);
    n[k] = clampi(part[k].count, 0, grid - part[k].first);
  }
  const int parts = n[0] + n[1];
  float m = -INFINITY, sum = 0.0f, x[8] = {};
  for (int i0 = SPLIT > 1 ? team : 0; i0 < parts; i0 += kAhead * SPLIT) {
    float2 ml[kAhead];
    f32x4 lo[kAhead], hi[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * SPLIT, k = i >= n[0], at = i - (k ? n[0] : 0);
      if (i < parts) {
        const bool whole = n[k] == 1 && (own.has & 1);  // in the row's own place
        const uint64_t p = whole ? k * all + r
                                 : (2 * (uint64_t)(part[k].first + at) + (at == 0 ? 1 : 0)) * ws.tile_rows + part[k].row;
        ml[j] = reinterpret_cast<const float2*>(whole ? ws.row_ml : ws.part_ml)[p];
        const f32x4* o = reinterpret_cast<const f32x4*>((whole ? ws.row_o : ws.part_o) + p * kPageDim + d);
        lo[j] = o[0], hi[j] = o[1];
      } else {
        ml[j] = float2{-INFINITY, 0.0f};
        lo[j] = hi[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
    float top = m;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) top = fmaxf(top, ml[j].x);
    const float ref = against(top), f = exp2_fast(m - ref);
    m = top, sum *= f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= f;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float w = exp2_fast(ml[j].x - ref);
      sum += w * ml[j].y;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += w * lo[j][e], x[4 + e] += w * hi[j][e];
    }
  }
  if constexpr (SPLIT > 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) got[team][d + e] = x[e];
    if (d == 0) got[team][kPageDim] = m, got[team][kPageDim + 1] = sum;
    __syncthreads();
    if (team) return;
    float top = -INFINITY;
    for (int k = 0; k < kTeams; ++k) top = fmaxf(top, got[k][kPageDim]);
    const float ref = against(top);
    m = top, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    for (int k = 0; k < kTeams; ++k) {
      const float w = exp2_fast(got[k][kPageDim] - ref);
      sum += w * got[k][kPageDim + 1];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] += w * got[k][d + e];
    }
  }
  const bool none = !(own.has & 2);
  write_out<DT>(a, row_at(a, a.os, row, h), d, x, none ? 0.0f : 1.0f / sum);
  if (a.lse && d == 0)
    a.lse[(int64_t)tok * a.Hq + h * a.G + row - tok * a.G] =
        none ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}

// ---- host ------------------------------------------------------------------------
int check_attend(const ferry_pages* p, const ferry_attend* a, PageView* v) {
  if (int rc = page_geometry(p, v)) return rc;
  if (!a) return report(FERRY_EINVAL, "null args");
  if (a->n_req < 0 || a->n_tokens < 0 || a->n_groups < 0 || a->n_groups > a->n_req)
    return report(FERRY_EINVAL, "n_req, n_tokens and n_groups must not be negative, n_groups at most n_req");
  if (a->q_heads < 1 || a->q_heads > 65535 || a->q_heads % p->kv_heads)
    return report(FERRY_EINVAL, "q_heads must be a multiple of kv_heads");
  if ((int64_t)a->n_tokens * (a->q_heads / p->kv_heads) > 0x3FFFFFFF)
    return report(FERRY_EINVAL, "too many query rows");
  if (!a->q_start && a->n_tokens != a->n_req)
    return report(FERRY_EINVAL, "without q_start a request has one token");
  return FERRY_OK;
}

uint64_t up256(uint64_t x) { return (x + 255) & ~255ull; }

// The tile forms a call may need: a segment has at most the rows of the whole batch,
// without groups and with one token per request those of one token.
int attend_forms(const ferry_pages* p, const ferry_attend* a) {
  const int64_t G = a->q_heads / p->kv_heads, rows = a->n_groups || a->q_start ? a->n_tokens * G : G;
  return p->dtype == FERRY_F32 || rows <= 16 ? 1 : rows <= 32 ? 2 : 3;
}

// Workgroups of a call, and its scratch at `base` (null: sizes only).
int plan_attend(const ferry_pages* p, const ferry_attend* a, uint8_t* base, Scratch* ws, uint64_t* bytes) {
  const int grid = kPerCu * gpu_cus(p->device);
  const uint64_t rows = (uint64_t)a->n_tokens * (a->q_heads / p->kv_heads), H = p->kv_heads;
  const uint64_t tile = p->dtype == FERRY_F32 ? 16 : std::min<uint64_t>(kWide, rows);
  uint64_t at = 0;
  auto take = [&](uint64_t n) {
    uint8_t* r = base + at;
    at += up256(n);
    return r;
  };
  ws->tile_rows = (int)tile;
  ws->where = reinterpret_cast<Where*>(take(2 * H * rows * sizeof(Where)));
  ws->part_ml = reinterpret_cast<float*>(take(2ull * grid * tile * 8));
  ws->part_o = reinterpret_cast<float*>(take(2ull * grid * tile * kPageDim * 4));
  const uint64_t twice = a->n_groups ? 2 * H * rows : 0;
  ws->row_ml = reinterpret_cast<float*>(take(twice * 8));
  ws->row_o = reinterpret_cast<float*>(take(twice * kPageDim * 4));
  *bytes = at;
  return grid;
}

template <int DT>
void launch_attend(const PageView& v, int layer, const AttendArgs& a, const Scratch& ws, int forms, int grid,
                   hipStream_t s) {
  if (forms == 1) k_attend<DT, 1><<<grid, kThreads, 0, s>>>(v, layer, a, ws);
  if constexpr (DT != FERRY_F32) {
    if (forms == 2) k_attend<DT, 2><<<grid, kThreads, 0, s>>>(v, layer, a, ws);
    if (forms == 3) k_attend<DT, 3><<<grid, kThreads, 0, s>>>(v, layer, a, ws);
  }
  // a workgroup per row where that does not fill the GPU twice
  const uint64_t all = (uint64_t)a.n_tokens * a.Hq;
  if (all <= 2ull * grid) {
    k_attend_join<DT, 16><<<(unsigned)all, kThreads, 0, s>>>(v, a, ws, grid, 0);
    return;
  }
  constexpr uint64_t kMost = 1ull << 27;  // rows of a launch, which has fewer than 2^32 threads
  for (uint64_t r0 = 0; r0 < all; r0 += kMost)
    k_attend_join<DT, 1><<<(unsigned)((std::min(all - r0, kMost) + 15) / 16), kThreads, 0, s>>>(v, a, ws, grid, r0);
}

}  // namespace

extern "C" {

int ferry_pages_attend_work_bytes(const ferry_pages* p, const ferry_attend* a, uint64_t* bytes) {
  return entry([&]() -> int {
    PageView v;
    if (int rc = check_attend(p, a, &v)) return rc;
    if (!bytes) return report(FERRY_EINVAL, "null bytes");
    Scratch ws;
    plan_attend(p, a, nullptr, &ws, bytes);
    return FERRY_OK;
  });
}

int ferry_pages_attend(const ferry_pages* p, int32_t layer, const ferry_attend* a, void* stream) {
  return entry([&]() -> int {
    PageView v;
    if (int rc = check_attend(p, a, &v)) return rc;
    if (layer < 0 || layer >= p->n_layers) return report(FERRY_EINVAL, "layer out of range");
    if (a->n_req == 0 || a->n_tokens == 0) return FERRY_OK;
    if (int rc = page_buffers(p, false)) return rc;
    if (int rc = check_all({{a->lanes, "lanes"}, {a->q, "q"}, {a->out, "out"}, {a->work, "work"}}, p->device)) return rc;
    if (a->q_start)
      if (int rc = check_on(a->q_start, "q_start", p->device)) return rc;
    if (a->n_groups)
      if (int rc = check_all({{a->group_start, "group_start"}, {a->shared, "shared"}}, p->device)) return rc;
    if (a->lse)
      if (int rc = check_on(a->lse, "lse", p->device)) return rc;
    if (a->q == a->out && (a->q_stride[0] != a->out_stride[0] || a->q_stride[1] != a->out_stride[1]))
      return report(FERRY_EINVAL, "out is q with other strides");
    Scratch ws;
    uint64_t need = 0;
    const int grid = plan_attend(p, a, static_cast<uint8_t*>(a->work), &ws, &need);
    if (a->work_bytes < need) return report(FERRY_EINVAL, "work is smaller than ferry_pages_attend_work_bytes");
    if (reinterpret_cast<uintptr_t>(a->work) % 256) return report(FERRY_EINVAL, "work must be 256-byte aligned");
    OnDevice on(p->device);
    if (!on.ok()) return report(FERRY_EHIP, "cannot use the cache's GPU");
    const int es = p->dtype == FERRY_F32 ? 4 : 2;
    uint64_t low = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out);
    for (int i = 0; i < 2; ++i) low |= (uint64_t)(a->q_stride[i] * es) | (uint64_t)(a->out_stride[i] * es);
    AttendArgs d{a->n_req, a->n_tokens, a->n_groups, a->q_heads, a->q_heads / p->kv_heads,
                 a->scale != 0.0f ? a->scale : 0.08838834764831845f, a->lanes, a->q_start, a->group_start,
                 a->shared, a->q, a->out, a->lse, {a->q_stride[0], a->q_stride[1]},
                 {a->out_stride[0], a->out_stride[1]}, low % 16 == 0, 0, 31};
    while (1 << (d.g_shift - 31) < d.G) ++d.g_shift;
    d.g_mul = (uint32_t)((1ull << d.g_shift) / d.G + 1);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int forms = attend_forms(p, a);
    if (p->dtype == FERRY_F32) launch_attend<FERRY_F32>(v, layer, d, ws, forms, grid, s);
    else if (p->dtype == FERRY_F16) launch_attend<FERRY_F16>(v, layer, d, ws, forms, grid, s);
    else if (p->dtype == FERRY_BF16) launch_attend<FERRY_BF16>(v, layer, d, ws, forms, grid, s);
    else launch_attend<FERRY_FP8_E4M3>(v, layer, d, ws, forms, grid, s);
    return launched("ferry_pages_attend");
  });
}

}  // extern "C"
