// pages_attn.hip -- attention of new query tokens over the pages of their lanes.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "pages.hpp"

using namespace ferry_amd;

namespace {

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
};

template <int DT>
__device__ inline float kv_elem(const uint8_t* p, int i) {
  if constexpr (DT == FERRY_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (DT == FERRY_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  else if constexpr (DT == FERRY_BF16) return bits_f32((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
  else {
    const uint32_t c = p[i];
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false);
    return (float)x[0];
  }
}

// A wavefront per (query row, head): two dims a lane, one token at a time.
template <int DT>
__global__ __launch_bounds__(64) void k_attend(PageView v, int layer, AttendArgs a) {
  const int row = blockIdx.x, h = blockIdx.y, l = threadIdx.x;
  // the request of this row
  int lo = 0, first = row, last = row + 1;
  if (a.q_start && row == 0 && h == 0)
    for (int i = l; i < a.n_req; i += 64)
      if (a.q_start[i] < 0 || a.q_start[i] > a.q_start[i + 1] || a.q_start[i + 1] > a.n_tokens)
        set_error(v.error, FERRY_ERANGE);
  if (a.q_start) {
    int hi = a.n_req - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (a.q_start[mid] <= row) lo = mid; else hi = mid - 1;
    }
    first = a.q_start[lo], last = a.q_start[lo + 1];
    if (row < first || row >= last) return;
  } else {
    lo = row;
    if (lo >= a.n_req) return;
  }
  const int lane = a.lanes[lo];
  int seen = 0, len = 0;
  if (lane >= 0 && lane < v.n_lanes) {
    len = v.len[lane];
    if (len > v.max_pages * kPageTokens) len = v.max_pages * kPageTokens, set_error(v.error, FERRY_ERANGE);
    seen = len - (last - first) + (row - first) + 1;
  } else if (lane != -1) {
    set_error(v.error, FERRY_ERANGE);
  }
  const int kvh = h / a.G;
  float q0, q1, m = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
  const int64_t qi = row * a.qs[0] + h * a.qs[1] + 2 * l;
  if constexpr (DT == FERRY_F32) q0 = static_cast<const float*>(a.q)[qi], q1 = static_cast<const float*>(a.q)[qi + 1];
  else if constexpr (DT == FERRY_F16) q0 = (float)static_cast<const _Float16*>(a.q)[qi], q1 = (float)static_cast<const _Float16*>(a.q)[qi + 1];
  else q0 = bits_f32((uint32_t)static_cast<const uint16_t*>(a.q)[qi] << 16), q1 = bits_f32((uint32_t)static_cast<const uint16_t*>(a.q)[qi + 1] << 16);
  for (int t = 0; t < seen; ++t) {
    uint32_t page = v.table[(uint64_t)lane * v.max_pages + t / kPageTokens];
    if (page >= (uint32_t)v.n_pages) page = 0, set_error(v.error, FERRY_ERANGE);
    const uint64_t rec = v.record(layer, page, kvh);
    const uint8_t* kp = v.pool + rec * v.bb;
    const int at = (t % kPageTokens) * kPageDim + 2 * l;
    const float ks = DT == FERRY_FP8_E4M3 ? v.scales[2 * rec] : 1.0f;
    const float vs = DT == FERRY_FP8_E4M3 ? v.scales[2 * rec + 1] : 1.0f;
    float s = q0 * kv_elem<DT>(kp, at) + q1 * kv_elem<DT>(kp, at + 1);
    for (int d = 32; d; d /= 2) s += __shfl_xor(s, d);
    s *= a.scale * ks;
    const float top = fmaxf(m, s), ref = top == -INFINITY ? 0.0f : top;
    const float keep = expf(m - ref), p = expf(s - ref);
    m = top;
    sum = sum * keep + p;
    o0 = o0 * keep + p * vs * kv_elem<DT>(kp, kPageTokens * kPageDim + at);
    o1 = o1 * keep + p * vs * kv_elem<DT>(kp, kPageTokens * kPageDim + at + 1);
  }
  const float inv = seen > 0 ? 1.0f / sum : 0.0f;
  const int64_t oi = row * a.os[0] + h * a.os[1] + 2 * l;
  o0 *= inv, o1 *= inv;
  if constexpr (DT == FERRY_F32) static_cast<float*>(a.out)[oi] = o0, static_cast<float*>(a.out)[oi + 1] = o1;
  else if constexpr (DT == FERRY_F16) static_cast<_Float16*>(a.out)[oi] = (_Float16)o0, static_cast<_Float16*>(a.out)[oi + 1] = (_Float16)o1;
  else static_cast<uint16_t*>(a.out)[oi] = f32_to_bf16(o0), static_cast<uint16_t*>(a.out)[oi + 1] = f32_to_bf16(o1);
  if (a.lse && l == 0) a.lse[(int64_t)row * a.Hq + h] = seen > 0 ? m + logf(sum) : -INFINITY;
}

int check_attend(const ferry_pages* p, const ferry_attend* a, PageView* v) {
  if (int rc = page_geometry(p, v)) return rc;
  if (!a) return report(FERRY_EINVAL, "null args");
  if (a->n_req < 0 || a->n_tokens < 0 || a->n_groups < 0 || a->n_groups > a->n_req)
    return report(FERRY_EINVAL, "n_req, n_tokens and n_groups must not be negative, n_groups at most n_req");
  if (a->q_heads < 1 || a->q_heads > 65535 || a->q_heads % p->kv_heads)
    return report(FERRY_EINVAL, "q_heads must be a multiple of kv_heads");
  if (!a->q_start && a->n_tokens != a->n_req)
    return report(FERRY_EINVAL, "without q_start a request has one token");
  return FERRY_OK;
}

}  // namespace

extern "C" {

int ferry_pages_attend_work_bytes(const ferry_pages* p, const ferry_attend* a, uint64_t* bytes) {
  return entry([&]() -> int {
    PageView v;
    if (int rc = check_attend(p, a, &v)) return rc;
    if (!bytes) return report(FERRY_EINVAL, "null bytes");
    *bytes = 256;
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
    OnDevice on(p->device);
    if (!on.ok()) return report(FERRY_EHIP, "cannot use the cache's GPU");
    AttendArgs d{a->n_req, a->n_tokens, a->n_groups, a->q_heads, a->q_heads / p->kv_heads,
                 a->scale != 0.0f ? a->scale : 0.08838834764831845f, a->lanes, a->q_start, a->group_start,
                 a->shared, a->q, a->out, a->lse, {a->q_stride[0], a->q_stride[1]}, {a->out_stride[0], a->out_stride[1]}};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(a->n_tokens, a->q_heads);
    if (p->dtype == FERRY_F32) k_attend<FERRY_F32><<<grid, 64, 0, s>>>(v, layer, d);
    else if (p->dtype == FERRY_F16) k_attend<FERRY_F16><<<grid, 64, 0, s>>>(v, layer, d);
    else if (p->dtype == FERRY_BF16) k_attend<FERRY_BF16><<<grid, 64, 0, s>>>(v, layer, d);
    else k_attend<FERRY_FP8_E4M3><<<grid, 64, 0, s>>>(v, layer, d);
    return launched("ferry_pages_attend");
  });
}

}  // extern "C"
