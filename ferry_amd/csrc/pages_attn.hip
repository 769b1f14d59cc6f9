// pages_attn.hip -- attention of new query tokens over the pages of their lanes
// (ferry_pages_attend): the call's checks, its plan and its launches.
#include "pages_attn.hpp"

namespace {

// ---- host ------------------------------------------------------------------------
int check_attend(const ferry_pages* p, const ferry_attend* a, const ferry_seen* seen, PageView* v) {
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
  if (seen) {
    if (seen->window < 0 || seen->sinks < 0) return report(FERRY_EINVAL, "window and sinks must not be negative");
    if (seen->sinks && !seen->window) return report(FERRY_EINVAL, "sinks go with a window");
    if (seen->window && a->n_groups) return report(FERRY_EINVAL, "a window goes with no groups");
    if (seen->tree_words < 0 || seen->tree_words > kTreeWords)
      return report(FERRY_EINVAL, "tree_words must be 0..64");
    if (a->n_tokens && (seen->tree_words > 0) != (seen->tree != nullptr))
      return report(FERRY_EINVAL, "tree and tree_words go together");
    if (reinterpret_cast<uintptr_t>(seen->tree) % 8) return report(FERRY_EINVAL, "tree must be 8-byte aligned");
  }
  return FERRY_OK;
}

uint64_t up256(uint64_t x) { return (x + 255) & ~255ull; }

// The tile forms a call may need: a segment has at most the rows of the whole batch,
// without groups and with one token per request those of one token.
int attend_forms(const ferry_pages* p, const ferry_attend* a) {
  const int64_t G = a->q_heads / p->kv_heads, rows = a->n_groups || a->q_start ? a->n_tokens * G : G;
  return p->dtype == FERRY_F32 || rows <= 16 ? 1 : rows <= 32 ? 2 : 3;
}

// Whether a call of form 3 goes to workgroups of eight wavefronts with tiles of up to 256
// rows, one per CU, rather than to those of four with 128, two per CU: where most tiles
// would read their pages for a second tile of the same request.  The rule is on the rows
// that a request has on average, as only the device knows each one's.  In us, wide and
// not, of 8 kv heads, 4 heads a kv head, 32 requests unless stated, bf16 (fp8):
//   drafts over 1,000 to 8,000 tokens: 12 to 24 of them 140 and 136 (125 and 114), 16 to 32
//   145 and 141 (136 and 119), 20 to 40 161 and 170 (173 and 160), 24 to 48 165 and 199
//   (176 and 182), 32 to 64 175 and 229 (179 and 203); 16 and 128 requests of 12 to 24 over
//   2,000: 47 and 42, 189 and 166 (46 and 42, 194 and 148).  In groups, whose shared pages
//   meet the rows of all members, over 8,000 shared tokens: 4 to 8 544 and 527 (542 and 540),
//   12 to 24 1,189 and 1,471 (1,259 and 1,423); over 1,000: 8 to 16 152 and 145 (163 and 160);
//   four groups over 4,000: 8 to 16 557 and 663 (561 and 623).  Up to four requests have fewer
//   parts to join: 4 x 8 over 700 18.1 and 19.1, 2 x 32 over 131,000 175 and 178.
//   windows of 4,096: 8 to 16 tokens 161 and 134 (140 and 105), 12 to 24 117 and 133 (105 and
//   111), 16 to 32 120 and 137 (107 and 119), 24 to 48 143 and 174 (157 and 180), 32 to 64 172
//   and 177 (179 and 192); of 1,024: 12 to 24 50 and 54 (49 and 54); of 1,000: 40 to 80 94 and
//   90 (107 and 101); 64 requests of 12 to 24 through 512 68 and 51, 8 of them through 4,096 53
//   and 48; 4 prompts of 1,500 157 and 137, as the tiles of a long request begin at other
//   pages each.
// So the rule is not the better side everywhere: it refuses windows of 12 to 32 tokens a request,
// where wide tiles take 5 to 14 % less if there is just one of them for each CU (32 requests
// of 8 heads) and more if not, and takes drafts of 20 to 40 in fp8 and windows of 40 to 80,
// at 5 to 8 % more.  It does not weigh the tiles against the CUs.
bool takes_wide(const ferry_pages* p, const ferry_attend* a, const ferry_seen* seen) {
  const int64_t rows = (int64_t)a->n_tokens * (a->q_heads / p->kv_heads), n = a->n_req;
  if (seen->window) return rows > 112 * n && rows <= 256 * n;
  return a->n_groups ? rows > 32 * n : n <= 4 || rows > 112 * n;
}

// Workgroups of a call, and its scratch at `base` (null: sizes only).
// wide: of one workgroup per CU, whose tiles have up to twice the rows; its parts take
// no more room.
int plan_attend(const ferry_pages* p, const ferry_attend* a, bool wide, uint8_t* base, Scratch* ws, uint64_t* bytes) {
  const int grid = (wide ? 1 : kPerCu) * gpu_cus(p->device);
  const uint64_t rows = (uint64_t)a->n_tokens * (a->q_heads / p->kv_heads), H = p->kv_heads;
  const uint64_t tile = p->dtype == FERRY_F32 ? 16 : std::min<uint64_t>(wide_of(wide ? kSeenWide : kCausal), rows);
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
void launch_attend(const PageView& v, int layer, const AttendArgs& a, const Scratch& ws, int forms, bool wide, int grid,
                   hipStream_t s) {
  if (a.seen.window || a.seen.words) launch_attend_seen(v, layer, DT, a, ws, forms, wide, grid, s);
  else launch_forms<DT, kCausal>(v, layer, a, ws, forms, grid, s);
  // a workgroup per row where that does not fill the GPU twice
  const uint64_t all = (uint64_t)a.n_tokens * a.Hq;
  if (all <= 2ull * (wide ? kPerCu : 1) * grid) {
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
    if (int rc = check_attend(p, a, nullptr, &v)) return rc;
    if (!bytes) return report(FERRY_EINVAL, "null bytes");
    Scratch ws;
    plan_attend(p, a, false, nullptr, &ws, bytes);
    return FERRY_OK;
  });
}

int ferry_pages_attend(const ferry_pages* p, int32_t layer, const ferry_attend* a, void* stream) {
  return ferry_pages_attend_seen(p, layer, a, nullptr, stream);
}

int ferry_pages_attend_seen(const ferry_pages* p, int32_t layer, const ferry_attend* a, const ferry_seen* seen,
                            void* stream) {
  return entry([&]() -> int {
    PageView v;
    if (int rc = check_attend(p, a, seen, &v)) return rc;
    if (seen && !seen->window && !seen->tree_words) seen = nullptr;  // the causal call, its grid and scratch too
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
    if (seen && seen->tree)
      if (int rc = check_on(seen->tree, "tree", p->device)) return rc;
    if (a->q == a->out && (a->q_stride[0] != a->out_stride[0] || a->q_stride[1] != a->out_stride[1]))
      return report(FERRY_EINVAL, "out is q with other strides");
    Scratch ws;
    uint64_t need = 0;
    const int forms = attend_forms(p, a);
    const bool wide = forms == 3 && seen && takes_wide(p, a, seen);
    const int grid = plan_attend(p, a, wide, static_cast<uint8_t*>(a->work), &ws, &need);
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
                 {a->out_stride[0], a->out_stride[1]}, low % 16 == 0, 0, 31, {}};
    constexpr int kAll = 1 << 25;  // more tokens than a lane holds
    if (seen) d.seen = SeenArgs{std::min(seen->window, kAll), std::min(seen->sinks, kAll), seen->tree_words, seen->tree};
    while (1 << (d.g_shift - 31) < d.G) ++d.g_shift;
    d.g_mul = (uint32_t)((1ull << d.g_shift) / d.G + 1);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->dtype == FERRY_F32) launch_attend<FERRY_F32>(v, layer, d, ws, forms, wide, grid, s);
    else if (p->dtype == FERRY_F16) launch_attend<FERRY_F16>(v, layer, d, ws, forms, wide, grid, s);
    else if (p->dtype == FERRY_BF16) launch_attend<FERRY_BF16>(v, layer, d, ws, forms, wide, grid, s);
    else launch_attend<FERRY_FP8_E4M3>(v, layer, d, ws, forms, wide, grid, s);
    return launched("ferry_pages_attend");
  });
}

}  // extern "C"
