// bkv_api.cpp - the C ABI (include/bkv.h): descriptor validation, partition planning, workspace
// layout and kernel dispatch. No allocation, no host synchronisation, no exception crosses out.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "../../include/bkv.h"
#include "bkv_internal.h"

namespace bkv {

static thread_local char g_hip_err[256] = "";

int hip_fail(hipError_t e) {
  if (e == hipSuccess) return BKV_OK;
  std::snprintf(g_hip_err, sizeof g_hip_err, "%s: %s", hipGetErrorName(e), hipGetErrorString(e));
  return BKV_EHIP;
}

static inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline int64_t next_pow2(int64_t x) {
  int64_t p = 1;
  while (p < x) p <<= 1;
  return p;
}
static inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
// the fewest keys a resident or stream workgroup takes (short contexts use fewer workgroups; at 4K
// keys, config 2: 128 (33 workgroups per group) 149.7-150.8 us per token, 96 150.9-152.4, 112
// 150.9-153.6, 64 154.0-156.0, 80 159.1-164.0; more than 128 leaves the short plan)
constexpr int64_t kResMinKeysPerWg = 128;

// Partition sizes of the split path. QK: the keys of one workgroup (256 q8_0 / 128 fp16). Probability chunks: kE2Chunk keys. PV: enough workgroups to cover the chip (512 at nkv = 4)
// with 16..512 keys each. Every array is sized
// by a bound that grows monotonically with n, so a workspace sized for max_ctx fits every n <= max_ctx.
// BKV_DECODE forces a decode implementation where its plan fits: "split" (four launches),
// "resident" or "stream" (single launches). Without it, q8_0 K + V plans that fit the stream kernel
// take it, other single-launch plans the resident kernel, the rest the split path. Read on every
// call, so tests can switch it.
enum { kPathSplit = 0, kPathResident = 2, kPathStream = 3 };
static int forced_path() {
  const char *e = std::getenv("BKV_DECODE");
  if (!e) return -1;
  if (std::strcmp(e, "split") == 0) return kPathSplit;
  if (std::strcmp(e, "resident") == 0) return kPathResident;
  if (std::strcmp(e, "stream") == 0) return kPathStream;
  return -1;
}

// Chunked prefill: 16 queries x 4 heads per workgroup; when that gives fewer than kPfFill
// workgroups the key range of every query block is split so that the chip fills (never into more
// splits than the first query block has 64-key tiles).
static int prefill_splits(int nkv, int nqb, int64_t first_keys) {
  const int64_t want = std::max<int64_t>(1, cdiv(kPfFill, (int64_t)nkv * nqb));
  return (int)std::min<int64_t>(want, std::max<int64_t>(1, cdiv(first_keys, kPfTile)));
}

// BKV_PREFILL=mfma selects the matrix-core prefill (scores and sums in MFMA order: within
// tolerance of the serial reference on long rows, not bit-identical probabilities); the default
// is the exact path.
static bool prefill_mfma_requested() {
  const char *e = std::getenv("BKV_PREFILL");
  return e && std::strcmp(e, "mfma") == 0;
}

// Prefill arrays start past every array a decode on the same workspace can use (the decode plan
// at the cache's full capacity): the resident decode polls its partials for generation tags, so no
// other path may leave bytes in that region.
PrefillPlan plan_prefill(int nh, int nkv, uint32_t pos0, int n_q, size_t base) {
  PrefillPlan p{};
  p.nqb = (int)cdiv(n_q, kPfQ);
  p.nsplit = prefill_splits(nkv, p.nqb, (int64_t)pos0 + std::min(n_q, kPfQ));
  const size_t rows = (size_t)n_q * nh;
  size_t o = base;
  p.off_stats = o;
  o = align256(o + (size_t)p.nsplit * rows * sizeof(float2));
  p.off_part = o;
  if (p.nsplit > 1) o = align256(o + (size_t)p.nsplit * rows * kHd * sizeof(float));
  p.total = o;
  return p;
}

// The exact prefill runs a chunk in slices of queries, whose scores it keeps: at least kPxSlice
// queries, more where their scores take at most kPxScratch (short contexts: fewer, fuller launches).
struct PxLayout {
  int64_t ld;                              // keys per query in the scratch (+ the exp sweep's overhang)
  size_t sums, part, total;
};
static PxLayout px_layout(int nh, int nkv, int64_t max_ctx, int64_t slice, size_t base) {
  PxLayout l;
  l.ld = cdiv(max_ctx, kPxTile16) * kPxTile16 + kPxTile16;
  const size_t units = (size_t)nkv * cdiv(slice, kPxQ);
  l.sums = base + align256(units * (size_t)l.ld * kPxRows * sizeof(float));
  l.part = l.sums + align256(units * kPxRows * sizeof(float));
  l.total = l.part + align256((size_t)kPvSplit * kPxSlice * nh * kHd * sizeof(float));
  return l;
}
static int64_t px_slice(int nkv, int64_t max_ctx, int64_t n_q) {
  const int64_t ld = cdiv(max_ctx, kPxTile16) * kPxTile16 + kPxTile16;
  const int64_t fit = (int64_t)(kPxScratch / ((size_t)nkv * ld * kGqa * sizeof(float))) / kPxQ * kPxQ;
  return std::min<int64_t>(n_q, std::max<int64_t>(kPxSlice, std::min<int64_t>(fit, BKV_PREFILL_MAX_Q)));
}
// the workspace for chunks ending at or before max_ctx: the largest any of them asks for
size_t prefill_exact_workspace(int nh, int nkv, int64_t max_ctx, size_t base) {
  const size_t least = px_layout(nh, nkv, max_ctx, kPxSlice, base).total;
  const int64_t most = std::min<int64_t>(max_ctx, BKV_PREFILL_MAX_Q);
  if (most <= kPxSlice) return least;
  const size_t scratch = std::min<size_t>(kPxScratch, px_layout(nh, nkv, max_ctx, most, 0).sums);
  return std::max(least, base + align256(scratch) + px_layout(nh, nkv, 1, BKV_PREFILL_MAX_Q, 0).total -
                             px_layout(nh, nkv, 1, BKV_PREFILL_MAX_Q, 0).sums);
}

// the largest plan_prefill(...).total over every chunk length and start position
size_t prefill_workspace_bound(int nh, int nkv, size_t base) {
  size_t worst = 0;
  for (int nqb = 1; nqb <= BKV_PREFILL_MAX_Q / kPfQ; ++nqb) {
    const int nsplit = (int)std::max<int64_t>(1, cdiv(kPfFill, (int64_t)nkv * nqb));
    const size_t rows = (size_t)nqb * kPfQ * nh;
    size_t o = align256(base + (size_t)nsplit * rows * sizeof(float2));
    if (nsplit > 1) o = align256(o + (size_t)nsplit * rows * kHd * sizeof(float));
    worst = std::max(worst, o);
  }
  return worst;
}

DecodePlan plan_decode(int nh, int nkv, int kfmt, int vfmt, int64_t n, int page) {
  DecodePlan p;
  p.qk_chunk = qk_keys_per_wg(kfmt);
  p.nch_qk = (int)cdiv(n, p.qk_chunk);
  p.nch_e = (int)cdiv(n, kE2Chunk);
  p.pv_chunk = (int)std::min<int64_t>(kPvMaxChunk, std::max<int64_t>(16, next_pow2(cdiv(n * nkv, 512))));
  p.nch_pv = (int)cdiv(n, p.pv_chunk);
  p.ld = cdiv(n, kE2Chunk) * kE2Chunk;
  const int64_t nq_bound = cdiv(n, 128);
  const int64_t np_bound = std::max<int64_t>(128, cdiv(n, kPvMaxChunk));
  // the single-launch kernels' tagged partials sit at a fixed offset that no other array of any
  // plan overlaps: a poll never sees bytes another path (or another context length) left there
  const size_t tagged_part = align256((size_t)nkv * kResMaxGroupWgs * kGqa * kHd * sizeof(unsigned long long));
  size_t o = kSyncBytes + tagged_part;
  p.off_score = o;  o += align256((size_t)nh * p.ld * sizeof(float));
  p.off_e = o;      o += align256((size_t)nh * p.ld * sizeof(float));
  p.off_stats = o;  o += align256((size_t)nh * nq_bound * sizeof(float2));
  p.off_rec = o;    o += align256((size_t)nh * p.nch_e * sizeof(ChunkRec));
  p.off_spec = o;   o += align256((size_t)nh * p.nch_e * kMaxSpecial * sizeof(Special));
  p.off_cnt = o;    o += align256((size_t)nh * kCounterStride * sizeof(unsigned));
  p.off_sum = o;    o += align256((size_t)nh * sizeof(float));
  p.off_status = o; o += align256((size_t)nh * sizeof(unsigned));
  p.off_dbg = o;    o += align256((size_t)nh * 8 * sizeof(unsigned long long));
  p.off_part = o;   o += align256((size_t)np_bound * nh * kHd * sizeof(float));
  size_t total = o;
  // the resident path: one workgroup per CU, up to kResMaxG per KV group, >= 128 keys each
  // (below 64 x kResMinKeysPerWg keys fewer workgroups per group, each with at least that many keys)
  p.rG = 0;
  p.rvres = p.rstream = false;
  const int rcap = resident_max_workgroups(kfmt, vfmt);
  const bool rsync_fits = kResSyncOffset + ((size_t)nkv * kResGroupLines + 1) * kCounterStride * sizeof(unsigned) <= kSyncBytes;
  const bool rtags_fit = kResTagOffset + (size_t)nh * kResMaxGroupWgs * 3 * sizeof(unsigned long long) <= kResSyncOffset;
  if (rcap >= nkv && rsync_fits && rtags_fit) {
    const int64_t gmax = std::min<int64_t>(rcap / nkv, kResMaxGroupWgs);
    const int64_t kpw = cdiv(n, std::min<int64_t>(gmax, cdiv(n, kResMinKeysPerWg)));
    // paged: a workgroup's keys must span at most kResPgMax pages (the kernel's LDS page table)
    const bool pages_fit = page <= 0 || cdiv(kpw, page) + 1 <= kResPgMax;
    if (kpw <= (int64_t)kResMaxPass * kResNT && pages_fit) {
      p.rkpw = (int)kpw;
      p.rG = (int)cdiv(n, kpw);
      p.rvres = vfmt == BKV_Q8_0 && kfmt == BKV_Q8_0 && kpw <= kResNT + kResTail;
      // the stream kernel: q8_0 V with q8_0 or fp16 K, one pass plus a tail per workgroup
      p.rstream = vfmt == BKV_Q8_0 && (kfmt == BKV_Q8_0 || kfmt == BKV_F16) && kpw <= kResNT + kResTail &&
                  p.rG * nkv <= stream_max_workgroups(page > 0);
      p.r_part = kSyncBytes;
      size_t f = kSyncBytes + tagged_part;
      p.r_spec = f;   f += align256((size_t)nh * gmax * kMaxSpecial * sizeof(Special));
      p.r_e = f;      f += align256((size_t)nh * p.ld * sizeof(float));
      p.r_sum = f;    f += align256((size_t)nh * sizeof(float));
      p.r_status = f; f += align256((size_t)nh * sizeof(unsigned));
      p.r_total = f;
      total = std::max(total, f);
    }
  }
#ifdef BKV_EXPERIMENT_TS
  total = align256(total) + 262144;
  p.ts_off = total - 262144;
#endif
  p.total = total;
  return p;
}

// BKV_KEEP_INTERMEDIATES=1: the resident path also writes every e_j into the workspace (where
// bkv_debug_layout says) for parity diagnostics; the other paths always do
static bool keep_intermediates() {
  const char *e = std::getenv("BKV_KEEP_INTERMEDIATES");
  return e && std::strcmp(e, "1") == 0;
}

// which implementation a decode of this plan takes
static int choose_path(const DecodePlan &p) {
  const int f = forced_path();
  if (f == kPathSplit) return kPathSplit;
  if (f == kPathResident && p.rG > 0) return kPathResident;
  if (p.rstream) return kPathStream;
  if (p.rG > 0) return kPathResident;
  return kPathSplit;
}

// Contexts a decode takes in one workgroup per KV group (bkv_short.hip): six V tiles with q8_0 V (seven with q8_0
// K, no pages and up to 4 KV heads), seven (pages, which cost it a lookup per load) or eight with fp16 V. us of
// one layer of 8 against the stream kernel, q8_0: 6.2 / 17.1 at 64 keys, 12.8 / 17.1 at 300, 16.5 / 17.1 at 400,
// 17.2 / 17.1 at 440 (8 KV heads 17.0 / 17.0 at 385, 17.5 / 17.0 at 420); with fp16 K 15.0 / 18.6 at 300; against
// the resident kernel, fp16 V: 14.9 / 22.0 at 300, 20.3 / 21.9 at 500.
static int short_decode_keys(int kfmt, int vfmt, bool paged, int nkv) {
  if (vfmt == BKV_Q8_0) return kfmt == BKV_Q8_0 && !paged && nkv <= 4 ? 448 : 384;
  return paged ? 448 : kShortKeys;
}

static bool aligned16(const void *p) { return p && ((uintptr_t)p & 15u) == 0; }

static uint64_t slot_bytes(const bkv_cache_desc *d, int which) {
  const int fmt = which < 2 ? d->k_fmt : d->v_fmt;
  const uint64_t hd = (uint64_t)d->hd, nkv = (uint64_t)d->nkv;
  switch (which) {
    case 0: case 2: return fmt == BKV_F16 ? nkv * hd * 2 : fmt == BKV_Q4_0 ? nkv * hd / 2 : nkv * hd;
    default: return fmt == BKV_F16 ? 0 : nkv * (hd / 32) * 2;
  }
}

static bool known(int fmt) { return fmt == BKV_F16 || fmt == BKV_Q8_0 || fmt == BKV_Q4_0; }

// the geometry, of any format
static int check_geom(const bkv_cache_desc *d) {
  if (!d) return BKV_EINVAL;
  if (d->n_layers < 1 || d->nkv < 1 || d->nh < 1 || d->hd < 1 || d->cap < 1) return BKV_EINVAL;
  if (!known(d->k_fmt) || !known(d->v_fmt)) return BKV_EINVAL;
  // KvGeom::check (runtime_vk/kv_guard.h:103-113)
  if (d->hd % 4 || d->hd % 32 || (d->hd / 32) % 2) return BKV_ESHAPE;
  if (d->nh % d->nkv) return BKV_ESHAPE;
  if (!(std::isfinite(d->scale)) || d->scale <= 0.0f) return BKV_EINVAL;
  if (d->page_tokens < 0) return BKV_EINVAL;
  if (d->page_tokens > 0) {
    if (d->cap % d->page_tokens || d->max_pages < 1 || !d->block_table) return BKV_EINVAL;
  }
  if (!d->k_data || !d->v_data) return BKV_EINVAL;
  if (d->k_fmt != BKV_F16 && !d->k_scales) return BKV_EINVAL;
  if (d->v_fmt != BKV_F16 && !d->v_scales) return BKV_EINVAL;
  const void *ptrs[4] = {d->k_data, d->k_scales, d->v_data, d->v_scales};
  for (int i = 0; i < 4; ++i) {
    const uint64_t sb = slot_bytes(d, i);
    if (!sb) continue;
    if (!aligned16(ptrs[i])) return BKV_EALIGN;
    if (d->n_layers > 1 && d->layer_stride_bytes[i] < sb * (uint64_t)d->cap) return BKV_EINVAL;
    if (d->layer_stride_bytes[i] % 16) return BKV_EALIGN;
  }
  return BKV_OK;
}

static bool any_q4(const bkv_cache_desc *d) { return d->k_fmt == BKV_Q4_0 || d->v_fmt == BKV_Q4_0; }

// the geometry, and formats that every kernel takes (the 4-bit one has its own calls)
static int check(const bkv_cache_desc *d) {
  const int rc = check_geom(d);
  return rc ? rc : any_q4(d) ? BKV_EUNSUPPORTED : BKV_OK;
}

// shapes the gfx950 kernels are specialised for: hd 256 and 4 query heads per KV head
static int check_kernels(const bkv_cache_desc *d) {
  if (d->hd != kHd || d->nh != kGqa * d->nkv) return BKV_EUNSUPPORTED;
  return BKV_OK;
}

static int64_t max_positions(const bkv_cache_desc *d) {
  return d->page_tokens > 0 ? (int64_t)d->max_pages * d->page_tokens : (int64_t)d->cap;
}

// where a prefill's own arrays begin: past the largest decode plan this cache allows
static size_t prefill_base(const bkv_cache_desc *d) {
  return align256(plan_decode(d->nh, d->nkv, d->k_fmt, d->v_fmt, max_positions(d), d->page_tokens).total);
}

static LayerView view(const bkv_cache_desc *d, int layer) {
  LayerView L;
  auto at = [&](void *base, int i) -> const uint8_t * {
    return base ? (const uint8_t *)base + (uint64_t)layer * d->layer_stride_bytes[i] : nullptr;
  };
  L.kd = at(d->k_data, 0);
  L.ks = at(d->k_scales, 1);
  L.vd = at(d->v_data, 2);
  L.vs = at(d->v_scales, 3);
  L.bt = d->page_tokens > 0 ? d->block_table + (int64_t)layer * d->max_pages : nullptr;
  L.page = d->page_tokens > 0 ? d->page_tokens : 0;
  L.base = 0;
  return L;
}

// q / gate: head rows qs / gs floats apart (hd for [nh][hd]; 2*hd for the engine's interleaved
// attn_q output, q then gate per head)
static int decode_common(const bkv_cache_desc *d, int layer, uint32_t nfill, const float *q,
                         const float *gate, float *out, float *out_gated, void *ws, size_t ws_bytes,
                         hipStream_t st, const AppendArgs *fused, int qs = kHd, int gs = kHd,
                         uint32_t kstart = 0) {
  int rc = check(d);
  if (rc) return rc;
  if ((rc = check_kernels(d))) return rc;
  if (layer < 0 || layer >= d->n_layers) return BKV_EINVAL;
  if (nfill == 0 || (int64_t)nfill > max_positions(d)) return BKV_ECAP;
  if (!aligned16(q) || !aligned16(out)) return q && out ? BKV_EALIGN : BKV_EINVAL;
  if ((gate == nullptr) != (out_gated == nullptr)) return BKV_EINVAL;
  if (gate && (!aligned16(gate) || !aligned16(out_gated))) return BKV_EALIGN;
  if (!ws) return BKV_EWORKSPACE;
  if (((uintptr_t)ws & 255u) != 0) return BKV_EALIGN;
  // a window [kstart, nfill): the kernels see nfill - kstart keys starting at position kstart
  if (kstart >= nfill) return BKV_EINVAL;
  nfill -= kstart;
  const DecodePlan p = plan_decode(d->nh, d->nkv, d->k_fmt, d->v_fmt, nfill, d->page_tokens);
  if (ws_bytes < p.total) return BKV_EWORKSPACE;
  char *w = (char *)ws;
  LayerView L = view(d, layer);
  L.base = kstart;

  const int path = choose_path(p);
  if (forced_path() < 0 && path != kPathSplit && nfill <= (uint32_t)short_decode_keys(d->k_fmt, d->v_fmt, d->page_tokens > 0, d->nkv)) {
    // the single launch of a short context: one workgroup per KV group
    ShortArgs sa{};
    sa.L = L; sa.nkv = d->nkv; sa.nh = d->nh; sa.pos0 = nfill - 1; sa.n_q = 1; sa.scale = d->scale;
    sa.q = q; sa.qs = qs; sa.gate = gate; sa.gs = gs; sa.out = out; sa.out_gated = out_gated;
    if (fused) sa.ap = *fused;
    sa.e = keep_intermediates() ? (float *)(w + p.r_e) : nullptr;
    sa.ld = p.ld;
    sa.sum = (float *)(w + p.r_sum);
    sa.status = (unsigned *)(w + p.r_status);
    return hip_fail(launch_short(sa, d->k_fmt, d->v_fmt, st));
  }
  if (path == kPathResident || path == kPathStream) {
    ResArgs ra{};
    ra.L = L; ra.nkv = d->nkv; ra.nh = d->nh; ra.nfill = nfill; ra.scale = d->scale;
    ra.G = p.rG; ra.kpw = p.rkpw; ra.ld = p.ld; ra.q = q; ra.qs = qs; ra.gs = gs;
    if (fused) ra.ap = *fused;
    ra.gate = gate; ra.out = out; ra.out_gated = out_gated;
    ra.tstats = (unsigned long long *)(w + kResTagOffset);
    ra.trec = ra.tstats + (size_t)d->nh * kResMaxGroupWgs;
    ra.spec = (Special *)(w + p.r_spec);
    ra.e = (float *)(w + p.r_e);
    ra.keep_e = keep_intermediates() ? 1 : 0;
    ra.sum = (float *)(w + p.r_sum);
    ra.status = (unsigned *)(w + p.r_status);
    ra.part = (unsigned long long *)(w + p.r_part);
    ra.sync = (unsigned *)(w + kResSyncOffset);
#ifdef BKV_EXPERIMENT_TS
    ra.ts = (unsigned *)w + 32768;
    ra.tsw = (unsigned *)(w + p.ts_off);
#endif
    if (path == kPathStream) return hip_fail(launch_stream(ra, d->k_fmt, st));
    return hip_fail(launch_resident(ra, d->k_fmt, d->v_fmt, p.rvres, st));
  }

  QkArgs qa{};
  qa.L = L; qa.nkv = d->nkv; qa.nfill = nfill; qa.nch = p.nch_qk; qa.ld = p.ld; qa.scale = d->scale;
  qa.q = q;
  qa.qs = qs;
  qa.score = (float *)(w + p.off_score);
  qa.stats = (float2 *)(w + p.off_stats);
  qa.counters = (unsigned *)(w + p.off_cnt);
  if (fused) qa.ap = *fused;
  EArgs ea{};
  ea.nh = d->nh; ea.nfill = nfill; ea.nch_qk = p.nch_qk; ea.qk_chunk = p.qk_chunk; ea.nch = p.nch_e;
  ea.ld = p.ld; ea.scale = d->scale; ea.score = qa.score; ea.stats = qa.stats;
  ea.e = (float *)(w + p.off_e);
  ea.rec = (ChunkRec *)(w + p.off_rec);
  ea.spec = (Special *)(w + p.off_spec);
  ea.counters = qa.counters;
  ea.sum = (float *)(w + p.off_sum);
  ea.status = (unsigned *)(w + p.off_status);
  ea.dbg = (unsigned long long *)(w + p.off_dbg);
  PvArgs pa{};
  pa.L = L; pa.nkv = d->nkv; pa.nh = d->nh; pa.nfill = nfill; pa.chunk = p.pv_chunk;
  pa.nch = p.nch_pv; pa.ld = p.ld; pa.e = ea.e; pa.sum = ea.sum;
  pa.part = (float *)(w + p.off_part);
  RedArgs ra{};
  ra.nh = d->nh; ra.nch = p.nch_pv; ra.part = pa.part; ra.gate = gate; ra.gs = gs; ra.out = out;
  ra.out_gated = out_gated;
  return hip_fail(launch_decode(qa, ea, pa, ra, d->k_fmt, d->v_fmt, fused != nullptr, st));
}

}  // namespace bkv

using namespace bkv;

extern "C" {

int bkv_geom_check(const bkv_cache_desc *d) { return check_geom(d); }

uint64_t bkv_slot_bytes(const bkv_cache_desc *d, int which) {
  if (!d || which < 0 || which > 3) return 0;
  return slot_bytes(d, which);
}

int64_t bkv_max_positions(const bkv_cache_desc *d) {
  if (check_geom(d)) return 0;
  return max_positions(d);
}

// the single-sequence calls on a 4-bit cache: token t at position pos0 + t
static SeqsView one_sequence(const bkv_cache_desc *d, const LayerView &L) {
  SeqsView v{};
  v.n_seq = 1;
  v.tables = L.bt;
  v.page = L.page;
  v.pool_pages = d->page_tokens > 0 ? d->cap / d->page_tokens : 0;
  v.max_pos = max_positions(d);
  return v;
}
static hipError_t append_q4(const bkv_cache_desc *d, int layer, uint32_t pos0, int n_tok, const bkv_rope &rope, Rows q, Rows k,
                            Rows v, const float *qn_w, const float *kn_w, float eps, const int32_t *positions, float *q_out,
                            hipStream_t stream) {
  SeqsRowArgs a{};
  a.L = view(d, layer);
  a.v = one_sequence(d, a.L);
  a.one = true;
  a.pos0 = pos0;
  a.nkv = d->nkv; a.nh = d->nh; a.n_tok = n_tok;
  a.q = q; a.k = k; a.v_rows = v;
  a.qn_w = qn_w; a.kn_w = kn_w;
  a.eps = eps;
  a.positions = positions;
  a.n_axes = 1;
  a.q_out = q_out;
  a.rope = rope;
  return launch_seqs_rope_append(a, d->k_fmt, d->v_fmt, stream);
}

int bkv_kv_append(const bkv_cache_desc *d, int layer, uint32_t pos, int n_tok, const float *k,
                  const float *v, hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = any_q4(d) ? (d->hd == kHd ? BKV_OK : BKV_EUNSUPPORTED) : check_kernels(d))) return rc;
  if (layer < 0 || layer >= d->n_layers || n_tok < 0) return BKV_EINVAL;
  if (n_tok == 0) return BKV_OK;
  if ((int64_t)pos + n_tok > max_positions(d)) return BKV_ECAP;
  if (!k || !v) return BKV_EINVAL;
  if (!aligned16(k) || !aligned16(v)) return BKV_EALIGN;
  if (any_q4(d)) {
    const bkv_rope none{0, BKV_ROPE_HALF, 1.0f, 0, {}};
    const int64_t tok = (int64_t)d->nkv * kHd;
    return hip_fail(append_q4(d, layer, pos, n_tok, none, Rows{}, Rows{k, tok, kHd}, Rows{v, tok, kHd}, nullptr, nullptr, 0.0f,
                              nullptr, nullptr, stream));
  }
  AppendArgs a{};
  a.L = view(d, layer);
  a.nkv = d->nkv;
  a.pos = pos;
  a.k = k;
  a.v = v;
  return hip_fail(launch_append(a, d->k_fmt, d->v_fmt, n_tok, stream));
}

int bkv_qk_norm_rope_append(const bkv_cache_desc *d, int layer, uint32_t pos0, int n_tok,
                            const float *q_in, const float *k_in, const float *v_in,
                            const float *qn_w, const float *kn_w, int nrot, float eps,
                            float freq_base, float *q_out, hipStream_t stream) {
  int rc = check(d);
  if (rc) return rc;
  if ((rc = check_kernels(d))) return rc;
  if (layer < 0 || layer >= d->n_layers || n_tok < 0) return BKV_EINVAL;
  if (nrot < 0 || nrot > d->hd || (nrot & 1)) return BKV_EINVAL;
  if (!(eps >= 0.0f) || !std::isfinite(freq_base) || freq_base <= 0.0f) return BKV_EINVAL;
  if (n_tok == 0) return BKV_OK;
  if ((int64_t)pos0 + n_tok > max_positions(d)) return BKV_ECAP;
  const void *ptrs[6] = {q_in, k_in, v_in, qn_w, kn_w, q_out};
  for (const void *p : ptrs) {
    if (!p) return BKV_EINVAL;
    if (!aligned16(p)) return BKV_EALIGN;
  }
  NormRopeArgs a{};
  a.L = view(d, layer);
  a.nkv = d->nkv;
  a.nh = d->nh;
  a.nrot = nrot;
  a.pos0 = pos0;
  a.eps = eps;
  a.freq_base = freq_base;
  a.q_in = q_in; a.k_in = k_in; a.v_in = v_in;
  a.qn_w = qn_w; a.kn_w = kn_w;
  a.q_out = q_out;
  return hip_fail(launch_norm_rope_append(a, d->k_fmt, d->v_fmt, n_tok, stream));
}

int bkv_attn_decode(const bkv_cache_desc *d, int layer, uint32_t nfill, const float *q,
                    const float *gate, float *out, float *out_gated, void *workspace,
                    size_t ws_bytes, hipStream_t stream) {
  return decode_common(d, layer, nfill, q, gate, out, out_gated, workspace, ws_bytes, stream,
                       nullptr);
}

static int decode_step_common(const bkv_cache_desc *d, int layer, uint32_t pos, const float *k,
                              const float *v, const float *q, const float *gate, float *out,
                              float *out_gated, void *workspace, size_t ws_bytes, hipStream_t stream,
                              int qs, int gs) {
  int rc = check(d);
  if (rc) return rc;
  if (layer < 0 || layer >= d->n_layers) return BKV_EINVAL;
  if ((int64_t)pos + 1 > max_positions(d)) return BKV_ECAP;
  if (!k || !v) return BKV_EINVAL;
  if (!aligned16(k) || !aligned16(v)) return BKV_EALIGN;
  AppendArgs a{};
  a.L = view(d, layer);
  a.nkv = d->nkv;
  a.pos = pos;
  a.k = k;
  a.v = v;
  return decode_common(d, layer, pos + 1, q, gate, out, out_gated, workspace, ws_bytes, stream, &a,
                       qs, gs);
}

int bkv_decode_step(const bkv_cache_desc *d, int layer, uint32_t pos, const float *k,
                    const float *v, const float *q, const float *gate, float *out,
                    float *out_gated, void *workspace, size_t ws_bytes, hipStream_t stream) {
  return decode_step_common(d, layer, pos, k, v, q, gate, out, out_gated, workspace, ws_bytes,
                            stream, kHd, kHd);
}

// the _qg variants read Q and the gate from the engine's attn_q output: per head, hd values of q
// then hd values of the gate (the layout deint_qg splits, runtime_vk/shaders/deint_qg.comp)
int bkv_attn_decode_window(const bkv_cache_desc *d, int layer, uint32_t kstart, uint32_t nfill,
                           const float *q, const float *gate, float *out, float *out_gated,
                           void *workspace, size_t ws_bytes, hipStream_t stream) {
  return decode_common(d, layer, nfill, q, gate, out, out_gated, workspace, ws_bytes, stream,
                       nullptr, kHd, kHd, kstart);
}

int bkv_attn_decode_qg(const bkv_cache_desc *d, int layer, uint32_t nfill, const float *qg,
                       float *out, float *out_gated, void *workspace, size_t ws_bytes,
                       hipStream_t stream) {
  if (!qg) return BKV_EINVAL;
  return decode_common(d, layer, nfill, qg, out_gated ? qg + kHd : nullptr, out, out_gated,
                       workspace, ws_bytes, stream, nullptr, 2 * kHd, 2 * kHd);
}

int bkv_decode_step_qg(const bkv_cache_desc *d, int layer, uint32_t pos, const float *k,
                       const float *v, const float *qg, float *out, float *out_gated,
                       void *workspace, size_t ws_bytes, hipStream_t stream) {
  if (!qg) return BKV_EINVAL;
  return decode_step_common(d, layer, pos, k, v, qg, out_gated ? qg + kHd : nullptr, out, out_gated,
                            workspace, ws_bytes, stream, 2 * kHd, 2 * kHd);
}

// Whether a chunk of two or more queries runs as one chunk (true; always from kPxMinQ on) or as decode rows:
// the chunk takes about 24 us and 6.2 ns per key of its last row (its serial sums) whatever its length, a decode
// row 17 us and 0.4 ns per key. us for the attention, rows / chunk, q8_0: 3 queries at 3000 keys 55 / 42, 6 at 3000
// 110 / 44, 6 at 8000 119 / 74, 3 at 8000 61 / 73, 8 at 8000 160 / 73, 6 at 32000 168 / 228, 12 at 32000 335 / 212;
// fp16: 6 at 8000 167 / 75. Over every format pair, 64-token pages, 1 to 16 KV heads, 520 to 64000 keys and 2 to 15
// queries (1216 combinations) the choice is nowhere behind the rows.
static bool px_worthwhile(int n_q, int64_t keys) {
  return n_q >= kPxMinQ || n_q * (170000 + 4 * keys) > 260000 + 62 * keys;
}

// Whether a chunk of a short context runs in the short kernel, whose workgroups (4 queries of a KV group) fill
// the chip in rounds of 256, or in the chunk kernels, whose time is nearly flat: up to about 860,000
// workgroup * (first + last key + 320). us, short / chunk kernels, q8_0 and fp16 K + V: 200 queries onto 100 keys,
// 16 KV heads (576,000) 47.7 / 53.4, 68.4 / 68.8; 512 onto none, 8 heads (850,000) 62.3 / 70.0, 85.9 / 87.7; 330
// onto none, 16 heads (863,000) 73.0 / 62.2, 103.7 / 77.7; 200 onto 300, 16 heads (896,000) 76.8 / 71.6,
// 102.4 / 89.5; 512 onto none, 32 heads 232 / 174, 323 / 230.
static bool short_chunk(int nkv, int64_t pos0, int64_t n_q) {
  return n_q < kPxMinQ || nkv * cdiv(n_q, kPxQ) * (2 * pos0 + n_q + 320) <= 860000;
}

static int prefill_common(const bkv_cache_desc *d, int layer, uint32_t pos0, int n_q,
                          const float *q, const float *gate, float *out, float *out_gated,
                          void *workspace, size_t ws_bytes, hipStream_t stream, int qs, int gs) {
  int rc = check(d);
  if (rc) return rc;
  if ((rc = check_kernels(d))) return rc;
  if (layer < 0 || layer >= d->n_layers) return BKV_EINVAL;
  if (n_q < 0 || n_q > BKV_PREFILL_MAX_Q) return BKV_EINVAL;
  if (n_q == 0) return BKV_OK;
  if ((int64_t)pos0 + n_q > max_positions(d)) return BKV_ECAP;
  if (!aligned16(q) || !aligned16(out)) return q && out ? BKV_EALIGN : BKV_EINVAL;
  if ((gate == nullptr) != (out_gated == nullptr)) return BKV_EINVAL;
  if (gate && (!aligned16(gate) || !aligned16(out_gated))) return BKV_EALIGN;
  if (!workspace) return BKV_EWORKSPACE;
  if (((uintptr_t)workspace & 255u) != 0) return BKV_EALIGN;
  const size_t base = prefill_base(d);
  // (a forced decode path also decides how the rows of a chunk below kPxMinQ queries run)
  const bool rows = n_q == 1 || (n_q < kPxMinQ && forced_path() >= 0);
  if (!prefill_mfma_requested() && !rows && (int64_t)pos0 + n_q <= kShortKeys && short_chunk(d->nkv, pos0, n_q)) {
    // a short context: one launch, 4 queries per workgroup (the workspace is asked for all the same, so
    // that a caller meets its size at the first chunk and not at a later one)
    const size_t need = n_q >= kPxMinQ ? px_layout(d->nh, d->nkv, (int64_t)pos0 + n_q, kPxSlice, base).total
                                       : plan_decode(d->nh, d->nkv, d->k_fmt, d->v_fmt, (int64_t)pos0 + n_q, d->page_tokens).total;
    if (ws_bytes < need) return BKV_EWORKSPACE;
    ShortArgs a{};
    a.L = view(d, layer); a.nkv = d->nkv; a.nh = d->nh; a.pos0 = pos0; a.n_q = n_q; a.scale = d->scale;
    a.q = q; a.qs = qs; a.gate = gate; a.gs = gs; a.out = out; a.out_gated = out_gated;
    return hip_fail(launch_short(a, d->k_fmt, d->v_fmt, stream));
  }
  if (!prefill_mfma_requested() && !rows && px_worthwhile(n_q, (int64_t)pos0 + n_q) &&
      (n_q >= kPxMinQ || ws_bytes >= px_layout(d->nh, d->nkv, (int64_t)pos0 + n_q, kPxSlice, base).total)) {
    // the exact kernels, in equal slices (of kPxSlice queries in a workspace without room for more)
    const int64_t ctx = (int64_t)pos0 + n_q;
    if (ws_bytes < px_layout(d->nh, d->nkv, ctx, kPxSlice, base).total) return BKV_EWORKSPACE;
    int64_t slice = px_slice(d->nkv, ctx, n_q);
    if (ws_bytes < px_layout(d->nh, d->nkv, ctx, slice, base).total) slice = kPxSlice;
    slice = cdiv(cdiv(n_q, cdiv(n_q, slice)), kPxQ) * kPxQ;
    const PxLayout l = px_layout(d->nh, d->nkv, ctx, slice, base);
    char *w = (char *)workspace;
    PrefillXArgs a{};
    a.L = view(d, layer);
    a.nkv = d->nkv;
    a.nh = d->nh;
    a.pos0 = pos0;
    a.chunk_q = n_q;
    a.scale = d->scale;
    a.ld = l.ld;
    a.q = q;
    a.qs = qs;
    a.gs = gs;
    a.sc = (float *)(w + base);
    a.sums = (float *)(w + l.sums);
    a.part = a.mx = (float *)(w + l.part);
    a.gate = gate;
    a.out = out;
    a.out_gated = out_gated;
    for (int qb = 0; qb < n_q; qb += (int)slice) {
      a.q_base = qb;
      a.n_q = std::min((int)slice, n_q - qb);
      a.nqb = (int)cdiv(a.n_q, kPxQ);
      if ((rc = hip_fail(launch_prefill_exact(a, d->k_fmt, d->v_fmt, stream)))) return rc;
    }
    return BKV_OK;
  }
  if (!prefill_mfma_requested()) {
    // short chunks (also in a workspace for decodes only): every row is the decode row at nfill = pos0 + i + 1
    const size_t rs = (size_t)d->nh * d->hd;
    for (int i = 0; i < n_q; ++i) {
      rc = decode_common(d, layer, pos0 + (uint32_t)i + 1u, q + i * (size_t)d->nh * qs,
                         gate ? gate + i * (size_t)d->nh * gs : nullptr, out + i * rs,
                         out_gated ? out_gated + i * rs : nullptr, workspace, ws_bytes, stream,
                         nullptr, qs, gs);
      if (rc) return rc;
    }
    return BKV_OK;
  }
  const PrefillPlan p = plan_prefill(d->nh, d->nkv, pos0, n_q, base);
  if (ws_bytes < p.total) return BKV_EWORKSPACE;
  char *w = (char *)workspace;
  PrefillArgs a{};
  a.L = view(d, layer);
  a.nkv = d->nkv;
  a.nh = d->nh;
  a.pos0 = pos0;
  a.n_q = n_q;
  a.scale = d->scale;
  a.nqb = p.nqb;
  a.nsplit = p.nsplit;
  a.q = q;
  a.gate = gate;
  a.out = out;
  a.out_gated = out_gated;
  a.stats = (float2 *)(w + p.off_stats);
  a.part = p.nsplit > 1 ? (float *)(w + p.off_part) : nullptr;
  a.qs = qs;
  a.gs = gs;
  return hip_fail(launch_prefill(a, d->k_fmt, d->v_fmt, stream));
}

int bkv_attn_prefill_chunk(const bkv_cache_desc *d, int layer, uint32_t pos0, int n_q,
                           const float *q, const float *gate, float *out, float *out_gated,
                           void *workspace, size_t ws_bytes, hipStream_t stream) {
  return prefill_common(d, layer, pos0, n_q, q, gate, out, out_gated, workspace, ws_bytes, stream,
                        kHd, kHd);
}

int bkv_prefill_step(const bkv_cache_desc *d, int layer, uint32_t pos0, int n_q, const float *k,
                     const float *v, const float *q, const float *gate, float *out,
                     float *out_gated, void *workspace, size_t ws_bytes, hipStream_t stream) {
  int rc = check(d);
  if (rc) return rc;
  if (n_q < 0 || n_q > BKV_PREFILL_MAX_Q) return BKV_EINVAL;
  if (layer < 0 || layer >= d->n_layers) return BKV_EINVAL;
  if ((int64_t)pos0 + n_q > max_positions(d)) return BKV_ECAP;
  if (!workspace) return BKV_EWORKSPACE;
  if (((uintptr_t)workspace & 255u) != 0) return BKV_EALIGN;
  if (!q || !out) return BKV_EINVAL;
  if ((rc = bkv_kv_append(d, layer, pos0, n_q, k, v, stream))) return rc;
  return bkv_attn_prefill_chunk(d, layer, pos0, n_q, q, gate, out, out_gated, workspace, ws_bytes,
                                stream);
}

int bkv_attn_prefill_chunk_qg(const bkv_cache_desc *d, int layer, uint32_t pos0, int n_q,
                              const float *qg, float *out, float *out_gated, void *workspace,
                              size_t ws_bytes, hipStream_t stream) {
  if (!qg) return BKV_EINVAL;
  return prefill_common(d, layer, pos0, n_q, qg, out_gated ? qg + kHd : nullptr, out, out_gated,
                        workspace, ws_bytes, stream, 2 * kHd, 2 * kHd);
}

// ------------------------------------------------------------------ drafted tokens
// head_dim 256, any number of query heads per KV head
static int check_hd(const bkv_cache_desc *d) { return d->hd == kHd ? BKV_OK : BKV_EUNSUPPORTED; }
// whether positions pos0 .. pos0 + n - 1 leave the cache (or the 32 bits of a position: a block table may span more)
static bool outside(const bkv_cache_desc *d, uint32_t pos0, int n) {
  return (int64_t)pos0 + n > std::min<int64_t>(max_positions(d), (int64_t(1) << 32) - 64);
}
static int pool_pages(const bkv_cache_desc *d) { return d->page_tokens > 0 ? d->cap / d->page_tokens : 0; }

static int check_rows(const bkv_rows *r) {
  if (!r || !r->p || r->tok < 0 || r->head < 0) return BKV_EINVAL;
  return aligned16(r->p) && r->tok % 4 == 0 && r->head % 4 == 0 ? BKV_OK : BKV_EALIGN;
}
static Rows rows_of(const bkv_rows *r) { return r ? Rows{r->p, r->tok, r->head} : Rows{nullptr, 0, 0}; }

int bkv_tree_mask(const int32_t *parent, int n, uint64_t *mask, int32_t *depth) {
  if (n < 0 || n > BKV_TREE_MAX_Q || (n > 0 && !parent)) return BKV_EINVAL;
  for (int i = 0; i < n; ++i)
    if (parent[i] < -1 || parent[i] >= i) return BKV_EINVAL;
  const int words = (n + 63) / 64;
  for (int i = 0; i < n; ++i) {
    const int p = parent[i];
    if (mask) {
      uint64_t *row = mask + (size_t)i * words;
      for (int w = 0; w < words; ++w) row[w] = p < 0 ? 0 : row[w + (std::ptrdiff_t)(p - i) * words];
      row[i / 64] |= uint64_t(1) << (i % 64);
    }
  }
  if (depth)
    for (int i = 0; i < n; ++i) depth[i] = parent[i] < 0 ? 0 : depth[parent[i]] + 1;
  return BKV_OK;
}

int bkv_attn_tree(const bkv_cache_desc *d, int layer, uint32_t pos0, int n_q, const bkv_rows *q,
                  const uint64_t *mask, const bkv_rows *gate, float *out, float *out_gated,
                  void *workspace, size_t ws_bytes, hipStream_t stream) {
  int rc = check(d);
  if (rc) return rc;
  if ((rc = check_hd(d))) return rc;
  if (layer < 0 || layer >= d->n_layers || n_q < 0 || n_q > BKV_TREE_MAX_Q) return BKV_EINVAL;
  if (n_q == 0) return BKV_OK;
  if (outside(d, pos0, n_q)) return BKV_ECAP;
  if ((int64_t)n_q * d->nh > INT32_MAX / 2) return BKV_EUNSUPPORTED;   // (rows are counted in 32 bits)
  for (int i = 0; i < 4; i += 2) {                 // (and so are the bytes of a step: 31 slots and a row)
    const uint64_t sb = slot_bytes(d, i);
    if (31 * sb + sb / d->nkv > UINT32_MAX) return BKV_EUNSUPPORTED;
  }
  if ((rc = check_rows(q))) return rc;
  if (!out || (gate == nullptr) != (out_gated == nullptr)) return BKV_EINVAL;
  if (gate && (rc = check_rows(gate))) return rc;
  if (!aligned16(out) || (out_gated && !aligned16(out_gated)) || ((uintptr_t)mask & 7u) != 0) return BKV_EALIGN;
  if (!workspace) return BKV_EWORKSPACE;
  if (((uintptr_t)workspace & 255u) != 0) return BKV_EALIGN;
  const TreePlan p = plan_tree(d->nh, d->nkv, d->k_fmt, d->v_fmt, d->page_tokens > 0, pos0, n_q, prefill_base(d));
  if (ws_bytes < p.total) return BKV_EWORKSPACE;
  char *w = (char *)workspace;
  TreeArgs a{};
  a.L = view(d, layer);
  a.pool_pages = pool_pages(d);
  a.nkv = d->nkv; a.nh = d->nh; a.grp = d->nh / d->nkv;
  a.pos0 = pos0;
  a.n_q = n_q;
  a.scale2 = (float)((double)d->scale * 1.4426950408889634);
  a.q = rows_of(q);
  a.gate = rows_of(gate);
  a.mask = mask;
  a.words = (n_q + 63) / 64;
  a.out = out;
  a.out_gated = out_gated;
  a.nrb = p.nrb;
  a.splits = p.splits;
  a.whole = d->nkv * p.splits / 8 * p.nrb;
  a.left = d->nkv * p.splits % 8 * p.nrb;
  a.share_out = (a.left + 7) / 8;
  a.share = p.share;
  a.spare = p.spare;
  a.ml = (float2 *)(w + p.off_ml);
  a.part = (float *)(w + p.off_part);
  return hip_fail(launch_tree(a, p, d->k_fmt, d->v_fmt, stream));
}

static bool positive(double x) { return std::isfinite(x) && x > 0.0; }

int bkv_rope_init(bkv_rope *r, int nrot, int layout, double freq_base, int scaling, double factor,
                  double trained_ctx, double beta_fast, double beta_slow) {
  if (!r || nrot < 0 || nrot > kHd || (nrot & 1)) return BKV_EINVAL;
  if (layout != BKV_ROPE_HALF && layout != BKV_ROPE_INTERLEAVED) return BKV_EINVAL;
  if (scaling < BKV_ROPE_PLAIN || scaling > BKV_ROPE_YARN) return BKV_EINVAL;
  if (!std::isfinite(freq_base) || freq_base <= 1.0) return BKV_EINVAL;
  if (scaling != BKV_ROPE_PLAIN && !positive(factor)) return BKV_EINVAL;
  if (scaling == BKV_ROPE_YARN && !(positive(trained_ctx) && positive(beta_slow) && std::isfinite(beta_fast) && beta_fast > beta_slow))
    return BKV_EINVAL;
  const double two_pi = 6.283185307179586476925;
  double base = freq_base;
  if (scaling == BKV_ROPE_NTK) {
    if (nrot == 2) return BKV_EINVAL;              // (the exponent nrot / (nrot - 2))
    if (nrot) base *= std::pow(factor, nrot / (nrot - 2.0));
    if (!std::isfinite(base) || base <= 0.0) return BKV_EINVAL;
  }
  double lo = 0.0, hi = 0.0;
  if (scaling == BKV_ROPE_YARN && nrot) {
    // the pair, as a real number, that turns so often in trained_ctx positions
    const double per = nrot / (2.0 * std::log(freq_base));
    lo = std::max(0.0, std::floor(per * std::log(trained_ctx / (two_pi * beta_fast))));
    hi = std::min(nrot - 1.0, std::ceil(per * std::log(trained_ctx / (two_pi * beta_slow))));
  }
  std::memset(r, 0, sizeof *r);
  r->nrot = nrot;
  r->layout = layout;
  r->mscale = scaling == BKV_ROPE_YARN && factor > 1.0 ? (float)(1.0 + 0.1 * std::log(factor)) : 1.0f;
  for (int p = 0; p < nrot / 2; ++p) {
    double th = std::pow(base, -2.0 * p / nrot);
    if (scaling == BKV_ROPE_LINEAR) th /= factor;
    if (scaling == BKV_ROPE_YARN) {
      const double ramp = std::min(1.0, std::max(0.0, (p - lo) / std::max(hi - lo, 1e-3)));
      th = th * (1.0 - ramp) + th / factor * ramp;
    }
    r->turns[p] = th / two_pi;
  }
  return BKV_OK;
}

static bool rope_fine(const bkv_rope *rope) {
  if (rope->nrot < 0 || rope->nrot > kHd || (rope->nrot & 1) || !std::isfinite(rope->mscale)) return false;
  if (rope->layout != BKV_ROPE_HALF && rope->layout != BKV_ROPE_INTERLEAVED) return false;
  for (int p = 0; p < rope->nrot / 2; ++p)
    if (!std::isfinite(rope->turns[p])) return false;
  return true;
}

int bkv_rope_append(const bkv_cache_desc *d, int layer, uint32_t pos0, int n_tok, const bkv_rope *rope,
                    const bkv_rows *q, const bkv_rows *k, const bkv_rows *v, const float *qn_w,
                    const float *kn_w, float eps, const int32_t *positions, float *q_out,
                    hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = check_hd(d))) return rc;
  if (layer < 0 || layer >= d->n_layers || n_tok < 0 || !rope) return BKV_EINVAL;
  if (!rope_fine(rope)) return BKV_EINVAL;
  if ((qn_w == nullptr) != (kn_w == nullptr) || (qn_w && !(eps >= 0.0f))) return BKV_EINVAL;
  if ((q == nullptr) != (q_out == nullptr)) return BKV_EINVAL;
  if (n_tok == 0) return BKV_OK;
  if (outside(d, pos0, n_tok)) return BKV_ECAP;
  if (q && (rc = check_rows(q))) return rc;
  if ((rc = check_rows(k)) || (rc = check_rows(v))) return rc;
  if ((q_out && !aligned16(q_out)) || (qn_w && (!aligned16(qn_w) || !aligned16(kn_w))) || ((uintptr_t)positions & 3u) != 0)
    return BKV_EALIGN;
  if (any_q4(d))
    return hip_fail(append_q4(d, layer, pos0, n_tok, *rope, rows_of(q), rows_of(k), rows_of(v), qn_w, kn_w, eps, positions, q_out,
                              stream));
  RopeArgs a{};
  a.L = view(d, layer);
  a.pool_pages = pool_pages(d);
  a.nkv = d->nkv; a.nh = d->nh;
  a.pos0 = pos0;
  a.q = rows_of(q); a.k = rows_of(k); a.v = rows_of(v);
  a.qn_w = qn_w; a.kn_w = kn_w;
  a.eps = eps;
  a.positions = positions;
  a.q_out = q_out;
  a.rope = *rope;
  return hip_fail(launch_rope_append(a, d->k_fmt, d->v_fmt, n_tok, stream));
}

// where values are written: rows that lie apart, whole tokens after one another or whole heads
static int check_out_rows(const bkv_cache_desc *d, int n, int out_type, const void *k_out, const void *v_out, int64_t tok_stride,
                          int64_t head_stride) {
  const bool tokens = tok_stride >= (__int128)(d->nkv - 1) * head_stride + kHd && head_stride >= kHd;
  const bool heads = head_stride >= (__int128)(n - 1) * tok_stride + kHd && tok_stride >= kHd;
  if (n > 1 && d->nkv > 1 ? !(tokens || heads) : (n > 1 && tok_stride < kHd) || (d->nkv > 1 && head_stride < kHd)) return BKV_EINVAL;
  const int64_t unit = out_type == BKV_OUT_F32 ? 4 : 8;
  if ((k_out && !aligned16(k_out)) || (v_out && !aligned16(v_out)) || (n > 1 && tok_stride % unit) || (d->nkv > 1 && head_stride % unit))
    return BKV_EALIGN;
  return BKV_OK;
}

int bkv_kv_read(const bkv_cache_desc *d, int layer, uint32_t pos0, int n, int out_type, void *k_out,
                void *v_out, int64_t tok_stride, int64_t head_stride, hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = check_hd(d))) return rc;
  if (layer < 0 || layer >= d->n_layers || n < 0) return BKV_EINVAL;
  if (out_type < BKV_OUT_F32 || out_type > BKV_OUT_BF16) return BKV_EINVAL;
  if (n == 0) return BKV_OK;
  if (outside(d, pos0, n)) return BKV_ECAP;
  if (!k_out && !v_out) return BKV_EINVAL;
  if ((rc = check_out_rows(d, n, out_type, k_out, v_out, tok_stride, head_stride))) return rc;
  if (any_q4(d)) {
    SeqsReadArgs s{};
    s.L = view(d, layer);
    s.v = one_sequence(d, s.L);
    s.one = true;
    s.pos0 = pos0;
    s.nkv = d->nkv;
    s.n_tok = n;
    s.k_out = k_out; s.v_out = v_out;
    s.tok = tok_stride; s.head = head_stride;
    return hip_fail(launch_seqs_read(s, d->k_fmt, d->v_fmt, out_type, stream));
  }
  ReadArgs a{};
  a.L = view(d, layer);
  a.pool_pages = pool_pages(d);
  a.nkv = d->nkv;
  a.pos0 = pos0;
  a.n = n;
  a.k_out = k_out; a.v_out = v_out;
  a.tok = tok_stride; a.head = head_stride;
  return hip_fail(launch_kv_read(a, d->k_fmt, d->v_fmt, out_type, stream));
}

int bkv_kv_commit(const bkv_cache_desc *d, uint32_t pos0, int n_draft, int n_keep, const int32_t *idx,
                  hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = check_hd(d))) return rc;
  if (n_draft < 0 || n_draft > BKV_TREE_MAX_Q || n_keep < 0 || n_keep > n_draft) return BKV_EINVAL;
  if (n_keep == 0) return BKV_OK;
  if (outside(d, pos0, n_draft)) return BKV_ECAP;
  if (slot_bytes(d, 0) > INT32_MAX || slot_bytes(d, 2) > INT32_MAX) return BKV_EUNSUPPORTED;   // (columns in 31 bits)
  if (!idx) return BKV_EINVAL;
  if (((uintptr_t)idx & 3u) != 0) return BKV_EALIGN;
  CommitArgs a{};
  void *bases[4] = {d->k_data, d->k_scales, d->v_data, d->v_scales};
  for (int i = 0; i < 4; ++i) {
    const uint64_t sb = slot_bytes(d, i);
    a.base[i] = sb ? (uint8_t *)bases[i] : nullptr;
    a.stride[i] = d->layer_stride_bytes[i];
    a.row[i] = (int)sb;
    a.units[i] = (int)cdiv((int64_t)sb, 64);
  }
  a.bt = d->block_table;
  a.max_pages = d->max_pages;
  a.page = d->page_tokens;
  a.pool_pages = pool_pages(d);
  a.pos0 = pos0;
  a.n_draft = n_draft; a.n_keep = n_keep;
  a.idx = idx;
  return hip_fail(launch_kv_commit(a, d->n_layers, stream));
}

// ------------------------------------------------------------------ several sequences
static int check_seqs(const bkv_cache_desc *d, const bkv_seqs *s) {
  if (!s || s->n_seq < 0 || s->n_seq > BKV_SEQS_MAX || s->n_tok < 0 || s->max_q < 0 || s->reserved != 0) return BKV_EINVAL;
  if (s->n_seq == 0 || s->n_tok == 0) return BKV_OK;
  if (!s->len || (!s->q_start && s->n_tok < s->n_seq)) return BKV_EINVAL;
  if (d->page_tokens > 0 ? !s->tables : s->n_seq > 1) return BKV_EINVAL;
  if (((uintptr_t)s->q_start | (uintptr_t)s->len | (uintptr_t)s->tables) & 3u) return BKV_EALIGN;
  // (rows and grids are counted in 31 bits, a step's bytes in 32)
  if ((int64_t)s->n_tok * d->nh > INT32_MAX / 2 || d->nkv > 65536) return BKV_EUNSUPPORTED;
  return BKV_OK;
}
static SeqsView seqs_view(const bkv_cache_desc *d, int layer, const bkv_seqs *s) {
  SeqsView v{};
  v.n_seq = s->n_seq;
  v.n_tok = s->n_tok;
  v.q_start = s->q_start;
  v.len = s->len;
  v.page = d->page_tokens > 0 ? d->page_tokens : 0;
  v.pool_pages = pool_pages(d);
  v.tables = v.page ? s->tables + (int64_t)layer * d->max_pages : nullptr;
  v.table_stride = (int64_t)d->n_layers * d->max_pages;
  v.max_pos = std::min<int64_t>(max_positions(d), INT32_MAX - 64);
  return v;
}

int bkv_rope_axes_init(bkv_rope_axes *x, int n_axes, const int32_t *pairs, int order) {
  if (!x || !pairs || n_axes < 1 || n_axes > BKV_ROPE_MAX_AXES) return BKV_EINVAL;
  if (order != BKV_AXES_BLOCKS && order != BKV_AXES_DEALT) return BKV_EINVAL;
  int left[BKV_ROPE_MAX_AXES], total = 0;
  for (int i = 0; i < n_axes; ++i) {
    if (pairs[i] < 0 || pairs[i] > kHd / 2 - total) return BKV_EINVAL;
    total += left[i] = pairs[i];
  }
  std::memset(x, 0, sizeof *x);
  x->n_axes = n_axes;
  x->n_pairs = total;
  for (int p = 0, i = 0; p < total; ++p) {
    while (left[i] == 0) i = (i + 1) % n_axes;
    x->axis[p] = (uint8_t)i;
    --left[i];
    if (order == BKV_AXES_DEALT) i = (i + 1) % n_axes;
  }
  return BKV_OK;
}

int bkv_seqs_rope_append(const bkv_cache_desc *d, int layer, const bkv_seqs *seqs, const bkv_rope *rope, const bkv_rope_axes *axes,
                         const bkv_rows *q, const bkv_rows *k, const bkv_rows *v, const float *qn_w, const float *kn_w, float eps,
                         const int32_t *positions, float *q_out, hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = check_hd(d))) return rc;
  if (layer < 0 || layer >= d->n_layers || !rope || !rope_fine(rope)) return BKV_EINVAL;
  if (axes) {
    if (axes->n_axes < 1 || axes->n_axes > BKV_ROPE_MAX_AXES || axes->n_pairs != rope->nrot / 2 || (axes->n_axes > 1 && !positions))
      return BKV_EINVAL;
    for (int p = 0; p < axes->n_pairs; ++p)
      if (axes->axis[p] >= axes->n_axes) return BKV_EINVAL;
  }
  if ((qn_w == nullptr) != (kn_w == nullptr) || (qn_w && !(eps >= 0.0f))) return BKV_EINVAL;
  if ((q == nullptr) != (q_out == nullptr)) return BKV_EINVAL;
  if ((rc = check_seqs(d, seqs))) return rc;
  if (seqs->n_seq == 0 || seqs->n_tok == 0) return BKV_OK;
  if (q && (rc = check_rows(q))) return rc;
  if ((rc = check_rows(k)) || (rc = check_rows(v))) return rc;
  if ((q_out && !aligned16(q_out)) || (qn_w && (!aligned16(qn_w) || !aligned16(kn_w))) || ((uintptr_t)positions & 3u) != 0)
    return BKV_EALIGN;
  SeqsRowArgs a{};
  a.L = view(d, layer);
  a.v = seqs_view(d, layer, seqs);
  a.nkv = d->nkv; a.nh = d->nh; a.n_tok = seqs->n_tok;
  a.q = rows_of(q); a.k = rows_of(k); a.v_rows = rows_of(v);
  a.qn_w = qn_w; a.kn_w = kn_w;
  a.eps = eps;
  a.positions = positions;
  a.n_axes = axes ? axes->n_axes : 1;
  a.q_out = q_out;
  a.rope = *rope;
  if (axes) std::memcpy(a.axis, axes->axis, sizeof a.axis);
  return hip_fail(launch_seqs_rope_append(a, d->k_fmt, d->v_fmt, stream));
}

int bkv_seqs_read(const bkv_cache_desc *d, int layer, const bkv_seqs *seqs, int out_type, void *k_out, void *v_out,
                  int64_t tok_stride, int64_t head_stride, hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = check_hd(d))) return rc;
  if (layer < 0 || layer >= d->n_layers || out_type < BKV_OUT_F32 || out_type > BKV_OUT_BF16) return BKV_EINVAL;
  if ((rc = check_seqs(d, seqs))) return rc;
  if (seqs->n_seq == 0 || seqs->n_tok == 0) return BKV_OK;
  if (!k_out && !v_out) return BKV_EINVAL;
  if ((rc = check_out_rows(d, seqs->n_tok, out_type, k_out, v_out, tok_stride, head_stride))) return rc;
  SeqsReadArgs a{};
  a.L = view(d, layer);
  a.v = seqs_view(d, layer, seqs);
  a.nkv = d->nkv;
  a.n_tok = seqs->n_tok;
  a.k_out = k_out; a.v_out = v_out;
  a.tok = tok_stride; a.head = head_stride;
  return hip_fail(launch_seqs_read(a, d->k_fmt, d->v_fmt, out_type, stream));
}

size_t bkv_seqs_workspace_bytes(const bkv_cache_desc *d, int n_seq, int n_tok) {
  if (check_geom(d) || n_seq < 1 || n_seq > BKV_SEQS_MAX || n_tok < 1 || (int64_t)n_tok * d->nh > INT32_MAX / 2 || d->nkv > 65536) return 0;
  return plan_seqs_attn(d->nh, d->nkv, n_seq, n_tok, 0).total;
}

int bkv_seqs_attn(const bkv_cache_desc *d, int layer, const bkv_seqs *seqs, const bkv_rows *q, const bkv_rows *gate, float *out,
                  float *out_gated, void *workspace, size_t ws_bytes, hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = check_hd(d))) return rc;
  if (d->k_fmt != BKV_Q4_0 || d->v_fmt != BKV_Q4_0) return BKV_EUNSUPPORTED;
  if (layer < 0 || layer >= d->n_layers) return BKV_EINVAL;
  if ((rc = check_seqs(d, seqs))) return rc;
  if (seqs->n_seq == 0 || seqs->n_tok == 0) return BKV_OK;
  // (row blocks of 16 times steps of 32 positions, and what a block's way in counts as, are counted in 31 bits)
  const int64_t blocks = (int64_t)seqs->n_tok * (d->nh / d->nkv) / 16 + seqs->n_seq;
  if ((int64_t)seqs->n_tok * d->nh > INT32_MAX / 2 || d->nkv > 65536) return BKV_EUNSUPPORTED;
  if (blocks > INT32_MAX / (std::min<int64_t>(max_positions(d), INT32_MAX) / 32 + 1 + kSeqWayIn)) return BKV_EUNSUPPORTED;
  if ((rc = check_rows(q))) return rc;
  if (!out || (gate == nullptr) != (out_gated == nullptr)) return BKV_EINVAL;
  if (gate && (rc = check_rows(gate))) return rc;
  if (!aligned16(out) || (out_gated && !aligned16(out_gated))) return BKV_EALIGN;
  if (!workspace) return BKV_EWORKSPACE;
  if (((uintptr_t)workspace & 255u) != 0) return BKV_EALIGN;
  const SeqsAttnPlan p = plan_seqs_attn(d->nh, d->nkv, seqs->n_seq, seqs->n_tok, seqs->max_q);
  if (ws_bytes < p.total) return BKV_EWORKSPACE;
  char *w = (char *)workspace;
  SeqsAttnArgs a{};
  a.L = view(d, layer);
  a.v = seqs_view(d, layer, seqs);
  a.nkv = d->nkv; a.nh = d->nh; a.grp = d->nh / d->nkv;
  a.scale2 = (float)((double)d->scale * 1.4426950408889634);
  a.q = rows_of(q);
  a.gate = rows_of(gate);
  a.out = out;
  a.out_gated = out_gated;
  a.lanes = p.lanes;
  a.by_nh = ByConst(d->nh);
  a.by_nkv = ByConst(d->nkv);
  a.by_grp = ByConst(a.grp);
  a.by_lanes = ByConst(p.lanes);
  a.by_page = ByConst(std::max(1, d->page_tokens));
  a.count = (unsigned *)w;
  a.few = p.few;
  a.way_in = p.way_in;
  a.tile_lanes = p.tile_lanes;
  a.by_tile_lanes = ByConst(p.tile_lanes);
  a.tile_part_rows = p.tile_part_rows;
  a.info = (uint4 *)(w + p.off_info);
  a.tile_ml = (float2 *)(w + p.off_tile_ml);
  a.tile_part = (float *)(w + p.off_tile_part);
  a.ml = (float2 *)(w + p.off_ml);
  a.part = (float *)(w + p.off_part);
  return hip_fail(launch_seqs_attn(a, p, stream));
}

// ------------------------------------------------------------------ pages
static int check_pages(const bkv_cache_desc *d, int n_seq, const void *tables, const void *refs) {
  if (n_seq < 0 || n_seq > BKV_SEQS_MAX || d->page_tokens <= 0 || !tables || !refs) return BKV_EINVAL;
  if (((uintptr_t)tables | (uintptr_t)refs) & 3u) return BKV_EALIGN;
  // (counts in 31 bits, pages by thousands at a time; a grid's rows)
  if ((int64_t)n_seq * d->max_pages > (1 << 30) || pool_pages(d) > (1 << 30) || d->n_layers > 65535) return BKV_EUNSUPPORTED;
  return BKV_OK;
}
static PagesArgs pages_args(const bkv_cache_desc *d, int n_seq) {
  PagesArgs a{};
  void *bases[4] = {d->k_data, d->k_scales, d->v_data, d->v_scales};
  for (int i = 0; i < 4; ++i) {
    a.slot[i] = slot_bytes(d, i);
    a.base[i] = a.slot[i] ? (uint8_t *)bases[i] : nullptr;
    a.stride[i] = d->layer_stride_bytes[i];
  }
  a.n_layers = d->n_layers;
  a.n_seq = n_seq;
  a.page = d->page_tokens;
  a.pool_pages = pool_pages(d);
  a.max_pages = d->max_pages;
  return a;
}
// The chunks of a page, all its arrays' one after another, are counted in 32 bits, and a workgroup's next piece is up to
// kPagePieces of kPagePiece of them further on: up to 2^31 chunks (32 GiB where positions go by 16 bytes, else 8).
static_assert((uint64_t)kPagePieces * kPagePiece + kPagePiece <= uint64_t(1) << 31, "a page's chunks and the step behind them in 32 bits");
static bool page_too_large(const bkv_cache_desc *d) {
  __int128 bytes = 0;
  for (int i = 0; i < 4; ++i) bytes += (__int128)slot_bytes(d, i) * d->page_tokens;
  return bytes / pages_chunk(pages_args(d, 0)) > (__int128(1) << 31);
}

size_t bkv_pages_workspace_bytes(const bkv_cache_desc *d) {
  if (check_geom(d) || d->page_tokens <= 0 || pool_pages(d) > (1 << 30)) return 0;
  return pages_workspace(d->n_layers, pool_pages(d));
}

int bkv_pages_fork(const bkv_cache_desc *d, int n_seq, int32_t *tables, int32_t *refs, int32_t *len, const int32_t *parent,
                   hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = check_pages(d, n_seq, tables, refs))) return rc;
  if (n_seq == 0) return BKV_OK;
  if (!parent) return BKV_EINVAL;
  if (((uintptr_t)parent | (uintptr_t)len) & 3u) return BKV_EALIGN;
  PagesArgs a = pages_args(d, n_seq);
  a.tables = a.tables_out = tables;
  a.refs = a.refs_out = refs;
  a.len = len;
  a.parent = parent;
  return hip_fail(launch_pages_fork(a, stream));
}

int bkv_pages_extend(const bkv_cache_desc *d, int n_seq, int32_t *tables, int32_t *refs, const int32_t *len, const int32_t *n_new,
                     int32_t *lack, void *workspace, size_t ws_bytes, hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = check_pages(d, n_seq, tables, refs))) return rc;
  if (!len || !n_new || !lack) return BKV_EINVAL;
  if (((uintptr_t)len | (uintptr_t)n_new | (uintptr_t)lack) & 3u) return BKV_EALIGN;
  if (page_too_large(d)) return BKV_EUNSUPPORTED;
  if (!workspace || ws_bytes < pages_workspace(d->n_layers, pool_pages(d))) return BKV_EWORKSPACE;
  if (((uintptr_t)workspace & 255u) != 0) return BKV_EALIGN;
  PagesArgs a = pages_args(d, n_seq);
  a.tables = a.tables_out = tables;
  a.refs = a.refs_out = refs;
  a.len = const_cast<int32_t *>(len);
  a.n_new = n_new;
  a.lack = lack;
  a.ws = (int32_t *)workspace;
  return hip_fail(launch_pages_extend(a, stream));
}

int bkv_pages_compact(const bkv_cache_desc *d, int n_seq, const int32_t *tables, const int32_t *refs, int32_t *tables_out,
                      int32_t *refs_out, void *workspace, size_t ws_bytes, hipStream_t stream) {
  int rc = check_geom(d);
  if (rc) return rc;
  if ((rc = check_pages(d, n_seq, tables, refs)) || (rc = check_pages(d, n_seq, tables_out, refs_out))) return rc;
  if (page_too_large(d)) return BKV_EUNSUPPORTED;
  if (!workspace || ws_bytes < pages_workspace(d->n_layers, pool_pages(d))) return BKV_EWORKSPACE;
  if (((uintptr_t)workspace & 255u) != 0) return BKV_EALIGN;
  PagesArgs a = pages_args(d, n_seq);
  a.tables = tables;
  a.refs = refs;
  a.tables_out = tables_out;
  a.refs_out = refs_out;
  a.ws = (int32_t *)workspace;
  return hip_fail(launch_pages_compact(a, stream));
}

size_t bkv_workspace_bytes(const bkv_cache_desc *d, int op, uint32_t max_ctx) {
  if (check(d) || max_ctx == 0) return 0;
  if (op == BKV_OP_TREE) return tree_workspace_bound(d->nh, prefill_base(d));
  if (op == BKV_OP_PREFILL)
    return std::max(prefill_workspace_bound(d->nh, d->nkv, prefill_base(d)),
                    prefill_exact_workspace(d->nh, d->nkv, max_ctx, prefill_base(d)));
  if (op != BKV_OP_DECODE) return 0;
  return plan_decode(d->nh, d->nkv, d->k_fmt, d->v_fmt, max_ctx, d->page_tokens).total;
}

const char *bkv_strerror(int err) {
  switch (err) {
    case BKV_OK: return "ok";
    case BKV_EINVAL: return "invalid argument";
    case BKV_ESHAPE: return "cache geometry rule broken (hd%4, hd%32, hd/32 even, nh%nkv)";
    case BKV_ECAP: return "position outside the cache (pos >= cap) or empty context";
    case BKV_EALIGN: return "pointer or stride not aligned (16 B; workspace 256 B)";
    case BKV_EWORKSPACE: return "workspace missing or smaller than bkv_workspace_bytes()";
    case BKV_ESCRATCH: return "decode plan larger than the static scratch (bkv_static_scratch_bytes())";
    case BKV_EHIP: return "HIP runtime error (see bkv_last_hip_error)";
    case BKV_EUNSUPPORTED: return "shape or format not supported by this call (hd 256, nh = 4*nkv, the cache's formats)";
    case BKV_ETIMEOUT: return "a decode kernel's workgroup wait timed out (its output is not valid)";
    default: return "unknown error";
  }
}

// byte offset of the single-launch kernels' error word (past their sync lines)
static uint64_t error_word_offset(int nkv) {
  return kResSyncOffset + (uint64_t)nkv * kResGroupLines * kCounterStride * sizeof(unsigned);
}

int bkv_error_words(const bkv_cache_desc *d, uint64_t out[1]) {
  const int rc = check(d);
  if (rc) return rc;
  if (!out) return BKV_EINVAL;
  out[0] = error_word_offset(d->nkv);
  return BKV_OK;
}

int bkv_workspace_error(const bkv_cache_desc *d, void *workspace, size_t ws_bytes, hipStream_t stream) {
  const int rc = check(d);
  if (rc) return rc;
  if (!workspace || ws_bytes < kSyncBytes) return BKV_EWORKSPACE;
  const uint64_t off[1] = {error_word_offset(d->nkv)};
  hipError_t e = hipStreamSynchronize(stream);
  if (e != hipSuccess) return hip_fail(e);
  int result = BKV_OK;
  for (uint64_t o : off) {
    unsigned v = 0;
    char *p = static_cast<char *>(workspace) + o;
    if ((e = hipMemcpy(&v, p, sizeof v, hipMemcpyDeviceToHost)) != hipSuccess) return hip_fail(e);
    if (v) result = BKV_ETIMEOUT;
  }
  if (result == BKV_ETIMEOUT) {
    // a call that gave up left its counters and tags mid-protocol: start the workspace afresh (this
    // also clears the error word), as bkv_workspace_init does
    if ((e = launch_workspace_init((unsigned *)workspace, ws_bytes / sizeof(unsigned), stream)) != hipSuccess ||
        (e = hipStreamSynchronize(stream)) != hipSuccess)
      return hip_fail(e);
  }
  return result;
}

int bkv_debug_layout(const bkv_cache_desc *d, uint32_t nfill, uint64_t out[6]) {
  const int rc = check(d);
  if (rc) return rc;
  if (!out || nfill == 0) return BKV_EINVAL;
  const DecodePlan p = plan_decode(d->nh, d->nkv, d->k_fmt, d->v_fmt, nfill, d->page_tokens);
  const int path = choose_path(p);
  out[0] = (uint64_t)p.ld;
  out[1] = path == kPathSplit ? p.off_score : 0;
  const bool res = path == kPathResident || path == kPathStream;
  out[2] = res ? p.r_e : p.off_e;
  out[3] = res ? p.r_sum : p.off_sum;
  out[4] = res ? p.r_status : p.off_status;
  out[5] = p.total;
  return BKV_OK;
}

int bkv_workspace_init(const bkv_cache_desc *d, void *workspace, size_t ws_bytes, hipStream_t stream) {
  const int rc = check_geom(d);
  if (rc) return rc;
  if (!workspace) return BKV_EWORKSPACE;
  if (((uintptr_t)workspace & 255u) != 0) return BKV_EALIGN;
  if (!any_q4(d) && ws_bytes < kSyncBytes) return BKV_EWORKSPACE;
  // the whole workspace: the sync words, and the tagged partials of the resident path (a tag is
  // the call generation, which starts at 1)
  return hip_fail(launch_workspace_init((unsigned *)workspace, ws_bytes / sizeof(unsigned), stream));
}

int bkv_kv_fill_synthetic(const bkv_cache_desc *d, hipStream_t stream) {
  const int rc = check_geom(d);
  if (rc) return rc;
  void *bases[4] = {d->k_data, d->k_scales, d->v_data, d->v_scales};
  for (int i = 0; i < 4; ++i) {
    const size_t bytes = (size_t)d->cap * slot_bytes(d, i);   // (0: the format has no such array)
    if (!bytes) continue;
    for (int l = 0; l < d->n_layers; ++l) {
      unsigned *p = (unsigned *)((char *)bases[i] + (uint64_t)l * d->layer_stride_bytes[i]);
      const hipError_t e = launch_fill_words(p, bytes / 4, 0x3C003C00u, stream);
      if (e != hipSuccess) return hip_fail(e);
    }
  }
  return BKV_OK;
}

int bkv_decode_path(const bkv_cache_desc *d, uint32_t nfill) {
  if (check(d) || nfill == 0) return -1;
  return choose_path(plan_decode(d->nh, d->nkv, d->k_fmt, d->v_fmt, nfill, d->page_tokens));
}

const char *bkv_last_hip_error(void) { return g_hip_err; }

const char *bkv_version(void) { return "bkv 0.1 gfx950"; }

}  // extern "C"
