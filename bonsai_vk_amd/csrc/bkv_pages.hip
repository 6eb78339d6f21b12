// bkv_pages.hip - the pages of a cache that several sequences share: fork, extend (copy on write) and compact.
//
// A sequence's table row names its pages, refs counts how many table entries name a page; a page that none names is free.
// Everything is decided on the device, in an order that the call's documentation fixes (the lowest free page first), so that
// the host neither waits nor reads anything back, and a captured graph allocates anew at every replay.

#include <algorithm>

#include "bkv_device.h"
#include "bkv_internal.h"

namespace bkv {

constexpr int kForkCols = 16;          // table columns of a fork workgroup
constexpr int kPlanThreads = 1024;
constexpr uint32_t kPiece = 16384;     // bytes that a workgroup copies at a time

__device__ __forceinline__ int64_t table_at(const PagesArgs &a, int s, int layer, int p) {
  return ((int64_t)s * a.n_layers + layer) * a.max_pages + p;
}

// ------------------------------------------------------------------ fork
// A workgroup has 16 columns of one layer's table in LDS, every sequence's: all are read before any is written. The counts
// are added to by atomics, whole numbers, whose order does not show.
__global__ __launch_bounds__(256) void pages_fork_kernel(PagesArgs a) {
  extern __shared__ int32_t s_tab[];               // [n_seq][kForkCols]
  const int layer = blockIdx.y, p0 = blockIdx.x * kForkCols, tid = threadIdx.x;
  const int col = tid % kForkCols, p = p0 + col, s0 = tid / kForkCols;
  constexpr int kStep = 256 / kForkCols;
  const bool mine = p < a.max_pages;
  for (int s = s0; s < a.n_seq; s += kStep) s_tab[s * kForkCols + col] = mine ? a.tables[table_at(a, s, layer, p)] : -1;
  const bool lens = a.len && blockIdx.x == 0 && layer == 0;
  int32_t len[BKV_SEQS_MAX / 256];
#pragma unroll
  for (int i = 0; i < BKV_SEQS_MAX / 256; ++i) {
    const int s = tid + 256 * i;
    len[i] = 0;
    if (lens && s < a.n_seq) {
      const uint32_t from = (uint32_t)a.parent[s];
      if (from < (uint32_t)a.n_seq) len[i] = a.len[from];
    }
  }
  __syncthreads();
  if (mine)
    for (int s = s0; s < a.n_seq; s += kStep) {
      const uint32_t from = (uint32_t)a.parent[s];
      const int32_t was = s_tab[s * kForkCols + col], now = from < (uint32_t)a.n_seq ? s_tab[from * kForkCols + col] : -1;
      if (was == now) continue;
      int32_t *refs = a.refs_out + (int64_t)layer * a.pool_pages;
      if ((uint32_t)was < (uint32_t)a.pool_pages) atomicAdd(refs + was, -1);
      if ((uint32_t)now < (uint32_t)a.pool_pages) atomicAdd(refs + now, 1);
      a.tables_out[table_at(a, s, layer, p)] = now;
    }
#pragma unroll
  for (int i = 0; i < BKV_SEQS_MAX / 256; ++i)
    if (lens && tid + 256 * i < a.n_seq) a.len[tid + 256 * i] = len[i];
}

hipError_t launch_pages_fork(const PagesArgs &a, hipStream_t st) {
  hipLaunchKernelGGL(pages_fork_kernel, dim3((a.max_pages + kForkCols - 1) / kForkCols, a.n_layers), dim3(256),
                     (size_t)a.n_seq * kForkCols * sizeof(int32_t), st, a);
  return hipGetLastError();
}

// ------------------------------------------------------------------ the workspace of extend and compact
// Per layer: a count (its own 64 bytes), then four lists of pool_pages numbers and one of pairs
//   extend   fresh pages, the lowest first | wanted[page] | last[page] | the pages before them, -1: none | (sequence, page of it)
//   compact  from | to | map[page]
struct PagesWs {
  int32_t *count, *list[4];
  int2 *pair;
  __host__ __device__ static size_t words(int pool_pages) { return 16 + (size_t)((pool_pages + 15) / 16 * 16) * 6; }
  __device__ __forceinline__ PagesWs(const PagesArgs &a, int layer) {
    const size_t n = (size_t)((a.pool_pages + 15) / 16 * 16);
    int32_t *p = a.ws + (size_t)layer * words(a.pool_pages);
    count = p;
    for (int i = 0; i < 4; ++i) list[i] = p + 16 + n * i;
    pair = reinterpret_cast<int2 *>(p + 16 + 4 * n);
  }
};
size_t pages_workspace(int n_layers, int pool_pages) { return (size_t)n_layers * PagesWs::words(pool_pages) * sizeof(int32_t); }

// `bytes` of each array's pages from -> to, or of the piece-th 16 KB of them: piece counts through the arrays' pieces
// of whole pages
struct CopyShape {
  int pieces[4], total;
  __host__ __device__ CopyShape(const PagesArgs &a) {
    total = 0;
    for (int i = 0; i < 4; ++i) total += pieces[i] = a.base[i] ? (int)((a.slot[i] * a.page + kPiece - 1) / kPiece) : 0;
  }
};
__device__ __forceinline__ void copy_piece(const PagesArgs &a, const CopyShape &c, int layer, int from, int to, int held, int piece) {
  int i = 0;
  while (i < 3 && piece >= c.pieces[i]) piece -= c.pieces[i++];
  const uint64_t page_bytes = a.slot[i] * a.page, bytes = a.slot[i] * held, off = (uint64_t)piece * kPiece;
  uint8_t *base = a.base[i] + (uint64_t)layer * a.stride[i];
  const uint4 *src = reinterpret_cast<const uint4 *>(base + (uint64_t)from * page_bytes + off);
  uint4 *dst = reinterpret_cast<uint4 *>(base + (uint64_t)to * page_bytes + off);
  const int n = off >= bytes ? 0 : (int)(min(bytes - off, (uint64_t)kPiece) / 16);
  if (n == 0) return;
  uint4 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = src[min((int)threadIdx.x + 256 * j, n - 1)];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if ((int)threadIdx.x + 256 * j < n) dst[threadIdx.x + 256 * j] = v[j];
}

// ------------------------------------------------------------------ extend
__device__ __forceinline__ int load_now(const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The pages that sequence s's next tokens lie in, p0 .. p1 (none: p1 < p0), and how many of them its row has no room for
struct Span {
  int len, p0, p1, over;
  __device__ __forceinline__ Span(const PagesArgs &a, int s) {
    len = max(a.len[s], 0);
    const int n = max(a.n_new[s], 0);
    p0 = len / a.page;
    const int64_t last = n == 0 ? (int64_t)p0 - 1 : ((int64_t)len + n - 1) / a.page;
    p1 = (int)min(last, (int64_t)a.max_pages - 1);
    over = (int)min(last - max(p1, p0 - 1), (int64_t)1 << 20);
  }
};

// One workgroup a layer decides; a wave takes a sequence at a time, a lane a page of it.
__global__ __launch_bounds__(kPlanThreads) void pages_extend_plan_kernel(PagesArgs a) {
  __shared__ int s_cnt[BKV_SEQS_MAX], s_scan[kPlanThreads / 64], s_over;
  const int layer = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  constexpr int NW = kPlanThreads / 64;
  const int32_t *refs = a.refs + (int64_t)layer * a.pool_pages;
  const PagesWs ws(a, layer);
  int32_t *const free_list = ws.list[0], *const wanted = ws.list[1], *const last = ws.list[2];
  if (tid == 0) s_over = 0;
  // each page that is wanted and shared: by how many of this call's sequences, and the last of them
  auto each = [&](auto &&f) {
    for (int s = w; s < a.n_seq; s += NW) {
      const Span at(a, s);
      f(s, at);
    }
  };
  auto entry_of = [&](int s, int p) { return (uint32_t)a.tables[table_at(a, s, layer, p)]; };
  auto shared = [&](uint32_t e) { return e < (uint32_t)a.pool_pages && refs[e] > 1; };
  __syncthreads();
  each([&](int s, const Span &at) {
    if (lane == 0 && at.over) atomicAdd(&s_over, at.over);
    for (int p = at.p0 + lane; p <= at.p1; p += 64) {
      const uint32_t e = entry_of(s, p);
      if (shared(e)) { wanted[e] = 0; last[e] = -1; }
    }
  });
  __threadfence();
  __syncthreads();
  each([&](int s, const Span &at) {
    for (int p = at.p0 + lane; p <= at.p1; p += 64) {
      const uint32_t e = entry_of(s, p);
      if (shared(e)) { atomicAdd(wanted + e, 1); atomicMax(last + e, s); }
    }
  });
  __threadfence();
  __syncthreads();
  // Whether page p of sequence s is a fresh one: there is none, or others have it too and will go on having it, or a later
  // one of those that want it keeps it.
  auto fresh = [&](int s, int p) {
    const uint32_t e = entry_of(s, p);
    if (e >= (uint32_t)a.pool_pages) return true;
    return refs[e] > 1 && !(load_now(wanted + e) == refs[e] && load_now(last + e) == s);
  };
  each([&](int s, const Span &at) {
    int n = 0;
    for (int p = at.p0; p <= at.p1; p += 64) n += __popcll(__ballot(p + lane <= at.p1 && fresh(s, p + lane)));
    if (lane == 0) s_cnt[s] = n;
  });
  __syncthreads();
  int total;
  const int before = block_excl_scan<kPlanThreads, int>(tid < a.n_seq ? s_cnt[tid] : 0, s_scan, &total);
  if (tid < a.n_seq) s_cnt[tid] = before;
  // the lowest `total` free pages
  int found = 0;
  for (int b = 0; b < a.pool_pages && found < total; b += 4 * kPlanThreads) {
    bool is[4];
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = b + 4 * tid + j;
      is[j] = p < a.pool_pages && refs[p] == 0;
      n += is[j];
    }
    int here, at = block_excl_scan<kPlanThreads, int>(n, s_scan, &here);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (is[j]) {
        if (found + at < total) free_list[found + at] = b + 4 * tid + j;
        ++at;
      }
    found += here;
  }
  const int lack = max(0, total - found) + s_over;
  if (tid == 0) {
    a.lack[layer] = lack;
    ws.count[0] = total;
  }
  if (lack) return;
  __syncthreads();
  each([&](int s, const Span &at) {
    int k = s_cnt[s];
    for (int p = at.p0; p <= at.p1; p += 64) {
      const bool is = p + lane <= at.p1 && fresh(s, p + lane);
      const uint64_t b = __ballot(is);
      if (is) {
        const int i = k + __popcll(b & ((1ull << lane) - 1));
        const uint32_t e = entry_of(s, p + lane);
        ws.pair[i] = make_int2(s, p + lane);
        ws.list[3][i] = e < (uint32_t)a.pool_pages ? (int)e : -1;
      }
      k += __popcll(b);
    }
  });
}

// Item (k, piece): the k-th fresh page takes its table entry and the bytes of the one before it.
__global__ __launch_bounds__(256) void pages_extend_apply_kernel(PagesArgs a, CopyShape c) {
  const int layer = blockIdx.y;
  for (int l = 0; l < a.n_layers; ++l)
    if (a.lack[l]) return;                         // (nothing at all where a layer lacks pages)
  const PagesWs ws(a, layer);
  const int count = ws.count[0];
  int32_t *refs = a.refs_out + (int64_t)layer * a.pool_pages;
  for (int64_t i = blockIdx.x; i < (int64_t)count * c.total; i += gridDim.x) {
    const int k = (int)(i / c.total), piece = (int)(i - (int64_t)k * c.total);
    const int2 sp = ws.pair[k];
    const int to = ws.list[0][k], len = max(a.len[sp.x], 0);
    // (the page before from the list: another piece's workgroup may have written the table)
    const int from = ws.list[3][k];
    if (from >= 0) copy_piece(a, c, layer, from, to, sp.y == len / a.page ? len % a.page : 0, piece);
    if (piece == 0 && threadIdx.x == 0) {
      a.tables_out[table_at(a, sp.x, layer, sp.y)] = to;
      refs[to] = 1;
      if (from >= 0) atomicAdd(refs + from, -1);
    }
  }
}

// workgroups of a layer that copy: 8 for each CU in all
static unsigned copy_grid(int64_t items, int n_layers) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(items, std::max(16, 2048 / n_layers))); }

hipError_t launch_pages_extend(const PagesArgs &a, hipStream_t st) {
  const CopyShape c(a);
  hipLaunchKernelGGL(pages_extend_plan_kernel, dim3(a.n_layers), dim3(kPlanThreads), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(pages_extend_apply_kernel, dim3(copy_grid((int64_t)a.pool_pages * c.total, a.n_layers), a.n_layers), dim3(256), 0, st, a, c);
  return hipGetLastError();
}

// ------------------------------------------------------------------ compact
// U pages are used: the i-th used one from U on moves to the i-th free one below U. One workgroup a layer lists them.
__global__ __launch_bounds__(kPlanThreads) void pages_compact_plan_kernel(PagesArgs a) {
  __shared__ long long s_scan[kPlanThreads / 64];
  const int layer = blockIdx.x, tid = threadIdx.x;
  const int32_t *refs = a.refs + (int64_t)layer * a.pool_pages;
  int32_t *out = a.refs_out + (int64_t)layer * a.pool_pages;
  const PagesWs ws(a, layer);
  int32_t *const from = ws.list[0], *const to = ws.list[1], *const map = ws.list[2];
  long long used = 0, all;
  for (int p = tid; p < a.pool_pages; p += kPlanThreads) used += refs[p] > 0;
  block_excl_scan<kPlanThreads, long long>(used, s_scan, &all);
  const int U = (int)all;
  long long base = 0;                              // pages listed: to move in the low half, free ones in the high half
  for (int b = 0; b < a.pool_pages; b += 4 * kPlanThreads) {
    long long n = 0;
    int kind[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = b + 4 * tid + j;
      const bool u = p < a.pool_pages && refs[p] > 0;
      kind[j] = p >= a.pool_pages ? 0 : u && p >= U ? 1 : !u && p < U ? 2 : 0;
      n += kind[j] == 1 ? 1ll : kind[j] == 2 ? 1ll << 32 : 0ll;
      if (p < a.pool_pages) map[p] = p;
    }
    long long here, at = block_excl_scan<kPlanThreads, long long>(n, s_scan, &here) + base;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (kind[j] == 1) { from[(int)at] = b + 4 * tid + j; at += 1; }
      if (kind[j] == 2) { to[(int)(at >> 32)] = b + 4 * tid + j; at += 1ll << 32; }
    }
    base += here;
  }
  const int moves = (int)base;
  if (tid == 0) ws.count[0] = moves;
  __syncthreads();
  // (refs_out may be refs: what is read of pages from U on is read before it is cleared)
  for (int i = tid; i < moves; i += kPlanThreads) {
    const int f = from[i], t = to[i];
    map[f] = t;
    out[t] = refs[f];
  }
  for (int p = tid; p < U; p += kPlanThreads) {
    const int32_t r = refs[p];
    if (r > 0) out[p] = r;
  }
  __syncthreads();
  for (int p = U + tid; p < a.pool_pages; p += kPlanThreads) out[p] = 0;
}

__global__ __launch_bounds__(256) void pages_compact_apply_kernel(PagesArgs a, CopyShape c) {
  const int layer = blockIdx.y;
  const PagesWs ws(a, layer);
  const int64_t items = (int64_t)ws.count[0] * c.total;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int k = (int)(i / c.total);
    copy_piece(a, c, layer, ws.list[0][k], ws.list[1][k], a.page, (int)(i - (int64_t)k * c.total));
  }
  const int64_t entries = (int64_t)a.n_seq * a.max_pages;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
    const int s = (int)(i / a.max_pages);
    const int64_t at = table_at(a, s, layer, (int)(i - (int64_t)s * a.max_pages));
    const int32_t e = a.tables[at];
    a.tables_out[at] = (uint32_t)e < (uint32_t)a.pool_pages ? ws.list[2][e] : e;
  }
}

hipError_t launch_pages_compact(const PagesArgs &a, hipStream_t st) {
  const CopyShape c(a);
  hipLaunchKernelGGL(pages_compact_plan_kernel, dim3(a.n_layers), dim3(kPlanThreads), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(pages_compact_apply_kernel, dim3(copy_grid((int64_t)(a.pool_pages + 1) / 2 * c.total, a.n_layers), a.n_layers), dim3(256), 0, st, a, c);
  return hipGetLastError();
}

}  // namespace bkv
