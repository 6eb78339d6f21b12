// bkv_pages.hip - the pages of a cache that several sequences share: fork, extend (copy on write) and compact.
//
// A sequence's table row names its pages, refs counts how many table entries name a page; a page that none names is free.
// Everything is decided on the device, in an order that the call's documentation fixes (the lowest free page first), so that
// the host neither waits nor reads anything back, and a captured graph allocates anew at every replay.

#include <algorithm>

#include "bkv_device.h"
#include "bkv_internal.h"

namespace bkv {

constexpr int kForkCols = 8;           // table columns of a fork workgroup
constexpr int kPlanThreads = 1024;
typedef uint32_t Four __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int64_t table_at(const PagesArgs &a, int s, int layer, int p) {
  return ((int64_t)s * a.n_layers + layer) * a.max_pages + p;
}

// ------------------------------------------------------------------ fork
// A workgroup has 8 columns of one layer's table in LDS, every sequence's: all are read before any is written. How many rows
// come to name a sequence's page is counted in LDS and added to the page's count at once (200 samples of one prompt: an addition
// a page, not 200), whole numbers by atomics, whose order does not show. Three trips to memory one after another: 3.5 us for 8
// sequences of 33 pages in 8 layers, 5.6 for 200 (14 where each row adds its own change).
__global__ __launch_bounds__(256) void pages_fork_kernel(PagesArgs a) {
  // [n_seq][kForkCols] entries; rows that come to name each, two columns' in 16 bits each (1024 at most); the parents
  extern __shared__ int32_t s_tab[];
  uint32_t *const s_gain = reinterpret_cast<uint32_t *>(s_tab) + a.n_seq * kForkCols;
  int32_t *const s_from = s_tab + a.n_seq * (kForkCols + kForkCols / 2);
  const int layer = blockIdx.y, p0 = blockIdx.x * kForkCols, tid = threadIdx.x;
  const int col = tid % kForkCols, p = p0 + col, s0 = tid / kForkCols;
  constexpr int kStep = 256 / kForkCols, kOwn = BKV_SEQS_MAX / 256;
  const bool mine = p < a.max_pages;
  int32_t from[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) from[i] = a.parent[min(tid + 256 * i, a.n_seq - 1)];
  for (int s = s0; s < a.n_seq; s += 8 * kStep) {
    int32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = a.tables[table_at(a, min(s + i * kStep, a.n_seq - 1), layer, min(p, a.max_pages - 1))];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (s + i * kStep < a.n_seq) s_tab[(s + i * kStep) * kForkCols + col] = e[i];
  }
  for (int i = tid; i < a.n_seq * (kForkCols / 2); i += 256) s_gain[i] = 0;
  const bool lens = a.len && blockIdx.x == 0 && layer == 0;
  int32_t len[kOwn] = {};
  if (lens) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      if (tid + 256 * i < a.n_seq && (uint32_t)from[i] < (uint32_t)a.n_seq) len[i] = a.len[from[i]];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOwn; ++i)
    if (tid + 256 * i < a.n_seq) {
      s_from[tid + 256 * i] = (uint32_t)from[i] < (uint32_t)a.n_seq ? from[i] : -1;
      if (lens) a.len[tid + 256 * i] = len[i];
    }
  __syncthreads();
  int32_t *const refs = a.refs_out + (int64_t)layer * a.pool_pages;
  if (mine)
    for (int s = s0; s < a.n_seq; s += kStep) {
      const int32_t f = s_from[s], was = s_tab[s * kForkCols + col], now = f >= 0 ? s_tab[f * kForkCols + col] : -1;
      if (was == now) continue;
      if (f >= 0) atomicAdd(s_gain + f * (kForkCols / 2) + col / 2, 1u << (16 * (col & 1)));
      if ((uint32_t)was < (uint32_t)a.pool_pages) atomicAdd(refs + was, -1);
      a.tables_out[table_at(a, s, layer, p)] = now;
    }
  __syncthreads();
  if (mine)
    for (int s = s0; s < a.n_seq; s += kStep) {
      const uint32_t gain = s_gain[s * (kForkCols / 2) + col / 2] >> (16 * (col & 1)) & 0xFFFFu, page = (uint32_t)s_tab[s * kForkCols + col];
      if (gain && page < (uint32_t)a.pool_pages) atomicAdd(refs + page, (int)gain);
    }
}

hipError_t launch_pages_fork(const PagesArgs &a, hipStream_t st) {
  hipLaunchKernelGGL(pages_fork_kernel, dim3((a.max_pages + kForkCols - 1) / kForkCols, a.n_layers), dim3(256),
                     (size_t)a.n_seq * (kForkCols + kForkCols / 2 + 1) * sizeof(int32_t), st, a);
  return hipGetLastError();
}

// ------------------------------------------------------------------ the workspace of extend and compact
// Per layer: a count (its own 64 bytes), then three lists of pool_pages numbers and one of fours
//   extend   fresh pages, the lowest first | wanted[page] | last[page] | sequence, page of it, the page before it (-1: none),
//            positions of that to be copied
//   compact  from | to | map[page]
struct PagesWs {
  int32_t *count, *list[3];
  int4 *item;
  __host__ __device__ static size_t words(int pool_pages) { return 16 + (size_t)((pool_pages + 15) / 16 * 16) * 7; }
  __device__ __forceinline__ PagesWs(const PagesArgs &a, int layer) {
    const size_t n = (size_t)((a.pool_pages + 15) / 16 * 16);
    int32_t *p = a.ws + (size_t)layer * words(a.pool_pages);
    count = p;
    for (int i = 0; i < 3; ++i) list[i] = p + 16 + n * i;
    item = reinterpret_cast<int4 *>(p + 16 + 3 * n);
  }
};
size_t pages_workspace(int n_layers, int pool_pages) { return (size_t)n_layers * PagesWs::words(pool_pages) * sizeof(int32_t); }

// The first `held` positions of a page's arrays from -> to, those of the four arrays one after another, in chunks T: of the pieces
// first, first + step, .. of kPagePiece chunks. (All arrays' chunks are counted in 32 bits, 2^31 at most: the calls refuse larger pages.)
template <class T>
__device__ __forceinline__ void copy_page(const PagesArgs &a, int layer, int from, int to, int held, int first, int step) {
  struct Array { uint64_t src, dst; uint32_t end; };   // (less the chunks of the arrays before)
  auto after = [&](uint32_t before, uint8_t *base, uint64_t stride, uint64_t slot) {
    const uint64_t at = (uint64_t)(uintptr_t)base + (uint64_t)layer * stride - sizeof(T) * (uint64_t)before, page = slot * a.page;
    return Array{at + from * page, at + to * page, before + (uint32_t)(slot * held / sizeof(T))};   // (slot: 0 where there is no such array)
  };
  const Array x0 = after(0, a.base[0], a.stride[0], a.slot[0]), x1 = after(x0.end, a.base[1], a.stride[1], a.slot[1]);
  const Array x2 = after(x1.end, a.base[2], a.stride[2], a.slot[2]), x3 = after(x2.end, a.base[3], a.stride[3], a.slot[3]);
  for (uint32_t c0 = (uint32_t)first * kPagePiece; c0 < x3.end; c0 += (uint32_t)step * kPagePiece) {
    T v[4];
    uint64_t to_at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = c0 + 256 * j + threadIdx.x, c = min(x, x3.end - 1);
      uint64_t s = x3.src, d = x3.dst;
      if (c < x2.end) { s = x2.src; d = x2.dst; }
      if (c < x1.end) { s = x1.src; d = x1.dst; }
      if (c < x0.end) { s = x0.src; d = x0.dst; }
      v[j] = *reinterpret_cast<const T *>(s + sizeof(T) * (uint64_t)c);
      to_at[j] = x < x3.end ? d + sizeof(T) * (uint64_t)c : 0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (to_at[j]) *reinterpret_cast<T *>(to_at[j]) = v[j];
  }
}
static uint32_t pieces_of(const PagesArgs &a) {
  uint64_t bytes = 0;
  for (int i = 0; i < 4; ++i) bytes += a.slot[i] * a.page;
  return (uint32_t)std::min<uint64_t>((bytes / pages_chunk(a) + kPagePiece - 1) / kPagePiece, kPagePieces);
}
// `count` pages shared out to the workgroups of a layer: `step` of them to a page, the workgroup's first of which is `k`
struct Shares {
  int step, every, k, first;
  __device__ __forceinline__ Shares(int count, int most) {
    step = min(max((int)(gridDim.x / (uint32_t)max(count, 1)), 1), most);
    every = (int)(gridDim.x / (uint32_t)step);
    k = (int)(blockIdx.x / (uint32_t)step);
    first = (int)blockIdx.x - k * step;
    if (k >= every) k = count;
  }
};

// ------------------------------------------------------------------ extend
__device__ __forceinline__ int load_now(const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void store_now(int32_t *p, int x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// the workgroup's atomics before it are seen by those behind it
__device__ __forceinline__ void atomics_barrier() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// One workgroup a layer decides. L lanes take a sequence, as many as the most pages that one of them needs (64 at most): all
// sequences of a step of single tokens at once. What the time goes to is trips to memory one after another; what a lane has read
// of its first page (most often its only one) it keeps. 7.5 us for 8 sequences in 8 layers, 10.2 for 200 (a wave a sequence,
// nothing kept: 14.8 and 58.7).
__global__ __launch_bounds__(kPlanThreads) void pages_extend_plan_kernel(PagesArgs a) {
  __shared__ int s_p0[BKV_SEQS_MAX], s_n[BKV_SEQS_MAX], s_len[BKV_SEQS_MAX], s_cnt[BKV_SEQS_MAX], s_scan[kPlanThreads / 64], s_over, s_most, s_any;
  const int layer = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int32_t *refs = a.refs + (int64_t)layer * a.pool_pages;
  const PagesWs ws(a, layer);
  int32_t *const free_list = ws.list[0], *const wanted = ws.list[1], *const last = ws.list[2];
  int32_t r4[4];                                   // the first counts that are looked through for free pages
#pragma unroll
  for (int j = 0; j < 4; ++j) r4[j] = refs[min(4 * tid + j, a.pool_pages - 1)];
  if (tid == 0) s_over = s_most = s_any = 0;
  __syncthreads();
  static_assert(kPlanThreads >= BKV_SEQS_MAX, "a thread a sequence");
  if (tid < a.n_seq) {                             // the pages p0 .. that its next tokens lie in, as far as its row has room
    const int len = max(a.len[tid], 0), n = max(a.n_new[tid], 0), p0 = len / a.page;
    const int64_t end = n == 0 ? p0 : ((int64_t)len + n - 1) / a.page + 1;
    const int here = max((int)min(end, (int64_t)a.max_pages) - p0, 0);
    s_p0[tid] = p0;
    s_len[tid] = len;
    s_n[tid] = here;
    s_cnt[tid] = 0;
    const int over = (int)min(end - p0 - here, (int64_t)1 << 20);
    if (over) atomicAdd(&s_over, over);
    if (here) atomicMax(&s_most, here);
  }
  __syncthreads();
  const int most = s_most;
  int L = 1;
  while (L < most && L < 64) L *= 2;
  const int group = tid / L, groups = kPlanThreads / L, li = tid & (L - 1);
  const uint64_t in_group = (L == 64 ? ~0ull : (1ull << L) - 1) << (lane & ~(L - 1));
  auto entry_of = [&](int s, int p) { return (uint32_t)a.tables[table_at(a, s, layer, p)]; };
  auto count_of = [&](uint32_t e) { return e < (uint32_t)a.pool_pages ? refs[e] : 0; };   // (0: there is no page)
  uint32_t e1 = ~0u;
  int r1 = 0;
  if (group < a.n_seq && li < s_n[group]) {
    e1 = entry_of(group, s_p0[group] + li);
    r1 = count_of(e1);
  }
  // f(sequence, page, entry, its count, whether it is the lane's first), a sequence's pages in order
  auto each = [&](auto &&f) {
    for (int s = group; s < a.n_seq; s += groups)
      for (int i = li; i < s_n[s]; i += L) {
        const bool kept = s == group && i == li;
        uint32_t e = e1;
        int r = r1;
        if (!kept) { e = entry_of(s, s_p0[s] + i); r = count_of(e); }
        f(s, s_p0[s] + i, e, r, kept);
      }
  };
  // each page that is wanted and shared: by how many of this call's sequences, and the last of them
  each([&](int, int, uint32_t e, int r, bool) {
    if (r > 1) { store_now(wanted + e, 0); store_now(last + e, -1); s_any = 1; }
  });
  atomics_barrier();
  if (s_any) {
    each([&](int s, int, uint32_t e, int r, bool) {
      if (r > 1) { atomicAdd(wanted + e, 1); atomicMax(last + e, s); }
    });
    atomics_barrier();
  }
  // Whether a page of sequence s is to be a fresh one: there is none, or others have it too and will go on having it, or a later
  // one of those that want it keeps it.
  auto fresh = [&](int s, uint32_t e, int r) {
    if (e >= (uint32_t)a.pool_pages) return true;
    return r > 1 && !(load_now(wanted + e) == r && load_now(last + e) == s);
  };
  bool fresh1 = false;
  each([&](int s, int, uint32_t e, int r, bool kept) {
    const bool is = fresh(s, e, r);
    if (kept) fresh1 = is;
    if (is) atomicAdd(&s_cnt[s], 1);
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
      is[j] = p < a.pool_pages && (b ? refs[p] : r4[j]) == 0;
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
  int k = 0, of = -1;                              // the fresh ones of sequence `of` so far
  each([&](int s, int p, uint32_t e, int r, bool kept) {
    if (of != s) { of = s; k = s_cnt[s]; }
    const bool is = kept ? fresh1 : fresh(s, e, r);
    const uint64_t b = __ballot(is) & in_group;
    if (is) {
      const int len = s_len[s], old = e < (uint32_t)a.pool_pages ? (int)e : -1;
      ws.item[k + __popcll(b & ((1ull << lane) - 1))] = make_int4(s, p, old, old >= 0 && p == s_p0[s] ? len - p * a.page : 0);
    }
    k += __popcll(b);
  });
}

// The k-th fresh page takes its table entry and what is held of the one before it. 5.0 us for 56 pages, 7.6 for 1592 of 9 KB each
// (24.5 where a workgroup goes through the arrays' pieces one by one, the empty ones too).
template <class T>
__global__ __launch_bounds__(256) void pages_extend_apply_kernel(PagesArgs a, int pieces) {
  const int layer = blockIdx.y;
  const PagesWs ws(a, layer);
  const int count = ws.count[0];
  int lack = 0;
  for (int l = threadIdx.x & 63; l < a.n_layers; l += 64) lack |= a.lack[l];
  if (__any(lack)) return;                         // (nothing at all where a layer lacks pages)
  int32_t *refs = a.refs_out + (int64_t)layer * a.pool_pages;
  const Shares mine(count, pieces);
  for (int k = mine.k; k < count; k += mine.every) {
    // (the page before from the list: another workgroup of this page may have written the table)
    const int4 x = ws.item[k];
    const int to = ws.list[0][k], from = x.z;
    if (from >= 0) copy_page<T>(a, layer, from, to, x.w, mine.first, mine.step);
    if (mine.first == 0 && threadIdx.x == 0) {
      a.tables_out[table_at(a, x.x, layer, x.y)] = to;
      refs[to] = 1;
      if (from >= 0) atomicAdd(refs + from, -1);
    }
  }
}

// workgroups of a layer that copy: 8 for each CU in all
static unsigned copy_grid(int64_t items, int n_layers) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(items, std::max(16, 2048 / n_layers))); }

hipError_t launch_pages_extend(const PagesArgs &a, hipStream_t st) {
  const uint32_t pieces = pieces_of(a);
  hipLaunchKernelGGL(pages_extend_plan_kernel, dim3(a.n_layers), dim3(kPlanThreads), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid(copy_grid((int64_t)a.pool_pages * pieces, a.n_layers), a.n_layers);
  if (pages_chunk(a) == 16) hipLaunchKernelGGL(pages_extend_apply_kernel<Four>, grid, dim3(256), 0, st, a, (int)pieces);
  else hipLaunchKernelGGL(pages_extend_apply_kernel<uint32_t>, grid, dim3(256), 0, st, a, (int)pieces);
  return hipGetLastError();
}

// ------------------------------------------------------------------ compact
// U pages are used: the i-th used one from U on moves to the i-th free one below U. One workgroup a layer lists them: 5.1 us for
// 77 pages, 6.7 for 2000.
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

// Bound by memory: 449 pages of 74 KB in each of 8 layers, 539 MB, in 117 us (4.6 TB/s; a large copy has 4.9).
template <class T>
__global__ __launch_bounds__(256) void pages_compact_apply_kernel(PagesArgs a, int pieces) {
  const int layer = blockIdx.y;
  const PagesWs ws(a, layer);
  const int count = ws.count[0];
  // table entries, the first of which is on its way while pages are copied
  const uint32_t entries = (uint32_t)a.n_seq * a.max_pages, i0 = blockIdx.x * 256 + threadIdx.x;   // (2^30 at most)
  auto at_of = [&](uint32_t i) {
    const uint32_t s = i / (uint32_t)a.max_pages;
    return table_at(a, (int)s, layer, (int)(i - s * a.max_pages));
  };
  const int32_t e0 = i0 < entries ? a.tables[at_of(i0)] : -1;
  const Shares mine(count, pieces);
  for (int k = mine.k; k < count; k += mine.every) copy_page<T>(a, layer, ws.list[0][k], ws.list[1][k], a.page, mine.first, mine.step);
  for (uint32_t i = i0; i < entries; i += gridDim.x * 256) {
    const int64_t at = at_of(i);
    const int32_t e = i == i0 ? e0 : a.tables[at];
    a.tables_out[at] = (uint32_t)e < (uint32_t)a.pool_pages ? ws.list[2][e] : e;
  }
}

hipError_t launch_pages_compact(const PagesArgs &a, hipStream_t st) {
  const uint32_t pieces = pieces_of(a);
  hipLaunchKernelGGL(pages_compact_plan_kernel, dim3(a.n_layers), dim3(kPlanThreads), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid(copy_grid((int64_t)(a.pool_pages + 1) / 2 * pieces, a.n_layers), a.n_layers);
  if (pages_chunk(a) == 16) hipLaunchKernelGGL(pages_compact_apply_kernel<Four>, grid, dim3(256), 0, st, a, (int)pieces);
  else hipLaunchKernelGGL(pages_compact_apply_kernel<uint32_t>, grid, dim3(256), 0, st, a, (int)pieces);
  return hipGetLastError();
}

}  // namespace bkv
