// bkv_read.hip - the cache read back as values (bkv_kv_read), and the accepted tokens of a draft moved
// together (bkv_kv_commit).

#include "bkv_device.h"
#include "bkv_internal.h"

namespace bkv {

// ------------------------------------------------------------------ read
// A head row is 256 values; 32 lanes take one, 8 values each, so that loads are 8 bytes (q8_0) or 16 (fp16) per
// lane and stores 16 or 32, all whole lines per row. Rows of one tensor run head first, then position. Bound by
// the memory; each thread asks for kReadRows rows before it stores the first. 32768 positions of q8_0 as bf16: 31.9 us,
// 206 MB at 6.4 TB/s; 777 of fp16 as fp32 5.4 us, 9.5 MB; a few positions 2.2 us, a launch.
constexpr int kReadRows = 4;

template <int OT>
__device__ __forceinline__ void store8(void *base, int64_t at, const float (&v)[8]) {
  if constexpr (OT == BKV_OUT_F32) {
    float4 *p = reinterpret_cast<float4 *>((float *)base + at);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (OT == BKV_OUT_F16) {
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16);
      } else {
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[2 * i]) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[2 * i + 1]) << 16);
      }
    }
    *reinterpret_cast<uint4 *>((uint16_t *)base + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int FMT, int OT>
__device__ __forceinline__ void read_rows(const ReadArgs &a, const uint8_t *data, const uint8_t *scales, void *out, int64_t first) {
  const int sub = threadIdx.x & 31;
  const int64_t rows = (int64_t)a.n * a.nkv;
  uint4 d[kReadRows];
  uint32_t s[kReadRows];
  int ok[kReadRows];
#pragma unroll
  for (int j = 0; j < kReadRows; ++j) {
    const int64_t r = min(first + 8 * j + (threadIdx.x >> 5), rows - 1);
    const uint32_t t = (uint32_t)(r / a.nkv), h = (uint32_t)(r - (int64_t)t * a.nkv);
    const int slot = slot_checked(a.L, a.pool_pages, a.pos0 + t);
    ok[j] = slot >= 0;
    const int64_t at = (int64_t)max(slot, 0) * a.nkv + h;
    if constexpr (FMT == BKV_Q8_0) {
      const uint2 w = reinterpret_cast<const uint2 *>(data + at * kHd)[sub];
      d[j] = make_uint4(w.x, w.y, 0, 0);
      s[j] = reinterpret_cast<const uint16_t *>(scales + at * kScaleRowBytes)[sub >> 2];
    } else {
      d[j] = reinterpret_cast<const uint4 *>(data + at * 2 * kHd)[sub];
      s[j] = 0;
    }
  }
#pragma unroll
  for (int j = 0; j < kReadRows; ++j) {
    const int64_t r = first + 8 * j + (threadIdx.x >> 5);
    if (r >= rows) continue;
    const int64_t t = r / a.nkv, h = r - t * a.nkv;
    float v[8];
    const uint32_t w[4] = {d[j].x, d[j].y, d[j].z, d[j].w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = FMT == BKV_Q8_0 ? sbyte(w[e >> 2], e & 3) * f16_to_f32(s[j]) : f16_to_f32((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
      if (!ok[j]) v[e] = 0.0f;
    }
    store8<OT>(out, t * a.tok + h * a.head + 8 * sub, v);
  }
}

template <int KF, int VF, int OT>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
  const int64_t first = (int64_t)blockIdx.x * (8 * kReadRows);
  if (blockIdx.y == 0 && a.k_out) read_rows<KF, OT>(a, a.L.kd, a.L.ks, a.k_out, first);
  else read_rows<VF, OT>(a, a.L.vd, a.L.vs, a.v_out, first);
}

hipError_t launch_kv_read(const ReadArgs &a, int kf, int vf, int out_type, hipStream_t st) {
  const int64_t rows = (int64_t)a.n * a.nkv;
  const dim3 grid((unsigned)((rows + 8 * kReadRows - 1) / (8 * kReadRows)), a.k_out && a.v_out ? 2 : 1);
  BKV_FMT_SWITCH(kf, vf, {
    if (out_type == BKV_OUT_F32) hipLaunchKernelGGL((kv_read_kernel<KF_, VF_, BKV_OUT_F32>), grid, dim3(256), 0, st, a);
    else if (out_type == BKV_OUT_F16) hipLaunchKernelGGL((kv_read_kernel<KF_, VF_, BKV_OUT_F16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv_read_kernel<KF_, VF_, BKV_OUT_BF16>), grid, dim3(256), 0, st, a);
  });
  return hipGetLastError();
}

// ------------------------------------------------------------------ commit
// A workgroup owns one 64-byte column of one array of one layer and all of the kept tokens: it reads every source
// into registers, and writes after a barrier, so that a source which another token's write covers has been read
// (positions of different columns, arrays and layers never meet). 4 lanes take the column's 16-byte pieces of a
// token, 64 tokens at a time, PT times. 5 tokens of 8 layers 2.9 us, 300 tokens of 8 fp16 layers 4.0 us: a launch and
// three latencies (the index, the page, the bytes); the 20 MB of the latter stay in the caches.
template <int PT>
__global__ __launch_bounds__(256) void kv_commit_kernel(CommitArgs a) {
  int u = blockIdx.x, arr = 0;
  while (arr < 3 && u >= a.units[arr]) u -= a.units[arr++];
  const int layer = blockIdx.y, col = 64 * u + 16 * (threadIdx.x & 3);
  uint8_t *base = a.base[arr] + (uint64_t)layer * a.stride[arr] + col;
  const bool mine = col < a.row[arr];
  LayerView L{};
  L.page = a.page;
  L.bt = a.page ? a.bt + (int64_t)layer * a.max_pages : nullptr;
  uint4 v[PT];
  int to[PT];
#pragma unroll
  for (int j = 0; j < PT; ++j) {
    const int i = 64 * j + (threadIdx.x >> 2);
    to[j] = -1;
    v[j] = make_uint4(0, 0, 0, 0);
    if (i < a.n_keep && mine) {
      const uint32_t k = (uint32_t)a.idx[i];
      if (k < (uint32_t)a.n_draft && k != (uint32_t)i) {
        const int from = slot_checked(L, a.pool_pages, a.pos0 + k);
        if (from >= 0) {
          to[j] = slot_checked(L, a.pool_pages, a.pos0 + (uint32_t)i);
          v[j] = *reinterpret_cast<const uint4 *>(base + (int64_t)from * a.row[arr]);
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PT; ++j)
    if (to[j] >= 0) *reinterpret_cast<uint4 *>(base + (int64_t)to[j] * a.row[arr]) = v[j];
}

hipError_t launch_kv_commit(const CommitArgs &a, int n_layers, hipStream_t st) {
  const dim3 grid(a.units[0] + a.units[1] + a.units[2] + a.units[3], n_layers);
  if (a.n_keep <= 64) hipLaunchKernelGGL((kv_commit_kernel<1>), grid, dim3(256), 0, st, a);
  else if (a.n_keep <= 256) hipLaunchKernelGGL((kv_commit_kernel<4>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((kv_commit_kernel<16>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace bkv
