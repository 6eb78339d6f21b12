// bkv_rope.hip - rotary positions with the quantising append (bkv_rope_append): strided projection rows,
// an optional per-head RMS norm, pairs in either layout at any position per token, K and V into the cache.
//
// Per row x of 256: n = x * (1 / sqrt(mean(x^2) + eps)) * w (or x), then for pair p of the first nrot dims
// with a = 2 pi * pos * turns[p]: y1 = (n1 cos a - n2 sin a) * mscale, y2 = (n2 cos a + n1 sin a) * mscale.
// The angle is reduced in fp64 in units of a turn, pos * turns[p] minus the nearest whole number, where an
// fp32 angle of a position past 2^17 would be off by 1e-2 radians; cosine and sine are rounded once to fp32.

#include "bkv_device.h"
#include "bkv_internal.h"

namespace bkv {

// One wave per row, 4 dims per lane; a workgroup takes 8 rows of one token (Q heads, then K, then V), so that a
// single token's 24 rows run on 3 workgroups and the token's sines are formed once for 8 rows. 1 token 4.4 us (a
// launch, the rows' latency and the fp64 sines), 501 tokens 6.1 us (22 MB read and written, 3.6 TB/s: the same chain,
// with the memory at two thirds of a copy's rate).
constexpr int kRopeRows = 8;

// the maximum over the 8 lanes that hold a q8_0 block
__device__ __forceinline__ float max8(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  return fmaxf(v, dpp<0x141>(v));
}

// a row of 4 values per lane into the cache, as append_row writes it
template <int FMT>
__device__ __forceinline__ void store_values(const float4 x, uint8_t *data, uint8_t *scales, int64_t row, int lane) {
  if constexpr (FMT == BKV_Q8_0) {
    const float amax = max8(fmaxf(fmaxf(fmaxf(fmaxf(0.0f, fabsf(x.x)), fabsf(x.y)), fabsf(x.z)), fabsf(x.w)));
    const float id = q8_iscale(amax);
    reinterpret_cast<uint32_t *>(data + row * kHd)[lane] =
        q8_byte<false>(x.x, id) | (q8_byte<false>(x.y, id) << 8) | (q8_byte<false>(x.z, id) << 16) | (q8_byte<false>(x.w, id) << 24);
    if ((lane & 7) == 0) reinterpret_cast<uint16_t *>(scales + row * kScaleRowBytes)[lane >> 3] = (uint16_t)f32_to_f16_rne(q8_scale(amax));
  } else {
    reinterpret_cast<uint2 *>(data + row * 2 * kHd)[lane] =
        make_uint2(f32_to_f16_rne(x.x) | (f32_to_f16_rne(x.y) << 16), f32_to_f16_rne(x.z) | (f32_to_f16_rne(x.w) << 16));
  }
}

template <int KF, int VF>
__global__ __launch_bounds__(256) void rope_append_kernel(RopeArgs a) {
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int nq = a.q.p ? a.nh : 0, nr = nq + 2 * a.nkv;
  __shared__ float s_cs[kHd / 2], s_sn[kHd / 2];
  __shared__ __attribute__((aligned(16))) float s_x[4][kHd];
  constexpr int RPW = kRopeRows / 4;
  float4 x[RPW];
  int row[RPW];
#pragma unroll
  for (int j = 0; j < RPW; ++j) {
    row[j] = blockIdx.y * kRopeRows + 4 * j + w;
    const int r = min(row[j], nr - 1);
    const float *p = r < nq ? a.q.at(t, r) : r < nq + a.nkv ? a.k.at(t, r - nq) : a.v.at(t, r - nq - a.nkv);
    x[j] = reinterpret_cast<const float4 *>(p)[lane];
  }
  const int half = a.rope.nrot / 2;
  if (tid < half) {
    const double pos = a.positions ? (double)a.positions[t] : (double)(a.pos0 + (uint32_t)t);
    const double turn = pos * a.rope.turns[tid];
    double sn, cs;
    sincospi(2.0 * (turn - rint(turn)), &sn, &cs);
    s_cs[tid] = (float)(cs * (double)a.rope.mscale);
    s_sn[tid] = (float)(sn * (double)a.rope.mscale);
  }
  __syncthreads();
  const int slot = slot_checked(a.L, a.pool_pages, a.pos0 + (uint32_t)t);
#pragma unroll
  for (int j = 0; j < RPW; ++j) {
    const int r = row[j];
    if (r >= nr) continue;                         // (wave-uniform)
    float4 y = x[j];
    if (r < nq + a.nkv) {
      const float *wt = r < nq ? a.qn_w : a.kn_w;
      if (wt) {
        const float4 g = reinterpret_cast<const float4 *>(wt)[lane];
        const float ss = wave_sum((y.x * y.x + y.y * y.y) + (y.z * y.z + y.w * y.w));
        const float inv = 1.0f / sqrtf(ss / (float)kHd + a.eps);
        y = make_float4(y.x * inv * g.x, y.y * inv * g.y, y.z * inv * g.z, y.w * inv * g.w);
      }
      if (a.rope.layout == BKV_ROPE_INTERLEAVED) {
        if (2 * lane < half) {
          const float c = s_cs[2 * lane], s = s_sn[2 * lane], lo = y.x, hi = y.y;
          y.x = lo * c - hi * s;
          y.y = hi * c + lo * s;
        }
        if (2 * lane + 1 < half) {
          const float c = s_cs[2 * lane + 1], s = s_sn[2 * lane + 1], lo = y.z, hi = y.w;
          y.z = lo * c - hi * s;
          y.w = hi * c + lo * s;
        }
      } else if (4 * lane < 2 * half) {            // (the other lanes' dims pass through, and no pair reads them)
        reinterpret_cast<float4 *>(s_x[w])[lane] = y;
        __builtin_amdgcn_wave_barrier();
        float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = 4 * lane + e;
          if (d < half) v[e] = v[e] * s_cs[d] - s_x[w][d + half] * s_sn[d];
          else if (d < 2 * half) v[e] = v[e] * s_cs[d - half] + s_x[w][d - half] * s_sn[d - half];
        }
        __builtin_amdgcn_wave_barrier();
        y = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    if (r < nq) {
      reinterpret_cast<float4 *>(a.q_out + ((size_t)t * a.nh + r) * kHd)[lane] = y;
    } else if (slot >= 0) {
      const int h = r - nq;
      if (h < a.nkv) store_values<KF>(y, const_cast<uint8_t *>(a.L.kd), const_cast<uint8_t *>(a.L.ks), (int64_t)slot * a.nkv + h, lane);
      else store_values<VF>(y, const_cast<uint8_t *>(a.L.vd), const_cast<uint8_t *>(a.L.vs), (int64_t)slot * a.nkv + h - a.nkv, lane);
    }
  }
}

hipError_t launch_rope_append(const RopeArgs &a, int kf, int vf, int n_tok, hipStream_t st) {
  const int nr = (a.q.p ? a.nh : 0) + 2 * a.nkv;
  BKV_FMT_SWITCH(kf, vf, hipLaunchKernelGGL((rope_append_kernel<KF_, VF_>), dim3(n_tok, (nr + kRopeRows - 1) / kRopeRows), dim3(256), 0, st, a));
  return hipGetLastError();
}

}  // namespace bkv
