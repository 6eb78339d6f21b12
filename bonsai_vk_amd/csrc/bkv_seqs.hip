// bkv_seqs.hip - the tokens of several sequences on their way into one cache (bkv_seqs_rope_append: rotary positions of
// up to 8 axes, any format) and back as values (bkv_seqs_read). The single-sequence appends and reads of a 4-bit cache run here
// too.
//
// Per row x of 256: n = x * (1 / sqrt(mean(x^2) + eps)) * w (or x), then for pair p of the first nrot dims with
// a = 2 pi * pos[axis[p]] * turns[p]: y1 = (n1 cos a - n2 sin a) * mscale, y2 = (n2 cos a + n1 sin a) * mscale. The
// norm's sum and the angle are formed in fp64, cosine and sine rounded once to fp32: a value next to the border of two
// codes, 1/16 of its block's largest apart, is then on the same side however the sum is ordered.

#include "bkv_device.h"
#include "bkv_internal.h"
#include "bkv_q4.h"

namespace bkv {

// ------------------------------------------------------------------ append
// One wave per row, 4 dims per lane; a workgroup takes 8 rows of one token (Q heads, then K, then V).
constexpr int kSeqRows = 8;

// over the 8 lanes that hold a block
__device__ __forceinline__ float block_max8(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  return fmaxf(v, dpp<0x141>(v));
}
__device__ __forceinline__ float block_min8(float v) { return -block_max8(-v); }

// a row of 4 values per lane into the cache
template <int FMT>
__device__ __forceinline__ void store_row(const float4 x, uint8_t *data, uint8_t *scales, int64_t row, int lane) {
  if constexpr (FMT == BKV_Q4_0) {
    const uint32_t d = q4_scale(block_max8(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w))), block_min8(fminf(fminf(x.x, x.y), fminf(x.z, x.w))));
    const float id = q4_iscale(d);
    uint32_t w = q4_code(x.x, id) | (q4_code(x.y, id) << 16) | (q4_code(x.z, id) << 4) | (q4_code(x.w, id) << 20);
    w <<= 8 * (lane & 1);
    w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xF, 0xF, false);
    if ((lane & 1) == 0) reinterpret_cast<uint32_t *>(data + row * kQ4RowBytes)[lane >> 1] = w;
    if ((lane & 7) == 0) reinterpret_cast<uint16_t *>(scales + row * kScaleRowBytes)[lane >> 3] = (uint16_t)d;
  } else if constexpr (FMT == BKV_Q8_0) {
    const float amax = block_max8(fmaxf(fmaxf(fmaxf(fmaxf(0.0f, fabsf(x.x)), fabsf(x.y)), fabsf(x.z)), fabsf(x.w)));
    const float id = q8_iscale(amax);
    reinterpret_cast<uint32_t *>(data + row * kHd)[lane] =
        q8_byte<false>(x.x, id) | (q8_byte<false>(x.y, id) << 8) | (q8_byte<false>(x.z, id) << 16) | (q8_byte<false>(x.w, id) << 24);
    if ((lane & 7) == 0) reinterpret_cast<uint16_t *>(scales + row * kScaleRowBytes)[lane >> 3] = (uint16_t)f32_to_f16_rne(q8_scale(amax));
  } else {
    reinterpret_cast<uint2 *>(data + row * 2 * kHd)[lane] =
        make_uint2(f32_to_f16_rne(x.x) | (f32_to_f16_rne(x.y) << 16), f32_to_f16_rne(x.z) | (f32_to_f16_rne(x.w) << 16));
  }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// the sequence and position of token t; false where it has none (a token behind the last sequence, a negative position, one
// past the cache)
__device__ __forceinline__ bool place_of(const SeqsRowArgs &a, int t, int &s, int64_t &pos) {
  if (a.one) {
    s = 0;
    pos = (int64_t)a.pos0 + t;
    return true;
  }
  s = a.v.sequence_of<64>(t);
  if (s < 0) return false;
  pos = (int64_t)a.v.len[s] - (a.v.q_begin(s + 1) - t);
  return true;
}

template <int KF, int VF>
__global__ __launch_bounds__(256) void seqs_rope_append_kernel(SeqsRowArgs a) {
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int nq = a.q.p ? a.nh : 0, nr = nq + 2 * a.nkv;
  __shared__ float s_cs[kHd / 2], s_sn[kHd / 2];
  __shared__ __attribute__((aligned(16))) float s_x[4][kHd];
  constexpr int RPW = kSeqRows / 4;
  float4 x[RPW];
  int row[RPW];
#pragma unroll
  for (int j = 0; j < RPW; ++j) {
    row[j] = blockIdx.y * kSeqRows + 4 * j + w;
    const int r = min(row[j], nr - 1);
    const float *p = r < nq ? a.q.at(t, r) : r < nq + a.nkv ? a.k.at(t, r - nq) : a.v_rows.at(t, r - nq - a.nkv);
    x[j] = reinterpret_cast<const float4 *>(p)[lane];
  }
  int s;
  int64_t pos;
  if (!place_of(a, t, s, pos)) return;             // (the whole workgroup)
  const int half = a.rope.nrot / 2;
  if (tid < half) {
    const double at = a.positions ? (double)a.positions[(int64_t)a.axis[tid] * a.n_tok + t] : (double)pos;
    const double turn = at * a.rope.turns[tid];
    double sn, cs;
    sincospi(2.0 * (turn - rint(turn)), &sn, &cs);
    s_cs[tid] = (float)(cs * (double)a.rope.mscale);
    s_sn[tid] = (float)(sn * (double)a.rope.mscale);
  }
  __syncthreads();
  const int slot = pos >= 0 && pos < a.v.max_pos ? a.v.slot(s, (uint32_t)pos) : -1;
#pragma unroll
  for (int j = 0; j < RPW; ++j) {
    const int r = row[j];
    if (r >= nr) continue;                         // (wave-uniform)
    float4 y = x[j];
    if (r < nq + a.nkv) {
      const float *wt = r < nq ? a.qn_w : a.kn_w;
      if (wt) {
        const float4 g = reinterpret_cast<const float4 *>(wt)[lane];
        const double sq = wave_sum_f64(((double)y.x * y.x + (double)y.y * y.y) + ((double)y.z * y.z + (double)y.w * y.w));
        const float inv = (float)(1.0 / sqrt(sq / kHd + (double)a.eps));
        y = make_float4(y.x * inv * g.x, y.y * inv * g.y, y.z * inv * g.z, y.w * inv * g.w);
      }
      if (a.rope.layout == BKV_ROPE_INTERLEAVED) {
        if (2 * lane < half) {
          const float c = s_cs[2 * lane], sn = s_sn[2 * lane], lo = y.x, hi = y.y;
          y.x = lo * c - hi * sn;
          y.y = hi * c + lo * sn;
        }
        if (2 * lane + 1 < half) {
          const float c = s_cs[2 * lane + 1], sn = s_sn[2 * lane + 1], lo = y.z, hi = y.w;
          y.z = lo * c - hi * sn;
          y.w = hi * c + lo * sn;
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
      if (h < a.nkv) store_row<KF>(y, const_cast<uint8_t *>(a.L.kd), const_cast<uint8_t *>(a.L.ks), (int64_t)slot * a.nkv + h, lane);
      else store_row<VF>(y, const_cast<uint8_t *>(a.L.vd), const_cast<uint8_t *>(a.L.vs), (int64_t)slot * a.nkv + h - a.nkv, lane);
    }
  }
}

hipError_t launch_seqs_rope_append(const SeqsRowArgs &a, int kf, int vf, hipStream_t st) {
  const int nr = (a.q.p ? a.nh : 0) + 2 * a.nkv;
  const dim3 grid(a.n_tok, (nr + kSeqRows - 1) / kSeqRows);
  BKV_ANY_FMT_SWITCH(kf, vf, hipLaunchKernelGGL((seqs_rope_append_kernel<KF_, VF_>), grid, dim3(256), 0, st, a));
  return hipGetLastError();
}

// ------------------------------------------------------------------ read
// A head row is 256 values; 32 lanes take one, 8 values each. Each thread asks for kSeqReadRows rows before it stores the
// first.
constexpr int kSeqReadRows = 4;

template <int OT>
__device__ __forceinline__ void store_out(void *base, int64_t at, const float (&v)[8]) {
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
__device__ __forceinline__ void seqs_read_rows(const SeqsReadArgs &a, const uint8_t *data, const uint8_t *scales, void *out, int64_t first) {
  const int sub = threadIdx.x & 31;
  const int64_t rows = (int64_t)a.n_tok * a.nkv;
  uint4 d[kSeqReadRows];
  uint32_t sc[kSeqReadRows];
  int there[kSeqReadRows];                         // 0: no sequence's row; 1: no position's; 2: a value
#pragma unroll
  for (int j = 0; j < kSeqReadRows; ++j) {
    const int64_t r = min(first + 8 * j + (threadIdx.x >> 5), rows - 1);
    const int t = (int)(r / a.nkv), h = (int)(r - (int64_t)t * a.nkv);
    int s = 0, slot = -1;
    int64_t pos = (int64_t)a.pos0 + t;
    if (!a.one) {
      s = a.v.sequence_of<32>(t);
      if (s >= 0) pos = (int64_t)a.v.len[s] - (a.v.q_begin(s + 1) - t);
    }
    if (s >= 0 && pos >= 0 && pos < a.v.max_pos) slot = a.v.slot(s, (uint32_t)pos);
    there[j] = s < 0 ? 0 : slot < 0 ? 1 : 2;
    const int64_t at = (int64_t)max(slot, 0) * a.nkv + h;
    d[j] = make_uint4(0, 0, 0, 0);
    sc[j] = 0;
    if constexpr (FMT == BKV_Q4_0) {
      d[j].x = reinterpret_cast<const uint32_t *>(data + at * kQ4RowBytes)[sub];
    } else if constexpr (FMT == BKV_Q8_0) {
      const uint2 w = reinterpret_cast<const uint2 *>(data + at * kHd)[sub];
      d[j].x = w.x;
      d[j].y = w.y;
    } else {
      d[j] = reinterpret_cast<const uint4 *>(data + at * 2 * kHd)[sub];
    }
    if constexpr (FMT != BKV_F16) sc[j] = reinterpret_cast<const uint16_t *>(scales + at * kScaleRowBytes)[sub >> 2];
  }
#pragma unroll
  for (int j = 0; j < kSeqReadRows; ++j) {
    const int64_t r = first + 8 * j + (threadIdx.x >> 5);
    if (r >= rows || there[j] == 0) continue;
    const int64_t t = r / a.nkv, h = r - t * a.nkv;
    float v[8];
    const uint32_t w[4] = {d[j].x, d[j].y, d[j].z, d[j].w};
    const float scale = f16_to_f32(FMT == BKV_Q4_0 ? q4_scales(sc[j]) & 0xFFFFu : sc[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (FMT == BKV_Q4_0) v[e] = (float)((int)((w[0] >> (16 * (e & 1) + 4 * (e >> 1))) & 15u) - 8) * scale;
      else if constexpr (FMT == BKV_Q8_0) v[e] = sbyte(w[e >> 2], e & 3) * scale;
      else v[e] = f16_to_f32((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
      if (there[j] != 2) v[e] = 0.0f;
    }
    store_out<OT>(out, t * a.tok + h * a.head + 8 * sub, v);
  }
}

template <int KF, int VF, int OT>
__global__ __launch_bounds__(256) void seqs_read_kernel(SeqsReadArgs a) {
  const int64_t first = (int64_t)blockIdx.x * (8 * kSeqReadRows);
  if (blockIdx.y == 0 && a.k_out) seqs_read_rows<KF, OT>(a, a.L.kd, a.L.ks, a.k_out, first);
  else seqs_read_rows<VF, OT>(a, a.L.vd, a.L.vs, a.v_out, first);
}

hipError_t launch_seqs_read(const SeqsReadArgs &a, int kf, int vf, int out_type, hipStream_t st) {
  const int64_t rows = (int64_t)a.n_tok * a.nkv;
  const dim3 grid((unsigned)((rows + 8 * kSeqReadRows - 1) / (8 * kSeqReadRows)), a.k_out && a.v_out ? 2 : 1);
  BKV_ANY_FMT_SWITCH(kf, vf, {
    if (out_type == BKV_OUT_F32) hipLaunchKernelGGL((seqs_read_kernel<KF_, VF_, BKV_OUT_F32>), grid, dim3(256), 0, st, a);
    else if (out_type == BKV_OUT_F16) hipLaunchKernelGGL((seqs_read_kernel<KF_, VF_, BKV_OUT_F16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((seqs_read_kernel<KF_, VF_, BKV_OUT_BF16>), grid, dim3(256), 0, st, a);
  });
  return hipGetLastError();
}

}  // namespace bkv
