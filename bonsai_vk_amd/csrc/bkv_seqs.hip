// bkv_seqs.hip - the tokens of several sequences on their way into one cache (bkv_seqs_rope_append: rotary positions of
// up to 8 axes, any format) and back as values (bkv_seqs_read). The single-sequence appends and reads of a 4-bit cache run here
// too.
//
// Per row x of 256: n = x * (1 / sqrt(mean(x^2) + eps)) * w (or x), then for pair p of the first nrot dims with
// a = 2 pi * pos[axis[p]] * turns[p]: y1 = (n1 cos a - n2 sin a) * mscale, y2 = (n2 cos a + n1 sin a) * mscale. The
// norm's sum and the angle are formed in fp64, cosine and sine rounded once to fp32: a value next to the border of two
// codes, 1/16 of its block's largest apart, is then on the same side however the sum is ordered.

#include <type_traits>

#include "bkv_device.h"
#include "bkv_internal.h"
#include "bkv_q4.h"

namespace bkv {

// ------------------------------------------------------------------ append
// One wave per row, 4 dims per lane; a workgroup takes up to 16 rows of one token (Q heads, then K, then V), 4 a wave.
constexpr int kSeqRows = 4;            // of a wave

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

// The sums over the lanes of 4 rows' values, of row j in the lanes 16 j .. (two rows at a time change halves, so that one
// addition serves both).
__device__ __forceinline__ double sums_of_4(const double (&v)[4]) {
  auto words = [](double x) { return __builtin_bit_cast(uint2, x); };
  auto number = [](uint32_t lo, uint32_t hi) { return __builtin_bit_cast(double, make_uint2(lo, hi)); };
  // lanes 0 .. 31: a's sum with the other half's, lanes 32 .. 63: b's
  auto halves = [&](double a, double b) {
    const auto lo = __builtin_amdgcn_permlane32_swap(words(a).x, words(b).x, false, false), hi = __builtin_amdgcn_permlane32_swap(words(a).y, words(b).y, false, false);
    return number(lo[0], hi[0]) + number(lo[1], hi[1]);
  };
  // of 32 lanes, the first 16: a's, the others: b's
  auto quarters = [&](double a, double b) {
    const auto lo = __builtin_amdgcn_permlane16_swap(words(a).x, words(b).x, false, false), hi = __builtin_amdgcn_permlane16_swap(words(a).y, words(b).y, false, false);
    return number(lo[0], hi[0]) + number(lo[1], hi[1]);
  };
  double x = quarters(halves(v[0], v[2]), halves(v[1], v[3]));
  auto more = [&](auto ctrl) {
    constexpr int C = decltype(ctrl)::value;
    const uint2 y = words(x);
    x += number((uint32_t)__builtin_amdgcn_update_dpp(0, (int)y.x, C, 0xF, 0xF, false), (uint32_t)__builtin_amdgcn_update_dpp(0, (int)y.y, C, 0xF, 0xF, false));
  };
  more(std::integral_constant<int, 0xB1>{});
  more(std::integral_constant<int, 0x4E>{});
  more(std::integral_constant<int, 0x141>{});
  more(std::integral_constant<int, 0x140>{});
  return x;
}
// 1 / sqrt(x): the instruction's 2^-26 and a step of Newton's, which leaves a square of that (Inf and NaN as they come)
__device__ __forceinline__ double rsqrt_f64(double x) {
  const double r = __builtin_amdgcn_rsq(x), y = fma(0.5 * r, fma(-x * r, r, 1.0), r);
  return y == y ? y : r;
}

// What bounds it: 40 KB a token in and out of 16 Q and 8 KV rows, and nearly as much the vector unit, in rows that are normed. So
// the four rows of a wave share a norm's reduction and root, a lane has its cosines and sines in registers for all its rows,
// and the small loads, which wait for one another, are asked for before the rows. One token 4.4 us (two trips to memory and the
// sines), 1201 of a picture without norms 12.5 (3.8 TB/s), 1100 with norms 14.1.
template <int KF, int VF>
__global__ __launch_bounds__(256) void seqs_rope_append_kernel(SeqsRowArgs a) {
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nq = a.q.p ? a.nh : 0, nr = nq + 2 * a.nkv, half = a.rope.nrot / 2;
  const int row0 = blockIdx.y * a.rows_per + w, rows = min(a.rows_per, nr - (int)blockIdx.y * a.rows_per);
  const int mine = (rows - w + 3) >> 2;            // rows w, w + 4, .. of the workgroup's
  __shared__ float s_cs[kHd / 2], s_sn[kHd / 2];
  __shared__ __attribute__((aligned(16))) float s_x[4][kHd];
  // ---- loads: of up to 64 sequences their ends and lengths, the token's positions, a pair's axis and turns
  const bool few = !a.one && a.v.n_seq <= 64;
  int end64 = 0, len64 = 0, begin0 = 0, pos_of_axis = 0, axis = 0;
  double turns = 0.0;
  if (few) {
    const int l = min(lane, a.v.n_seq - 1);
    end64 = a.v.q_start ? a.v.q_start[l + 1] : l + 1;
    len64 = a.v.len[l];
    begin0 = a.v.q_start ? a.v.q_start[0] : 0;
  }
  if (a.positions) pos_of_axis = a.positions[(int64_t)min(lane, a.n_axes - 1) * a.n_tok + t];
  if (tid < half) {
    axis = a.axis[tid];
    turns = a.rope.turns[tid];
  }
  float4 x[kSeqRows], wq = {}, wk = {};
  if (a.qn_w) wq = reinterpret_cast<const float4 *>(a.qn_w)[lane];
  if (a.kn_w) wk = reinterpret_cast<const float4 *>(a.kn_w)[lane];
#pragma unroll
  for (int j = 0; j < kSeqRows; ++j) {
    x[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (j >= mine) continue;
    const int r = row0 + 4 * j;
    const float *p = r < nq ? a.q.at(t, r) : r < nq + a.nkv ? a.k.at(t, r - nq) : a.v_rows.at(t, r - nq - a.nkv);
    x[j] = reinterpret_cast<const float4 *>(p)[lane];
  }
  // ---- the sequence and position of the token; none: one behind the last sequence
  int s = 0;
  int64_t pos = (int64_t)a.pos0 + t;
  if (few) {
    s = (int)__popcll(__ballot(lane < a.v.n_seq && end64 <= t));
    if (s >= a.v.n_seq) return;                    // (the whole workgroup)
    const int last = __builtin_amdgcn_readlane(end64, s), begin = s ? __builtin_amdgcn_readlane(end64, s - 1) : begin0;
    if (min(max(begin, 0), a.v.n_tok) > t) return;
    pos = (int64_t)__builtin_amdgcn_readlane(len64, s) - (min(max(last, 0), a.v.n_tok) - t);
  } else if (!a.one) {
    s = __builtin_amdgcn_readfirstlane(a.v.sequence_of<64>(t));
    if (s < 0) return;
    pos = (int64_t)a.v.len[s] - (a.v.q_begin(s + 1) - t);
  }
  const int slot = pos >= 0 && pos < a.v.max_pos ? a.v.slot(s, (uint32_t)pos) : -1;
  if (w < (half + 63) >> 6) {                      // (whole waves: the axes' positions are in their lanes)
    const int at_axis = __shfl(pos_of_axis, axis);
    const double at = a.positions ? (double)at_axis : (double)pos;
    const double turn = at * turns;
    double sn, cs;
    sincospi(2.0 * (turn - rint(turn)), &sn, &cs);
    if (tid < half) {
      s_cs[tid] = (float)(cs * (double)a.rope.mscale);
      s_sn[tid] = (float)(sn * (double)a.rope.mscale);
    }
  }
  // ---- norms
  float inv[kSeqRows];
  if (a.qn_w || a.kn_w) {
    double sq[kSeqRows];
#pragma unroll
    for (int j = 0; j < kSeqRows; ++j) sq[j] = ((double)x[j].x * x[j].x + (double)x[j].y * x[j].y) + ((double)x[j].z * x[j].z + (double)x[j].w * x[j].w);
    const float r = (float)rsqrt_f64(sums_of_4(sq) / kHd + (double)a.eps);
#pragma unroll
    for (int j = 0; j < kSeqRows; ++j) inv[j] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(r), 16 * j));
  }
  __syncthreads();
  // ---- the lane's turns: y[e] = x[e] c[e] + partner's s[e]
  const bool pairs = a.rope.layout == BKV_ROPE_INTERLEAVED, by4 = (half & 3) == 0;
  float c[4], sn[4];
  int partner[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = 4 * lane + e, p = min(pairs ? d >> 1 : d < half ? d : d - half, kHd / 2 - 1);
    const bool first = pairs ? (e & 1) == 0 : d < half;
    c[e] = s_cs[p];
    sn[e] = first ? -s_sn[p] : s_sn[p];
    partner[e] = (first ? d + half : d - half) & (kHd - 1);
  }
  const int turned = 2 * half - 4 * lane;          // of the lane's dims, the first; the others pass through
#pragma unroll
  for (int j = 0; j < kSeqRows; ++j) {
    if (j >= mine) break;                          // (the whole wave)
    const int r = row0 + 4 * j;
    float y[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
    if (r < nq + a.nkv) {
      if (r < nq ? a.qn_w : a.kn_w) {
        const float4 g = r < nq ? wq : wk;
        y[0] = y[0] * inv[j] * g.x; y[1] = y[1] * inv[j] * g.y; y[2] = y[2] * inv[j] * g.z; y[3] = y[3] * inv[j] * g.w;
      }
      float o[4] = {y[1], y[0], y[3], y[2]};
      if (!pairs) {
        if (by4) {                                 // (a lane's partners are one lane's)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = __shfl(y[e], partner[0] >> 2);
        } else {
          reinterpret_cast<float4 *>(s_x[w])[lane] = make_float4(y[0], y[1], y[2], y[3]);
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = s_x[w][partner[e]];
          __builtin_amdgcn_wave_barrier();
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = e < turned ? y[e] * c[e] + o[e] * sn[e] : y[e];
    }
    const float4 z = make_float4(y[0], y[1], y[2], y[3]);
    if (r < nq) {
      reinterpret_cast<float4 *>(a.q_out + ((size_t)t * a.nh + r) * kHd)[lane] = z;
    } else if (slot >= 0) {
      const int h = r - nq;
      if (h < a.nkv) store_row<KF>(z, const_cast<uint8_t *>(a.L.kd), const_cast<uint8_t *>(a.L.ks), (int64_t)slot * a.nkv + h, lane);
      else store_row<VF>(z, const_cast<uint8_t *>(a.L.vd), const_cast<uint8_t *>(a.L.vs), (int64_t)slot * a.nkv + h - a.nkv, lane);
    }
  }
}

hipError_t launch_seqs_rope_append(const SeqsRowArgs &in, int kf, int vf, hipStream_t st) {
  SeqsRowArgs a = in;
  // 4 rows a wave where that leaves the card a workgroup a CU (1201 tokens of 24 rows: 12.5 us; at 2 rows a wave 13.1), 2 of
  // fewer tokens' (one: 4.4 us; at 4 rows 4.8)
  const int nr = (a.q.p ? a.nh : 0) + 2 * a.nkv, per = (int64_t)a.n_tok * nr >= 4096 ? 4 * kSeqRows : 2 * kSeqRows;
  const int blocks = (nr + per - 1) / per;
  a.rows_per = (nr + blocks - 1) / blocks;
  const dim3 grid(a.n_tok, blocks);
  BKV_ANY_FMT_SWITCH(kf, vf, hipLaunchKernelGGL((seqs_rope_append_kernel<KF_, VF_>), grid, dim3(256), 0, st, a));
  return hipGetLastError();
}

// ------------------------------------------------------------------ read
// A head row is 256 values; 32 lanes take one, 8 values each. A row a thread: with four, asked for together, 1201 tokens take
// 7.8 us instead of 5.2 and one token 5.1 instead of 2.8.
constexpr int kSeqReadRows = 8;        // of a workgroup

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
__device__ __forceinline__ void seqs_read_row(const SeqsReadArgs &a, const uint8_t *data, const uint8_t *scales, void *out, int64_t r) {
  const int sub = threadIdx.x & 31;
  const int64_t rows = (int64_t)a.n_tok * a.nkv, rr = min(r, rows - 1);
  const int t = (int)(rr / a.nkv), h = (int)(rr - (int64_t)t * a.nkv);
  int s = 0, slot = -1;
  int64_t pos = (int64_t)a.pos0 + t;
  if (!a.one) {
    s = a.v.sequence_of<32>(t);
    if (s >= 0) pos = (int64_t)a.v.len[s] - (a.v.q_begin(s + 1) - t);
  }
  if (s >= 0 && pos >= 0 && pos < a.v.max_pos) slot = a.v.slot(s, (uint32_t)pos);
  if (r >= rows || s < 0) return;                  // (no sequence's row: left as it was)
  const int64_t at = (int64_t)max(slot, 0) * a.nkv + h;
  uint4 d = make_uint4(0, 0, 0, 0);
  uint32_t sc = 0;
  if constexpr (FMT == BKV_Q4_0) {
    d.x = reinterpret_cast<const uint32_t *>(data + at * kQ4RowBytes)[sub];
  } else if constexpr (FMT == BKV_Q8_0) {
    const uint2 w = reinterpret_cast<const uint2 *>(data + at * kHd)[sub];
    d.x = w.x;
    d.y = w.y;
  } else {
    d = reinterpret_cast<const uint4 *>(data + at * 2 * kHd)[sub];
  }
  if constexpr (FMT != BKV_F16) sc = reinterpret_cast<const uint16_t *>(scales + at * kScaleRowBytes)[sub >> 2];
  float v[8];
  const uint32_t w[4] = {d.x, d.y, d.z, d.w};
  const float scale = f16_to_f32(FMT == BKV_Q4_0 ? q4_scales(sc) & 0xFFFFu : sc);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (FMT == BKV_Q4_0) v[e] = (float)((int)((w[0] >> (16 * (e & 1) + 4 * (e >> 1))) & 15u) - 8) * scale;
    else if constexpr (FMT == BKV_Q8_0) v[e] = sbyte(w[e >> 2], e & 3) * scale;
    else v[e] = f16_to_f32((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
    if (slot < 0) v[e] = 0.0f;                     // (no position's)
  }
  store_out<OT>(out, t * a.tok + h * a.head + 8 * sub, v);
}

template <int KF, int VF, int OT>
__global__ __launch_bounds__(256) void seqs_read_kernel(SeqsReadArgs a) {
  const int64_t r = (int64_t)blockIdx.x * kSeqReadRows + (threadIdx.x >> 5);
  if (blockIdx.y == 0 && a.k_out) seqs_read_row<KF, OT>(a, a.L.kd, a.L.ks, a.k_out, r);
  else seqs_read_row<VF, OT>(a, a.L.vd, a.L.vs, a.v_out, r);
}

hipError_t launch_seqs_read(const SeqsReadArgs &a, int kf, int vf, int out_type, hipStream_t st) {
  const int64_t rows = (int64_t)a.n_tok * a.nkv;
  const dim3 grid((unsigned)((rows + kSeqReadRows - 1) / kSeqReadRows), a.k_out && a.v_out ? 2 : 1);
  BKV_ANY_FMT_SWITCH(kf, vf, {
    if (out_type == BKV_OUT_F32) hipLaunchKernelGGL((seqs_read_kernel<KF_, VF_, BKV_OUT_F32>), grid, dim3(256), 0, st, a);
    else if (out_type == BKV_OUT_F16) hipLaunchKernelGGL((seqs_read_kernel<KF_, VF_, BKV_OUT_F16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((seqs_read_kernel<KF_, VF_, BKV_OUT_BF16>), grid, dim3(256), 0, st, a);
  });
  return hipGetLastError();
}

}  // namespace bkv
