// bkv_tree.hip - attention of a tree of drafted tokens over the cache (bkv_attn_tree).
//
// The rows of one KV head are its n_q * grp (token, query head) pairs; row r sees the keys below pos0 and the
// drafted keys of its token's mask. With s = q16 . k (fp16 products, exact in the matrix cores, summed in fp32)
// and x = s * scale * log2(e):
//   out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m)   over the visible j, for any m near the largest x_j.
// One pass over the keys: every wave keeps a reference m, a sum and 256 unnormalised outputs per row, and lifts m
// only when a row's score exceeds it by kLift (the sums then stay below 2^(kLift + 1) per key, far from fp32's
// range). The key axis is split over workgroups, whose partial results tree_merge_kernel joins.
//
// P V on the fp16 matrix cores keeps fp32's precision by splitting both factors: 2^(x - m) * 2^9 = ph + pl, two
// fp16 (22 bits; the factor keeps pl normal down to p = 2^-14 of the largest), and q8_0's d * b = vh + vl, two fp16
// (exact: 19 bits); out = ph vh + pl vh + ph vl, what is left out is below 2^-22 of the result. A single fp16 per
// factor would leave 1e-4. q8_0 scales are brought near 2^7 by a power of two that a wave keeps for its keys, so
// that neither a large scale leaves fp16 nor a small one loses vl.
//
// Keys that a row does not see enter the products with p = 0. Where such a key's V is Inf or NaN the product is NaN,
// and so are Inf V under a visible key (ph and pl may have opposite signs) and non-finite scores: whatever is not
// finite at the end is computed again by tree_careful_row, key by key, in fp32, without the keys that are not seen.

#include <algorithm>

#include "bkv_device.h"
#include "bkv_internal.h"
#include "bkv_mfma16.h"

namespace bkv {

constexpr float kLift = 6.0f;          // a score this far (in powers of two) above the reference lifts it
constexpr float kPScale = 9.0f;        // log2 of the factor on p: 2^(kLift + kPScale) is within fp16
constexpr int kTreeKeys = 32;          // keys of a step
constexpr int kTreeFill = 512;         // workgroups that the key split aims for
constexpr int kTreeMaxSplit = 128;     // (the merge holds a row's partial references two to a lane)

// the 32 keys from kb on that row token i sees, one bit each; keys from nk on are not there
__device__ __forceinline__ uint32_t tree_window(const TreeArgs &a, int i, int64_t kb) {
  const int64_t rel = kb - a.pos0;                 // > -32: some of the keys are drafted ones
  const int nq = a.n_q;
  uint32_t win;
  if (a.mask == nullptr) {
    const int64_t last = i - rel;                  // bits 0 .. last
    win = last < 0 ? 0u : last >= 31 ? ~0u : (2u << (int)last) - 1u;
  } else {
    const uint64_t *row = a.mask + (int64_t)i * a.words;
    if (rel < 0) {
      const int c = (int)-rel;
      win = ((uint32_t)row[0] << c) | ((1u << c) - 1u);
    } else {
      const int w = (int)(rel >> 6), sh = (int)(rel & 63);
      uint64_t v = row[w] >> sh;
      if (sh > 32 && w + 1 < a.words) v |= row[w + 1] << (64 - sh);
      win = (uint32_t)v;
    }
  }
  const int64_t there = nq - rel;                  // keys before nk
  return there >= 32 ? win : win & ((1u << (int)there) - 1u);
}

// ------------------------------------------------------------------ joining the key ranges
// Row r = i * nh + h by itself: 4 waves take every fourth key, a lane 4 dims. Only reached for rows whose partial
// results are not finite, so its time (about 1 us per 30 keys) is not that of ordinary calls.
template <int KF, int VF>
__device__ void tree_careful_row(const TreeArgs &a, int i, int h, float *s_o, float *s_ml, float4 &o, float &l) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hk = h / a.grp;
  const float4 qv = reinterpret_cast<const float4 *>(a.q.at(i, h))[lane];
  const float q[4] = {round_f16(qv.x), round_f16(qv.y), round_f16(qv.z), round_f16(qv.w)};
  const uint32_t nk = a.pos0 + (uint32_t)a.n_q;
  float m = -INFINITY, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  l = 0.0f;
  auto row4 = [&](const uint8_t *data, const uint8_t *scales, int fmt, int64_t row, float (&x)[4]) {
    if (fmt == BKV_Q8_0) {
      const uint32_t b = reinterpret_cast<const uint32_t *>(data + row * kHd)[lane];
      const float d = f16_to_f32(reinterpret_cast<const uint16_t *>(scales + row * kScaleRowBytes)[lane >> 3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = sbyte(b, e) * d;
    } else {
      const uint2 b = reinterpret_cast<const uint2 *>(data + row * 2 * kHd)[lane];
      x[0] = f16_to_f32(b.x & 0xFFFFu); x[1] = f16_to_f32(b.x >> 16);
      x[2] = f16_to_f32(b.y & 0xFFFFu); x[3] = f16_to_f32(b.y >> 16);
    }
  };
  for (uint32_t k = (uint32_t)w; k < nk; k += 4) {
    if (k >= a.pos0 && !(tree_window(a, i, k) & 1u)) continue;
    const int slot = slot_checked(a.L, a.pool_pages, k);
    if (slot < 0) continue;
    const int64_t row = (int64_t)slot * a.nkv + hk;
    float x[4], v[4];
    row4(a.L.vd, a.L.vs, VF, row, v);
    float s;
    if constexpr (KF == BKV_Q8_0) {                // per block (8 lanes) the scale times the bytes' sum, as the other kernels
      const uint32_t b = reinterpret_cast<const uint32_t *>(a.L.kd + row * kHd)[lane];
      s = (q[0] * sbyte(b, 0) + q[1] * sbyte(b, 1)) + (q[2] * sbyte(b, 2) + q[3] * sbyte(b, 3));
      s += dpp<0xB1>(s);
      s += dpp<0x4E>(s);
      s += dpp<0x141>(s);
      s *= f16_to_f32(reinterpret_cast<const uint16_t *>(a.L.ks + row * kScaleRowBytes)[lane >> 3]);
      s += dpp<0x140>(s);
      s += __shfl_xor(s, 16);
      s = (s + __shfl_xor(s, 32)) * a.scale2;
    } else {
      row4(a.L.kd, a.L.ks, KF, row, x);
      s = wave_sum((q[0] * x[0] + q[1] * x[1]) + (q[2] * x[2] + q[3] * x[3])) * a.scale2;
    }
    const float mn = s > m ? s : m;
    const float al = m == mn ? 1.0f : exp2f(m - mn);
    // (a score of -Inf counts for nothing beside others; alone it leaves 0 / 0)
    const float p = s == -INFINITY ? 0.0f : exp2f(s - mn);
    l = l * al + p;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = acc[e] * al + p * v[e];
    m = mn;
  }
  reinterpret_cast<float4 *>(s_o + w * kHd)[lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  if (lane == 0) { s_ml[2 * w] = m; s_ml[2 * w + 1] = l; }
  __syncthreads();
  float mm = fmaxf(fmaxf(s_ml[0], s_ml[2]), fmaxf(s_ml[4], s_ml[6]));
  l = 0.0f;
  o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int j = 0; j < 4; ++j) {
    const float mj = s_ml[2 * j], lj = s_ml[2 * j + 1];
    const float f = mj == mm ? 1.0f : exp2f(mj - mm);
    const float4 t = reinterpret_cast<const float4 *>(s_o + j * kHd)[lane];
    if (mj == -INFINITY && lj == 0.0f) continue;
    l += lj * f;
    o.x += t.x * f; o.y += t.y * f; o.z += t.z * f; o.w += t.w * f;
  }
  __syncthreads();
}

// whether row i's token sees any key
__device__ __forceinline__ bool tree_sees(const TreeArgs &a, int i) {
  const uint32_t nk = a.pos0 + (uint32_t)a.n_q;
  if (a.L.page == 0) {
    if (a.pos0 > 0 || a.mask == nullptr) return true;
    for (int j = 0; j < a.n_q; j += 32)
      if (tree_window(a, i, j)) return true;
    return false;
  }
  for (uint32_t k = 0; k < nk; ++k) {
    if (k >= a.pos0 && !(tree_window(a, i, k) & 1u)) continue;
    if (slot_checked(a.L, a.pool_pages, k) >= 0) return true;
  }
  return false;
}

// One workgroup per row: wave w sums the ranges w, w + 4, .. (a lane 4 dims, kB ranges requested together), then
// the waves' sums meet in LDS.
template <int KF, int VF>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t rows = (int64_t)a.n_q * a.nh, r = blockIdx.x;
  const int i = (int)(r / a.nh), h = (int)(r - (int64_t)i * a.nh);
  __shared__ __attribute__((aligned(16))) float s_o[4 * kHd];
  __shared__ float s_ml[8];
  const float2 none = make_float2(-INFINITY, 0.0f);
  const float2 m0 = lane < a.splits ? a.ml[(int64_t)lane * rows + r] : none;
  const float2 m1 = lane + 64 < a.splits ? a.ml[(int64_t)(lane + 64) * rows + r] : none;
  const float mm = wave_max(fmaxf(m0.x, m1.x));
  const float f0 = m0.x == -INFINITY ? 0.0f : exp2f(m0.x - mm), f1 = m1.x == -INFINITY ? 0.0f : exp2f(m1.x - mm);
  float l = wave_sum(m0.y * f0 + m1.y * f1);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  constexpr int kB = 8;
  for (int s0 = w; s0 < a.splits; s0 += 4 * kB) {
    float4 t[kB];
#pragma unroll
    for (int j = 0; j < kB; ++j)
      t[j] = reinterpret_cast<const float4 *>(a.part + ((int64_t)min(s0 + 4 * j, a.splits - 1) * rows + r) * kHd)[lane];
#pragma unroll
    for (int j = 0; j < kB; ++j) {
      const int s = s0 + 4 * j;
      if (s >= a.splits) break;
      const float f = __shfl(s < 64 ? f0 : f1, s & 63);
      o.x = fmaf(t[j].x, f, o.x); o.y = fmaf(t[j].y, f, o.y); o.z = fmaf(t[j].z, f, o.z); o.w = fmaf(t[j].w, f, o.w);
    }
  }
  reinterpret_cast<float4 *>(s_o + w * kHd)[lane] = o;
  __syncthreads();
  o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 t = reinterpret_cast<const float4 *>(s_o + j * kHd)[lane];
    o.x += t.x; o.y += t.y; o.z += t.z; o.w += t.w;
  }
  __syncthreads();
  // (every wave holds the whole row: the decision is the workgroup's)
  const float big = fmaxf(fmaxf(fabsf(o.x), fabsf(o.y)), fmaxf(fabsf(o.z), fabsf(o.w)));
  bool fine = l > 0.0f && l < INFINITY && !__any(!(big < INFINITY) || o.x != o.x || o.y != o.y || o.z != o.z || o.w != o.w);
  // fp16 V of subnormal size (kTiny is below 2^-14 by the averaging of a few keys): the matrix cores keep such a
  // product to about 2^-37 of p's unit and not to 24 bits of itself (V of 1e-6: 7e-6 off; of 1e-4: 3e-7)
  constexpr float kTiny = 0x1p-17f;
  if (VF == BKV_F16 && fine) {
    const float top = wave_max(big);
    fine = top == 0.0f || !(top < kTiny * l);
  }
  bool empty = false;
  if (!fine) {
    empty = !tree_sees(a, i);
    if (!empty) tree_careful_row<KF, VF>(a, i, h, s_o, s_ml, o, l);
  }
  if (w == 0) {
    const float4 v = empty ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
    reinterpret_cast<float4 *>(a.out + r * kHd)[lane] = v;
    if (a.gate.p) {
      const float4 g = reinterpret_cast<const float4 *>(a.gate.at(i, h))[lane];
      reinterpret_cast<float4 *>(a.out_gated + r * kHd)[lane] =
          make_float4(v.x / (1.0f + expf(-g.x)), v.y / (1.0f + expf(-g.y)), v.z / (1.0f + expf(-g.z)), v.w / (1.0f + expf(-g.w)));
    }
  }
}

// ------------------------------------------------------------------ few rows: keys straight into registers
// A workgroup holds 16 rows; each of its 4 waves streams a key range of its own, 32 keys a step, without LDS or
// barriers until the ranges are joined. Bound by the memory: a wave has a step's K and V (17 KB in q8_0) in flight.
//
// Scores are computed transposed, S^T = K Q^T: lane (n, g) = (lane % 16, lane / 16) then holds keys 4 g .. 4 g + 3 of
// a 16-key tile for row n, which is P^T's operand of O^T = V^T P^T as it stands if slot (g, j) of the 32-key
// contraction stands for key 4 g + j (j < 4) or 16 + 4 g + j - 4, for both operands. V's operand wants one dim of 8
// keys per lane: lane (m, g) loads its 8 keys' bytes of dims 16 m .. 16 m + 15 (whole 256-byte rows per 16 lanes), and
// product dt takes byte dt of each, so that row m of product dt is dim 16 m + dt (fp16 V: 8 dims per load, dim
// 128 (dt / 8) + 8 m + dt % 8). No transposition goes through LDS.
template <int VF>
__device__ __forceinline__ int tree_dim(int dt, int m) {
  return VF == BKV_Q8_0 ? 16 * m + dt : 128 * (dt >> 3) + 8 * m + (dt & 7);
}

// fp16 pair (low half of a's selected half or byte, then b's)
template <int SEL>
__device__ __forceinline__ uint32_t pair_bytes(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x0C000C00u | (uint32_t)SEL | ((uint32_t)(SEL + 4) << 16));
}

// keys 4 g + i of the tile for all lanes of row group g: lane (r, g) holds the scales of key 4 g + r % 4
template <int I>
__device__ __forceinline__ uint32_t row_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x150 + I, 0xF, 0xF, false);
}

template <int KF, int VF, bool PG>
__global__ __launch_bounds__(256, KF == BKV_F16 && VF == BKV_F16 ? 1 : 2) void tree_stream_kernel(TreeArgs a, int nrb) {
  constexpr int KRB = row_bytes(KF), VRB = row_bytes(VF);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  // workgroups 8 apart run on the same XCD: the row blocks of one key range are neighbours there
  const int unit = (int)(blockIdx.x / (8 * nrb)) * 8 + (blockIdx.x & 7), rb = (blockIdx.x >> 3) % nrb;
  if (unit >= a.nkv * a.splits) return;
  const int hk = unit / a.splits, split = unit - hk * a.splits;
  const int R = a.n_q * a.grp, r = min(16 * rb + n, R - 1), tok = r / a.grp, hq = hk * a.grp + r - tok * a.grp;
  const uint32_t nk = a.pos0 + (uint32_t)a.n_q;
  const int64_t steps = (nk + kTreeKeys - 1) / kTreeKeys, wi = split * 4 + w, nw = a.splits * 4;
  const int64_t t0 = steps * wi / nw, t1 = steps * (wi + 1) / nw;

  h8 qh[8];                                        // row n, dims 32 b + 8 g ..
  {
    const float *q = a.q.at(tok, hq) + 8 * g;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const float4 x = *reinterpret_cast<const float4 *>(q + 32 * b), y = *reinterpret_cast<const float4 *>(q + 32 * b + 4);
      qh[b] = h8{(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w, (_Float16)y.x, (_Float16)y.y, (_Float16)y.z, (_Float16)y.w};
    }
  }
  f4 o[16] = {};
  float m = -INFINITY, l = 0.0f;                   // m: the reference less kPScale
  int ve = 100;                                    // q8_0 V: the outputs are in units of 2^-ve (100: none yet)
  uint4 kr[2][KF ? 4 : 8], ks[2], vr[8][VF ? 1 : 2];
  uint32_t vs[4];
  const size_t krow = (size_t)a.nkv * KRB, vrow = (size_t)a.nkv * VRB, srow = (size_t)a.nkv * kScaleRowBytes;
  const uint8_t *kd = a.L.kd + (size_t)hk * KRB, *vd = a.L.vd + (size_t)hk * VRB;
  const uint8_t *ksc = KF ? a.L.ks + (size_t)hk * kScaleRowBytes : nullptr, *vsc = VF ? a.L.vs + (size_t)hk * kScaleRowBytes : nullptr;

  // lane l's slot of key kb + l % 32 (keys from nk on: the last one's), -1 outside the pool
  auto slots = [&](int64_t kb) { return slot_checked(a.L, a.pool_pages, (uint32_t)min(kb + (lane & 31), (int64_t)nk - 1)); };
  auto slot = [&](int sl, int64_t kb, int j) -> int64_t {
    if constexpr (PG) return max(__shfl(sl, j), 0);
    else return min(kb + j, (int64_t)nk - 1);
  };
  auto load_k = [&](int64_t kb, int sl) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t *p = kd + (size_t)slot(sl, kb, 16 * t + n) * krow;
      if constexpr (KF) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint2 x = *reinterpret_cast<const uint2 *>(p + 64 * b + 8 * g), y = *reinterpret_cast<const uint2 *>(p + 64 * b + 32 + 8 * g);
          kr[t][b] = make_uint4(x.x, x.y, y.x, y.y);
        }
        ks[t] = *reinterpret_cast<const uint4 *>(ksc + (size_t)slot(sl, kb, 16 * t + 4 * g + (n & 3)) * srow);
      } else {
#pragma unroll
        for (int b = 0; b < 8; ++b) kr[t][b] = *reinterpret_cast<const uint4 *>(p + 64 * b + 16 * g);
      }
    }
  };
  auto load_v = [&](int64_t kb, int sl) {
    uint32_t s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const size_t at = (size_t)slot(sl, kb, (j & 4) * 4 + 4 * g + (j & 3));
      const uint8_t *p = vd + at * vrow + 16 * n;
      vr[j][0] = *reinterpret_cast<const uint4 *>(p);
      if constexpr (VF) s[j] = *reinterpret_cast<const uint16_t *>(vsc + at * srow + 2 * (n >> 1));
      else vr[j][VF ? 0 : 1] = *reinterpret_cast<const uint4 *>(p + 256);
    }
    if constexpr (VF)
#pragma unroll
      for (int j = 0; j < 4; ++j) vs[j] = s[2 * j] | (s[2 * j + 1] << 16);
  };

  int sl = 0;
  if (t0 < t1) {
    if constexpr (PG) sl = slots(t0 * kTreeKeys);
    load_k(t0 * kTreeKeys, sl);
    load_v(t0 * kTreeKeys, sl);
  }
#pragma unroll 1
  for (int64_t t = t0; t < t1; ++t) {
    const int64_t kb = t * kTreeKeys;
    const int64_t kn = min(t + 1, t1 - 1) * kTreeKeys;
    // ---- scores
    f4 s[2] = {};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (KF) {
        const uint32_t sw[4] = {ks[u].x, ks[u].y, ks[u].z, ks[u].w};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint32_t x[4] = {kr[u][b].x ^ 0x80808080u, kr[u][b].y ^ 0x80808080u, kr[u][b].z ^ 0x80808080u, kr[u][b].w ^ 0x80808080u};
          const uint32_t d[4] = {row_lane<0>(sw[b]), row_lane<1>(sw[b]), row_lane<2>(sw[b]), row_lane<3>(sw[b])};
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) {
            uint4 kv;
            kv.x = as_u(bytes_h2<0x04010400u>(x[2 * hb])); kv.y = as_u(bytes_h2<0x04030402u>(x[2 * hb]));
            kv.z = as_u(bytes_h2<0x04010400u>(x[2 * hb + 1])); kv.w = as_u(bytes_h2<0x04030402u>(x[2 * hb + 1]));
            const f4 p = mfma16(__builtin_bit_cast(h8, kv), qh[2 * b + hb], f4{});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              s[u][i] = __builtin_fmaf(p[i], (float)__builtin_bit_cast(_Float16, (uint16_t)(d[i] >> (16 * hb))), s[u][i]);
          }
        }
      } else {
#pragma unroll
        for (int b = 0; b < 8; ++b) s[u] = mfma16(__builtin_bit_cast(h8, kr[u][b]), qh[b], s[u]);
      }
    }
    uint32_t there = ~0u;                          // keys whose page is in the pool
    if constexpr (PG) there = (uint32_t)__ballot(sl >= 0);
    int sn = 0;
    if constexpr (PG) sn = slots(kn);
    load_k(kn, sn);
    // ---- probabilities
    uint32_t win = there;
    if (kb + kTreeKeys > a.pos0) win &= tree_window(a, tok, kb);
    win >>= 4 * g;                                 // bit i: key 4 g + i of tile 0, bit 16 + i: of tile 1
    float x[8], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = s[j >> 2][j & 3] * a.scale2;
      if (!((win >> ((j & 4) * 4 + (j & 3))) & 1u)) x[j] = -INFINITY;
      top = fmaxf(top, x[j]);
    }
    if (__any(top > m + (kLift + kPScale))) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, top - kPScale);
      const float f = mn == m ? 1.0f : exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < 16; ++dt) o[dt] *= f;
    }
    h8 ph, pl;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool seen = (win >> ((j & 4) * 4 + (j & 3))) & 1u;
      const float p = seen ? __builtin_amdgcn_exp2f(x[j] - m) : 0.0f;
      l += p;
      ph[j] = (_Float16)p;
      pl[j] = (_Float16)(p - (float)ph[j]);
    }
    // ---- V
    if constexpr (VF) {
      // the factor 2^ve that brings the largest scale to [2^7, 2^8) of the keys so far
      uint32_t b = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) b = max(b, max(vs[j] & 0x7FFFu, (vs[j] >> 16) & 0x7FFFu));
      const int e = b ? 7 + 15 - (int)max(b >> 10, 1u) : 15;
      if (__any(e < ve)) {
        int en = min(e, 15);
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) en = min(en, __shfl_xor(en, k));
        if (ve != 100) {
          const float f = __builtin_ldexpf(1.0f, en - ve);
#pragma unroll
          for (int dt = 0; dt < 16; ++dt) o[dt] *= f;
        }
        ve = en;
      }
      const _Float16 vf = (_Float16)__builtin_ldexpf(1.0f, ve);
      h2 d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = as_h2(vs[j]) * h2{vf, vf};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t wv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) wv[j] = (&vr[j][0].x)[c];
#pragma unroll
        for (int by = 0; by < 4; ++by) {
          uint32_t ah[4], al[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = wv[2 * j], hi = wv[2 * j + 1];
            const uint32_t pb = by == 0 ? pair_bytes<0>(lo, hi) : by == 1 ? pair_bytes<1>(lo, hi) : by == 2 ? pair_bytes<2>(lo, hi) : pair_bytes<3>(lo, hi);
            h2 h, lw;
            split_prod(as_h2(pb ^ 0x64806480u) - h2{(_Float16)1152.0f, (_Float16)1152.0f}, d[j], h, lw);
            ah[j] = as_u(h);
            al[j] = as_u(lw);
          }
          const h8 vh = __builtin_bit_cast(h8, make_uint4(ah[0], ah[1], ah[2], ah[3]));
          const h8 vl = __builtin_bit_cast(h8, make_uint4(al[0], al[1], al[2], al[3]));
          f4 &z = o[4 * c + by];
          z = mfma16(vl, ph, z);
          z = mfma16(vh, pl, z);
          z = mfma16(vh, ph, z);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t wv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) wv[j] = (&vr[j][VF ? 0 : c >> 2].x)[c & 3];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t av[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) av[j] = __builtin_amdgcn_perm(wv[2 * j + 1], wv[2 * j], hf ? 0x07060302u : 0x05040100u);
          const h8 vh = __builtin_bit_cast(h8, make_uint4(av[0], av[1], av[2], av[3]));
          f4 &z = o[2 * c + hf];
          z = mfma16(vh, pl, z);
          z = mfma16(vh, ph, z);
        }
      }
    }
    load_v(kn, sn);
    sl = sn;
  }

  // ---- the 4 ranges joined, one partial result per row and workgroup
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  constexpr int kOS = kHd + 4;
  __shared__ __attribute__((aligned(16))) float s_o[4][16][kOS];
  __shared__ float s_m[4][16], s_l[4][16];
  if (g == 0) { s_m[w][n] = m; s_l[w][n] = l; }
  __syncthreads();
  const float mm = fmaxf(fmaxf(s_m[0][n], s_m[1][n]), fmaxf(s_m[2][n], s_m[3][n]));
  const float f = m == -INFINITY ? 0.0f : exp2f(m - mm), fo = VF && ve != 100 ? __builtin_ldexpf(f, -ve) : f;
#pragma unroll
  for (int dt = 0; dt < 16; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) s_o[w][n][tree_dim<VF>(dt, 4 * g + i)] = o[dt][i] * fo;
  __syncthreads();
  const int row = threadIdx.x >> 4, c = threadIdx.x & 15, rr = 16 * rb + row;
  if (rr < R) {
    const int64_t rows = (int64_t)a.n_q * a.nh;
    const int ti = rr / a.grp;
    const int64_t at = (int64_t)split * rows + (int64_t)ti * a.nh + hk * a.grp + rr - ti * a.grp;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 t = *reinterpret_cast<const float4 *>(&s_o[j][row][4 * c + 64 * k]);
        v.x += t.x; v.y += t.y; v.z += t.z; v.w += t.w;
      }
      *reinterpret_cast<float4 *>(a.part + at * kHd + 4 * c + 64 * k) = v;
    }
    if (c == 0) {
      const float mr = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
      float lr = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) lr += s_m[j][row] == -INFINITY ? s_l[j][row] : s_l[j][row] * exp2f(s_m[j][row] - mr);
      a.ml[at] = make_float2(mr, lr);
    }
  }
}

// ------------------------------------------------------------------ host side
static inline int64_t cdiv(int64_t x, int64_t y) { return (x + y - 1) / y; }
static inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

TreePlan plan_tree(int nh, int nkv, int64_t pos0, int n_q, size_t base) {
  TreePlan p{};
  const int64_t rows = (int64_t)n_q * (nh / nkv), steps = cdiv(pos0 + n_q, kTreeKeys);
  p.nrb = (int)cdiv(rows, 16);
  p.splits = (int)std::min<int64_t>(std::min<int64_t>(kTreeMaxSplit, cdiv(steps, 4)), std::max<int64_t>(1, kTreeFill / ((int64_t)nkv * p.nrb)));
  p.off_ml = base;
  p.off_part = up256(base + (size_t)p.splits * n_q * nh * sizeof(float2));
  p.total = up256(p.off_part + (size_t)p.splits * n_q * nh * kHd * sizeof(float));
  return p;
}

// the largest plan of any call: split row blocks are at most kTreeFill of 16 rows, others write every row once
size_t tree_workspace_bound(int nh, int nkv, size_t base) {
  const size_t rows = std::max<size_t>((size_t)kTreeFill * 16, (size_t)BKV_TREE_MAX_Q * nh);
  (void)nkv;
  return base + up256(rows * sizeof(float2)) + up256(rows * kHd * sizeof(float)) + 256;
}

hipError_t launch_tree(const TreeArgs &a, const TreePlan &p, int kf, int vf, hipStream_t st) {
  const unsigned grid = (unsigned)(cdiv((int64_t)a.nkv * a.splits, 8) * 8 * p.nrb);
  BKV_FMT_SWITCH(kf, vf, {
    if (a.L.page) hipLaunchKernelGGL((tree_stream_kernel<KF_, VF_, true>), dim3(grid), dim3(256), 0, st, a, p.nrb);
    else hipLaunchKernelGGL((tree_stream_kernel<KF_, VF_, false>), dim3(grid), dim3(256), 0, st, a, p.nrb);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((tree_merge_kernel<KF_, VF_>), dim3((unsigned)((int64_t)a.n_q * a.nh)), dim3(256), 0, st, a);
  });
  return hipGetLastError();
}

}  // namespace bkv
