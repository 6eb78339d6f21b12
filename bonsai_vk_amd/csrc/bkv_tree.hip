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
// factor would leave 1e-4; against the formula in 64 bits the results are 3e-7 to 6e-7 off (2-norm). scale_level says
// how q8_0 scales of any size stay within fp16.
//
// Keys that a row does not see enter the products with p = 0. Where such a key's V is Inf or NaN the product is NaN,
// and so are Inf V under a visible key (ph and pl may have opposite signs) and non-finite scores: whatever is not
// finite at the end is computed again by tree_careful_row, key by key, in fp32, without the keys that are not seen.
//
// Two launches whatever the sizes: tree_stream_kernel (16 rows a workgroup) or tree_tile_kernel (128 or 256), whichever
// plan_tree expects to take less time, then the join.

#include <algorithm>
#include <cmath>

#include "bkv_device.h"
#include "bkv_internal.h"
#include "bkv_mfma16.h"

namespace bkv {

constexpr float kLift = 6.0f;          // a score this far (in powers of two) above the reference lifts it
constexpr float kPScale = 9.0f;        // log2 of the factor on p: 2^(kLift + kPScale) is within fp16
constexpr int kTreeKeys = 32;          // keys of a step
constexpr int kTreeMaxSplit = 128;     // (the merge holds a row's partial references two to a lane)

// the 32 keys from kb on that row token i sees, one bit each; keys from nk on are not there
__device__ __forceinline__ uint32_t tree_window(const TreeArgs &a, int i, int64_t kb) {
  const int rel = (int)(kb - a.pos0);              // > -32: some of the keys are drafted ones
  uint32_t win;
  if (a.mask == nullptr) {
    const int last = i - rel;                      // bits 0 .. last
    win = last < 0 ? 0u : last >= 31 ? ~0u : (2u << last) - 1u;
  } else {
    const uint32_t row = (uint32_t)(i * a.words);
    if (rel < 0) {
      win = ((uint32_t)a.mask[row] << -rel) | ((1u << -rel) - 1u);
    } else {
      const int w = rel >> 6, sh = rel & 63;
      uint64_t v = a.mask[row + w] >> sh;
      if (sh > 32 && w + 1 < a.words) v |= a.mask[row + w + 1] << (64 - sh);
      win = (uint32_t)v;
    }
  }
  const int there = a.n_q - rel;                   // keys before nk
  return there >= 32 ? win : win & ((1u << there) - 1u);
}

// ------------------------------------------------------------------ joining the key ranges
// Row (i, h) by itself: each wave takes every NWV-th key, a lane 4 dims. Only reached for rows whose partial
// results are not finite, so its time is not that of ordinary calls: a latency after the other, 1.1 us per key of a wave.
// 8 tokens, one of whose V is NaN, onto 8192 and 32768 keys take 1.2 and 4.6 ms (22 and 38 us without), on 8 waves a row;
// 1024 tokens, which have one wave a row, 17 and 66 ms (0.37 and 1.1).
template <int KF, int VF, int NWV>
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
  for (uint32_t k = (uint32_t)w; k < nk; k += NWV) {
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
  float mm = -INFINITY;
  for (int j = 0; j < NWV; ++j) mm = fmaxf(mm, s_ml[2 * j]);
  l = 0.0f;
  o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int j = 0; j < NWV; ++j) {
    const float mj = s_ml[2 * j], lj = s_ml[2 * j + 1];
    const float f = mj == mm ? 1.0f : exp2f(mj - mm);
    const float4 t = reinterpret_cast<const float4 *>(s_o + j * kHd)[lane];
    if (mj == -INFINITY && lj == 0.0f) continue;
    l += lj * f;
    o.x += t.x * f; o.y += t.y * f; o.z += t.z * f; o.w += t.w * f;
  }
  __syncthreads();
}

// whether row i's token sees any key (a lane a page, then a lane a drafted token)
__device__ __forceinline__ bool tree_sees(const TreeArgs &a, int i) {
  const int lane = threadIdx.x & 63;
  if (a.L.page == 0 && a.pos0 > 0) return true;
  bool some = false;
  if (a.L.page > 0)
    for (uint64_t k = (uint64_t)lane * (uint32_t)a.L.page; k < a.pos0; k += 64ull * (uint32_t)a.L.page)
      some |= slot_checked(a.L, a.pool_pages, (uint32_t)k) >= 0;
  for (int j = lane; j < a.n_q; j += 64)
    some |= (tree_window(a, i, (int64_t)a.pos0 + j) & 1u) && slot_checked(a.L, a.pool_pages, a.pos0 + (uint32_t)j) >= 0;
  return __any(some);
}

// One workgroup of NWV waves per row: wave w sums the ranges w, w + NWV, .. (a lane 4 dims, 8 ranges requested
// together), then the waves' sums meet in LDS. The launch takes as many waves as leave each 8 ranges: one row's 128
// ranges on 4 waves took 12.4 us, a latency after the other. 4 us for a few rows, a launch and two latencies; 15 us for
// 1024 rows of 64 ranges, whose 67 MB it reads at 4.5 TB/s.
template <int KF, int VF, int NWV>
__global__ __launch_bounds__(64 * NWV) void tree_merge_kernel(TreeArgs a) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t rows = (int64_t)a.n_q * a.nh, r = blockIdx.x;
  const int i = (int)(r / a.nh), h = (int)(r - (int64_t)i * a.nh);
  __shared__ __attribute__((aligned(16))) float s_o[NWV * kHd];
  __shared__ float s_ml[2 * NWV];
  const float2 none = make_float2(-INFINITY, 0.0f);
  const float2 m0 = lane < a.splits ? a.ml[(int64_t)lane * rows + r] : none;
  const float2 m1 = lane + 64 < a.splits ? a.ml[(int64_t)(lane + 64) * rows + r] : none;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f), t[8];
  float mm = 0.0f, f0 = 0.0f, f1 = 0.0f;
  for (int s0 = w; s0 < a.splits; s0 += 8 * NWV) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (s0 + j * NWV < a.splits) t[j] = reinterpret_cast<const float4 *>(a.part + ((int64_t)(s0 + j * NWV) * rows + r) * kHd)[lane];
    if (s0 == w) {
      mm = wave_max(fmaxf(m0.x, m1.x));
      f0 = m0.x == -INFINITY ? 0.0f : exp2f(m0.x - mm);
      f1 = m1.x == -INFINITY ? 0.0f : exp2f(m1.x - mm);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int s = s0 + j * NWV;
      if (s >= a.splits) break;
      const float f = __shfl(s < 64 ? f0 : f1, s & 63);
      o.x = fmaf(t[j].x, f, o.x); o.y = fmaf(t[j].y, f, o.y); o.z = fmaf(t[j].z, f, o.z); o.w = fmaf(t[j].w, f, o.w);
    }
  }
  if (w >= a.splits) {                             // (a wave without ranges: the row's sum all the same)
    mm = wave_max(fmaxf(m0.x, m1.x));
    f0 = m0.x == -INFINITY ? 0.0f : exp2f(m0.x - mm);
    f1 = m1.x == -INFINITY ? 0.0f : exp2f(m1.x - mm);
  }
  const float l0 = fabsf(m0.y) * f0, l1 = fabsf(m1.y) * f1;   // (the sign: see marked_sum)
  float l = wave_sum(l0 + l1);
  reinterpret_cast<float4 *>(s_o + w * kHd)[lane] = o;
  __syncthreads();
  o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int j = 0; j < NWV; ++j) {
    const float4 x = reinterpret_cast<const float4 *>(s_o + j * kHd)[lane];
    o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
  }
  __syncthreads();
  // (every wave holds the whole row: the decision is the workgroup's)
  const float big = fmaxf(fmaxf(fabsf(o.x), fabsf(o.y)), fmaxf(fabsf(o.z), fabsf(o.w)));
  bool fine = l > 0.0f && l < INFINITY && !__any(!(big < INFINITY) || o.x != o.x || o.y != o.y || o.z != o.z || o.w != o.w);
  // Rows whose outputs are all small are formed again: what is left subnormal of V (below), and of p 2^-34 whatever its
  // size, is cut; beside a step of level 2, whose V are large, sooner.
  if (fine) {
    const float top = wave_max(big);
    const bool high = __any((m0.y < 0.0f && f0 > 0.0f) || (m1.y < 0.0f && f1 > 0.0f));
    fine = top == 0.0f ? !high : top >= l * (high ? 0x1p-9f : 0x1p-17f);
  }
  bool empty = false;
  if (!fine) {
    empty = !tree_sees(a, i);
    if (!empty) tree_careful_row<KF, VF, NWV>(a, i, h, s_o, s_ml, o, l);
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

// where the i-th key range begins, in steps (the host has divided: a division here is 200 cycles before the first load)
__device__ __forceinline__ int range_begin(const TreeArgs &a, int i) { return __builtin_amdgcn_readfirstlane(i * a.share + min(i, a.spare)); }

// Which KV head, key range and row block a workgroup takes. Workgroups 8 apart run on the same XCD, whose L2 reads a
// range once for its row blocks: range u of all KV heads' goes to XCD u % 8 with every row block, and the row blocks of
// the last nkv * splits % 8 ranges are shared out evenly. (Those by whole ranges as well: 3 row blocks of 84 ranges put 33
// workgroups on 4 XCDs' 32 CUs, 66 us in place of 33. Every XCD a run of neighbouring ranges instead: 131072 keys took
// 52 us in place of 48.)
__device__ __forceinline__ bool tree_place(const TreeArgs &a, int &hk, int &split, int &rb) {
  const int xcd = (int)(blockIdx.x & 7);
  int at = (int)(blockIdx.x >> 3), unit;
  const bool whole = at < a.whole;
  if (!whole) {
    at = xcd * a.share_out + at - a.whole;
    if (at >= a.left) return false;
  }
  unit = a.nrb == 1 ? at : at / a.nrb;
  rb = at - unit * a.nrb;
  unit = whole ? 8 * unit + xcd : a.nkv * a.splits / 8 * 8 + unit;
  hk = unit / a.splits;
  split = unit - hk * a.splits;
  return true;
}

// The rows r, r + 1, .. of a KV head as (token, query head of the group), r < rows
struct RowWalk {
  int tok, h;
  __device__ __forceinline__ RowWalk(int r, int grp) : tok(r / grp), h(r - tok * grp) {}
  __device__ __forceinline__ void next(int grp) {
    if (++h == grp) { h = 0; ++tok; }
  }
};

// 8 probabilities as ph + pl: ph cut to fp16 (two in one instruction), pl the rest, rounded (one instruction each)
__device__ __forceinline__ void split_p(const float (&p)[8], h8 &ph, h8 &pl) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const auto c = __builtin_amdgcn_cvt_pkrtz(p[j], p[j + 1]);
    ph[j] = (_Float16)c[0];
    ph[j + 1] = (_Float16)c[1];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) pl[j] = (_Float16)__builtin_fmaf((float)ph[j], -1.0f, p[j]);
}

// q8_0 scales are taken times 2^9, so that vl of the smallest is no subnormal product; a step with one above 2^-1 takes
// all of its times 2^1, with one above 2^7 times 2^-7 (its level: 0, 1, 2), which keeps vh within fp16, and the outputs
// are brought to the step's unit. vh and vl hold d * b exactly where the scaled d is exact: always at levels 0 and 1,
// at level 2 from d = 2^-7 on. Smaller ones beside such large ones (16256 beside 1, in 32 neighbouring keys) leave NaN
// in place of the range's sum, so that its rows are computed key by key.
// fp16 V is taken as it is, but for steps in which a lane's 8 keys have nothing but subnormals (and zeros) in some dim:
// those are taken times 2^10 (level 1). The matrix cores align the products of a sum by their exponents, a subnormal's
// taken as 2^-14, and lose what is 2^-22 below the largest: dims of 1e-7 beside ordinary ones came out 1e-4 off. Looking
// for these dims takes 0 to 2 % of the kernels' time; all steps times 2^10 if their values allow it took 2 to 14 %.
// What is left subnormal loses up to 2^-36 of the largest weight: fp16 V beside a larger value in its own dim and 8 keys,
// or beside values of 64 or more, which the factor would take past fp16; q8_0 V of scales below 2^-15 beside ones above
// 1/2 (level 1).
// the level of the largest of fp16 scales (bits, sign cleared): above 2^-1, above 2^7
__device__ __forceinline__ int scale_level(uint32_t top) { return (top > 0x3800u) + (top > 0x5800u); }
// whether a step of level 2 loses bits of one of the scales
__device__ __forceinline__ bool scale_lost(const uint32_t (&sc)[8]) {
  bool lost = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) lost |= ((sc[j] & 0x7FFFu) - 1u) < 0x1FFFu;
  return __any(lost);
}
constexpr int kLostBits = 4;                       // (beside the level)
// V's operands are V * 2^(unit - step * level)
constexpr int v_unit(int vf) { return vf ? 9 : 0; }
constexpr int v_step(int vf) { return vf ? 8 : -10; }
// the level of fp16 V of 8 keys and 2 W dims per lane
template <int W>
__device__ __forceinline__ int f16_level(const uint32_t (&r)[8][W]) {
  typedef uint16_t u2 __attribute__((ext_vector_type(2)));
  // (3 of the keys first: a dim whose or-ed exponent is not 0 has a value that is not subnormal)
  uint32_t x[W];
  u2 least = {0xFFFF, 0xFFFF};
#pragma unroll
  for (int c = 0; c < W; ++c) {
    x[c] = (r[0][c] | r[1][c] | r[2][c]) & 0x7FFF7FFFu;
    least = __builtin_elementwise_min(least, __builtin_bit_cast(u2, x[c]));
  }
  if (__builtin_expect(!__any(least[0] < 0x400 || least[1] < 0x400), 1)) return 0;
  bool some = false;                               // (dims of zeros need nothing)
#pragma unroll
  for (int c = 0; c < W; ++c) {
#pragma unroll
    for (int j = 3; j < 8; ++j) x[c] |= r[j][c];
    some |= (x[c] & 0x7FFFu) - 1u < 0x3FFu || (x[c] >> 16 & 0x7FFFu) - 1u < 0x3FFu;
  }
  if (!__any(some)) return 0;
  float sq = 0.0f;                                 // (64^2 or more, or NaN, where a value is 64 or more)
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int c = 0; c < W; ++c) sq = __builtin_amdgcn_fdot2(as_h2(r[j][c]), as_h2(r[j][c]), sq, false);
  return __any(!(sq < 4096.0f)) ? 0 : 1;
}
template <int W>
__device__ __forceinline__ void f16_lift(uint32_t (&r)[8][W]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int c = 0; c < W; ++c) r[j][c] = as_u(as_h2(r[j][c]) * h2{(_Float16)0x1p10f, (_Float16)0x1p10f});
}
// a range's sum of p as it is left for the join: below zero where a step of q8_0 V had level 2
__device__ __forceinline__ float marked_sum(float l, uint32_t levels) {
  return levels & kLostBits ? __builtin_nanf("") : levels & 2 ? -l : l;
}

// fp16 pair: the SEL-th byte of lo in the low half and of hi in the high one
template <int SEL>
__device__ __forceinline__ uint32_t pair_bytes(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x0C000C00u | (uint32_t)SEL | ((uint32_t)(SEL + 4) << 16));
}

// ------------------------------------------------------------------ few rows: every wave a key range of its own
// A workgroup holds 16 rows; each of its 4 waves streams a key range, 32 keys a step, without barriers until the
// ranges are joined. A step's K is asked for as soon as the last one's has been read, its V likewise, so that a wave has
// nearly a whole step (17 KB in q8_0) on its way into its own part of LDS at all times. Bound by the memory over long
// contexts (4 rows of q8_0: 131072 keys 49 us, 5.8 TB/s; 32768 17.5 us, 4.1) and by latencies over short ones (600
// keys: 7 us with 4 rows, 8.2 with 28, most of it the first step's). Loads into registers took 27.9 us where this took
// 17.8; 8 waves a workgroup, for half the ranges to join, 18.9 (53 against 48 at 131072 keys); 32 rows a workgroup, which
// read the cache once, 31.4 where two blocks of 16 take 28.4 and the second reads L2.
//
// Scores are computed transposed, S^T = K Q^T: lane (n, g) = (lane % 16, lane / 16) then holds keys 4 g .. 4 g + 3 of
// a 16-key tile for row n, which is P^T's operand of O^T = V^T P^T as it stands if slot (g, j) of the 32-key
// contraction stands for key 4 g + j (j < 4) or 16 + 4 g + j - 4, for both operands. V's operand wants one dim of 8
// keys per lane: lane (m, g) reads its 8 keys' bytes of dims 16 m .. 16 m + 15, and product dt takes byte dt of each,
// so that row m of product dt is dim 16 m + dt (fp16 V: 8 dims per read, dim 128 (dt / 8) + 8 m + dt % 8).
// LDS: V rows as they are; 16-byte piece c of K's row k at place c ^ k % 16, so that 16 rows' pieces lie in 16 banks'
// widths (the lanes of the load ask for the pieces in that order).
template <int VF>
__device__ __forceinline__ int tree_dim(int dt, int m) {
  return VF == BKV_Q8_0 ? 16 * m + dt : 128 * (dt >> 3) + 8 * m + (dt & 7);
}

// PG, here and below: 0 a contiguous cache; 1 pages of whole steps (a multiple of 32 tokens: a step's keys are neighbours,
// at one base for the whole workgroup); 2 any pages (a slot of its own for every key)
template <int KF, int VF, int PG>
__global__ __launch_bounds__(256, KF == BKV_Q8_0 && VF == BKV_Q8_0 ? 2 : 1) void tree_stream_kernel(TreeArgs a) {
  constexpr int KRB = row_bytes(KF), VRB = row_bytes(VF), RB = 16;
  constexpr uint32_t oV = kTreeKeys * KRB, oSK = oV + kTreeKeys * VRB, oSV = oSK + (KF ? 512 : 0), kWave = oSV + (VF ? 512 : 0);
  constexpr int kOS = kHd + 4;                     // a row of the join
  constexpr uint32_t kJoin = 4 * RB * kOS * 4;
  __shared__ __attribute__((aligned(128))) uint8_t sm[4 * kWave > kJoin ? 4 * kWave : kJoin];
  __shared__ float s_m[4][RB], s_l[4][RB];
  __shared__ uint32_t s_lv[4];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  int hk, split, rb;
  if (!tree_place(a, hk, split, rb)) return;
  const int R = a.n_q * a.grp;
  const uint32_t nk = a.pos0 + (uint32_t)a.n_q;
  const int t0 = range_begin(a, split * 4 + w), t1 = range_begin(a, split * 4 + w + 1);
  const uint32_t krow = (uint32_t)a.nkv * KRB, vrow = (uint32_t)a.nkv * VRB, srow = (uint32_t)a.nkv * kScaleRowBytes;
  const uint8_t *kd = a.L.kd + (size_t)hk * KRB, *vd = a.L.vd + (size_t)hk * VRB;
  const uint8_t *ksc = KF ? a.L.ks + (size_t)hk * kScaleRowBytes : nullptr, *vsc = VF ? a.L.vs + (size_t)hk * kScaleRowBytes : nullptr;
  uint8_t *const my = sm + kWave * w;
  const uint32_t my0 = lds_addr(sm) + kWave * w;

  // ---- a step's bytes on their way
  uint32_t there = ~0u, there_next = ~0u;          // keys whose pages are in the pool: this step's, the next's
  int sl = 0;                                      // PG 2: the slot of key lane % 32 of the step asked for
  size_t s0 = 0;
  auto look_up = [&](int t) {
    const uint32_t kb = (uint32_t)t * kTreeKeys;
    s0 = kb;
    if constexpr (PG == 1) {
      const int first = __builtin_amdgcn_readfirstlane(slot_checked(a.L, a.pool_pages, kb));
      there_next = first >= 0 ? ~0u : 0u;
      s0 = (size_t)max(first, 0);
    }
    if constexpr (PG == 2) {
      sl = slot_checked(a.L, a.pool_pages, min(kb + ((uint32_t)lane & 31), nk - 1));
      there_next = (uint32_t)__ballot(sl >= 0);
    }
  };
  // (offsets within a step are 32 bits: 31 rows)
  auto take = [&](int t, const uint8_t *base, int key, uint32_t row, uint32_t col, uint32_t dst) {
    if constexpr (PG == 2) load_to_lds(base + (size_t)max(__shfl(sl, key), 0) * row + col, __builtin_amdgcn_readfirstlane(dst));
    else load_to_lds(base + s0 * row, min((uint32_t)key, nk - 1 - (uint32_t)t * kTreeKeys) * row + col, __builtin_amdgcn_readfirstlane(dst));
  };
  constexpr int NK = KF ? 9 : 16, NV = VF ? 9 : 16;   // loads of a step's K, of its V
  auto scales = [&](int t, const uint8_t *base, uint32_t dst) {
    const uint32_t key = (uint32_t)lane & 31;
    const uint8_t *src = PG == 2 ? base + (size_t)max(__shfl(sl, (int)key), 0) * srow : base + s0 * srow + min(key, nk - 1 - (uint32_t)t * kTreeKeys) * srow;
    if (lane < 32) load_to_lds(src, __builtin_amdgcn_readfirstlane(dst));
  };
  auto request_k = [&](int t) {
    constexpr int LR = KF ? 16 : 32;               // lanes of a row
#pragma unroll
    for (int u = 0; u < 32 * LR / 64; ++u) {
      const int key = (64 / LR) * u + lane / LR;
      take(t, kd, key, krow, 16 * ((lane % LR) ^ (key & 15)), my0 + 1024 * u);
    }
    if constexpr (KF) scales(t, ksc, my0 + oSK);
  };
  auto request_v = [&](int t) {
    constexpr int LR = VF ? 16 : 32;
#pragma unroll
    for (int u = 0; u < 32 * LR / 64; ++u) take(t, vd, (64 / LR) * u + lane / LR, vrow, 16 * (lane % LR), my0 + oV + 1024 * u);
    if constexpr (VF) scales(t, vsc, my0 + oSV);
  };
  // the workgroup's rows of Q first, 4 of them by each wave into the place of its V (piece c of row r at c ^ r % 16),
  // then K; V once the rows have been read
  {
    RowWalk at(min(RB * rb + 4 * w, R - 1), a.grp);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = 4 * w + j;
      load_to_lds(reinterpret_cast<const uint8_t *>(a.q.at(at.tok, hk * a.grp + at.h)) + 16 * (lane ^ (row & 15)), __builtin_amdgcn_readfirstlane(my0 + oV + 1024 * j));
      if (RB * rb + row + 1 < R) at.next(a.grp);
    }
  }
  if (t0 < t1) {
    look_up(t0);
    request_k(t0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK) : "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  lds_barrier();

  const int tok = min(RB * rb + n, R - 1) / a.grp;
  h8 qh[8];                                        // row n, dims 32 b + 8 g ..
  const uint8_t *q = sm + kWave * (n / 4) + oV + 1024 * (n % 4);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const float4 x = *reinterpret_cast<const float4 *>(q + 16 * ((8 * b + 2 * g) ^ n)), y = *reinterpret_cast<const float4 *>(q + 16 * ((8 * b + 2 * g + 1) ^ n));
    qh[b] = h8{(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w, (_Float16)y.x, (_Float16)y.y, (_Float16)y.z, (_Float16)y.w};
  }
  lds_barrier();
  if (t0 < t1) request_v(t0);
  f4 o[16] = {};
  float m = -INFINITY, l = 0.0f;                   // m: the reference less kPScale
  int lv = 0;                                      // the outputs' level
  uint32_t lv_any = 0;                             // all that were taken, or-ed

#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
    const int64_t kb = (int64_t)t * kTreeKeys;
    there = there_next;
    // which keys the rows see: lane (n, g)'s bit i is key 4 g + i, bit 16 + i key 16 + 4 g + i
    const bool whole = kb + kTreeKeys <= a.pos0 && (!PG || there == ~0u);
    const uint32_t win = (whole ? ~0u : kb + kTreeKeys > a.pos0 ? there & tree_window(a, tok, kb) : there) >> (4 * g);
    // ---- scores
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NV) : "memory");   // (this step's V may still be on its way)
    f4 s[2] = {};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (KF) {
        uint4 sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[i] = *reinterpret_cast<const uint4 *>(my + oSK + 16 * (16 * u + 4 * g + i));
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const uint2 r = *reinterpret_cast<const uint2 *>(my + KRB * (16 * u + n) + 16 * ((2 * b + (g >> 1)) ^ n) + 8 * (g & 1));
          const uint32_t x = r.x ^ 0x80808080u, y = r.y ^ 0x80808080u;
          const uint4 kv = make_uint4(as_u(bytes_h2<0x04010400u>(x)), as_u(bytes_h2<0x04030402u>(x)), as_u(bytes_h2<0x04010400u>(y)), as_u(bytes_h2<0x04030402u>(y)));
          const f4 z = mfma16(__builtin_bit_cast(h8, kv), qh[b], f4{});
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[u][i] = __builtin_fmaf(z[i], (float)__builtin_bit_cast(_Float16, (uint16_t)((&sc[i].x)[b >> 1] >> (16 * (b & 1)))), s[u][i]);
        }
      } else {
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const h8 kf = *reinterpret_cast<const h8 *>(my + KRB * (16 * u + n) + 16 * ((4 * b + g) ^ n));
          s[u] = mfma16(kf, qh[b], s[u]);
        }
      }
    }
    asm volatile("" : "+v"(s[0]), "+v"(s[1]));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + 1 < t1) {
      look_up(t + 1);
      request_k(t + 1);
    }
    // ---- probabilities
    h8 ph, pl;
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!((win >> ((j & 4) * 4 + (j & 3))) & 1u)) s[j >> 2][j & 3] = -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                      fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))) * a.scale2;
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
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], a.scale2, -m));
    if (!whole) {                                  // (where nothing was seen yet, -Inf - -Inf)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!((win >> ((j & 4) * 4 + (j & 3))) & 1u)) p[j] = 0.0f;
    }
    l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    split_p(p, ph, pl);
    // ---- P V
    if (t + 1 < t1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK) : "memory");   // (the next step's K may still be on its way)
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint8_t *vp = my + oV + 16 * n;
    auto key_of = [&](int j) { return (j & 4) * 4 + 4 * g + (j & 3); };
    if constexpr (VF) {
      uint32_t sc[8], top = 0;
      uint4 r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sc[j] = *reinterpret_cast<const uint16_t *>(my + oSV + 16 * key_of(j) + 2 * (n >> 1));
        r[j] = *reinterpret_cast<const uint4 *>(vp + VRB * key_of(j));
        top = max(top, sc[j] & 0x7FFFu);
      }
      const int level = __any(scale_level(top) != 0) ? (__any(scale_level(top) == 2) ? 2 : 1) : 0;
      const _Float16 f = level == 0 ? (_Float16)0x1p9f : level == 1 ? (_Float16)0x1p1f : (_Float16)0x1p-7f;
      if (level == 2) lv_any |= 2u | (scale_lost(sc) ? kLostBits : 0);
      if (level != lv) {
        const float x = __builtin_ldexpf(1.0f, 8 * (lv - level));
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) o[dt] *= x;
        lv = level;
      }
      h2 d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = as_h2(sc[2 * j] | (sc[2 * j + 1] << 16)) * h2{f, f};
#pragma unroll
      for (int dt = 0; dt < 16; ++dt) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lo = (&r[2 * j].x)[dt >> 2], hi = (&r[2 * j + 1].x)[dt >> 2];
          const uint32_t pb = (dt & 3) == 0 ? pair_bytes<0>(lo, hi) : (dt & 3) == 1 ? pair_bytes<1>(lo, hi) : (dt & 3) == 2 ? pair_bytes<2>(lo, hi) : pair_bytes<3>(lo, hi);
          h2 h, lw;
          split_prod(as_h2(pb ^ 0x64806480u) - h2{(_Float16)1152.0f, (_Float16)1152.0f}, d[j], h, lw);
          ah[j] = as_u(h);
          al[j] = as_u(lw);
        }
        const h8 vh = __builtin_bit_cast(h8, make_uint4(ah[0], ah[1], ah[2], ah[3]));
        const h8 vl = __builtin_bit_cast(h8, make_uint4(al[0], al[1], al[2], al[3]));
        o[dt] = mfma16(vl, ph, o[dt]);
        o[dt] = mfma16(vh, pl, o[dt]);
        o[dt] = mfma16(vh, ph, o[dt]);
      }
    } else {
      uint32_t r[8][8];                            // dims 8 n .. and 128 + 8 n ..
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint4 x = *reinterpret_cast<const uint4 *>(vp + VRB * key_of(j & 7) + 256 * (j >> 3));
#pragma unroll
        for (int c = 0; c < 4; ++c) r[j & 7][4 * (j >> 3) + c] = (&x.x)[c];
      }
      const int level = f16_level(r);
      if (__builtin_expect(level | lv, 0)) {
        const float x = __builtin_ldexpf(1.0f, v_step(VF) * (lv - level));
        // (the outputs are accumulation registers; without the asm they are read ahead of the branch, 64 instructions a
        // step: 25 tokens onto 8192 q8_0 K 27.1 us in place of 25.9)
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) {
          asm volatile("" : "+a"(o[dt]));
          o[dt] *= x;
          asm volatile("" : "+a"(o[dt]));
        }
        lv = level;
        if (lv) f16_lift(r);
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint32_t av[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            av[j] = __builtin_amdgcn_perm(r[2 * j + 1][4 * hf + (e >> 1)], r[2 * j][4 * hf + (e >> 1)], e & 1 ? 0x07060302u : 0x05040100u);
          const h8 vh = __builtin_bit_cast(h8, make_uint4(av[0], av[1], av[2], av[3]));
          o[8 * hf + e] = mfma16(vh, pl, o[8 * hf + e]);
          o[8 * hf + e] = mfma16(vh, ph, o[8 * hf + e]);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + 1 < t1) request_v(t + 1);
  }

  // ---- the 4 ranges joined, one partial result per row and workgroup
  float *s_o = reinterpret_cast<float *>(sm);
  const int64_t rows = (int64_t)a.n_q * a.nh;
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) { s_m[w][n] = m; s_l[w][n] = l; }
  if (lane == 0) s_lv[w] = lv_any;
  __syncthreads();                                 // (and the waves' own parts have been read)
  const float mm = fmaxf(fmaxf(s_m[0][n], s_m[1][n]), fmaxf(s_m[2][n], s_m[3][n]));
  const float f = m == -INFINITY ? 0.0f : exp2f(m - mm), fo = __builtin_ldexpf(f, v_step(VF) * lv - v_unit(VF));
#pragma unroll
  for (int dt = 0; dt < 16; dt += 4)               // (4 products' dims are neighbours)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<float4 *>(&s_o[(RB * w + n) * kOS + tree_dim<VF>(dt, 4 * g + i)]) =
          make_float4(o[dt][i] * fo, o[dt + 1][i] * fo, o[dt + 2][i] * fo, o[dt + 3][i] * fo);
  __syncthreads();
  const int row = threadIdx.x >> 4, c = threadIdx.x & 15, r = RB * rb + row;
  if (r < R) {
    const int ti = r / a.grp;
    const int64_t at = (int64_t)split * rows + (int64_t)ti * a.nh + hk * a.grp + r - ti * a.grp;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 x = *reinterpret_cast<const float4 *>(&s_o[(RB * j + row) * kOS + 4 * c + 64 * k]);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
      }
      *reinterpret_cast<float4 *>(a.part + at * kHd + 4 * c + 64 * k) = v;
    }
    if (c == 0) {
      const float mr = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
      float lr = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) lr += s_m[j][row] == -INFINITY ? s_l[j][row] : s_l[j][row] * exp2f(s_m[j][row] - mr);
      a.ml[at] = make_float2(mr, marked_sum(lr, s_lv[0] | s_lv[1] | s_lv[2] | s_lv[3]));
    }
  }
}

// ------------------------------------------------------------------ many rows: key tiles in LDS
// 8 waves hold 16 MT rows each with all 256 outputs in registers, and step through the workgroup's key range 32 keys at
// a time. A step's cache bytes are loaded straight into LDS while the step before it is computed, and turned once into
// the products' operands for all of the workgroup's rows: K's bytes into fp16 (fp16 K needs nothing: its pieces land
// where they are wanted), V transposed, so that a lane's 8 keys of one dim are 16 bytes, as vh (and vl for q8_0). S^T and
// O^T are formed as in the kernel above, so P never leaves its lane. Two waves share a SIMD, and the second one's P V
// runs a step late, beside the first one's scores: hence two steps' operands of K and three of V. With 128 rows the
// registers leave room for 4 more waves, which bring and turn the bytes.
//
// Bound by what two waves a SIMD can overlap: of a step's 7500 cycles (256 rows, q8_0) the matrix cores work 4096, the
// vector unit (softmax, the scales of K's blocks, the operands) 4200, LDS about as many. q8_0 takes 4 products and fp16
// 3 where the formula has 2. 1024 rows onto 32768 keys: 81 us (34 GFLOP, 0.42 PFLOP/s), 8192 onto 8192 164 us (71
// GFLOP, 0.43), 1008 onto 65536 in fp16 112 us (68 GFLOP, 0.60). Of 81 us 25 are the rows' first bytes and the partial
// results (67 MB written).
//
// LDS positions, in 16-byte pieces: K piece c of key k at 32 k + (c ^ k % 16); V piece g of dim d (keys 4 g .. 4 g + 3
// and 16 + 4 g .. 16 + 4 g + 3) at 8 (d / 2) + ((4 (d % 2) + g) ^ kx(d)), kx chosen so that both the 8 dims next to
// one another that a read takes and the 8 dims 4 apart that a write takes lie in different banks.
//
__device__ __forceinline__ uint32_t v_piece(int d, int g) {
  const int kx = ((d >> 4) & 1) << 2 | ((d >> 2) & 1) << 1 | (((d >> 1) ^ (d >> 3)) & 1);
  return (uint32_t)(128 * (d >> 1) + 16 * ((4 * (d & 1) + g) ^ kx));
}

// 8 waves with rows, and 4 more where the registers allow them
constexpr int tree_tile_threads(int mt) { return mt == 1 ? 768 : 512; }

template <int KF, int VF, int PG, int MT>
__global__ __launch_bounds__(tree_tile_threads(MT), MT == 1 ? 3 : 2) void tree_tile_kernel(TreeArgs a) {
  constexpr int NW = 8, KRB = row_bytes(KF), VRB = row_bytes(VF), RB = 16 * MT * NW;
  constexpr uint32_t kOp = kTreeKeys * 2 * kHd;    // an operand: 32 keys of 256 fp16
  // three steps' V operands (vh, vl, their levels) and two steps' of K (with its scales); behind them the bytes as
  // they came, a wave's own
  constexpr uint32_t kVB = kOp * (VF ? 2 : 1) + 128, kKB = kOp + (KF ? 512 : 0), oLV = kVB - 128;
  constexpr uint32_t oK = 3 * kVB, oRV = oK + 2 * kKB, oRK = oRV + kTreeKeys * VRB, oSV = oRK + (KF ? kTreeKeys * KRB : 0), oSK = oSV + (VF ? 512 : 0);
  __shared__ __attribute__((aligned(128))) uint8_t sm[oSK + (KF ? 512 : 0)];
  const uint32_t sm0 = lds_addr(sm);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  int hk, split, rb;
  if (!tree_place(a, hk, split, rb)) return;
  const int R = a.n_q * a.grp;
  const uint32_t nk = a.pos0 + (uint32_t)a.n_q;
  const int t0 = range_begin(a, split), t1 = range_begin(a, split + 1);

  // (the lane's number, opaque where addresses are formed from it: kept from step to step they would take the
  // registers that the outputs need)
  auto my_lane = [&]() {
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  const uint32_t krow = (uint32_t)a.nkv * KRB, vrow = (uint32_t)a.nkv * VRB, srow = (uint32_t)a.nkv * kScaleRowBytes;
  const uint8_t *kd = a.L.kd + (size_t)hk * KRB, *vd = a.L.vd + (size_t)hk * VRB;
  const uint8_t *ksc = KF ? a.L.ks + (size_t)hk * kScaleRowBytes : nullptr, *vsc = VF ? a.L.vs + (size_t)hk * kScaleRowBytes : nullptr;

  // ---- a step's bytes on their way, and later into operands: 4 waves V (64 dims each), 4 waves K (8 keys each). A wave
  // brings what it will make into operands itself, so it waits for its own loads only. With 256 rows waves 0 .. 3 take
  // V and waves 4 .. 7 K beside their rows; with 128 the registers leave room for 4 more waves, which take both and have
  // no rows.
  const int wk = w & 3;
  const bool does_v = MT == 1 ? w >= NW : w < 4, does_k = MT == 1 ? w >= NW : w >= 4;
  uint32_t there = ~0u, there_next = ~0u, there_after = ~0u;   // keys whose pages are in the pool: this step's, the next's, ..
  int sl = 0;                                      // PG 2: the slot of the key lane % 32 of the step asked for next
  auto look_up = [&](int t) {
    if constexpr (PG == 2) sl = slot_checked(a.L, a.pool_pages, min((uint32_t)t * kTreeKeys + ((uint32_t)lane & 31), nk - 1));
  };
  auto request = [&](int t, int buf) {
    const int lane = my_lane();
    const uint32_t kb = (uint32_t)t * kTreeKeys, last = min(nk - 1 - kb, (uint32_t)kTreeKeys - 1);
    size_t s0 = kb;
    if constexpr (PG == 1) {
      const int first = __builtin_amdgcn_readfirstlane(slot_checked(a.L, a.pool_pages, kb));
      there_after = first >= 0 ? ~0u : 0u;
      s0 = (size_t)max(first, 0);
    }
    if constexpr (PG == 2) there_after = (uint32_t)__ballot(sl >= 0);
    // (offsets within a step are 32 bits: 31 rows)
    auto take = [&](const uint8_t *base, int key, uint32_t row, uint32_t col, uint32_t dst) {
      if constexpr (PG == 2) load_to_lds(base + (size_t)max(__shfl(sl, key), 0) * row + col, __builtin_amdgcn_readfirstlane(dst));
      else load_to_lds(base + s0 * row, min((uint32_t)key, last) * row + col, __builtin_amdgcn_readfirstlane(dst));
    };
    if (does_v) {
      // [place][64 dims], 4 or 8 lanes of 16 bytes per key; place 4 j + g is key slot (g, j) of the contraction, so that
      // the 4 groups' reads of one j are neighbours
      constexpr int LR = VF ? 4 : 8;
      auto key_of = [](int p) { return (p & 16) + 4 * (p & 3) + ((p >> 2) & 3); };
#pragma unroll
      for (int u = 0; u < (VF ? 2 : 4); ++u)
        take(vd, key_of((64 / LR) * u + lane / LR), vrow, 16 * (LR * wk + lane % LR), sm0 + oRV + 32 * 16 * LR * wk + 1024 * u);
      if constexpr (VF) {                          // its two blocks' scales: 4 bytes of each key's row
        const int key = key_of(lane & 31);
        const uint8_t *src = PG == 2 ? vsc + (size_t)max(__shfl(sl, key), 0) * srow : vsc + s0 * srow + min((uint32_t)key, last) * srow;
        if (lane < 32) load4_to_lds(src + 4 * wk, __builtin_amdgcn_readfirstlane(sm0 + oSV + 128 * wk));
      }
    }
    if (does_k) {
      constexpr int LR = KF ? 16 : 32;             // lanes of a row
#pragma unroll
      for (int u = 0; u < (KF ? 2 : 4); ++u) {
        const int first = 8 * wk + (64 / LR) * u, key = first + lane / LR, c = lane % LR;
        if constexpr (KF) take(kd, key, krow, 16 * c, sm0 + oRK + KRB * first);
        else take(kd, key, krow, 16 * (c ^ (key & 15)), sm0 + oK + kKB * buf + KRB * first);
      }
      if constexpr (KF) {                          // (the shuffle with every lane there, the load with 8)
        const int key = (8 * wk + lane) & 31;
        const uint8_t *src = PG == 2 ? ksc + (size_t)max(__shfl(sl, key), 0) * srow : ksc + s0 * srow + min((uint32_t)key, last) * srow;
        if (lane < 8) load_to_lds(src, __builtin_amdgcn_readfirstlane(sm0 + oSK + 128 * wk));
      }
    }
  };

  if (t0 < t1) {
    look_up(t0);
    request(t0, 1);
    there = there_after;
  }
  const bool has_rows = w < NW;
  h8 qh[MT][8];
  auto token_of = [&](int mt) { return min(RB * rb + 16 * MT * w + 16 * mt + (my_lane() & 15), R - 1) / a.grp; };
  // the rows of Q, whole rows at a time (a row's pieces lane by lane would ask for each line four times), to fp16 and
  // through LDS, 8 KB of the operands' place per wave, to the lanes that want them; pieces as K's
  static_assert(oRV >= 8 * 8192 && (KF || oK + kKB >= 8 * 8192), "the rows end before the bytes that are on their way");
  RowWalk at(min(RB * rb + 16 * MT * w, R - 1), a.grp);   // (the same in all lanes)
  if (has_rows)
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float4 x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      x[j] = reinterpret_cast<const float4 *>(a.q.at(at.tok, hk * a.grp + at.h))[lane];
      if (RB * rb + 16 * (MT * w + mt) + j + 1 < R) at.next(a.grp);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const h2 lo = {(_Float16)x[j].x, (_Float16)x[j].y}, hi = {(_Float16)x[j].z, (_Float16)x[j].w};
      *reinterpret_cast<uint2 *>(sm + 8192 * w + 512 * j + 16 * ((lane >> 1) ^ j) + 8 * (lane & 1)) = make_uint2(as_u(lo), as_u(hi));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int b = 0; b < 8; ++b) qh[mt][b] = *reinterpret_cast<const h8 *>(sm + 8192 * w + 512 * n + 16 * ((4 * b + g) ^ n));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  f4 o[MT][16] = {};
  float m[MT], l[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) { m[mt] = -INFINITY; l[mt] = 0.0f; }
  uint32_t lv = 0, lv_any = 0;                     // the outputs' levels, a byte per 64 dims; all that were taken, or-ed

  // ---- the wave's bytes, landed, made into operands
  uint32_t levels = 0;                             // fp16 V: those of the wave's 64 dims, the last step's first
  auto convert = [&](uint8_t *kto, uint8_t *vto) {
    const int lane = my_lane(), n = lane & 15, g = lane >> 4;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (does_k) {
      if constexpr (KF) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int key = 8 * wk + 4 * u + g;
#pragma unroll
          for (int e = 0; e < 2; ++e) {            // pieces n and 16 + n: 16 lanes write 16 banks' worth
            const uint2 r = *reinterpret_cast<const uint2 *>(sm + oRK + KRB * key + 8 * n + 128 * e);
            const uint32_t x = r.x ^ 0x80808080u, y = r.y ^ 0x80808080u;
            *reinterpret_cast<uint4 *>(kto + 512 * key + 16 * ((n ^ (key & 15)) + 16 * e)) =
                make_uint4(as_u(bytes_h2<0x04010400u>(x)), as_u(bytes_h2<0x04030402u>(x)), as_u(bytes_h2<0x04010400u>(y)), as_u(bytes_h2<0x04030402u>(y)));
          }
        }
        const int key = 8 * wk + (lane >> 3);      // scales: [key / 4][block][key % 4]
        reinterpret_cast<uint16_t *>(kto + kOp)[32 * (key >> 2) + 4 * (lane & 7) + (key & 3)] =
            reinterpret_cast<const uint16_t *>(sm + oSK)[64 * wk + lane];
      }
    }
    if (!does_v) return;
    if constexpr (VF) {
      uint32_t r[8], sc[8], top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[j] = *reinterpret_cast<const uint32_t *>(sm + oRV + 2048 * wk + 64 * (4 * j + g) + 4 * n);
        sc[j] = *reinterpret_cast<const uint16_t *>(sm + oSV + 128 * wk + 4 * (4 * j + g) + 2 * (n >> 3));
        top = max(top, sc[j] & 0x7FFFu);
      }
      const int level = __any(scale_level(top) != 0) ? (__any(scale_level(top) == 2) ? 2 : 1) : 0;
      const _Float16 f = level == 0 ? (_Float16)0x1p9f : level == 1 ? (_Float16)0x1p1f : (_Float16)0x1p-7f;
      const int lost = level == 2 && scale_lost(sc) ? kLostBits : 0;
      if (lane == 0) vto[oLV + wk] = (uint8_t)(level | lost);
      h2 d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = as_h2(sc[2 * j] | (sc[2 * j + 1] << 16)) * h2{f, f};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lo = r[2 * j], hi = r[2 * j + 1];
          const uint32_t pb = e == 0 ? pair_bytes<0>(lo, hi) : e == 1 ? pair_bytes<1>(lo, hi) : e == 2 ? pair_bytes<2>(lo, hi) : pair_bytes<3>(lo, hi);
          h2 h, lw;
          split_prod(as_h2(pb ^ 0x64806480u) - h2{(_Float16)1152.0f, (_Float16)1152.0f}, d[j], h, lw);
          ah[j] = as_u(h);
          al[j] = as_u(lw);
        }
        const uint32_t at = v_piece(64 * wk + 4 * n + e, g);
        *reinterpret_cast<uint4 *>(vto + at) = make_uint4(ah[0], ah[1], ah[2], ah[3]);
        *reinterpret_cast<uint4 *>(vto + (VF ? kOp : 0u) + at) = make_uint4(al[0], al[1], al[2], al[3]);
      }
    } else {
      uint32_t r[8][2];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint2 x = *reinterpret_cast<const uint2 *>(sm + oRV + 4096 * wk + 128 * (4 * j + g) + 8 * n);
        r[j][0] = x.x;
        r[j][1] = x.y;
      }
      auto write = [&]() {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t ah[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            ah[j] = __builtin_amdgcn_perm(r[2 * j + 1][e >> 1], r[2 * j][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
          *reinterpret_cast<uint4 *>(vto + v_piece(64 * wk + 4 * n + e, g)) = make_uint4(ah[0], ah[1], ah[2], ah[3]);
        }
      };
      write();                                     // (once more where they are to be lifted: the look waits for no write)
      const int level = f16_level(r);
      if (__builtin_expect(level, 0)) {
        f16_lift(r);
        write();
      }
      // (the place's level is that of three steps ago)
      if (__builtin_expect(level != (int)(levels >> 2 & 1u), 0) && lane == 0) vto[oLV + wk] = (uint8_t)level;
      levels = levels << 1 | (uint32_t)level;
    }
  };

  h8 ph[MT], pl[MT];
  uint32_t now = 0;                                // the levels of the step whose products are next
  auto scores = [&](int t, const uint8_t *kbuf, const uint8_t *vb) {
    const int64_t kb = (int64_t)t * kTreeKeys;
    // which keys the rows see: lane (n, g)'s bit i is key 4 g + i, bit 16 + i key 16 + 4 g + i
    const int g4 = 4 * (my_lane() >> 4);
    const bool whole = kb + kTreeKeys <= a.pos0 && (!PG || there == ~0u);
    uint32_t win[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) win[mt] = ~0u;
    if (!whole) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) win[mt] = (kb + kTreeKeys > a.pos0 ? there & tree_window(a, token_of(mt), kb) : there) >> g4;
    }
    __builtin_amdgcn_sched_barrier(0);
    // ---- scores; the operands of product ub + AK are asked for before product ub, and no further ahead (the
    // registers hold no more)
    constexpr int AK = KF ? (MT == 2 ? 1 : 2) : 2;
    f4 s[MT][2] = {};
    const int lane = my_lane(), n = lane & 15, g = lane >> 4;
    const uint8_t *kop = kbuf + 512 * n;
    const uint32_t kx = 16 * (g ^ n);              // piece 4 b + g at (4 b + g) ^ n
    const uint8_t *sp = kbuf + kOp + 64 * g;
    auto k_at = [&](int ub) { return *reinterpret_cast<const h8 *>(kop + (kx ^ (64u * (ub & 3))) + 8192 * (ub >> 3) + 256 * ((ub & 7) >> 2)); };
    auto s_at = [&](int ub) { return *reinterpret_cast<const h8 *>(sp + 256 * (ub >> 3) + 16 * ((ub & 7) >> 1)); };   // two blocks
    h8 kf[AK + 1], sc = {}, sn = {};
    f4 p[MT] = {};                                 // q8_0: the last block's products, still to be scaled and added
    uint32_t mine = 0;                             // (fp16 V: there when K is; q8_0 V's are read with its products)
    if constexpr (!VF) mine = *reinterpret_cast<const uint32_t *>(vb + oLV);
    if constexpr (KF) sn = s_at(0);
#pragma unroll
    for (int j = 0; j < AK; ++j) kf[j] = k_at(j);
    if constexpr (!VF) now = __builtin_amdgcn_readfirstlane(mine);
    auto add = [&](int ub) {                       // block ub's products (its pair's scales are in sc)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[mt][ub >> 3][i] = __builtin_fmaf(p[mt][i], (float)sc[4 * (ub & 1) + i], s[mt][ub >> 3][i]);
    };
#pragma unroll
    for (int ub = 0; ub < 16; ++ub) {
      if (ub + AK < 16) kf[(ub + AK) % (AK + 1)] = k_at(ub + AK);
      if constexpr (KF) {
        f4 z[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) z[mt] = mfma16(kf[ub % (AK + 1)], qh[mt][ub & 7], f4{});
        if (ub > 0) add(ub - 1);
        if (!(ub & 1)) {
          sc = sn;
          if (ub < 14) sn = s_at(ub + 2);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) p[mt] = z[mt];
      } else {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][ub >> 3] = mfma16(kf[ub % (AK + 1)], qh[mt][ub & 7], s[mt][ub >> 3]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (KF) add(15);
    // (here, and not where the second row tile's are first used, with every block's product kept until then)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) asm volatile("" : "+v"(s[mt][0]), "+v"(s[mt][1]));
    // ---- probabilities
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!((win[mt] >> ((j & 4) * 4 + (j & 3))) & 1u)) s[mt][j >> 2][j & 3] = -INFINITY;
      }
      float top = fmaxf(fmaxf(fmaxf(s[mt][0][0], s[mt][0][1]), fmaxf(s[mt][0][2], s[mt][0][3])),
                        fmaxf(fmaxf(s[mt][1][0], s[mt][1][1]), fmaxf(s[mt][1][2], s[mt][1][3]))) * a.scale2;
      if (__any(top > m[mt] + (kLift + kPScale))) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float mn = fmaxf(m[mt], top - kPScale);
        const float f = mn == m[mt] ? 1.0f : exp2f(m[mt] - mn);
        m[mt] = mn;
        l[mt] *= f;
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) o[mt][dt] *= f;
      }
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][j >> 2][j & 3], a.scale2, -m[mt]));
      if (!whole) {                                // (where nothing was seen yet, -Inf - -Inf)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!((win[mt] >> ((j & 4) * 4 + (j & 3))) & 1u)) p[j] = 0.0f;
      }
      l[mt] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      split_p(p, ph[mt], pl[mt]);
    }
  };
  auto products = [&](const uint8_t *vb) {
    const int lane = my_lane(), n = lane & 15, g = lane >> 4;
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (VF) now = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const uint32_t *>(vb + oLV));
    if (__builtin_expect(now != lv, 0)) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float f = __builtin_ldexpf(1.0f, v_step(VF) * ((int)((lv >> (8 * c)) & 3u) - (int)((now >> (8 * c)) & 3u)));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) o[mt][4 * c + dt] *= f;
      }
      lv = now;
      lv_any |= now;
    }
    const uint32_t vp[2] = {v_piece(n, g), v_piece(16 + n, g) - 1024u};
    auto v_at = [&](int dt, int lo) { return *reinterpret_cast<const h8 *>(vb + lo * kOp + vp[dt & 1] + 1024 * dt); };
    constexpr int AH = 2;
    h8 vh[AH + 1], vl[VF ? AH + 1 : 1];
#pragma unroll
    for (int j = 0; j < AH; ++j) {
      vh[j] = v_at(j, 0);
      if constexpr (VF) vl[j] = v_at(j, 1);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) {
      const int c = dt % (AH + 1), f = (dt + AH) % (AH + 1);
      if (dt + AH < 16) {
        vh[f] = v_at(dt + AH, 0);
        if constexpr (VF) vl[f] = v_at(dt + AH, 1);
      }
      if constexpr (VF) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[mt][dt] = mfma16(vl[c], ph[mt], o[mt][dt]);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt][dt] = mfma16(vh[c], pl[mt], o[mt][dt]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt][dt] = mfma16(vh[c], ph[mt], o[mt][dt]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Waves 4 .. 7, which share their SIMDs with waves 0 .. 3, take P V of a step at the beginning of the next one: while
  // one wave's scores and probabilities keep the vector unit busy, the other's products keep the matrix cores busy.
  const bool late = w >= 4, works = has_rows && RB * rb + 16 * MT * w < R;   // (a wave whose rows are all past the last only brings bytes)
  lds_barrier();                                   // (every wave has its rows)
  if (t0 < t1) {
    if constexpr (!VF) {
      if (does_v && lane < 3) sm[kVB * lane + oLV + wk] = 0;
    }
    convert(sm + oK + kKB, sm);
    look_up(min(t0 + 1, t1 - 1));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t0 + 1 < t1) request(t0 + 1, 0);
    there_next = there_after;
    lds_barrier();
  }
  uint32_t v_last = 0, v_now = 0, v_next = kVB;    // V's operands of the last step, of this one, of the next
  for (int t = t0; t < t1; ++t) {                  // (the same count in the whole workgroup)
    const int b = (t - t0 + 1) & 1;              // (the first step's K lies in the second place, clear of the rows)
    // (the products, a stream of matrix instructions, go on where the other wave leaves room)
    __builtin_amdgcn_s_setprio(0);
    if (works && late && t > t0) products(sm + v_last);
    __builtin_amdgcn_s_setprio(2);
    __builtin_amdgcn_sched_barrier(0);
    if (works) scores(t, sm + oK + kKB * b, sm + v_now);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    if (works && !late) products(sm + v_now);
    __builtin_amdgcn_s_setprio(2);
    __builtin_amdgcn_sched_barrier(0);
    if (t + 1 < t1) {
      // the next step's operands, in places whose readers have passed the barrier; then, with the wave's bytes used,
      // those of the step after it
      convert(sm + oK + kKB * (b ^ 1), sm + v_next);
      look_up(min(t + 2, t1 - 1));
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if constexpr (KF) {
        if (t + 2 < t1) request(t + 2, 0);
      }
    }
    lds_barrier();
    if constexpr (!KF) {                           // (fp16 K lands where this step's was read)
      if (t + 2 < t1) request(t + 2, b);
    }
    there = there_next;
    there_next = there_after;
    v_last = v_now;
    v_now = v_next;
    v_next = v_next == 2 * kVB ? 0 : v_next + kVB;
  }
  if (works && late && t0 < t1) products(sm + v_last);

  // ---- one partial result per row (through LDS, so that whole rows are written at once, took 2 us more)
  if (!works) return;
  const int64_t rows = (int64_t)a.n_q * a.nh;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = RB * rb + 16 * MT * w + 16 * mt + n, tok = min(r, R - 1) / a.grp;
    float sum = l[mt];
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (r < R) {
      const int64_t at = (int64_t)split * rows + (int64_t)tok * a.nh + hk * a.grp + r - tok * a.grp;
      if (g == 0) a.ml[at] = make_float2(m[mt], marked_sum(sum, lv_any | lv_any >> 16 | (lv_any | lv_any >> 16) >> 8));
    }
    // A store of one product's outputs would reach 16 rows' 64 bytes, half a line each, at a third of the rate of whole
    // lines: so lanes n and n ^ 1 exchange halves of two products, and a store reaches 8 rows' 128 bytes.
    const int64_t mine = r < R ? (int64_t)split * rows + (int64_t)tok * a.nh + hk * a.grp + r - tok * a.grp : -1;
    const int64_t other = __shfl_xor(mine, 1);
    const bool odd = n & 1;
    const int64_t even_row = odd ? other : mine, odd_row = odd ? mine : other;
#pragma unroll
    for (int dt = 0; dt < 16; dt += 2) {
      const float f = __builtin_ldexpf(1.0f, v_step(VF) * (int)((lv >> (8 * (dt >> 2))) & 3u) - v_unit(VF));
      f4 a0 = o[mt][dt] * f, a1 = o[mt][dt + 1] * f, e, d;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = dpp<0xB1>(odd ? a0[i] : a1[i]);          // the other row's half
        e[i] = odd ? x : a0[i];
        d[i] = odd ? a1[i] : x;
      }
      const int col = 16 * (dt + (odd ? 1 : 0)) + 4 * g;
      if (even_row >= 0) *reinterpret_cast<f4 *>(a.part + even_row * kHd + col) = e;
      if (odd_row >= 0) *reinterpret_cast<f4 *>(a.part + odd_row * kHd + col) = d;
    }
  }
}

// ------------------------------------------------------------------ host side
static inline int64_t cdiv(int64_t x, int64_t y) { return (x + y - 1) / y; }
static inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

// Which kernel a call takes: the one with the least estimate of its time in us. The estimates' constants are this card's,
// and choose what was faster wherever two kernels differ by more than 2 us of (kernel + join), as a profiler times them
// (0 to 4 us more than the same call takes among others). Among them, 4 KV heads of q8_0, blocks of 16 / tiles of 128 / of
// 256:
//   onto 600 keys      8 tokens 11.9 / 13.0,  25 tokens 13.2 / 17.9 / 19.6
//   onto 2000         33 tokens 19.4 / 25.7 / 30.6,  128 tokens 35.5 / 35.9 / 43.9
//   onto 8192          8 tokens 17.6 / 20.8,  25 tokens 31.6 / 30.1 / 33.1,  64 tokens .. / 42.2 / 50.2,  300 .. / 134 / 119
//   onto 32768         8 tokens 32.8 / 40.1,  12 tokens 42.9 / 42.4,  33 tokens .. / 93 / 79,  64 tokens .. / 101 / 93
// (of fp16, whose tiles have 3 products a step and no scales: 64 tokens onto 32768 68 in tiles of 128, 76 in 256; onto
// 65536 124 / 119, in pages 137 / 127.)
enum { kTree16, kTree128, kTree256 };
// workgroups that the key split aims for: one per CU (two of the stream kernel's would fit in q8_0, and leave twice the
// ranges to join: 1 token onto 32768 keys 18.7 + 7.6 us against 18.2 + 5.6, onto 131072 56.0 + 7.5 against 48.4 + 5.4)
constexpr int kTreeFill = 256;

TreePlan plan_tree(int nh, int nkv, int kf, int vf, bool paged, int64_t pos0, int n_q, size_t base) {
  TreePlan p{};
  const int64_t rows = (int64_t)n_q * (nh / nkv), steps = cdiv(pos0 + n_q, kTreeKeys);
  const int kq = kf == BKV_Q8_0, vq = vf == BKV_Q8_0;
  const double mb = (double)n_q * nh / 1024.0;       // of partial results, for a key range
  const double read = (double)(pos0 + n_q) * nkv * ((kq ? 272 : 512) + (vq ? 272 : 512)) / 5.5e6;
  double least = 0.0;
  for (int kind = kTree16; kind <= kTree256; ++kind) {
    const int rb = kind == kTree16 ? 16 : kind == kTree128 ? 128 : 256, waves = kind == kTree16 ? 4 : 1;
    const int64_t nrb = cdiv(rows, rb), full = std::min<int64_t>(rows, rb);
    // A step of a wave (stream kernel) or of a workgroup, and what is there without any. q8_0 adds the scales and the
    // products of vl, pages their look-up; 64 rows leave every SIMD of the tile of 128 one wave.
    const double step = (paged ? 0.2 : 0.0) +
                        (kind == kTree16    ? 2.2 + 0.5 * vq
                         : kind == kTree128 ? (1.55 + 0.35 * kq + 0.5 * vq) * (full <= 64 ? 2.0 / 3.0 : 1.0)
                                            : 2.6 + 0.8 * kq + 0.9 * vq - 0.6 * kq * vq);
    const double start = kind == kTree16 ? 5.0 : kind == kTree128 ? 6.0 + 7.0 * (double)full / 128.0 : 12.0 + 8.0 * (double)full / 256.0;
    // A wave of the stream kernel takes a step at least. The tiles: a step fewer per workgroup saves `step`, a key range
    // more costs 0.2 us per MB of partial results to write and join; the least of their sum.
    const int64_t most = kind == kTree16 ? cdiv(steps, waves) : std::max<int64_t>(1, (int64_t)std::sqrt(step * (double)steps / (0.2 * mb)));
    const int64_t splits = std::min(std::min<int64_t>(std::min<int64_t>(kTreeMaxSplit, steps), most), std::max<int64_t>(1, kTreeFill / (nkv * nrb)));
    const double rounds = (double)cdiv(nkv * nrb * splits, kTreeFill);
    const double n_steps = kind == kTree16 ? (double)cdiv(steps, splits * waves) : (double)steps / (double)splits;
    const double cost = std::max(rounds * (start + step * n_steps), 3.0 + read) + 0.2 * mb * (double)splits;
    if (kind > kTree16 && cost >= least) continue;
    least = cost;
    p.kind = kind;
    p.nrb = (int)nrb;
    p.splits = (int)splits;
    p.share = (int)(steps / (splits * waves));
    p.spare = (int)(steps % (splits * waves));
  }
  p.off_ml = base;
  p.off_part = up256(base + (size_t)p.splits * n_q * nh * sizeof(float2));
  p.total = up256(p.off_part + (size_t)p.splits * n_q * nh * kHd * sizeof(float));
  return p;
}

// the largest plan of any call: 65536 rows where the keys are split (at most 256 workgroups of at most 256 rows),
// otherwise every row once
size_t tree_workspace_bound(int nh, size_t base) {
  const size_t rows = std::max<size_t>(65536, (size_t)BKV_TREE_MAX_Q * nh);
  return base + up256(rows * sizeof(float2)) + up256(rows * kHd * sizeof(float)) + 256;
}

template <int KF, int VF, int PG>
static hipError_t launch_tree_main(const TreeArgs &a, const TreePlan &p, hipStream_t st) {
  const dim3 grid(8 * (unsigned)(a.whole + a.share_out));
  switch (p.kind) {
    case kTree16: hipLaunchKernelGGL((tree_stream_kernel<KF, VF, PG>), grid, dim3(256), 0, st, a); break;
    case kTree128: hipLaunchKernelGGL((tree_tile_kernel<KF, VF, PG, 1>), grid, dim3(tree_tile_threads(1)), 0, st, a); break;
    default: hipLaunchKernelGGL((tree_tile_kernel<KF, VF, PG, 2>), grid, dim3(tree_tile_threads(2)), 0, st, a); break;
  }
  return hipGetLastError();
}

hipError_t launch_tree(const TreeArgs &a, const TreePlan &p, int kf, int vf, hipStream_t st) {
  BKV_FMT_SWITCH(kf, vf, {
    const hipError_t e = a.L.page == 0 ? launch_tree_main<KF_, VF_, 0>(a, p, st)
                         : a.L.page % kTreeKeys == 0 ? launch_tree_main<KF_, VF_, 1>(a, p, st)
                                                     : launch_tree_main<KF_, VF_, 2>(a, p, st);
    if (e != hipSuccess) return e;
    const dim3 rows((unsigned)((int64_t)a.n_q * a.nh));
    if (a.splits <= 8) hipLaunchKernelGGL((tree_merge_kernel<KF_, VF_, 1>), rows, dim3(64), 0, st, a);
    else if (a.splits <= 32) hipLaunchKernelGGL((tree_merge_kernel<KF_, VF_, 4>), rows, dim3(256), 0, st, a);
    else if (a.splits <= 64) hipLaunchKernelGGL((tree_merge_kernel<KF_, VF_, 8>), rows, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((tree_merge_kernel<KF_, VF_, 16>), rows, dim3(1024), 0, st, a);
  });
  return hipGetLastError();
}

}  // namespace bkv
