// bkv_seqs_attn.hip - attention of the tokens of several sequences over a 4-bit cache (bkv_seqs_attn).
//
// The rows of one KV head and sequence are its n * grp (token, query head) pairs; the row of token i sees the keys below
// len - n + i + 1. With s = q16 . k and x = s * scale * log2(e): out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m) over the
// visible j, for any m near the largest x_j. One pass over the keys: every wave keeps a reference m, a sum and 256
// unnormalised outputs per row, and lifts m only when a row's score exceeds it by kLift.
//
// Products on the fp16 matrix cores, summed in fp32: q and k are exact operands (bkv_q4.h), v too, and
// 2^(x - m) * 2^9 = ph + pl, two fp16 (22 bits; the factor keeps pl normal down to p = 2^-14 of the largest). One product
// for the scores, two for the outputs, where the formula has one each; a single fp16 p would leave 1e-4 in place of 1e-6.
// Everything in the cache is finite whatever its bytes, so that keys that a row does not see, p = 0, have no effect.
//
// The work is cut evenly however long the sequences are: the 32-key steps of all row blocks, one sequence after the other,
// are one line, of which every workgroup takes an equal piece. A piece that ends inside a row block leaves unnormalised
// partial results, which seqs_merge_kernel joins; a row block that lies in one piece is written as it is.

#include <algorithm>

#include "bkv_device.h"
#include "bkv_internal.h"
#include "bkv_mfma16.h"
#include "bkv_q4.h"

namespace bkv {

constexpr float kLift = 6.0f;          // a score this far (in powers of two) above the reference lifts it
constexpr float kPScale = 9.0f;        // log2 of the factor on p: 2^(kLift + kPScale) is within fp16
constexpr int kSeqKeys = 32;           // keys of a step
constexpr int kSeqBlock = 16;          // rows of a row block

__device__ __forceinline__ int cdiv_d(int a, int b) { return (a + b - 1) / b; }

// 4 h2 (8 elements in order) of a word of codes: 0x4C00 | q << 6 is the fp16 number 16 + q, and (16 + q + 8 - 24) * d, in one
// fused step, is exact: both 24 d and the result have 11 bits at most.
template <int S>
__device__ __forceinline__ h2 q4_pair(uint32_t w, h2 d, h2 c) {
  const uint32_t x = S == 0 ? w << 6 : S == 1 ? w << 2 : S == 2 ? w >> 2 : w >> 6;
  return __builtin_elementwise_fma(as_h2((x & 0x03C003C0u) | 0x4C004C00u), d, c);
}
__device__ __forceinline__ h2 q4_offset(h2 d) { return d * h2{(_Float16)-24.0f, (_Float16)-24.0f}; }
__device__ __forceinline__ h8 q4_eight(uint32_t w, h2 d, h2 c) {
  return __builtin_bit_cast(h8, make_uint4(as_u(q4_pair<0>(w, d, c)), as_u(q4_pair<1>(w, d, c)), as_u(q4_pair<2>(w, d, c)), as_u(q4_pair<3>(w, d, c))));
}

// 8 probabilities as ph + pl: ph cut to fp16 (two in one instruction), pl the rest, rounded
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

// ------------------------------------------------------------------ the line of steps
// A sequence's row blocks, and the steps of each (one at least, so that rows that see nothing are written too)
__device__ __forceinline__ int blocks_of(const SeqsAttnArgs &a, int s) { return cdiv_d(a.v.tokens(s) * a.grp, kSeqBlock); }
__device__ __forceinline__ int steps_of(const SeqsAttnArgs &a, int s) { return max(1, (a.v.length(s) + kSeqKeys - 1) / kSeqKeys); }

// the line's length for one KV head (by every wave alike)
__device__ __forceinline__ int64_t line_length(const SeqsAttnArgs &a) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  for (int s0 = 0; s0 < a.v.n_seq; s0 += 64) {
    const int s = s0 + lane;
    int64_t v = s < a.v.n_seq ? (int64_t)blocks_of(a, s) * steps_of(a, s) : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    total += v;
  }
  return total;
}
// how the line is cut: nl pieces of share steps, the first spare of one more
struct Cut {
  int64_t share, spare;
  int nl;
  __device__ __forceinline__ Cut(int64_t total, int lanes, int least) {
    nl = (int)min((int64_t)lanes, max((int64_t)1, total / least));
    share = total / nl;
    spare = total - share * nl;
  }
  __device__ __forceinline__ int64_t begin(int i) const { return i * share + min((int64_t)i, spare); }
  __device__ __forceinline__ int piece_of(int64_t x) const {
    const int64_t longer = spare * (share + 1);
    return (int)(x < longer ? x / (share + 1) : spare + (x - longer) / share);
  }
};

// ------------------------------------------------------------------ few rows a block
// A workgroup of 4 waves takes its piece of the line for one KV head; of each row block in it the waves take a quarter of
// the steps each and meet in LDS. Scores are computed transposed, S^T = K Q^T: lane (n, g) = (lane % 16, lane / 16) holds
// keys 4 g .. 4 g + 3 of a 16-key tile for row n, which is P^T's operand of O^T = V^T P^T as it stands if slot (g, j) of the
// 32-key contraction stands for key 4 g + j (j < 4) or 16 + 4 g + j - 4, for both operands. Product c of the scores takes
// word 8 g + c of a key, dims 64 g + 8 c .., so that a lane's 8 words are 32 bytes; product dt of the outputs dim 16 m + dt,
// so that a lane's dims of a key are 8 bytes.
// PG: 0 a contiguous cache; 1 pages of whole steps (a multiple of 32 tokens); 2 any pages
template <int PG>
__global__ __launch_bounds__(256, 2) void seqs_attn_kernel(SeqsAttnArgs a) {
  constexpr int kOS = kHd + 4;                     // a row of the join
  __shared__ __attribute__((aligned(16))) float s_o[4 * kSeqBlock * kOS];
  __shared__ float s_m[4][kSeqBlock], s_l[4][kSeqBlock];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  // pieces 8 apart on the same XCD; a piece's KV heads next to one another there, whose scales share lines
  const int at8 = (int)(blockIdx.x >> 3), hk = at8 % a.nkv, piece = at8 / a.nkv * 8 + (int)(blockIdx.x & 7);
  const int64_t total = line_length(a);
  const Cut cut(total, a.lanes, a.least);
  if (piece >= cut.nl) return;
  int64_t at = cut.begin(piece);
  const int64_t end = cut.begin(piece + 1);
  // the sequence that position `at` of the line lies in, and what lies before that
  int seq = 0, tile0 = 0;
  int64_t line0 = 0;
  for (int s0 = 0; s0 < a.v.n_seq; s0 += 64) {
    const int s = s0 + lane;
    const int nb = s < a.v.n_seq ? blocks_of(a, s) : 0;
    const int64_t v = s < a.v.n_seq ? (int64_t)nb * steps_of(a, s) : 0;
    const int64_t inc = wave_incl_scan(v, lane);
    const int binc = wave_incl_scan(nb, lane);
    const uint64_t past = __ballot(line0 + inc > at);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      seq = s0 + l;
      line0 += __shfl(inc - v, l);
      tile0 += __shfl(binc - nb, l);
      break;
    }
    line0 += __shfl(inc, 63);
    tile0 += __shfl(binc, 63);
  }
  seq = __builtin_amdgcn_readfirstlane(seq);

  const uint32_t krow = (uint32_t)a.nkv * kQ4RowBytes, srow = (uint32_t)a.nkv * kScaleRowBytes;
  const uint8_t *kd = a.L.kd + (size_t)hk * kQ4RowBytes, *vd = a.L.vd + (size_t)hk * kQ4RowBytes;
  const uint8_t *ksc = a.L.ks + (size_t)hk * kScaleRowBytes, *vsc = a.L.vs + (size_t)hk * kScaleRowBytes;

  while (at < end && seq < a.v.n_seq) {
    // ---- the piece's part of one row block
    const int q0 = a.v.q_begin(seq), nt = a.v.tokens(seq), len = a.v.length(seq), steps = steps_of(a, seq);
    if (nt == 0) { ++seq; continue; }              // (there is a sequence with rows: at < end)
    const int R = nt * a.grp, rb = (int)((at - line0) / steps), st0 = (int)(at - line0 - (int64_t)rb * steps);
    const int st1 = (int)min((int64_t)steps, st0 + (end - at)), m4 = st1 - st0;
    const int t0 = st0 + m4 * w / 4, t1 = st0 + m4 * (w + 1) / 4;
    const int last = max(len - 1, 0);              // (the last key that there are bytes of)
    const int r0 = kSeqBlock * rb, row = min(r0 + n, R - 1), tok = row / a.grp;
    const int lim = len - nt + tok + 1;            // keys below it are seen
    const int lim_all = len - nt + r0 / a.grp + 1; // by all rows of the block

    uint32_t there = ~0u, there_next = ~0u;        // keys whose pages are in the pool: this step's, the next's
    int sl = 0;                                    // PG 2: the slot of key lane % 32
    size_t s0 = 0;
    auto look_up = [&](int t) {
      const uint32_t kb = (uint32_t)t * kSeqKeys;
      s0 = kb;
      if constexpr (PG == 1) {
        const int first = __builtin_amdgcn_readfirstlane(a.v.slot(seq, min(kb, (uint32_t)last)));
        there_next = first >= 0 ? ~0u : 0u;
        s0 = (size_t)max(first, 0);
      }
      if constexpr (PG == 2) {
        sl = a.v.slot(seq, min(kb + ((uint32_t)lane & 31), (uint32_t)last));
        there_next = (uint32_t)__ballot(sl >= 0);
      }
    };
    // a lane's bytes of a key, `stride` from a key to the next
    auto from = [&](const uint8_t *base, int t, int key, uint32_t stride) -> const uint8_t * {
      if constexpr (PG == 2) return base + (size_t)max(__shfl(sl, key), 0) * stride;
      else return base + s0 * stride + min((uint32_t)key, (uint32_t)last - (uint32_t)t * kSeqKeys) * stride;
    };
    uint4 kr[2][2];
    uint32_t ks[2];
    uint2 vr[8];
    uint32_t vs[8];
    auto key_of = [&](int j) { return (j & 4) * 4 + 4 * g + (j & 3); };
    auto load_k = [&](int t) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 *p = reinterpret_cast<const uint4 *>(from(kd, t, 16 * u + n, krow) + 32 * g);
        kr[u][0] = p[0];
        kr[u][1] = p[1];
        ks[u] = *reinterpret_cast<const uint32_t *>(from(ksc, t, 16 * u + n, srow) + 4 * g);
      }
    };
    auto load_v = [&](int t) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        vr[j] = *reinterpret_cast<const uint2 *>(from(vd, t, key_of(j), krow) + 8 * n);
        vs[j] = *reinterpret_cast<const uint16_t *>(from(vsc, t, key_of(j), srow) + 2 * (n >> 1));
      }
    };
    if (t0 < t1) {
      look_up(t0);
      load_k(t0);
      load_v(t0);
    }
    h8 qh[8];                                      // row n, dims 64 g + 8 c ..
    {
      const float4 *q = reinterpret_cast<const float4 *>(a.q.at(q0 + tok, hk * a.grp + row - tok * a.grp)) + 16 * g;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float4 x = q[2 * c], y = q[2 * c + 1];
        qh[c] = h8{(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w, (_Float16)y.x, (_Float16)y.y, (_Float16)y.z, (_Float16)y.w};
      }
    }
    f4 o[16] = {};
    float m = -INFINITY, l = 0.0f;                 // m: the reference less kPScale

#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      const int kb = t * kSeqKeys;
      there = there_next;
      // which keys the rows see: lane (n, g)'s bit i is key 4 g + i, bit 16 + i key 16 + 4 g + i
      const bool whole = kb + kSeqKeys <= lim_all && (!PG || there == ~0u);
      uint32_t win = there;
      if (!whole) {
        const int seen = lim - kb;                 // of the step's keys the first `seen`
        win &= seen <= 0 ? 0u : seen >= 32 ? ~0u : (1u << seen) - 1u;
      }
      win >>= 4 * g;
      // ---- scores
      f4 s[2] = {};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const h2 two = as_h2(q4_scales(ks[u]));
        const h2 d[2] = {h2{two[0], two[0]}, h2{two[1], two[1]}};
        const h2 c[2] = {q4_offset(d[0]), q4_offset(d[1])};
#pragma unroll
        for (int i = 0; i < 8; ++i) s[u] = mfma16(q4_eight((&kr[u][i >> 2].x)[i & 3], d[i >> 2], c[i >> 2]), qh[i], s[u]);
      }
      if (t + 1 < t1) {
        look_up(t + 1);
        load_k(t + 1);
      }
      // ---- probabilities
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
      if (!whole) {                                // (where nothing was seen yet, -Inf - -Inf)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!((win >> ((j & 4) * 4 + (j & 3))) & 1u)) p[j] = 0.0f;
      }
      l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      h8 ph, pl;
      split_p(p, ph, pl);
      // ---- P V
      h2 d[4], c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d[j] = as_h2(q4_scales(vs[2 * j] | (vs[2 * j + 1] << 16)));
        c[j] = q4_offset(d[j]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {                // the 16-bit halves of the lane's two words: dims 8 (e / 2) + e % 2 + 0, 2, 4, 6
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = __builtin_amdgcn_perm(e & 2 ? vr[2 * j + 1].y : vr[2 * j + 1].x, e & 2 ? vr[2 * j].y : vr[2 * j].x, e & 1 ? 0x07060302u : 0x05040100u);
        auto product = [&](const h2 (&v)[4], int i) {
          const int dt = 8 * (e >> 1) + 2 * i + (e & 1);
          const h8 vh = __builtin_bit_cast(h8, make_uint4(as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3])));
          o[dt] = mfma16(vh, pl, o[dt]);
          o[dt] = mfma16(vh, ph, o[dt]);
        };
        const h2 v0[4] = {q4_pair<0>(x[0], d[0], c[0]), q4_pair<0>(x[1], d[1], c[1]), q4_pair<0>(x[2], d[2], c[2]), q4_pair<0>(x[3], d[3], c[3])};
        const h2 v1[4] = {q4_pair<1>(x[0], d[0], c[0]), q4_pair<1>(x[1], d[1], c[1]), q4_pair<1>(x[2], d[2], c[2]), q4_pair<1>(x[3], d[3], c[3])};
        const h2 v2[4] = {q4_pair<2>(x[0], d[0], c[0]), q4_pair<2>(x[1], d[1], c[1]), q4_pair<2>(x[2], d[2], c[2]), q4_pair<2>(x[3], d[3], c[3])};
        const h2 v3[4] = {q4_pair<3>(x[0], d[0], c[0]), q4_pair<3>(x[1], d[1], c[1]), q4_pair<3>(x[2], d[2], c[2]), q4_pair<3>(x[3], d[3], c[3])};
        product(v0, 0);
        product(v1, 1);
        product(v2, 2);
        product(v3, 3);
      }
      if (t + 1 < t1) load_v(t + 1);
    }

    // ---- the 4 waves' parts joined
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) { s_m[w][n] = m; s_l[w][n] = l; }
    __syncthreads();
    const float mm = fmaxf(fmaxf(s_m[0][n], s_m[1][n]), fmaxf(s_m[2][n], s_m[3][n]));
    const float f = m == -INFINITY ? 0.0f : exp2f(m - mm);
#pragma unroll
    for (int dt = 0; dt < 16; dt += 4)             // (4 products' dims are neighbours)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4 *>(&s_o[(kSeqBlock * w + n) * kOS + 16 * (4 * g + i) + dt]) =
            make_float4(o[dt][i] * f, o[dt + 1][i] * f, o[dt + 2][i] * f, o[dt + 3][i] * f);
    __syncthreads();
    const int jr = threadIdx.x >> 4, c = threadIdx.x & 15, r = r0 + jr;
    if (r < R) {
      const int ti = r / a.grp, h = hk * a.grp + r - ti * a.grp;
      const float mr = fmaxf(fmaxf(s_m[0][jr], s_m[1][jr]), fmaxf(s_m[2][jr], s_m[3][jr]));
      float lr = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) lr += s_m[j][jr] == -INFINITY ? 0.0f : s_l[j][jr] * exp2f(s_m[j][jr] - mr);
      const bool alone = m4 == steps;
      const float inv = lr > 0.0f || lr != lr ? lr : 1.0f;
      const uint32_t part = ((uint32_t)(piece + tile0 + rb) * a.nkv + hk) * kSeqBlock + jr;
      const int64_t dst = (int64_t)(q0 + ti) * a.nh + h;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 x = *reinterpret_cast<const float4 *>(&s_o[(kSeqBlock * j + jr) * kOS + 4 * c + 64 * k]);
          v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        const int col = 4 * c + 64 * k;
        if (alone) {
          v = make_float4(v.x / inv, v.y / inv, v.z / inv, v.w / inv);
          *reinterpret_cast<float4 *>(a.out + dst * kHd + col) = v;
          if (a.gate.p) {
            const float4 gt = *reinterpret_cast<const float4 *>(a.gate.at(q0 + ti, h) + col);
            *reinterpret_cast<float4 *>(a.out_gated + dst * kHd + col) =
                make_float4(v.x / (1.0f + expf(-gt.x)), v.y / (1.0f + expf(-gt.y)), v.z / (1.0f + expf(-gt.z)), v.w / (1.0f + expf(-gt.w)));
          }
        } else if (part < a.part_rows) {
          *reinterpret_cast<float4 *>(a.part + (int64_t)part * kHd + col) = v;
        }
      }
      if (c == 0) {
        if (!alone && part < a.part_rows) a.ml[part] = make_float2(mr, lr);
        if (st0 == 0) {
          const int count = cut.piece_of(line0 + (int64_t)(rb + 1) * steps - 1) - piece + 1;
          a.info[dst] = make_uint4(part, (uint32_t)a.nkv * kSeqBlock, (uint32_t)count, 0);
        }
      }
    }
    __syncthreads();                               // (LDS is the next part's)
    at += m4;
    if (rb + 1 == blocks_of(a, seq) && st1 == steps) {
      line0 += (int64_t)(rb + 1) * steps;
      tile0 += rb + 1;
      ++seq;
    }
  }
}

// ------------------------------------------------------------------ the join
// One workgroup of NWV waves per row: wave w sums the partial results w, w + NWV, .. (a lane 4 dims, 8 of them requested
// together), then the waves' sums meet in LDS.
template <int NWV>
__global__ __launch_bounds__(64 * NWV) void seqs_merge_kernel(SeqsAttnArgs a) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = blockIdx.x;
  const int t = (int)(r / a.nh), h = (int)(r - (int64_t)t * a.nh);
  __shared__ __attribute__((aligned(16))) float s_o[NWV * kHd];
  const uint4 in = a.info[r];
  if (a.v.sequence_of<64>(t) < 0) return;          // (no sequence's row: nothing was left for it)
  const uint32_t first = in.x, stride = in.y, count = in.z;
  if (count <= 1 || (uint64_t)first + (uint64_t)stride * (count - 1) >= a.part_rows) return;
  float mm = -INFINITY;
  for (uint32_t i = lane; i < count; i += 64) mm = fmaxf(mm, a.ml[first + i * stride].x);
  mm = wave_max(mm);
  float l = 0.0f;
  for (uint32_t i = lane; i < count; i += 64) {
    const float2 x = a.ml[first + i * stride];
    l += x.x == -INFINITY ? 0.0f : x.y * exp2f(x.x - mm);
  }
  l = wave_sum(l);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f), x[8];
  for (uint32_t i0 = w; i0 < count; i0 += 8 * NWV) {
    float m8[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t i = min(i0 + j * NWV, count - 1);
      x[j] = reinterpret_cast<const float4 *>(a.part + (int64_t)(first + i * stride) * kHd)[lane];
      m8[j] = a.ml[first + i * stride].x;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i0 + j * NWV >= count) break;
      const float f = m8[j] == -INFINITY ? 0.0f : exp2f(m8[j] - mm);
      o.x = fmaf(x[j].x, f, o.x); o.y = fmaf(x[j].y, f, o.y); o.z = fmaf(x[j].z, f, o.z); o.w = fmaf(x[j].w, f, o.w);
    }
  }
  reinterpret_cast<float4 *>(s_o + w * kHd)[lane] = o;
  __syncthreads();
  if (w != 0) return;
  o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int j = 0; j < NWV; ++j) {
    const float4 y = reinterpret_cast<const float4 *>(s_o + j * kHd)[lane];
    o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
  }
  const float inv = l > 0.0f || l != l ? l : 1.0f;
  const float4 v = make_float4(o.x / inv, o.y / inv, o.z / inv, o.w / inv);
  reinterpret_cast<float4 *>(a.out + r * kHd)[lane] = v;
  if (a.gate.p) {
    const float4 gt = reinterpret_cast<const float4 *>(a.gate.at(t, h))[lane];
    reinterpret_cast<float4 *>(a.out_gated + r * kHd)[lane] =
        make_float4(v.x / (1.0f + expf(-gt.x)), v.y / (1.0f + expf(-gt.y)), v.z / (1.0f + expf(-gt.z)), v.w / (1.0f + expf(-gt.w)));
  }
}

// ------------------------------------------------------------------ host side
static inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
constexpr int kSeqFill = 512;          // workgroups of all KV heads that the line is cut for
constexpr int kSeqLeast = 4;           // steps of a piece at least

SeqsAttnPlan plan_seqs_attn(int nh, int nkv, int n_seq, int n_tok) {
  SeqsAttnPlan p{};
  p.lanes = std::max(1, kSeqFill / nkv);
  p.least = kSeqLeast;
  // a partial result's number is its piece plus its row block, both counted from 0
  const uint64_t tiles = (uint64_t)n_tok * (nh / nkv) / kSeqBlock + n_seq;
  p.part_rows = (p.lanes + tiles) * nkv * kSeqBlock;
  p.off_ml = up256((size_t)n_tok * nh * sizeof(uint4));
  p.off_part = up256(p.off_ml + p.part_rows * sizeof(float2));
  p.total = up256(p.off_part + p.part_rows * kHd * sizeof(float));
  return p;
}

hipError_t launch_seqs_attn(const SeqsAttnArgs &a, const SeqsAttnPlan &p, hipStream_t st) {
  const dim3 grid((unsigned)((p.lanes + 7) / 8 * 8 * a.nkv));
  if (a.v.page == 0) hipLaunchKernelGGL((seqs_attn_kernel<0>), grid, dim3(256), 0, st, a);
  else if (a.v.page % kSeqKeys == 0) hipLaunchKernelGGL((seqs_attn_kernel<1>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((seqs_attn_kernel<2>), grid, dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 rows((unsigned)((int64_t)a.v.n_tok * a.nh));
  if (rows.x > 2048) hipLaunchKernelGGL((seqs_merge_kernel<1>), rows, dim3(64), 0, st, a);
  else if (rows.x > 256) hipLaunchKernelGGL((seqs_merge_kernel<4>), rows, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((seqs_merge_kernel<16>), rows, dim3(1024), 0, st, a);
  return hipGetLastError();
}

}  // namespace bkv
