// bkv_seqs_attn.hip - attention of the tokens of several sequences over a 4-bit cache (bkv_seqs_attn).
//
// The rows of one KV head and sequence are its n * grp (token, query head) pairs; the row of token i sees the keys below
// len - n + i + 1 that the cache has room for (len may be past that). With s = q16 . k and x = s * scale * log2(e):
// out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m) over the visible j, for any m near the largest x_j. One pass over the
// keys: every wave keeps a reference m, a sum and 256 unnormalised outputs per row, and lifts m only when a row's score
// exceeds it by kLift.
//
// Products on the fp16 matrix cores, summed in fp32: q and k are exact operands (bkv_q4.h), v too, and
// 2^(x - m) * 2^9 = ph + pl, two fp16 (22 bits; the factor keeps pl normal down to p = 2^-14 of the largest). One product
// for the scores, two for the outputs, where the formula has one each; a single fp16 p would leave 1e-4 in place of 1e-6.
// Everything in the cache is finite whatever its bytes, so that keys that a row does not see, p = 0, have no effect.
//
// The work is cut evenly however long the sequences are: the 32-key steps of all row blocks, one sequence after the other,
// are one line, of which every workgroup takes an equal piece. A piece that ends inside a row block leaves unnormalised
// partial results, which are joined; a row block that lies in one piece is written as it is.

#include <algorithm>
#include <type_traits>

#include "bkv_device.h"
#include "bkv_internal.h"
#include "bkv_mfma16.h"
#include "bkv_q4.h"

namespace bkv {

constexpr float kLift = 6.0f;          // a score this far (in powers of two) above the reference lifts it
constexpr float kPScale = 9.0f;        // log2 of the factor on p: 2^(kLift + kPScale) is within fp16
constexpr int kSeqKeys = 32;           // keys of a step
constexpr int kSeqBlock = 16;          // rows of a row block
constexpr int kSeqLeast = 8;           // steps of a piece at least

__device__ __forceinline__ int cdiv_d(int a, int b) { return (a + b - 1) / b; }
// the positions of a sequence that there are bytes of
__device__ __forceinline__ int keys_of(const SeqsAttnArgs &a, int len) { return min(len, (int)a.v.max_pos); }

// 4 h2 (8 elements in order) of a word of codes: 0x4C00 | q << 6 is the fp16 number 16 + q, and (16 + q + 8 - 24) * d, in one
// fused step, is exact: both 24 d and the result have 11 bits at most.
// (the constants in registers, one scalar and one vector, so that taking the bits and the or is one instruction)
struct Q4Bits {
  uint32_t mask = 0x03C003C0u, ones = 0x4C004C00u;
  __device__ __forceinline__ Q4Bits() {
    asm volatile("" : "+s"(mask));
    asm volatile("" : "+v"(ones));
  }
  template <int S>
  __device__ __forceinline__ h2 pair(uint32_t w, h2 d, h2 c) const {
    const uint32_t x = S == 0 ? w << 6 : S == 1 ? w << 2 : S == 2 ? w >> 2 : w >> 6;
    return __builtin_elementwise_fma(as_h2((x & mask) | ones), d, c);
  }
  __device__ __forceinline__ h8 eight(uint32_t w, h2 d, h2 c) const {
    return __builtin_bit_cast(h8, make_uint4(as_u(pair<0>(w, d, c)), as_u(pair<1>(w, d, c)), as_u(pair<2>(w, d, c)), as_u(pair<3>(w, d, c))));
  }
};
__device__ __forceinline__ h2 q4_offset(h2 d) { return d * h2{(_Float16)-24.0f, (_Float16)-24.0f}; }

// 8 probabilities as ph + pl: ph cut to fp16 (two in one instruction), pl the rest, rounded (one mixed-precision instruction
// each, if the compiler does not see that the factor is -1)
__device__ __forceinline__ void split_p(const float (&p)[8], h8 &ph, h8 &pl) {
  float minus = -1.0f;
  asm volatile("" : "+s"(minus));
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const auto c = __builtin_amdgcn_cvt_pkrtz(p[j], p[j + 1]);
    ph[j] = (_Float16)c[0];
    ph[j + 1] = (_Float16)c[1];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) pl[j] = (_Float16)__builtin_fmaf((float)ph[j], minus, p[j]);
}

// the kernel's arguments (its first and only one), read anew
template <typename T>
__device__ __forceinline__ T arguments_again() {
  uint32_t raw[sizeof(T) / 4];
#ifdef __HIP_DEVICE_COMPILE__
  const __attribute__((address_space(4))) uint32_t *p = (const __attribute__((address_space(4))) uint32_t *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; ++i) raw[i] = p[i];
#endif
  return __builtin_bit_cast(T, raw);
}

// The lines that the kernel's arguments lie in, asked for at once: where each use waits for its own, a launch's first
// microseconds are such waits one after another.
template <typename T>
__device__ __forceinline__ void arguments_near() {
#ifdef __HIP_DEVICE_COMPILE__
  const __attribute__((address_space(4))) uint32_t *p = (const __attribute__((address_space(4))) uint32_t *)__builtin_amdgcn_kernarg_segment_ptr();
  uint32_t x = 0;
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; i += 16) x |= p[i];
  asm volatile("" ::"s"(x));
#endif
}

// ------------------------------------------------------------------ the line of steps
// inclusive sums over the wave
__device__ __forceinline__ int wave_sums(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}
__device__ __forceinline__ int of_lane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }

// Lane l's of 64 sequences: where its rows begin, how many tokens and positions it has, its row blocks and the steps of
// each (one at least, so that rows that see nothing are written too)
struct SeqLanes {
  int q0, nt, len, steps, blocks;
  bool bad;                                        // some sequence's rows begin behind the next one's
  __device__ __forceinline__ SeqLanes(const SeqsAttnArgs &a, int s0) {
    const int s = s0 + (int)(threadIdx.x & 63), in = min(s, a.v.n_seq - 1);
    int e = in + 1;
    q0 = in;
    if (a.v.q_start) {
      q0 = a.v.q_start[in];
      e = a.v.q_start[in + 1];
    }
    bad = __any(e < q0);
    len = a.v.length(in);
    q0 = min(max(q0, 0), a.v.n_tok);
    nt = s < a.v.n_seq ? max(min(max(e, 0), a.v.n_tok) - q0, 0) : 0;
    steps = max(1, (int)((uint32_t)(keys_of(a, len) + kSeqKeys - 1) / kSeqKeys));
    blocks = (int)((uint32_t)(nt * a.grp + kSeqBlock - 1) / kSeqBlock);
  }
  // (of the sequences of few rows)
  __device__ __forceinline__ int line(const SeqsAttnArgs &a) const { return nt * a.grp <= a.few ? blocks * (a.way_in + steps) : 0; }
};

// how the line is cut: nl pieces of share steps, the first spare of one more
struct Cut {
  int share, spare, nl;
  __device__ __forceinline__ Cut(int total, int lanes, const ByConst &by_lanes, int least) {
    const int most = max(1, (int)((uint32_t)(total + least - 1) / (uint32_t)least));
    nl = min(lanes, most);
    share = nl == lanes ? by_lanes.div(total) : (int)((uint32_t)total / (uint32_t)nl);
    spare = total - share * nl;
  }
  __device__ __forceinline__ int begin(int i) const { return i * share + min(i, spare); }
  __device__ __forceinline__ int piece_of(int x) const {
    const int longer = spare * (share + 1);
    return x < longer ? (int)((uint32_t)x / (uint32_t)(share + 1)) : spare + (int)((uint32_t)(x - longer) / (uint32_t)share);
  }
};

// ------------------------------------------------------------------ few rows a block
// A workgroup of 8 waves takes its piece of the line for one KV head; of each row block in it the waves take an eighth of
// the steps each and meet in LDS. Scores are computed transposed, S^T = K Q^T: lane (n, g) = (lane % 16, lane / 16) holds
// keys 4 g .. 4 g + 3 of a 16-key tile for row n, which is P^T's operand of O^T = V^T P^T as it stands if slot (g, j) of the
// 32-key contraction stands for key 4 g + j (j < 4) or 16 + 4 g + j - 4, for both operands. Product c of the scores takes
// word 8 g + c of a key, dims 64 g + 8 c .., so that a lane's 8 words are 32 bytes; product dt of the outputs dim 16 m + dt,
// so that a lane's dims of a key are 8 bytes.
//
// A row block cut into several pieces: each leaves its partial results in memory, past the caches of its XCD, and counts
// itself; the last of every 8 pieces joins theirs, and the last of those joins these.
//
// What bounds it: the vector unit in the steps (553 instructions a wave and step, 384 of them codes on their way to fp16; a wave
// and step takes 3.3 thousand cycles of its SIMD), and around them latencies: arguments, lengths, Q and the first bytes
// 3.5 us, the waves' join 2, the pieces' 3 a round of 8. One token of 16 heads at 600 / 32,768 positions 11.6 / 20 us
// (1.9 TB/s), 29 sequences of 40 to 12,000 28 (2.7 TB/s).
// PG: 0 a contiguous cache; 1 pages of whole steps (a multiple of 32 tokens); 2 any pages
constexpr int kSeqWaves = 8;
constexpr int kSeqFill = 256;          // pieces of all KV heads: a workgroup a CU
constexpr int kJoin = 8;               // partial results that are joined at a time
constexpr int kJoinLevels = 3;         // counters: of each level, a piece's two row blocks
static_assert(kJoin * kJoin * kJoin >= kSeqFill, "levels of joins");

__device__ __forceinline__ void st_part(void *p, float2 v) { st_agent(reinterpret_cast<unsigned long long *>(p), __builtin_bit_cast(unsigned long long, v)); }
__device__ __forceinline__ float2 ld_part(const void *p) { return __builtin_bit_cast(float2, ld_agent(reinterpret_cast<const unsigned long long *>(p))); }

// N outputs of a row, from dim col on
template <int N>
__device__ __forceinline__ void write_out(const SeqsAttnArgs &a, int t, int h, int col, const float (&v)[N], float l) {
  typedef float V __attribute__((ext_vector_type(N)));
  const float by = l > 0.0f || l != l ? l : 1.0f;
  const int64_t at = ((int64_t)t * a.nh + h) * kHd + col;
  V o;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = v[i] / by;
  *reinterpret_cast<V *>(a.out + at) = o;
  if (a.gate.p) {
    const V g = *reinterpret_cast<const V *>(a.gate.at(t, h) + col);
    V y;
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = o[i] / (1.0f + expf(-g[i]));
    *reinterpret_cast<V *>(a.out_gated + at) = y;
  }
}

template <int PG>
__global__ __launch_bounds__(64 * kSeqWaves, 2) void seqs_attn_kernel(SeqsAttnArgs a) {
  constexpr int NT = 64 * kSeqWaves;
  // a wave's two steps: K and V rows of 128 bytes, then their scales, 16 bytes a key; later its rows of the join
  constexpr uint32_t oV = kSeqKeys * kQ4RowBytes, oKS = 2 * oV, oVS = oKS + 512, kStep = oVS + 512, kWave = 2 * kStep;
  constexpr int kOS = kHd + 4;                     // a row of the join
  static_assert(kSeqBlock * kOS * 4 <= kWave && 2 * 1024 <= kStep, "the join's rows and two rows of Q in the steps' place");
  __shared__ __attribute__((aligned(128))) uint8_t sm[kSeqWaves * kWave];
  __shared__ int32_t s_tab[PG ? 2 * kSeqWaves : 1][64];   // table entries of a wave's steps
  __shared__ float s_m[kSeqWaves][kSeqBlock], s_l[kSeqWaves][kSeqBlock];
  __shared__ int s_last;
  arguments_near<SeqsAttnArgs>();
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const Q4Bits bits;
  // pieces 8 apart on the same XCD; a piece's KV heads next to one another there, whose scales share lines
  const int at8 = (int)(blockIdx.x >> 3), round = a.by_nkv.div(at8), hk = at8 - round * a.nkv, piece = 8 * round + (int)(blockIdx.x & 7);
  // the line, by every wave alike: 64 sequences at a time
  SeqLanes my(a, 0);
  int inc = wave_sums(my.line(a)), total = of_lane(inc, 63);
  bool bad = my.bad;
  for (int s0 = 64; s0 < a.v.n_seq; s0 += 64) {
    const SeqLanes more(a, s0);
    total += of_lane(wave_sums(more.line(a)), 63);
    bad |= more.bad;
  }
  if (bad) return;                                 // (starts that go back: their sums would have no bound)
  const Cut cut(total, a.lanes, a.by_lanes, kSeqLeast);
  if (piece >= cut.nl) return;
  int at = cut.begin(piece);
  const int end = cut.begin(piece + 1);
  // the sequence that step `at` of the line lies in, and where that begins
  int s0 = 0, in64 = 0, line0 = 0;
  for (;;) {
    const uint64_t past = __ballot(line0 + inc > at);
    if (past) {
      in64 = __ffsll((unsigned long long)past) - 1;
      line0 += of_lane(inc - my.line(a), in64);
      break;
    }
    line0 += of_lane(inc, 63);
    s0 += 64;
    if (s0 >= a.v.n_seq) return;
    my = SeqLanes(a, s0);
    inc = wave_sums(my.line(a));
  }

  const uint32_t krow = (uint32_t)a.nkv * kQ4RowBytes, srow = (uint32_t)a.nkv * kScaleRowBytes;
  const uint8_t *kd = a.L.kd + (size_t)hk * kQ4RowBytes, *vd = a.L.vd + (size_t)hk * kQ4RowBytes;
  const uint8_t *ksc = a.L.ks + (size_t)hk * kScaleRowBytes, *vsc = a.L.vs + (size_t)hk * kScaleRowBytes;
  uint8_t *const mine = sm + kWave * w;
  const uint32_t mine0 = lds_addr(sm) + kWave * w;
  // A lane's 16 bytes of the 8 keys that a load brings: key lane / 8, piece lane % 8 of V's row, that ^ key % 8 of K's (so
  // that 8 keys' pieces of one number lie in different banks)
  const uint32_t key8 = (uint32_t)lane >> 3, vcol = 16u * (lane & 7), kcol = 16u * ((lane & 7) ^ key8);
  const uint8_t *const scales = lane < 32 ? ksc : vsc;      // the scales' load: K's keys by the lower lanes, V's by the others

  while (at < end) {
    // ---- the piece's part of one row block
    const int q0 = of_lane(my.q0, in64), nt = of_lane(my.nt, in64), len = of_lane(my.len, in64), steps = of_lane(my.steps, in64);
    const int blocks = nt * a.grp <= a.few ? of_lane(my.blocks, in64) : 0, seq = s0 + in64;
    const int way_in = a.way_in, long_steps = way_in + steps;
    if (at - line0 >= blocks * long_steps) {       // the next sequence
      line0 += blocks * long_steps;
      if (++in64 == 64) {
        in64 = 0;
        s0 += 64;
        if (s0 >= a.v.n_seq) break;
        my = SeqLanes(a, s0);
      } else if (s0 + in64 >= a.v.n_seq) {
        break;
      }
      continue;
    }
    const int R = nt * a.grp, rb = blocks == 1 ? 0 : (at - line0) / long_steps, x0 = at - line0 - rb * long_steps;
    const int x1 = min(long_steps, x0 + (end - at)), st0 = max(x0 - way_in, 0), st1 = max(x1 - way_in, 0), m4 = st1 - st0;
    at += x1 - x0;
    if (m4 == 0) continue;
    const int t0 = st0 + (int)((uint32_t)(m4 * w) / kSeqWaves), t1 = st0 + (int)((uint32_t)(m4 * (w + 1)) / kSeqWaves);
    const int last = max(keys_of(a, len) - 1, 0), before = len - nt;   // (the last key that there are bytes of; none: len - nt + tok < 0)
    // Blocks of 8 rows or fewer: columns n and n + 8 of the products are the same row, and one product of the outputs takes ph in
    // the one and pl in the other, whose sum the join forms
    const int r0 = kSeqBlock * rb, real = min(R - r0, kSeqBlock);
    const bool halves = real <= kSeqBlock / 2;
    const int col = halves ? n & 7 : n, row = min(r0 + col, R - 1), tok = a.by_grp.div(row);
    const int lim = min(before + tok, last) + 1;   // keys below it are seen
    const int lim_all = min(before + a.by_grp.div(r0), last) + 1;   // by all rows of the block

    // ---- a step's bytes on their way: 9 loads straight into LDS, and before them, in pages, the next step's table entries (a
    // load into a register would be waited for with everything that is on its way)
    constexpr int NL = PG ? 10 : 9;
    uint32_t there = ~0u, there_next = ~0u;        // keys whose pages are in the pool: this step's, the next's
    const int32_t *const table = PG ? a.v.tables + (int64_t)seq * a.v.table_stride : nullptr;
    auto ask_entries = [&](int t) {
      const uint32_t key = PG == 2 ? min((uint32_t)t * kSeqKeys + ((uint32_t)lane & 31), (uint32_t)last) : (uint32_t)t * kSeqKeys;
      load4_to_lds(reinterpret_cast<const uint8_t *>(table + a.by_page.div(key)), __builtin_amdgcn_readfirstlane(lds_addr(s_tab[2 * w + (t & 1)])));
    };
    auto request = [&](int t) {                    // (of its entries, asked for before)
      const uint32_t kb = (uint32_t)t * kSeqKeys, dst = mine0 + kStep * (t & 1), left = (uint32_t)last - kb;
      uint32_t entry = 0;
      if constexpr (PG != 0) {
        if (t != t0) asm volatile("s_waitcnt vmcnt(9)" ::: "memory");   // (what was asked for since its entries: a step)
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        entry = (uint32_t)s_tab[2 * w + (t & 1)][lane];
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(entry)::"memory");
        ask_entries(min(t + 1, t1 - 1));           // (always one, for the counts of what is on its way)
      }
      if constexpr (PG == 2) {
        const uint32_t key = min(kb + ((uint32_t)lane & 31), (uint32_t)last);
        const int sl = entry < (uint32_t)a.v.pool_pages ? (int)(entry * (uint32_t)a.v.page + a.by_page.rest(key, a.v.page)) : -1;
        there_next = (uint32_t)__ballot(sl >= 0);
        size_t slot[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) slot[u] = (size_t)max(__shfl(sl, 8 * u + (int)key8), 0);
        load_to_lds_at<0>(kd + slot[0] * krow + kcol, dst);
        load_to_lds_at<1024>(kd + slot[1] * krow + kcol, dst);
        load_to_lds_at<2048>(kd + slot[2] * krow + kcol, dst);
        load_to_lds_at<3 * 1024>(kd + slot[3] * krow + kcol, dst);
        load_to_lds_at<oKS>(scales + (size_t)max(sl, 0) * srow, dst);
        load_to_lds_at<oV>(vd + slot[0] * krow + vcol, dst);
        load_to_lds_at<oV + 1024>(vd + slot[1] * krow + vcol, dst);
        load_to_lds_at<oV + 2048>(vd + slot[2] * krow + vcol, dst);
        load_to_lds_at<oV + 3 * 1024>(vd + slot[3] * krow + vcol, dst);
      } else {
        uint32_t base = kb;
        if constexpr (PG == 1) {
          const uint32_t b = (uint32_t)__builtin_amdgcn_readfirstlane((int)entry);
          there_next = b < (uint32_t)a.v.pool_pages ? ~0u : 0u;
          base = there_next ? b * (uint32_t)a.v.page + a.by_page.rest(kb, a.v.page) : 0;
        }
        const uint8_t *const kp = kd + (uint64_t)base * krow, *const vp = vd + (uint64_t)base * krow;
        uint32_t at[4] = {key8, key8 + 8, key8 + 16, key8 + 24}, sk = lane & 31;
        if (left < kSeqKeys - 1) {                 // (the last step: keys past the end take the last one's bytes)
#pragma unroll
          for (int u = 0; u < 4; ++u) at[u] = min(at[u], left);
          sk = min(sk, left);
        }
        load_to_lds_at<0>(kp, at[0] * krow + kcol, dst);
        load_to_lds_at<1024>(kp, at[1] * krow + kcol, dst);
        load_to_lds_at<2048>(kp, at[2] * krow + kcol, dst);
        load_to_lds_at<3 * 1024>(kp, at[3] * krow + kcol, dst);
        load_to_lds_at<oKS>(scales + (uint64_t)(base + sk) * srow, dst);
        load_to_lds_at<oV>(vp, at[0] * krow + vcol, dst);
        load_to_lds_at<oV + 1024>(vp, at[1] * krow + vcol, dst);
        load_to_lds_at<oV + 2048>(vp, at[2] * krow + vcol, dst);
        load_to_lds_at<oV + 3 * 1024>(vp, at[3] * krow + vcol, dst);
      }
    };
    // ---- the block's rows of Q, two by each wave, whole rows at a time (a lane's pieces of a row would ask for each line
    // four times, in every wave), into the place of the second step; piece c of row r at c ^ r % 8
    const uint32_t q_at = kStep * ((t0 & 1) ^ 1);
    if (PG && t0 < t1) ask_entries(t0);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = min(r0 + 2 * w + j, R - 1), ti = a.by_grp.div(r);
      load_to_lds(reinterpret_cast<const uint8_t *>(a.q.at(q0 + ti, hk * a.grp + r - ti * a.grp)) + 16 * (lane ^ ((2 * w + j) & 7)),
                  __builtin_amdgcn_readfirstlane(mine0 + q_at + 1024 * j));
    }
    if (t0 < t1) {
      request(t0);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(9) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    lds_barrier();
    h8 qh[8];                                      // row n, dims 64 g + 8 c ..
    {
      // (row col lies with wave col / 2, whose second step's place is its own)
      const int wt0 = st0 + (int)((uint32_t)(m4 * (col >> 1)) / kSeqWaves);
      const uint8_t *q = sm + kWave * (col >> 1) + kStep * ((wt0 & 1) ^ 1) + 1024 * (col & 1);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float4 x = *reinterpret_cast<const float4 *>(q + 16 * ((16 * g + 2 * c) ^ (col & 7))), y = *reinterpret_cast<const float4 *>(q + 16 * ((16 * g + 2 * c + 1) ^ (col & 7)));
        qh[c] = h8{(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w, (_Float16)y.x, (_Float16)y.y, (_Float16)y.z, (_Float16)y.w};
      }
    }
    lds_barrier();
    f4 o[16] = {};
    float m = -INFINITY, l = 0.0f;                 // m: the reference less kPScale

    auto sweep = [&](auto in_halves) {
    constexpr bool HALVES = decltype(in_halves)::value;
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      const int kb = t * kSeqKeys;
      const uint8_t *const at_k = mine + kStep * (t & 1), *const at_v = at_k + oV;
      there = there_next;
      if (t + 1 < t1) {
        request(t + 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      // all of the step's bytes to registers at once: its LDS latency once
      auto key_of = [&](int j) { return (j & 4) * 4 + 4 * g + (j & 3); };
      uint4 kr[2][2];
      uint32_t ks[2];
      uint2 vr[8];
      uint32_t vs[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        ks[u] = *reinterpret_cast<const uint32_t *>(at_k + oKS + 16 * (16 * u + n) + 4 * g);
#pragma unroll
        for (int i = 0; i < 2; ++i) kr[u][i] = *reinterpret_cast<const uint4 *>(at_k + kQ4RowBytes * (16 * u + n) + 16 * ((2 * g + i) ^ (n & 7)));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) vr[j] = *reinterpret_cast<const uint2 *>(at_v + kQ4RowBytes * key_of(j) + 8 * n);
#pragma unroll
      for (int j = 0; j < 8; ++j) vs[j] = *reinterpret_cast<const uint16_t *>(at_k + oVS + 16 * key_of(j) + 2 * (n >> 1));
      __builtin_amdgcn_sched_barrier(0);
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
        for (int i = 0; i < 8; ++i) s[u] = mfma16(bits.eight((&kr[u][i >> 2].x)[i & 3], d[i >> 2], c[i >> 2]), qh[i], s[u]);
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
        const float mn = top > m + (kLift + kPScale) ? top - kPScale : m;   // (by the row alone: others leave it as it is)
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
      if (HALVES) ph = n < 8 ? ph : pl;
      __builtin_amdgcn_s_setprio(0);               // (the other wave's scores go first: the two take turns)
      // ---- P V
      h2 d[4], c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d[j] = as_h2(q4_scales(vs[2 * j] | (vs[2 * j + 1] << 16)));
        c[j] = q4_offset(d[j]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {                // a 16-bit half of the lane's two words: dims 8 (e / 2) + e % 2 + 0, 2, 4, 6
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = __builtin_amdgcn_perm(e & 2 ? vr[2 * j + 1].y : vr[2 * j + 1].x, e & 2 ? vr[2 * j].y : vr[2 * j].x, e & 1 ? 0x07060302u : 0x05040100u);
        // (two products' small parts, then their large ones: a product does not wait for the one before it)
        auto products = [&](const h2 (&v)[4], const h2 (&z)[4], int i) {
          const int dt = 8 * (e >> 1) + 2 * i + (e & 1);
          const h8 vh = __builtin_bit_cast(h8, make_uint4(as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3])));
          const h8 zh = __builtin_bit_cast(h8, make_uint4(as_u(z[0]), as_u(z[1]), as_u(z[2]), as_u(z[3])));
          if constexpr (!HALVES) {
            o[dt] = mfma16(vh, pl, o[dt]);
            o[dt + 2] = mfma16(zh, pl, o[dt + 2]);
          }
          o[dt] = mfma16(vh, ph, o[dt]);
          o[dt + 2] = mfma16(zh, ph, o[dt + 2]);
        };
        const h2 v0[4] = {bits.pair<0>(x[0], d[0], c[0]), bits.pair<0>(x[1], d[1], c[1]), bits.pair<0>(x[2], d[2], c[2]), bits.pair<0>(x[3], d[3], c[3])};
        const h2 v1[4] = {bits.pair<1>(x[0], d[0], c[0]), bits.pair<1>(x[1], d[1], c[1]), bits.pair<1>(x[2], d[2], c[2]), bits.pair<1>(x[3], d[3], c[3])};
        products(v0, v1, 0);
        const h2 v2[4] = {bits.pair<2>(x[0], d[0], c[0]), bits.pair<2>(x[1], d[1], c[1]), bits.pair<2>(x[2], d[2], c[2]), bits.pair<2>(x[3], d[3], c[3])};
        const h2 v3[4] = {bits.pair<3>(x[0], d[0], c[0]), bits.pair<3>(x[1], d[1], c[1]), bits.pair<3>(x[2], d[2], c[2]), bits.pair<3>(x[3], d[3], c[3])};
        products(v2, v3, 2);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the step's place is the next request's)
      __builtin_amdgcn_s_setprio(1);
    }
    };
    if (halves) sweep(std::true_type{});
    else sweep(std::false_type{});

    // (what only the end needs is read here, and holds no register before)
    const SeqsAttnArgs z = arguments_again<SeqsAttnArgs>();
    // ---- the waves' parts joined
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) s_m[w][n] = m;
    __syncthreads();
    float *const s_o = reinterpret_cast<float *>(sm);
    constexpr int kWF = kWave / 4;                 // (a wave's rows in the place of its steps)
    {
      float mm = s_m[0][n];
#pragma unroll
      for (int j = 1; j < kSeqWaves; ++j) mm = fmaxf(mm, s_m[j][n]);
      const float f = m == -INFINITY ? 0.0f : exp2f(m - mm);
      if (g == 0) s_l[w][n] = l * f;
#pragma unroll
      for (int dt = 0; dt < 16; ++dt) o[dt] *= f;
      if (halves) {                                // (the large parts' sums and the small parts')
#pragma unroll
        for (int dt = 0; dt < 16; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[dt][i] += dpp<0x128>(o[dt][i]);
      }
      if (n < real) {
#pragma unroll
        for (int dt = 0; dt < 16; dt += 4)         // (4 products' dims are neighbours)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4 *>(&s_o[kWF * w + n * kOS + 16 * (4 * g + i) + dt]) = make_float4(o[dt][i], o[dt + 1][i], o[dt + 2][i], o[dt + 3][i]);
      }
    }
    __syncthreads();
    const bool alone = m4 == steps;
    // the row block's pieces, this one among them, and where partial results of piece i lie
    const int tile_line = line0 + rb * long_steps + way_in;
    const int first = alone ? piece : cut.piece_of(tile_line), count = alone ? 1 : cut.piece_of(tile_line + steps - 1) - first + 1;
    // (a piece is the first of one cut row block, whose beginning it holds the last of, and a later one of one other)
    auto part_of = [&](int i) { return (uint32_t)((2 * (first + i) + (i == 0)) * z.nkv + hk); };
    // (two dims a thread: 4 rows are the whole workgroup's)
    for (int x = threadIdx.x; x < real * (kHd / 2); x += NT) {
      const int jr = x / (kHd / 2), col = 2 * (x % (kHd / 2));
      float v[2] = {}, lr = 0.0f;
#pragma unroll
      for (int j = 0; j < kSeqWaves; ++j) {
        const float2 y = *reinterpret_cast<const float2 *>(&s_o[kWF * j + jr * kOS + col]);
        v[0] += y.x; v[1] += y.y;
        lr += s_l[j][jr];
      }
      if (alone) {
        const int ti = z.by_grp.div(r0 + jr);
        write_out(z, q0 + ti, hk * z.grp + r0 + jr - ti * z.grp, col, v, lr);
      } else {
        const uint32_t p = part_of(piece - first) * kSeqBlock + jr;
        st_part(z.part + (int64_t)p * kHd + col, make_float2(v[0], v[1]));
        if (col == 0) {
          float mr = s_m[0][jr];
#pragma unroll
          for (int j = 1; j < kSeqWaves; ++j) mr = fmaxf(mr, s_m[j][jr]);
          st_part(z.ml + p, make_float2(mr, lr));
        }
      }
    }
    // ---- the pieces joined: 8 at a time, then those
    if (!alone) {
      int mine = piece - first, groups = count, unit = 1;   // this one among the results of a level; pieces that one stands for
      for (unsigned *counters = z.count;; counters += 2 * kSeqFill) {
        const int g0 = mine / kJoin * kJoin, size = min(kJoin, groups - g0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // (the results are in memory)
        __syncthreads();
        unsigned *const counter = counters + part_of(g0 * unit);
        if (threadIdx.x == 0) s_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)size - 1;
        __syncthreads();
        if (!s_last) break;
        if (threadIdx.x == 0) st_agent(counter, 0u);        // (for the next call)
        const bool done = size == groups;
        for (int x = threadIdx.x; x < real * (kHd / 2); x += NT) {
          const int jr = x / (kHd / 2), col = 2 * (x % (kHd / 2));
          float2 v[kJoin], ml[kJoin];
          float o2[2] = {};
#pragma unroll
          for (int j = 0; j < kJoin; ++j) {
            const uint32_t p = part_of((g0 + min(j, size - 1)) * unit) * kSeqBlock + jr;
            ml[j] = ld_part(z.ml + p);
            v[j] = ld_part(z.part + (int64_t)p * kHd + col);
          }
          float mr = ml[0].x, lr = 0.0f;
#pragma unroll
          for (int j = 1; j < kJoin; ++j) mr = fmaxf(mr, ml[j].x);
#pragma unroll
          for (int j = 0; j < kJoin; ++j) {
            const float f = j >= size || ml[j].x == -INFINITY ? 0.0f : exp2f(ml[j].x - mr);
            if (j < size) {
              lr = fmaf(ml[j].y, f, lr);
              o2[0] = fmaf(v[j].x, f, o2[0]);
              o2[1] = fmaf(v[j].y, f, o2[1]);
            }
          }
          if (done) {
            const int ti = z.by_grp.div(r0 + jr);
            write_out(z, q0 + ti, hk * z.grp + r0 + jr - ti * z.grp, col, o2, lr);
          } else {                                 // in the place of its first: what a thread writes it alone has read,
            const uint32_t p = part_of(g0 * unit) * kSeqBlock + jr;
            st_part(z.part + (int64_t)p * kHd + col, make_float2(o2[0], o2[1]));
            s_o[2 * jr] = mr;                      // but for the reference and the sum, written behind a barrier
            s_o[2 * jr + 1] = lr;
          }
        }
        if (done) break;
        __syncthreads();
        if (threadIdx.x < real)
          st_part(z.ml + part_of(g0 * unit) * kSeqBlock + threadIdx.x, make_float2(s_o[2 * threadIdx.x], s_o[2 * threadIdx.x + 1]));
        mine /= kJoin;
        groups = (groups + kJoin - 1) / kJoin;
        unit *= kJoin;
      }
    }
    __syncthreads();                               // (LDS is the next part's)
  }
}

// ------------------------------------------------------------------ many rows: key tiles in LDS
// 4 waves hold 32 rows each, with all 256 outputs of a row in registers, and step through the even 32-key steps of the
// workgroup's piece; 4 more waves have the same rows and the odd steps, and the two halves of the outputs meet in LDS at the
// end. (As two workgroups, each a piece of its own, they read Q and write partial results twice.) A step's cache bytes are
// loaded straight into LDS two rounds ahead and turned once into the products' operands for all 128 rows, the round before
// they are wanted: K as it is, V transposed, so that a lane's 8 keys of one dim are 16 bytes. (Were the one four to turn bytes
// at a round's beginning and the other at its end, pages of 48 tokens would take 120 us instead of 103, a round's bytes being
// asked for later.) S^T and O^T are formed as in the kernel above, P never leaves its lane.
//
// What bounds it: 96 matrix instructions (16 cycles) and 480 vector ones (4) a wave and step, of which little runs side by side:
// the two waves of a SIMD reach the same phase together, and a round of two steps takes 8.2 thousand cycles where the sum
// is 6.9. The way in and out is 15 us, 128 KB of partial results a piece among it. 512 tokens of 16 heads onto 8,192
// positions 140 us (0.5 PFLOP/s of the formula's operations).
//
// LDS positions, in 16-byte pieces: K piece c (8 dims) of key k at 32 k + (c ^ k % 16); V piece g of dim d (keys 4 g .. 4 g + 3
// and 16 + 4 g .. 16 + 4 g + 3) at 4 d + (g ^ vx(d)); both so that 8 neighbouring lanes' reads and writes lie in different banks.
constexpr int kTileRows = 128, kTileWaves = 8, kTileLeast = 16;
constexpr int kTileFill = 256;         // pieces of all KV heads: a workgroup a CU
constexpr int kTileShort = 4;          // steps of a piece of a tile at least, where tiles are cut
constexpr int kTileWayIn = 8;          // steps that a tile's way in and out takes as long as
__device__ __forceinline__ uint32_t v_piece(int d, int g) { return (uint32_t)(64 * d + 16 * (g ^ (((d >> 1) ^ (d >> 3)) & 3))); }

// tiles of a sequence, and steps of tile rb: up to its last row's last key (one at least)
struct Tiles {
  int nt, len, grp, most;                          // most: positions that the cache has room for
  __device__ __forceinline__ int count() const { return (int)((uint32_t)(nt * grp + kTileRows - 1) / kTileRows); }
  __device__ __forceinline__ int steps(const ByConst &by_grp, int rb) const {
    const int toks = min(nt, by_grp.div((uint32_t)(kTileRows * (rb + 1) + grp - 1)));
    return (int)((uint32_t)(min(max(len - nt + toks, 1), most) + kSeqKeys - 1) / kSeqKeys);
  }
};

template <int PG>
__global__ __launch_bounds__(64 * kTileWaves, 2) void seqs_tile_kernel(SeqsAttnArgs a) {
  constexpr uint32_t kOp = kSeqKeys * 2 * kHd;     // an operand: 32 keys of 256 fp16
  // two steps' operands of K and of V; behind them the bytes as they came, each wave's own: 8 keys' rows of K, 64 dims of V,
  // 8 keys' scales of K, 2 blocks' scales of V
  constexpr uint32_t oVop = 2 * kOp, oRaw = 4 * kOp, kRawV = 1024, kRawKS = 2048, kRawVS = 2176, kRaw = 2304, kFour = oRaw + 4 * kRaw;
  __shared__ __attribute__((aligned(128))) uint8_t all[2 * kFour];   // (of each four waves)
  __shared__ float s_m[2][kTileRows], s_l[2][kTileRows];
  __shared__ int s_tile[kTileFill], s_steps[kTileFill];   // of up to as many tiles as pieces: sequence and number in it; steps
  __shared__ int s_seq[3][64];                     // rows' beginnings, tokens and lengths of the 64 sequences at hand
  __shared__ int32_t s_tab[PG ? kTileWaves : 1][64];
  arguments_near<SeqsAttnArgs>();
  const int lane = threadIdx.x & 63, w8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = w8 & 3, odd = w8 >> 2, n = lane & 15, g = lane >> 4;
  uint8_t *const sm = all + kFour * odd;
  const Q4Bits bits;
  // (the lane's number, opaque where addresses are formed from it: kept from step to step they would take the registers that
  // the outputs need)
  auto my_lane = [&]() {
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  const int at8 = (int)(blockIdx.x >> 3), round = a.by_nkv.div(at8), hk = at8 - round * a.nkv;
  // ---- the line: all tiles' steps, 64 sequences at a time
  auto line_of = [&](const SeqLanes &s) {
    const Tiles t{s.nt, s.len, a.grp, (int)a.v.max_pos};
    int sum = 0;
    if (s.nt * a.grp > a.few)
      for (int rb = 0; rb < t.count(); ++rb) sum += t.steps(a.by_grp, rb);
    return sum;
  };
  auto tiles_of = [&](const SeqLanes &s) { return s.nt * a.grp > a.few ? Tiles{s.nt, s.len, a.grp, (int)a.v.max_pos}.count() : 0; };
  SeqLanes my(a, 0);
  int mine_line = line_of(my), inc = wave_sums(mine_line), total = of_lane(inc, 63), n_tiles = of_lane(wave_sums(tiles_of(my)), 63);
  bool bad = my.bad;
  for (int s0 = 64; s0 < a.v.n_seq; s0 += 64) {
    const SeqLanes more(a, s0);
    total += of_lane(wave_sums(line_of(more)), 63);
    n_tiles += of_lane(wave_sums(tiles_of(more)), 63);
    bad |= more.bad;
  }
  if (bad || total == 0) return;
  const Cut cut(total, a.tile_lanes, a.by_tile_lanes, kTileLeast);
  // an XCD has neighbouring pieces: those of one tile read the same rows of Q, each of which comes to its L2 once
  int piece = 0;
  auto none = [&](int nl) {
    const int rounds = (nl + 7) / 8;
    piece = rounds * (int)(blockIdx.x & 7) + round;
    return round >= rounds || piece >= nl;
  };
  int at = 0, end = 0, s0 = 0, in64 = 0, line0 = 0, rb = 0;   // the sequence and tile that `at` lies in, and where that begins
  // ---- Where there are no more tiles than pieces: each tile cut into equal pieces, the longest of which are as short as their
  // number allows, so that a piece has one way in and out. (Unless the longest have more than another way in and out over an
  // equal share.)
  int parts = 0;                                   // of the tile, 0: the line is cut
  if (n_tiles <= a.tile_lanes) {
    if (w8 == 0) {
      int before = 0;
      for (int q = 0; q < a.v.n_seq; q += 64) {
        const SeqLanes s(a, q);
        const Tiles t{s.nt, s.len, a.grp, (int)a.v.max_pos};
        const int c = tiles_of(s), c_inc = wave_sums(c);
        for (int i = 0; i < c; ++i) {
          s_tile[before + c_inc - c + i] = (q + lane) << 8 | i;
          s_steps[before + c_inc - c + i] = t.steps(a.by_grp, i);
        }
        before += of_lane(c_inc, 63);
      }
    }
    lds_barrier();
    constexpr int NC = kTileFill / 64;
    int st[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) st[j] = 64 * j + lane < n_tiles ? s_steps[64 * j + lane] : 0;
    // pieces of x steps of s at most (s is no less than an equal share: the quotient is small, and its error less than 1)
    auto pieces_of = [&](int x, int s) {
      const int y = x + s - 1;
      int n = (int)((float)y * (1.0f / (float)s));
      n += (n + 1) * s <= y ? 1 : 0;
      return n - (n * s > y ? 1 : 0);
    };
    auto in_all = [&](int s) {
      int n = 0;
#pragma unroll
      for (int j = 0; j < NC; ++j) n += pieces_of(st[j], s);
      return of_lane(wave_sums(n), 63);
    };
    int lo = max(kTileShort, (int)((uint32_t)(total + a.tile_lanes - 1) / (uint32_t)a.tile_lanes)), hi = lo + kTileWayIn;
    if (in_all(hi) <= a.tile_lanes) {
      while (lo < hi) {                            // (the least that is enough: hi always is)
        const int mid = (lo + hi) / 2;
        if (in_all(mid) <= a.tile_lanes) hi = mid;
        else lo = mid + 1;
      }
      if (none(in_all(hi))) return;
      int before = 0, tile = 0, steps = 0;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int k = pieces_of(st[j], hi), k_inc = wave_sums(k);
        const uint64_t past = __ballot(before + k_inc > piece);
        if (parts == 0 && past) {
          const int l = __ffsll((unsigned long long)past) - 1;
          tile = 64 * j + l;
          steps = of_lane(st[j], l);
          parts = of_lane(k, l);
          at = piece - (before + of_lane(k_inc - k, l));
        }
        before += of_lane(k_inc, 63);
      }
      const int each = steps / parts, longer = steps - each * parts, part = at;
      at = part * each + min(part, longer);
      end = at + each + (part < longer ? 1 : 0);
      const int where = __builtin_amdgcn_readfirstlane(s_tile[tile]);
      rb = where & 255;
      in64 = (where >> 8) & 63;
      s0 = (where >> 8) - in64;
      if (s0) my = SeqLanes(a, s0);
    }
  }
  // A piece of the line that would begin or end a little inside a tile begins or ends at the tile's own end: its rows' way in and out costs
  // as much as near steps (15 sequences with chunks among them: 92 us; with an eighth of a piece 101).
  const int near = parts ? -1 : min(cut.share / 4, 8);
  auto last_piece = [&](int begin, int steps) {    // of a tile
    const int p = cut.piece_of(begin + steps - 1), b = cut.begin(p);
    return b > begin && b - begin > near && begin + steps - b <= near ? p - 1 : p;
  };
  if (!parts) {
    if (none(cut.nl)) return;
    at = cut.begin(piece);
    end = cut.begin(piece + 1);
    for (;;) {
      const uint64_t past = __ballot(line0 + inc > at);
      if (past) {
        in64 = __ffsll((unsigned long long)past) - 1;
        line0 += of_lane(inc - mine_line, in64);
        break;
      }
      line0 += of_lane(inc, 63);
      s0 += 64;
      if (s0 >= a.v.n_seq) return;
      my = SeqLanes(a, s0);
      mine_line = line_of(my);
      inc = wave_sums(mine_line);
    }
    // the tile of that sequence: 64 at a time
    {
      const Tiles t{of_lane(my.nt, in64), of_lane(my.len, in64), a.grp, (int)a.v.max_pos};
      for (;;) {
        const int i = rb + lane, st = i < t.count() ? t.steps(a.by_grp, i) : 0, tinc = wave_sums(st);
        const uint64_t past = __ballot(line0 + tinc > at);
        if (past) {
          const int l = __ffsll((unsigned long long)past) - 1;
          line0 += of_lane(tinc - st, l);
          rb += l;
          break;
        }
        line0 += of_lane(tinc, 63);
        rb += 64;
        if (rb >= t.count()) return;
      }
    }
  }
  bool first = true;
  auto keep = [&](const SeqLanes &x) {             // (by every wave alike)
    s_seq[0][lane] = x.q0;
    s_seq[1][lane] = x.nt;
    s_seq[2][lane] = x.len;
  };
  keep(my);
  lds_barrier();

  const uint32_t krow = (uint32_t)a.nkv * kQ4RowBytes, srow = (uint32_t)a.nkv * kScaleRowBytes;
  const uint8_t *kd = a.L.kd + (size_t)hk * kQ4RowBytes, *vd = a.L.vd + (size_t)hk * kQ4RowBytes;
  const uint8_t *ksc = a.L.ks + (size_t)hk * kScaleRowBytes, *vsc = a.L.vs + (size_t)hk * kScaleRowBytes;
  uint8_t *const raw = sm + oRaw + kRaw * w;
  const uint32_t raw0 = lds_addr(sm) + oRaw + kRaw * w;
  // Where the lane finds its bytes and puts its operands. K: words i + 8 j of key 8 w + k lie in raw piece (i / 4 + 2 j) ^ k and go
  // to piece (i + 8 j) ^ key % 16: the number j changes bits by itself. V: dims d0 + 2 s, whose piece's place s changes likewise.
  const int lk = lane >> 3, li = lane & 7;
  const uint32_t k_raw = 128 * lk + 16 * ((li >> 2) ^ lk) + 4 * (li & 3);
  const uint32_t k_op = 512 * (8 * w + lk) + 16 * (li ^ lk) + 128 * (w & 1);
  const uint32_t v_raw = kRawV + 32 * g + 2 * n;
  const uint32_t v_op = 64 * (64 * w + 8 * (n >> 1) + (n & 1)) + 16 * (g ^ ((n >> 1) & 3));

  while (at < end) {
    // ---- the piece's part of one tile
    const int q0 = __builtin_amdgcn_readfirstlane(s_seq[0][in64]), nt = __builtin_amdgcn_readfirstlane(s_seq[1][in64]), len = __builtin_amdgcn_readfirstlane(s_seq[2][in64]), seq = s0 + in64;
    const Tiles tiles{nt, len, a.grp, (int)a.v.max_pos};
    if (nt * a.grp <= a.few || rb == tiles.count()) {   // the next sequence
      rb = 0;
      if (++in64 == 64) {
        in64 = 0;
        s0 += 64;
        if (s0 >= a.v.n_seq) break;
        lds_barrier();
        keep(SeqLanes(a, s0));
        lds_barrier();
      } else if (s0 + in64 >= a.v.n_seq) {
        break;
      }
      continue;
    }
    const int R = nt * a.grp, steps = tiles.steps(a.by_grp, rb);
    // (the boundaries moved: of a piece's beginning in the first tile that it meets, of its end in the last)
    auto moved = [&](int x) { return x - line0 <= near ? line0 : line0 + steps - x <= near ? line0 + steps : x; };
    if (first && piece > 0) at = moved(at);
    first = false;
    const int stop = end < line0 + steps && piece + 1 < cut.nl ? moved(end) : end;
    if (at >= line0 + steps) {                     // (all of it is the piece's before)
      line0 += steps;
      ++rb;
      continue;
    }
    if (stop <= at) break;                         // (what is left of it is the next piece's)
    const int t0 = __builtin_amdgcn_readfirstlane(at - line0), t1 = __builtin_amdgcn_readfirstlane(min(steps, t0 + (stop - at)));
    const int last = max(keys_of(a, len) - 1, 0), before = len - nt, r0 = kTileRows * rb, rw = r0 + 32 * w;
    const bool works = rw < R;                     // (a wave whose rows are all past the last only brings bytes)
    // keys below lim are seen: by a row of the lane's, by all of the wave's, by any
    auto lim_of = [&](int mt) { return min(before + a.by_grp.div((uint32_t)min(rw + 16 * mt + (my_lane() & 15), R - 1)), last) + 1; };
    const int lim_all = min(before + a.by_grp.div((uint32_t)min(rw, R - 1)), last) + 1, lim_any = min(before + a.by_grp.div((uint32_t)min(rw + 31, R - 1)), last) + 1;

    // ---- bytes on their way: the wave's own, of step t
    uint32_t there = ~0u, there_next = ~0u;        // keys whose pages are in the pool: this step's, the next's
    const int32_t *const table = PG ? a.v.tables + (int64_t)seq * a.v.table_stride : nullptr;
    auto ask_entries = [&](int t) {
      const int lane = my_lane();
      const uint32_t key = PG == 2 ? min((uint32_t)t * kSeqKeys + ((uint32_t)lane & 31), (uint32_t)last) : min((uint32_t)t * kSeqKeys, (uint32_t)last);
      load4_to_lds(reinterpret_cast<const uint8_t *>(table + a.by_page.div(key)), __builtin_amdgcn_readfirstlane(lds_addr(s_tab[PG ? w8 : 0])));
    };
    // V's keys lie in the order of the contraction's slots: place 4 j + g is slot (g, j), so that the 4 groups' reads of one j
    // are neighbours
    auto key_of = [](int p) { return (p & 16) + 4 * (p & 3) + ((p >> 2) & 3); };
    uint32_t there_after = ~0u;
    auto request = [&](int t) {                    // (of its entries, landed)
      const int lane = my_lane();
      const uint32_t kb = (uint32_t)t * kSeqKeys, left = (uint32_t)last - min(kb, (uint32_t)last);
      const int kk = 8 * w + (lane >> 3), kv = key_of(lane >> 1), ksk = (8 * w + lane) & 31, kvs = key_of(lane & 31);
      if constexpr (PG == 2) {
        const uint32_t key = min(kb + ((uint32_t)lane & 31), (uint32_t)last), e = (uint32_t)s_tab[w8][lane];
        const int sl = e < (uint32_t)a.v.pool_pages ? (int)(e * (uint32_t)a.v.page + a.by_page.rest(key, a.v.page)) : -1;
        there_after = (uint32_t)__ballot(sl >= 0);
        const size_t sk = (size_t)max(__shfl(sl, kk), 0), sv = (size_t)max(__shfl(sl, kv), 0), s1 = (size_t)max(__shfl(sl, ksk), 0), s2 = (size_t)max(__shfl(sl, kvs), 0);
        load_to_lds_at<0>(kd + sk * krow + 16 * ((lane ^ (lane >> 3)) & 7), raw0);
        load_to_lds_at<kRawV>(vd + sv * krow + 32 * w + 16 * (lane & 1), raw0);
        if (lane < 8) load_to_lds_at<kRawKS>(ksc + s1 * srow, raw0);
        if (lane < 32) load4_to_lds(vsc + s2 * srow + 4 * w, __builtin_amdgcn_readfirstlane(raw0 + kRawVS));
      } else {
        uint32_t base = min(kb, (uint32_t)last);
        if constexpr (PG == 1) {
          const uint32_t e = (uint32_t)__builtin_amdgcn_readfirstlane(s_tab[w8][lane]);
          there_after = e < (uint32_t)a.v.pool_pages ? ~0u : 0u;
          base = there_after ? e * (uint32_t)a.v.page + a.by_page.rest(base, a.v.page) : 0;
        }
        const uint64_t off = (uint64_t)base * krow, soff = (uint64_t)base * srow;
        load_to_lds_at<0>(kd + off, min((uint32_t)kk, left) * krow + 16 * ((lane ^ (lane >> 3)) & 7), raw0);
        load_to_lds_at<kRawV>(vd + off, min((uint32_t)kv, left) * krow + 32 * w + 16 * (lane & 1), raw0);
        if (lane < 8) load_to_lds_at<kRawKS>(ksc + soff, min((uint32_t)ksk, left) * srow, raw0);
        if (lane < 32) load4_to_lds(vsc + soff + min((uint32_t)kvs, left) * srow + 4 * w, __builtin_amdgcn_readfirstlane(raw0 + kRawVS));
      }
    };
    // ---- the wave's bytes, landed, made into operands
    auto convert = [&](int buf) {
      typedef uint16_t u2 __attribute__((ext_vector_type(2)));
      uint32_t k_raw_ = k_raw, k_op_ = k_op, v_op_ = v_op;   // (opaque: their variants are formed here, not kept)
      asm volatile("" : "+v"(k_raw_), "+v"(k_op_), "+v"(v_op_));
      const int lane = my_lane();
      const uint32_t ks_raw = kRawKS + 16 * (lane >> 3), k_half = lane & 4 ? 0x03020302u : 0x01000100u, vs_raw = kRawVS + 4 * (lane >> 4) + 2 * ((lane >> 3) & 1);
      {                                            // K: words i, i + 8, .. of key lane / 8 (word i + 8 j: block 2 j + i / 4)
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const uint32_t *>(raw + (k_raw_ ^ (32u * j)));
        const uint4 sc = *reinterpret_cast<const uint4 *>(raw + ks_raw);
        uint8_t *const to = sm + kOp * buf;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t two = q4_scales((&sc.x)[j]);
          const h2 d = as_h2(__builtin_amdgcn_perm(two, two, k_half));
          *reinterpret_cast<h8 *>(to + (k_op_ ^ (128u * (j & 1))) + 256 * (j >> 1)) = bits.eight(x[j], d, q4_offset(d));
        }
      }
      {                                            // V: 4 dims of 8 keys: a half of word n / 2 of the wave's 8
        uint32_t x[4];
        h2 d[4], c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint8_t *const p = raw + v_raw + 256 * j, *const q = raw + vs_raw + 32 * j;
          x[j] = __builtin_bit_cast(uint32_t, u2{*reinterpret_cast<const uint16_t *>(p), *reinterpret_cast<const uint16_t *>(p + 128)});
          d[j] = as_h2(q4_scales(__builtin_bit_cast(uint32_t, u2{*reinterpret_cast<const uint16_t *>(q), *reinterpret_cast<const uint16_t *>(q + 16)})));
          c[j] = q4_offset(d[j]);
        }
        uint8_t *const to = sm + oVop + kOp * buf;
        auto put = [&](int s, const h2 (&v)[4]) {
          *reinterpret_cast<uint4 *>(to + (v_op_ ^ (16u * s)) + 128 * s) = make_uint4(as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3]));
        };
        put(0, {bits.pair<0>(x[0], d[0], c[0]), bits.pair<0>(x[1], d[1], c[1]), bits.pair<0>(x[2], d[2], c[2]), bits.pair<0>(x[3], d[3], c[3])});
        put(1, {bits.pair<1>(x[0], d[0], c[0]), bits.pair<1>(x[1], d[1], c[1]), bits.pair<1>(x[2], d[2], c[2]), bits.pair<1>(x[3], d[3], c[3])});
        put(2, {bits.pair<2>(x[0], d[0], c[0]), bits.pair<2>(x[1], d[1], c[1]), bits.pair<2>(x[2], d[2], c[2]), bits.pair<2>(x[3], d[3], c[3])});
        put(3, {bits.pair<3>(x[0], d[0], c[0]), bits.pair<3>(x[1], d[1], c[1]), bits.pair<3>(x[2], d[2], c[2]), bits.pair<3>(x[3], d[3], c[3])});
      }
    };

    // ---- Q: 16 rows by each wave, to fp16 and through LDS (the operands' place), piece c of row r at c ^ r % 16
    if (PG) {
      ask_entries(min(t0 + odd, t1 - 1));
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    request(t0 + odd);
    there_next = there_after;
    h8 qh[2][8];
    {
      float4 x[16];
      const int first = r0 + 16 * w8;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int r = min(first + j, R - 1), ti = a.by_grp.div((uint32_t)r);
        x[j] = reinterpret_cast<const float4 *>(a.q.at(q0 + ti, hk * a.grp + r - ti * a.grp))[lane];
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const h2 lo = {(_Float16)x[j].x, (_Float16)x[j].y}, hi = {(_Float16)x[j].z, (_Float16)x[j].w};
        *reinterpret_cast<uint2 *>(all + 8192 * w8 + 512 * j + 16 * ((lane >> 1) ^ j) + 8 * (lane & 1)) = make_uint2(as_u(lo), as_u(hi));
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (PG) ask_entries(min(t0 + 2 + odd, t1 - 1));
    lds_barrier();                                 // (the rows are there)
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int b = 0; b < 8; ++b) qh[mt][b] = *reinterpret_cast<const h8 *>(all + 8192 * (2 * w + mt) + 512 * n + 16 * ((4 * b + g) ^ n));
    static_assert(8 * 8192 <= oRaw, "the rows end before the bytes that are on their way");
    f4 o[2][16] = {};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();                                 // (every wave has its rows)
    convert(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    auto ask = [&](int t) {                        // the bytes of step t, where there is one, and the entries of the one after it
      if (t >= t1) return;
      request(t);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (PG) ask_entries(min(t + 2, t1 - 1));
    };
    ask(t0 + 2 + odd);
    lds_barrier();

    // the next round's operands, in places whose readers have passed the barrier; then, with the wave's bytes used, those of
    // the round after it
    auto bring = [&](int t, int buf) {
      if (t + 2 < t1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        convert(buf ^ 1);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        ask(t + 4);
      }
    };
#pragma unroll 1
    for (int tt = t0; tt < t1; tt += 2) {          // (the same count in the whole workgroup)
      const int t = tt + odd, kb = t * kSeqKeys, buf = ((tt - t0) >> 1) & 1;
      there = there_next;
      there_next = there_after;
      if (works && t < t1 && kb < lim_any) {
        const int lane = my_lane(), n = lane & 15, g = lane >> 4;
        const uint8_t *const kop = sm + kOp * buf + 512 * n, *const vop = sm + oVop + kOp * buf + 64 * n;
        const uint32_t kx = 16 * (g ^ n);          // piece 4 b + g at (4 b + g) ^ n
        const uint32_t vx[2] = {v_piece(n, g) - 64 * n, v_piece(16 + n, g) - 64 * (16 + n)};
        auto k_at = [&](int ub) { return *reinterpret_cast<const h8 *>(kop + (kx ^ (64u * (ub & 3))) + 8192 * (ub >> 3) + 256 * ((ub & 7) >> 2)); };
        auto v_at = [&](int dt) { return *reinterpret_cast<const h8 *>(vop + vx[dt & 1] + 1024 * dt); };
        const bool whole = kb + kSeqKeys <= lim_all && (!PG || there == ~0u);
        // ---- scores
        // (the operands of product ub + AK are asked for before product ub, and no further ahead: the registers hold no more)
        constexpr int AK = 2;
        f4 s[2][2] = {};
        h8 kf[AK + 1];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < AK; ++j) kf[j] = k_at(j);
#pragma unroll
        for (int ub = 0; ub < 16; ++ub) {
          if (ub + AK < 16) kf[(ub + AK) % (AK + 1)] = k_at(ub + AK);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) s[mt][ub >> 3] = mfma16(kf[ub % (AK + 1)], qh[mt][ub & 7], s[mt][ub >> 3]);
          __builtin_amdgcn_sched_barrier(0);
        }
        // ---- probabilities
        h8 ph[2], pl[2];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t win = ~0u;
          if (!whole) {
            const int seen = lim_of(mt) - kb;
            win = there & (seen <= 0 ? 0u : seen >= 32 ? ~0u : (1u << seen) - 1u);
            win >>= 4 * g;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (!((win >> ((j & 4) * 4 + (j & 3))) & 1u)) s[mt][j >> 2][j & 3] = -INFINITY;
          }
          float top = fmaxf(fmaxf(fmaxf(s[mt][0][0], s[mt][0][1]), fmaxf(s[mt][0][2], s[mt][0][3])),
                            fmaxf(fmaxf(s[mt][1][0], s[mt][1][1]), fmaxf(s[mt][1][2], s[mt][1][3]))) * a.scale2;
          if (__any(top > m[mt] + (kLift + kPScale))) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float mn = top > m[mt] + (kLift + kPScale) ? top - kPScale : m[mt];   // (by the row alone: others leave it as it is)
            const float f = mn == m[mt] ? 1.0f : exp2f(m[mt] - mn);
            m[mt] = mn;
            l[mt] *= f;
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) o[mt][dt] *= f;
          }
          float p[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][j >> 2][j & 3], a.scale2, -m[mt]));
          if (!whole) {                            // (where nothing was seen yet, -Inf - -Inf)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (!((win >> ((j & 4) * 4 + (j & 3))) & 1u)) p[j] = 0.0f;
          }
          l[mt] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
          split_p(p, ph[mt], pl[mt]);
        }
        // ---- P V
        constexpr int AV = 2;
        h8 vf[AV + 1];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < AV; ++j) vf[j] = v_at(j);
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) {
          if (dt + AV < 16) vf[(dt + AV) % (AV + 1)] = v_at(dt + AV);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) o[mt][dt] = mfma16(vf[dt % (AV + 1)], pl[mt], o[mt][dt]);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) o[mt][dt] = mfma16(vf[dt % (AV + 1)], ph[mt], o[mt][dt]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      bring(t, buf);
      lds_barrier();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    const SeqsAttnArgs z = arguments_again<SeqsAttnArgs>();
    // ---- the two fours' outputs joined: each sends the half of the dims that the other finishes
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      l[mt] += __shfl_xor(l[mt], 16);
      l[mt] += __shfl_xor(l[mt], 32);
      if (g == 0) { s_m[odd][32 * w + 16 * mt + n] = m[mt]; s_l[odd][32 * w + 16 * mt + n] = l[mt]; }
    }
    lds_barrier();
    float f[2], by[2];                             // of the wave's own outputs; the sums
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const float mo = s_m[odd ^ 1][32 * w + 16 * mt + n], mm = fmaxf(m[mt], mo), fo = mo == -INFINITY ? 0.0f : exp2f(mo - mm);
      f[mt] = m[mt] == -INFINITY ? 0.0f : exp2f(m[mt] - mm);
      by[mt] = (m[mt] == -INFINITY && l[mt] == 0.0f ? 0.0f : l[mt] * f[mt]) + (mo == -INFINITY ? 0.0f : s_l[odd ^ 1][32 * w + 16 * mt + n] * fo);
      m[mt] = mm;
    }
    auto send = [&](auto from) {                   // 16 bytes a lane and product, one after another
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
          *reinterpret_cast<f4 *>(all + 65536 * odd + 16384 * w + 1024 * (8 * mt + dt) + 16 * lane) = o[mt][decltype(from)::value + dt] * f[mt];
    };
    if (odd) send(std::integral_constant<int, 0>{});
    else send(std::integral_constant<int, 8>{});
    lds_barrier();
    static_assert(2 * 65536 <= 2 * kFour, "the outputs in the operands' place");
    // ---- the outputs, or a partial result for each row of a tile that several pieces share
    const bool alone = t1 - t0 == steps;
    // (a piece leaves partial results of two tiles at most: the one that it begins inside, and the one whose beginning it has
    // but not its end)
    const uint32_t part0 = ((uint32_t)(2 * piece + (t0 == 0)) * z.nkv + hk) * kTileRows + 32 * w;
    auto finish = [&](auto from) {
      constexpr int D0 = decltype(from)::value;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int r = rw + 16 * mt + n, ti = z.by_grp.div((uint32_t)min(r, R - 1)), h = hk * z.grp + min(r, R - 1) - ti * z.grp;
        const int64_t dst = (int64_t)(q0 + ti) * z.nh + h;
        const uint32_t part = part0 + 16 * mt + n;
        const float sum = by[mt], div = !alone ? 1.0f : sum > 0.0f || sum != sum ? sum : 1.0f;
        if (D0 == 0 && r < R && g == 0) {
          if (t0 == 0) z.info[dst] = make_uint4(part, 2u * (uint32_t)z.nkv * kTileRows, (uint32_t)(alone ? 1 : parts ? parts : last_piece(line0, steps) - piece + 1), 0);
          if (!alone) z.tile_ml[part] = make_float2(m[mt], sum);
        }
        // lanes n and n ^ 1 exchange halves of two products, so that a store reaches 8 rows' whole lines
        const bool odd_n = n & 1;
        float *const mine = r < R ? (alone ? z.out + dst * kHd : z.tile_part + (int64_t)part * kHd) : nullptr;
        const uint64_t other = __shfl_xor((unsigned long long)(uintptr_t)mine, 1);
        float *const even_row = odd_n ? (float *)(uintptr_t)other : mine, *const odd_row = odd_n ? mine : (float *)(uintptr_t)other;
        const float *const gate = z.gate.p && alone && r < R ? z.gate.at(q0 + ti, h) : nullptr;
        const uint64_t gother = __shfl_xor((unsigned long long)(uintptr_t)gate, 1);
        const float *const even_gate = odd_n ? (const float *)(uintptr_t)gother : gate, *const odd_gate = odd_n ? gate : (const float *)(uintptr_t)gother;
#pragma unroll
        for (int dt = 0; dt < 8; dt += 2) {
          const uint8_t *const in = all + 65536 * (odd ^ 1) + 16384 * w + 1024 * (8 * mt + dt) + 16 * lane;
          f4 v0 = o[mt][D0 + dt] * f[mt] + *reinterpret_cast<const f4 *>(in), v1 = o[mt][D0 + dt + 1] * f[mt] + *reinterpret_cast<const f4 *>(in + 1024);
          if (alone) { v0 /= div; v1 /= div; }
          f4 e, d;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = dpp<0xB1>(odd_n ? v0[i] : v1[i]);      // the other row's half
            e[i] = odd_n ? x : v0[i];
            d[i] = odd_n ? v1[i] : x;
          }
          const int col = 16 * (D0 + dt + (odd_n ? 1 : 0)) + 4 * g;
          auto write = [&](float *row, const float *gt, f4 v) {
            if (!row) return;
            *reinterpret_cast<f4 *>(row + col) = v;
            if (gt) {
              const f4 x = *reinterpret_cast<const f4 *>(gt + col);
              f4 y;
#pragma unroll
              for (int i = 0; i < 4; ++i) y[i] = v[i] / (1.0f + expf(-x[i]));
              *reinterpret_cast<f4 *>(z.out_gated + (row - z.out) + col) = y;
            }
          };
          write(even_row, even_gate, e);
          write(odd_row, odd_gate, d);
        }
      }
    };
    if (works) {
      if (odd) finish(std::integral_constant<int, 8>{});
      else finish(std::integral_constant<int, 0>{});
    }
    lds_barrier();                                 // (LDS is the next part's)
    at += t1 - t0;
    if (t1 == steps) {
      line0 += steps;
      ++rb;
    }
  }
}

// ------------------------------------------------------------------ the join of the tiles' partial results
// A row by SW waves: wave w of them sums the partial results w, w + SW, .. (a lane 4 dims, 8 of them requested together), then
// the waves' sums meet in LDS. Bound by memory: 33 MB of partial results and 8 MB of outputs in 9.5 us.
constexpr int kMergeWaves = 4;
template <int SW>
__global__ __launch_bounds__(64 * kMergeWaves) void seqs_merge_kernel(SeqsAttnArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave % SW;
  const int64_t r = (int64_t)blockIdx.x * (kMergeWaves / SW) + wave / SW;
  if (r >= (int64_t)a.v.n_tok * a.nh) return;      // (all SW waves of it)
  const int t = a.by_nh.div((uint32_t)r), h = (int)r - t * a.nh;
  __shared__ __attribute__((aligned(16))) float s_o[SW > 1 ? SW * kHd : 4];
  const uint4 in = a.info[r];
  const int s = a.v.sequence_of<64>(t);
  if (s < 0 || a.v.tokens(s) * a.grp <= a.few) return;     // (no row of a tile: nothing was left for it)
  const uint32_t first = in.x, stride = in.y, count = in.z;
  if (count <= 1 || (uint64_t)first + (uint64_t)stride * (count - 1) >= a.tile_part_rows) return;
  auto row_of = [&](uint32_t i) { return first + i * stride - (i ? stride / 2 : 0); };
  auto part = [&](uint32_t i) { return reinterpret_cast<const float4 *>(a.tile_part + (int64_t)row_of(i) * kHd)[lane]; };
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f), x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = part(min((uint32_t)(w + j * SW), count - 1));
  float2 ml = a.tile_ml[row_of(min((uint32_t)lane, count - 1))];
  float mm = ml.x;
  for (uint32_t i = 64 + lane; i < count; i += 64) mm = fmaxf(mm, a.tile_ml[row_of(i)].x);
  mm = wave_max(mm);
  float l = 0.0f;
  for (uint32_t i0 = 0; i0 < count; i0 += 64) {    // 64 partial results' weights at a time
    if (i0) ml = a.tile_ml[row_of(min(i0 + lane, count - 1))];
    const float f = i0 + lane >= count || ml.x == -INFINITY ? 0.0f : exp2f(ml.x - mm);
    l += i0 + lane >= count || ml.x == -INFINITY ? 0.0f : ml.y * f;
    const uint32_t n64 = min(count - i0, 64u);
    for (uint32_t i = w; i < n64; i += 8 * SW) {
      if (i0 + i >= 8 * SW) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = part(min(i0 + i + j * SW, count - 1));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (i + j * SW >= n64) break;
        const float fj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), (int)(i + j * SW)));
        o.x = fmaf(x[j].x, fj, o.x); o.y = fmaf(x[j].y, fj, o.y); o.z = fmaf(x[j].z, fj, o.z); o.w = fmaf(x[j].w, fj, o.w);
      }
    }
  }
  l = wave_sum(l);
  if constexpr (SW > 1) {
    reinterpret_cast<float4 *>(s_o + w * kHd)[lane] = o;
    __syncthreads();
    if (w != 0) return;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < SW; ++j) {
      const float4 y = reinterpret_cast<const float4 *>(s_o + j * kHd)[lane];
      o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
    }
  }
  write_out(a, t, h, 4 * lane, {o.x, o.y, o.z, o.w}, l);
}

// ------------------------------------------------------------------ host side
static inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
// A sequence of more rows goes by tiles, where the call has more than kFewInAll (in fewer, no workgroup has much to do by
// either, and a block's way in and out is the shorter). One sequence in blocks / in tiles: 128 rows 17 / 39 us at 1000
// positions, 29 / 44 at 8000, 56 / 51 at 32000; 192 rows 19 / 40, 35 / 54, 80 / 82; 256 rows 20 / 41, 39 / 58, 92 / 84.
// 16 sequences at 3000: 64 rows each 47 / 71, 96 77 / 78, 128 87 / 79, 192 127 / 97.
constexpr int kFewRows = 96, kFewInAll = 192;

SeqsAttnPlan plan_seqs_attn(int nh, int nkv, int n_seq, int n_tok, int max_q) {
  SeqsAttnPlan p{};
  const int grp = nh / nkv;
  p.lanes = std::max(1, kSeqFill / nkv);
  const size_t parts = (size_t)2 * p.lanes * nkv * kSeqBlock;
  p.off_ml = up256((size_t)kJoinLevels * 2 * kSeqFill * sizeof(unsigned));
  p.off_part = up256(p.off_ml + parts * sizeof(float2));
  p.total = up256(p.off_part + parts * kHd * sizeof(float));
  // Both kernels where there may be sequences of both kinds; of a single one's only the size that it may have is known here,
  // and either kernel takes it whatever it has.
  const int most = max_q > 0 ? std::min(max_q, n_tok) : n_tok;
  const int few = (int64_t)n_tok * grp <= kFewInAll ? kFewInAll : kFewRows;
  p.tiles = (int64_t)most * grp > few;
  p.blocks = !p.tiles || n_seq > 1;
  p.few = !p.tiles ? INT32_MAX : p.blocks ? few : 0;
  p.way_in = n_seq > 1 || (int64_t)most * grp > kSeqBlock ? kSeqWayIn : 0;
  p.tile_lanes = std::max(1, kTileFill / nkv);
  if ((int64_t)n_tok * grp > few) {                // (whatever max_q says: one workspace for all of a size)
    p.tile_part_rows = p.tile_lanes > 1 ? (uint64_t)2 * p.tile_lanes * nkv * kTileRows : 0;   // (a single piece shares no tile)
    p.off_info = p.total;
    p.off_tile_ml = up256(p.off_info + (size_t)n_tok * nh * sizeof(uint4));
    p.off_tile_part = up256(p.off_tile_ml + p.tile_part_rows * sizeof(float2));
    p.total = up256(p.off_tile_part + p.tile_part_rows * kHd * sizeof(float));
  }
  return p;
}

template <int PG>
static hipError_t launch_seqs_attn_pg(const SeqsAttnArgs &a, const SeqsAttnPlan &p, hipStream_t st) {
  if (p.tiles) {
    hipLaunchKernelGGL((seqs_tile_kernel<PG>), dim3((unsigned)((p.tile_lanes + 7) / 8 * 8 * a.nkv)), dim3(64 * kTileWaves), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.blocks) hipLaunchKernelGGL((seqs_attn_kernel<PG>), dim3((unsigned)((p.lanes + 7) / 8 * 8 * a.nkv)), dim3(64 * kSeqWaves), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_seqs_attn(const SeqsAttnArgs &a, const SeqsAttnPlan &p, hipStream_t st) {
  const hipError_t e = a.v.page == 0 ? launch_seqs_attn_pg<0>(a, p, st) : a.v.page % kSeqKeys == 0 ? launch_seqs_attn_pg<1>(a, p, st) : launch_seqs_attn_pg<2>(a, p, st);
  if (e != hipSuccess || !p.tiles) return e;
  const unsigned rows = (unsigned)((int64_t)a.v.n_tok * a.nh);
  if (rows > 2048) hipLaunchKernelGGL((seqs_merge_kernel<1>), dim3((rows + kMergeWaves - 1) / kMergeWaves), dim3(64 * kMergeWaves), 0, st, a);
  else hipLaunchKernelGGL((seqs_merge_kernel<kMergeWaves>), dim3(rows), dim3(64 * kMergeWaves), 0, st, a);
  return hipGetLastError();
}

}  // namespace bkv
