// bkv_q4.h - the 4-bit cache format BKV_Q4_0 and the view of several sequences over one cache.
//
// A block of 32 values has a scale d and whole numbers q = -8 .. 7; a value is d * q. d is kept to 8 significant bits (an
// fp16 word whose low 3 bits are 0), so that d * q, at most 11 bits, is an exact fp16 number: the matrix products take the
// cache's values as they are, one fp16 operand each, where d of 11 bits would leave a rounding or need two. What that costs
// is up to 2^-9 of a scale, a thirtieth of half a step at q = 8.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bkv_common.h"

namespace bkv {

constexpr int kQ4RowBytes = kHd / 2;               // a head row: 32 words of 8 values, element 2 s + h at bit 16 h + 4 s
constexpr uint32_t kQ4MaxScale = 0x6800;           // 2048: (16 + q) * d and 24 * d stay within fp16

// bytes of one head row of the data array, any format
__host__ __device__ constexpr int any_row_bytes(int fmt) { return fmt == BKV_Q4_0 ? kQ4RowBytes : row_bytes(fmt); }

// ------------------------------------------------------------------ writing
// The scale of a block whose largest and smallest values are hi and lo, as fp16 bits: the value furthest from 0 (the
// positive one of two as far) is -8 steps. Rounded to fp16, then to the upper 13 bits of it. A block whose scale would be
// beyond 2048 (values beyond 16384) saturates; 0 is +0.
__device__ __forceinline__ uint32_t q4_scale(float hi, float lo) {
  const uint32_t h = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)((hi >= -lo ? hi : lo) * -0.125f));
  uint32_t m = h & 0x7FFFu;
  m = min((m + 3u + ((m >> 3) & 1u)) & 0x7FF8u, kQ4MaxScale);
  return m ? m | (h & 0x8000u) : 0u;
}
__device__ __forceinline__ float q4_iscale(uint32_t scale) {
  const float d = f16_to_f32(scale);
  return d != 0.0f ? 1.0f / d : 0.0f;
}
// q + 8 (a NaN is 0)
__device__ __forceinline__ uint32_t q4_code(float x, float id) {
  float r = __builtin_rintf(x * id);
  r = (r != r) ? 0.0f : fminf(fmaxf(r, -8.0f), 7.0f);
  return (uint32_t)((int)r + 8);
}

// ------------------------------------------------------------------ reading
// Two scales as they count: the low 3 bits do not, and magnitudes past 2048 (Inf and NaN patterns among them) are 2048, so
// that whatever the bytes of a position are, its values are finite.
__device__ __forceinline__ uint32_t q4_scales(uint32_t two) {
  typedef uint16_t u2 __attribute__((ext_vector_type(2)));
  const u2 m = __builtin_elementwise_min(__builtin_bit_cast(u2, two & 0x7FF87FF8u), u2{(uint16_t)kQ4MaxScale, (uint16_t)kQ4MaxScale});
  return __builtin_bit_cast(uint32_t, m) | (two & 0x80008000u);
}

// Division of 0 .. 2^31 - 1 by a number that the host knows: x / d = x * m >> (32 + s) with m = ceil(2^(32 + s) / d) and 2^s
// < d <= 2^(s + 1): m d is less than d past 2^(32 + s), so that x (m d - 2^(32 + s)) < 2^(32 + s): the quotient is exact.
// (d = 1 has m = 0 and adds x.)
struct ByConst {
  uint32_t m, one;
  int s;
  ByConst() = default;
  explicit ByConst(uint32_t d) : m(0), one(d == 1 ? ~0u : 0u), s(0) {
    while ((uint64_t(2) << s) < d) ++s;
    if (d > 1) m = (uint32_t)(((uint64_t(1) << (32 + s)) + d - 1) / d);
  }
  __device__ __forceinline__ int div(uint32_t x) const { return (int)((__umulhi(x, m) + (x & one)) >> s); }
  __device__ __forceinline__ uint32_t rest(uint32_t x, uint32_t d) const { return x - (uint32_t)div(x) * d; }
};

// ------------------------------------------------------------------ several sequences
// Sequence s has the tokens q_begin(s) .. q_begin(s + 1) - 1 of a call and length(s) positions, its tokens' the last. What
// is read from device memory is held against the call's sizes: whatever it says, no access leaves them.
struct SeqsView {
  int n_seq, n_tok;
  const int32_t *q_start;                          // [n_seq + 1], or null: one token each
  const int32_t *len;                              // [n_seq]
  const int32_t *tables;                           // this layer's row of sequence 0, or null (contiguous)
  int64_t table_stride;                            // from a sequence's row to the next's
  int page, pool_pages;
  int64_t max_pos;                                 // positions that a sequence can have

  __device__ __forceinline__ int q_begin(int s) const { return min(max(q_start ? q_start[s] : s, 0), n_tok); }
  __device__ __forceinline__ int tokens(int s) const { return max(q_begin(s + 1) - q_begin(s), 0); }
  __device__ __forceinline__ int length(int s) const { return max(len[s], 0); }   // (it may be past max_pos: those tokens are not there)
  // the slot of a position (0 <= pos < max_pos), -1 where its page is not in the pool
  __device__ __forceinline__ int slot(int s, uint32_t pos) const {
    if (page == 0) return (int)pos;
    const uint32_t pg = pos / (uint32_t)page, b = (uint32_t)tables[s * table_stride + pg];
    return b < (uint32_t)pool_pages ? (int)(b * (uint32_t)page + (pos - pg * (uint32_t)page)) : -1;
  }
  // The sequence of token t, -1 where it is none's, by W lanes (32 or 64) that ask for the starts side by side: a search
  // would be one latency after the other.
  template <int W>
  __device__ __forceinline__ int sequence_of(int t) const {
    if (!q_start) return t < n_seq ? t : -1;
    const int lane = threadIdx.x & 63, sub = lane & (W - 1);
    int before = 0;                                // sequences that end at or before t
    for (int s = 0; s < n_seq; s += W) {
      const uint64_t b = __ballot(s + sub < n_seq && q_start[min(s + sub, n_seq - 1) + 1] <= t);
      before += W == 64 ? __popcll(b) : __popc((uint32_t)(b >> (lane & 32)));
    }
    return before < n_seq && q_begin(before) <= t ? before : -1;
  }
};

// FORMAT = what KF, VF of the kernels stand for
#define BKV_ANY_FMT_SWITCH(KF, VF, ...)                                                            \
  do {                                                                                             \
    if ((KF) == BKV_Q4_0) BKV_ANY_V_SWITCH(BKV_Q4_0, VF, __VA_ARGS__);                              \
    else if ((KF) == BKV_Q8_0) BKV_ANY_V_SWITCH(BKV_Q8_0, VF, __VA_ARGS__);                         \
    else BKV_ANY_V_SWITCH(BKV_F16, VF, __VA_ARGS__);                                                \
  } while (0)
#define BKV_ANY_V_SWITCH(K, VF, ...)                                                               \
  do {                                                                                             \
    if ((VF) == BKV_Q4_0) { constexpr int KF_ = K, VF_ = BKV_Q4_0; __VA_ARGS__; }                   \
    else if ((VF) == BKV_Q8_0) { constexpr int KF_ = K, VF_ = BKV_Q8_0; __VA_ARGS__; }              \
    else { constexpr int KF_ = K, VF_ = BKV_F16; __VA_ARGS__; }                                     \
  } while (0)

}  // namespace bkv
