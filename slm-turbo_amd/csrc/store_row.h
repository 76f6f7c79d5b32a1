// A token's (kv head) row in the packed per-token 4-bit format: its ruler and codes, 8 dims per
// lane (shared by the quantize-on-write store and the store that rotates its keys first).
#pragma once

#include "slmt_internal.h"

namespace slmt {
namespace {

__device__ __forceinline__ f16x2 pair_min(f16x2 a, f16x2 b) { return __builtin_elementwise_min(a, b); }
__device__ __forceinline__ f16x2 pair_max(f16x2 a, f16x2 b) { return __builtin_elementwise_max(a, b); }
template <int CTRL>
__device__ __forceinline__ f16x2 pair_dpp(f16x2 h) {
  return __builtin_bit_cast(f16x2, dpp_u<CTRL>(__builtin_bit_cast(uint32_t, h)));
}

// Eight fp16 values from an address that is a multiple of 4 only (the hardware
// takes 16-byte loads there).
struct Eight {
  f16x2 h[4];
};
__device__ __forceinline__ Eight load_eight(const uint16_t* p) {
  Eight v;
  __builtin_memcpy(&v, __builtin_assume_aligned(p, 4), 16);
  return v;
}

// Ruler of a row spread over LANES lanes: minimum and step (1 where the range is 0
// or no number).  NaNs are passed over; a row of nothing else has the minimum
// infinity at head_dim 64 and 80 (`seed`) and NaN at 128.
template <int LANES, bool SEED>
__device__ __forceinline__ void row_ruler(const Eight& x, float& mn, float& step) {
#pragma clang fp contract(off)
  f16x2 lo = pair_min(pair_min(x.h[0], x.h[1]), pair_min(x.h[2], x.h[3]));
  f16x2 hi = pair_max(pair_max(x.h[0], x.h[1]), pair_max(x.h[2], x.h[3]));
  lo = pair_min(lo, pair_dpp<DPP_QUAD_XOR1>(lo));
  hi = pair_max(hi, pair_dpp<DPP_QUAD_XOR1>(hi));
  lo = pair_min(lo, pair_dpp<DPP_QUAD_XOR2>(lo));
  hi = pair_max(hi, pair_dpp<DPP_QUAD_XOR2>(hi));
  if (LANES == 8) {
    lo = pair_min(lo, pair_dpp<DPP_ROW_HALF_MIRROR>(lo));
    hi = pair_max(hi, pair_dpp<DPP_ROW_HALF_MIRROR>(hi));
  } else {
    lo = pair_min(lo, pair_dpp<DPP_ROW_ROR4>(lo));
    hi = pair_max(hi, pair_dpp<DPP_ROW_ROR4>(hi));
    lo = pair_min(lo, pair_dpp<DPP_ROW_ROR8>(lo));
    hi = pair_max(hi, pair_dpp<DPP_ROW_ROR8>(hi));
  }
  mn = fminf((float)lo[0], (float)lo[1]);
  float mx = fmaxf((float)hi[0], (float)hi[1]);
  if (SEED) {
    mn = fminf(mn, INFINITY);
    mx = fmaxf(mx, -INFINITY);
  }
  step = (mx - mn) / 15.0f;
  if (!(step > 0.0f)) step = 1.0f;
}

// Codes (int)((x - mn) / step + 0.5) of eight values, two a byte.  The quotient is
// correctly rounded as a division's: r is 1 / step correctly rounded, the first
// residual step leaves less than an ulp of error and the second, from there, the
// rounded quotient (Markstein).  Nothing under- or overflows: x - mn is 0 or at
// least 2^-24, and step lies in [2^-24 / 15, 8734].  Half the compiler's division.
// Infinite steps and NaNs, which the division takes to 0 or NaN, come out NaN, and
// NaN is code 0; a number's quotient is at most 15 (1 + 2^-22) and needs no clamp.
__device__ __forceinline__ uint32_t codes(const Eight& x, float mn, float step, float r) {
#pragma clang fp contract(off)
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = (float)x.h[i >> 1][i & 1] - mn;
    float q = a * r;
    q = __builtin_fmaf(__builtin_fmaf(-q, step, a), r, q);
    q = __builtin_fmaf(__builtin_fmaf(-q, step, a), r, q);
    out |= (uint32_t)fmaxf(q + 0.5f, 0.0f) << (4 * i);
  }
  return out;
}

}  // namespace
}  // namespace slmt
