// The scales of e4m3 codes, in rules that kernels and host share.
//
// Each group of 128 values of a row (of weights: each block of 128 x 128) has a scale
// s = 2^e in 8 bits (e8m0: the biased exponent e + 127; 255 is NaN).  s is the smallest
// power of two from 2^-126 on with largest <= 448 s: what a scaled MFMA takes, and x / s
// is exact, so a code is one rounding of x.
//
// Scales lie [words, rows, 4]: word i of a row has the scales of its groups 4 i .. 4 i + 3,
// so that the rows of an MFMA operand read theirs for 512 values in one coalesced dword.
// Groups past the last one have the scale of zeros.
#pragma once

#include <stdint.h>

#include "../../include/ttlhip.h"

#if defined(__HIPCC__)
#define TTLH_FP8_HD __host__ __device__ inline
#else
#define TTLH_FP8_HD inline
#endif

namespace ttlh {

constexpr int kFp8Group = 128;   // values that share a scale
constexpr int kFp8Word = 512;    // values whose scales are one dword
constexpr int kScaleNan = 255;   // the code of values that are not finite
constexpr int kScaleLeast = 1;   // 2^-126

// the scale's code for a largest magnitude given by its bits as fp32
TTLH_FP8_HD int scale_code(uint32_t largest) {
  const int e = static_cast<int>(largest >> 23);
  if (e >= 255) return kScaleNan;
  // 448 = 1.75 x 2^8
  const int s = e - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);
  return s < kScaleLeast ? kScaleLeast : s;
}

// the same for a finite largest magnitude given by its bits as fp64
TTLH_FP8_HD int scale_code64(uint64_t largest) {
  const int e = static_cast<int>(largest >> 52) - 1023 + 127;
  const int s = e - 8 + ((largest & 0xfffffffffffffull) > 0xc000000000000ull ? 1 : 0);
  return s < kScaleLeast ? kScaleLeast : s > 254 ? 254 : s;
}

// Whether a largest magnitude that is right to 32 units in its last place leaves the
// scale open: 1.75 x 2^n lies that near.
TTLH_FP8_HD bool scale_open(uint32_t largest) {
  return static_cast<uint32_t>((largest & 0x7fffffu) - 0x600000u + 32u) <= 64u;
}

// 1 / s as fp32 bits (s finite; codes of fp32 values are at most 247)
TTLH_FP8_HD uint32_t inverse_scale_bits(int code) {
  return static_cast<uint32_t>(254 - code) << 23;
}

// Codes as bf16 operands of a product (results in fp32), times powers of two whose product is that of
// their scales 2^(ex - 127) and 2^(ew - 127).  bf16 has neither 256 x 2^120 nor 2^-9 x 2^-126, so ex and ew
// themselves will not do: w's operand gets half of ew's exponent and 2^-21 (it is between 2^-94 and 2^51 then,
// whatever ew is), and x's the rest.  Where that is below 2^-117, x's operand may lose bits (or is held at
// 2^-126), but w's is less than 2^-25 then: products that are off are off by less than 2^-149.  Where it
// is above 2^119 bf16 may not hold it: wide_far.  (NaN scales, ex or ew 255: the caller's.)
constexpr int kWideMost = 246;  // 448 x 2^(246 - 127) is the largest that bf16 holds

TTLH_FP8_HD int wide_w(int ew) { return (ew >> 1) + 42; }
TTLH_FP8_HD int wide_rest(int ex, int ew) { return ex + (ew - wide_w(ew)); }  // before its limits
TTLH_FP8_HD int wide_x(int rest) {
  return rest < kScaleLeast ? kScaleLeast : rest > kWideMost ? kWideMost : rest;
}
TTLH_FP8_HD bool wide_far(int rest) { return rest > kWideMost; }

}  // namespace ttlh
