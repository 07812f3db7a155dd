// Device helpers of the 8-bit key/value cache's kernels.
#pragma once

#include <type_traits>

#include "ttlh_common.h"
#include "ttlh_kvcache.h"

namespace ttlh {

// checks a cache and its call's sizes (kvcache.hip)
int check_cache(const char* fn, const ttlh_kv_cache* c, CacheArgs* a);

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return bf16_to_f32(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ uint16_t from_f32<uint16_t>(float x) {
  return static_cast<uint16_t>(cvt_pk_bf16x2(x, x));
}

// values, at most the largest code in magnitude, rounded to four codes
template <int FMT>
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {
  if constexpr (FMT == TTLH_CACHE_INT8) {
    const int i = static_cast<int>(rintf(a)), j = static_cast<int>(rintf(b));
    const int k = static_cast<int>(rintf(c)), l = static_cast<int>(rintf(d));
    return (i & 255) | (j & 255) << 8 | (k & 255) << 16 | static_cast<uint32_t>(l) << 24;
  } else {
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
  }
}
template <int FMT>
__device__ __forceinline__ float from_code(uint8_t c) {
  if constexpr (FMT == TTLH_CACHE_INT8)
    return static_cast<float>(static_cast<int8_t>(c));
  else
    return __builtin_amdgcn_cvt_f32_fp8(c, 0);
}

// Lane i gets x of lane i - SHIFT of its row of 16 (SHIFT < 16), or of the last lane
// of the rows before it (kRowBcast15, kRowBcast31); `none` where there is none.
constexpr int kRowShr1 = 0x111, kRowShr2 = 0x112, kRowShr4 = 0x114, kRowShr8 = 0x118;
constexpr int kRowBcast15 = 0x142, kRowBcast31 = 0x143;
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int dpp(int x, int none) {
  return __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xf, false);
}
// sum of x over lanes 0 .. own
__device__ __forceinline__ int prefix_sum(int x) {
  x += dpp<kRowShr1>(x, 0);
  x += dpp<kRowShr2>(x, 0);
  x += dpp<kRowShr4>(x, 0);
  x += dpp<kRowShr8>(x, 0);
  x += dpp<kRowBcast15, 0xa>(x, 0);
  x += dpp<kRowBcast31, 0xc>(x, 0);
  return x;
}
// sum over the wave, the same in every lane (and in every wave with the same x)
__device__ __forceinline__ float wave_total(float x) {
  const auto add = [&](auto ctrl, auto rows) {
    x += __int_as_float(dpp<decltype(ctrl)::value, decltype(rows)::value>(__float_as_int(x), 0));
  };
  typedef std::integral_constant<int, 0xf> all;
  add(std::integral_constant<int, kRowShr1>(), all());
  add(std::integral_constant<int, kRowShr2>(), all());
  add(std::integral_constant<int, kRowShr4>(), all());
  add(std::integral_constant<int, kRowShr8>(), all());
  add(std::integral_constant<int, kRowBcast15>(), std::integral_constant<int, 0xa>());
  add(std::integral_constant<int, kRowBcast31>(), std::integral_constant<int, 0xc>());
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  const auto step = [&](auto ctrl, auto rows) {
    x = max(x, static_cast<uint32_t>(
                   dpp<decltype(ctrl)::value, decltype(rows)::value>(static_cast<int>(x), 0)));
  };
  typedef std::integral_constant<int, 0xf> all;
  step(std::integral_constant<int, kRowShr1>(), all());
  step(std::integral_constant<int, kRowShr2>(), all());
  step(std::integral_constant<int, kRowShr4>(), all());
  step(std::integral_constant<int, kRowShr8>(), all());
  step(std::integral_constant<int, kRowBcast15>(), std::integral_constant<int, 0xa>());
  step(std::integral_constant<int, kRowBcast31>(), std::integral_constant<int, 0xc>());
  return __builtin_amdgcn_readlane(static_cast<int>(x), 63);
}

// Item `item` of the sequences' items, count(b) of sequence b: its sequence and its
// number there, or false past the last one.  Every lane of a wave gets the same
// answer; the wave counts 64 sequences at a time, so the host need not know how
// many items there are, only a bound for the grid (less than 2^31).
template <typename F>
__device__ __forceinline__ bool find_item(int seqs, int item, F count, int& b, int& local) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < seqs; b0 += 64) {
    const int n = b0 + lane < seqs ? count(b0 + lane) : 0;
    const int end = prefix_sum(n);
    const unsigned long long past = __ballot(before + end > item);
    if (past) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
      b = b0 + l;
      local = item - before - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(n, l));
      return true;
    }
    before += __builtin_amdgcn_readlane(end, 63);
  }
  return false;
}

}  // namespace ttlh
