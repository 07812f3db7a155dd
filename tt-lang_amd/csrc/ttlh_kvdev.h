// Device helpers of the 8-bit key/value cache's kernels.
#pragma once

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

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int i = 32; i; i >>= 1) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), i)));
  return x;
}

// Item `item` of the sequences' items, count(b) of sequence b: its sequence and its
// number there, or false past the last one.  Every lane of a wave gets the same
// answer; the wave counts 64 sequences at a time, so the host need not know how
// many items there are, only a bound for the grid.
template <typename F>
__device__ __forceinline__ bool find_item(int seqs, int64_t item, F count, int& b, int& local) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int b0 = 0; b0 < seqs; b0 += 64) {
    const int n = b0 + lane < seqs ? count(b0 + lane) : 0;
    int64_t end = n;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
      const int64_t o = __shfl_up(end, i);
      if (lane >= i) end += o;
    }
    const unsigned long long past = __ballot(before + end > item);
    if (past) {
      const int l = __ffsll(past) - 1;
      b = b0 + l;
      local = static_cast<int>(item - before - (__shfl(end, l) - __shfl(n, l)));
      b = __builtin_amdgcn_readfirstlane(b);
      local = __builtin_amdgcn_readfirstlane(local);
      return true;
    }
    before += __shfl(end, 63);
  }
  return false;
}

}  // namespace ttlh
