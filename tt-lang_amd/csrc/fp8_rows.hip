// Rows of values into e4m3 codes with a scale for each 128 of them, for gfx950: as they
// are, through a root-mean-square norm, or through a gated activation.
//
// All three read their operands once and write a byte for each value: HBM bound.  A lane
// has eight neighbouring values, 16 lanes a group, a wave four groups: their scales are
// one dword, and the group's largest magnitude is found by rotations within a row of 16
// lanes, without LDS.
//
// Values are computed in fp32.  A scale, though, steps by two where its group's largest
// value crosses 448 x 2^n, so that an error of one unit in the last place there changes
// 128 codes; a group whose largest value comes within 32 units of such a border (one in
// 10^5) is therefore decided in fp64.  Scales are those of the exact values.

#include <cmath>
#include <type_traits>

#include "ttlh_common.h"
#include "ttlh_fp8.h"
#include "ttlh_kvdev.h"

namespace ttlh {
namespace {

constexpr int kThreads = 256;

// Eight neighbouring values of a row.  Addresses need only the alignment of an element
// (gfx950 under HSA takes unaligned vector accesses).
typedef u32x4 u32x4u __attribute__((aligned(2)));
typedef uint2 uint2u __attribute__((aligned(1)));

template <typename T>
struct Eight {
  float v[8];
  // n: how many of them there are; zeros in the place of the others
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= 8) {
      if constexpr (sizeof(T) == 2) {
        const u32x4 w = *reinterpret_cast<const u32x4u*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 w = *reinterpret_cast<const u32x4u*>(p + 4 * h);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * h + i] = __uint_as_float(w[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
    }
  }
  __device__ __forceinline__ void store(T* p, int n) const {
    if (n >= 8) {
      if constexpr (sizeof(T) == 2) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = cvt_pk_bf16x2(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<u32x4u*>(p) = w;
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[4 * h + i]);
          *reinterpret_cast<u32x4u*>(p + 4 * h) = w;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = from_f32<T>(v[i]);
    }
  }
};

// the largest x of a row of 16 lanes, in each of them
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  const auto step = [&](auto ctrl) {
    x = max(x, static_cast<uint32_t>(dpp<decltype(ctrl)::value>(static_cast<int>(x), 0)));
  };
  step(std::integral_constant<int, 0x128>());  // rotated by 8
  step(std::integral_constant<int, 0x124>());
  step(std::integral_constant<int, 0x122>());
  step(std::integral_constant<int, 0x121>());
  return x;
}

struct Out {
  uint8_t* codes;
  uint32_t* scales;
  int64_t codes_ld, scales_ld;  // bytes; dwords from a word of all rows to the next
};

// The codes of a wave's 512 values (n of a lane's eight exist) and their scales, to
// `codes` (the lane's) and `word`.  exact(i): value i in fp64, where fp32 does not decide
// a scale.
template <bool EXACT, typename F>
__device__ __forceinline__ void emit(const float (&y)[8], F exact, int n, uint8_t* codes,
                                     uint32_t* word) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
  m = row_max(m);
  int s = scale_code(m);
  if constexpr (!EXACT) {
    if (__any(scale_open(m) && s != kScaleNan)) {
      double big = 0.0;
#pragma unroll 1
      for (int i = 0; i < n; ++i) big = fmax(big, fabs(exact(i)));
#pragma unroll
      for (int i = 8; i; i >>= 1) big = fmax(big, __shfl_xor(big, i));
      if (scale_open(m) && s != kScaleNan)
        s = scale_code64(static_cast<uint64_t>(__double_as_longlong(big)));
    }
  }
  const float inv = __uint_as_float(inverse_scale_bits(s));
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = s == kScaleNan ? 0.0f : y[i] * inv;
  const uint2 w = {four_codes<TTLH_CACHE_E4M3>(v[0], v[1], v[2], v[3]),
                   four_codes<TTLH_CACHE_E4M3>(v[4], v[5], v[6], v[7])};
  if (n >= 8) {
    *reinterpret_cast<uint2u*>(codes) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) codes[i] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
  }
  const uint32_t four = static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 0)) |
                        static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 16)) << 8 |
                        static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 32)) << 16 |
                        static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 48)) << 24;
  if ((threadIdx.x & 63) == 0) *word = four;
}

// --- as they are, and gated -----------------------------------------------------

constexpr int kActNone = -1;

// exp(x): 2^(x log2 e) with the product's rounding error and the constant's tail put back
// (one unit in the last place; x at most 88 in magnitude where that matters)
__device__ __forceinline__ float exp_f32(float x) {
  constexpr float kL2E = 1.44269502e+00f, kL2ELo = 1.92596299e-08f, kLn2 = 6.93147182e-01f;
  const float t = x * kL2E;
  const float lo = __builtin_fmaf(x, kL2ELo, __builtin_fmaf(x, kL2E, -t));
  const float p = __builtin_amdgcn_exp2f(t);
  return fabsf(t) < 128.0f ? __builtin_fmaf(p, lo * kLn2, p) : p;
}

template <int ACT>
__device__ __forceinline__ float gated(float g, float u) {
  if constexpr (ACT == TTLH_GLU_SILU)
    return g / (1.0f + exp_f32(-g)) * u;
  else {
    // erfc(z + lo) = erfc(z) (1 - 2 z lo) to 2^-24 where z > 0, whose rounding error lo
    // would count 2 z^2 times
    constexpr float kC = -0.707106769f, kCLo = -1.21016175e-08f;  // -1 / sqrt 2
    const float z = g * kC;
    const float lo = __builtin_fmaf(g, kCLo, __builtin_fmaf(g, kC, -z));
    const float e = erfcf(z);
    return 0.5f * g * (z > 0.0f && z < 16.0f ? __builtin_fmaf(-2.0f * z * lo, e, e) : e) * u;
  }
}
template <int ACT>
__device__ __forceinline__ double gated64(double g, double u) {
  if constexpr (ACT == TTLH_GLU_SILU)
    return g / (1.0 + exp(-g)) * u;
  else
    return 0.5 * g * erfc(g * -0.70710678118654752440) * u;
}

struct UnitArgs {
  const void* a;
  const void* b;
  int64_t a_ld, b_ld;
  Out o;
  int32_t rows, dim, words;
  int32_t blocks;  // workgroups of a row
};

template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void fp8_units_kernel(const UnitArgs p) {
  const int row = blockIdx.x / p.blocks;
  const int word = (blockIdx.x - row * p.blocks) * (kThreads / 64) +
                   __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (word >= p.words) return;
  const int at = word * kFp8Word + (threadIdx.x & 63) * 8, n = p.dim - at;
  const T* pa = static_cast<const T*>(p.a) + row * p.a_ld + at;
  const T* pb = static_cast<const T*>(p.b) + row * p.b_ld + at;
  uint8_t* codes = p.o.codes + row * p.o.codes_ld + at;
  uint32_t* to = p.o.scales + word * p.o.scales_ld + row;
  Eight<T> a;
  a.load(pa, n);
  if constexpr (ACT == kActNone) {
    emit<true>(a.v, 0, n, codes, to);
  } else {
    Eight<T> b;
    b.load(pb, n);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = gated<ACT>(a.v[i], b.v[i]);
    emit<false>(y, [&](int i) {
      return gated64<ACT>(static_cast<double>(to_f32(pa[i])), static_cast<double>(to_f32(pb[i])));
    }, min(n, 8), codes, to);
  }
}

// --- the norm --------------------------------------------------------------------

struct NormArgs {
  const void* x;
  const void* residual;  // may be null
  void* total;           // may be null
  const void* weight;
  int64_t x_ld, residual_ld, total_ld;
  Out o;
  int32_t rows, dim;
  int32_t weight_f32;
  float eps;
};

// the sum of x over the LANES (64, or all of a workgroup of 256) that have a row
template <int LANES>
__device__ __forceinline__ double row_sum(double x) {
#pragma unroll
  for (int i = 32; i; i >>= 1) x += __shfl_xor(x, i);
  if constexpr (LANES > 64) {
    __shared__ double part[LANES / 64];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = part[0];
#pragma unroll
    for (int w = 1; w < LANES / 64; ++w) x += part[w];
  }
  return x;
}

// LANES lanes have a row, SWEEPS x 8 values each, which stay in registers between the sum
// of squares (in fp64: a group near a scale's border needs the exact norm) and the codes.
// SWEEPS 0: any length, read twice.
template <typename T, int LANES, int SWEEPS>
__global__ __launch_bounds__(kThreads) void fp8_norm_kernel(const NormArgs p) {
  constexpr int kStep = LANES * 8;
  const int row = blockIdx.x * (kThreads / LANES) + (LANES == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  const int lane = threadIdx.x & (LANES - 1);
  if (row >= p.rows) return;  // (a whole wave of its own where LANES is 64)
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_ld : nullptr;
  T* total = p.total ? static_cast<T*>(p.total) + row * p.total_ld : nullptr;
  const auto read = [&](int at, Eight<T>& t) {
    const int n = p.dim - at;
    t.load(x + at, n);
    if (r) {
      Eight<T> more;
      more.load(r + at, n);
#pragma unroll
      for (int i = 0; i < 8; ++i) t.v[i] += more.v[i];
    }
  };
  double sum = 0.0;
  const auto add = [&](const Eight<T>& t) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fma(static_cast<double>(t.v[i]), static_cast<double>(t.v[i]), sum);
  };
  Eight<T> t[SWEEPS ? SWEEPS : 1];
  if constexpr (SWEEPS > 0) {
#pragma unroll
    for (int i = 0; i < SWEEPS; ++i) read(lane * 8 + i * kStep, t[i]);
#pragma unroll
    for (int i = 0; i < SWEEPS; ++i) add(t[i]);
  } else {
    for (int at = lane * 8; at < p.dim; at += kStep) {
      read(at, t[0]);
      add(t[0]);
    }
  }
  sum = row_sum<LANES>(sum);
  const double by = 1.0 / sqrt(sum / p.dim + static_cast<double>(p.eps));
  const float by32 = static_cast<float>(by);
  const auto write = [&](int at, const Eight<T>& t) {
    const int n = p.dim - at;
    float w[8], y[8];
    if (p.weight_f32) {
      Eight<float> e;
      e.load(static_cast<const float*>(p.weight) + at, n);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = e.v[i];
    } else {
      Eight<uint16_t> e;
      e.load(static_cast<const uint16_t*>(p.weight) + at, n);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = e.v[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = t.v[i] * by32 * w[i];
    emit<false>(y, [&](int i) {
      double v = to_f32(x[at + i]);
      if (r) v += static_cast<double>(to_f32(r[at + i]));
      const double g = p.weight_f32 ? static_cast<const float*>(p.weight)[at + i]
                                    : to_f32(static_cast<const uint16_t*>(p.weight)[at + i]);
      return v * by * g;
    }, min(n, 8), p.o.codes + row * p.o.codes_ld + at,
                p.o.scales + (at / kFp8Word) * p.o.scales_ld + row);
    if (total) t.store(total + at, n);  // (after the values are read: total may be x or residual)
  };
  // (whole waves: one has a word of the row or is past it)
  if constexpr (SWEEPS > 0) {
#pragma unroll
    for (int i = 0; i < SWEEPS; ++i)
      if ((lane & ~63) * 8 + i * kStep < p.dim) write(lane * 8 + i * kStep, t[i]);
  } else {
    for (int at = lane * 8; at - (lane & 63) * 8 < p.dim; at += kStep) {
      read(at, t[0]);
      write(at, t[0]);
    }
  }
}

int check_rows(const char* fn, int64_t rows, int64_t dim, int dtype) {
  TTLH_REQUIRE(rows >= 0 && dim > 0, TTLH_EINVAL, "%s: bad sizes", fn);
  TTLH_REQUIRE(dtype == TTLH_BF16 || dtype == TTLH_F32, TTLH_EINVAL, "%s: bf16 or f32 values", fn);
  TTLH_REQUIRE(rows < (int64_t(1) << 31) && dim <= (int64_t(1) << 30), TTLH_EUNSUPPORTED,
               "%s: too many rows or values", fn);
  return TTLH_OK;
}

int check_out(const char* fn, int64_t rows, void* codes, int64_t codes_ld, void* scales,
              int64_t scales_ld, Out* o) {
  TTLH_REQUIRE(codes && scales, TTLH_EINVAL, "%s: null pointer", fn);
  TTLH_REQUIRE((reinterpret_cast<uintptr_t>(scales) & 3) == 0, TTLH_EINVAL,
               "%s: the scales must be 4-byte aligned", fn);
  o->codes = static_cast<uint8_t*>(codes);
  o->scales = static_cast<uint32_t*>(scales);
  o->codes_ld = codes_ld;
  o->scales_ld = scales_ld;
  return TTLH_OK;
}

int run_units(const char* fn, const void* a, int64_t a_ld, const void* b, int64_t b_ld, int dtype,
              int act, void* codes, int64_t codes_ld, void* scales, int64_t scales_ld, int64_t rows,
              int64_t dim, void* stream) {
  int st = check_rows(fn, rows, dim, dtype);
  if (st != TTLH_OK || rows == 0) return st;
  UnitArgs p;
  st = check_out(fn, rows, codes, codes_ld, scales, scales_ld, &p.o);
  if (st != TTLH_OK) return st;
  TTLH_REQUIRE(a && b, TTLH_EINVAL, "%s: null pointer", fn);
  p.a = a;
  p.b = b;
  p.a_ld = a_ld;
  p.b_ld = b_ld;
  p.rows = static_cast<int32_t>(rows);
  p.dim = static_cast<int32_t>(dim);
  p.words = static_cast<int32_t>((dim + kFp8Word - 1) / kFp8Word);
  p.blocks = (p.words + kThreads / 64 - 1) / (kThreads / 64);
  TTLH_REQUIRE(rows * p.blocks < (int64_t(1) << 31), TTLH_EUNSUPPORTED, "%s: too many rows or values", fn);
  const dim3 grid(static_cast<uint32_t>(rows * p.blocks));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, p); };
  const auto pick = [&](auto value) {
    typedef decltype(value) T;
    if (act == TTLH_GLU_SILU)
      run(fp8_units_kernel<T, TTLH_GLU_SILU>);
    else if (act == TTLH_GLU_GELU)
      run(fp8_units_kernel<T, TTLH_GLU_GELU>);
    else
      run(fp8_units_kernel<T, kActNone>);
  };
  dtype == TTLH_BF16 ? pick(uint16_t()) : pick(float());
  return check_launch("fp8_units_kernel");
}

}  // namespace
}  // namespace ttlh

using namespace ttlh;

extern "C" int ttlh_fp8_quant(const void* x, int64_t x_ld, int dtype, void* codes, int64_t codes_ld,
                              void* scales, int64_t scales_ld, int64_t rows, int64_t dim,
                              void* stream) {
  clear_error();
  return run_units("ttlh_fp8_quant", x, x_ld, x, x_ld, dtype, kActNone, codes, codes_ld, scales,
                   scales_ld, rows, dim, stream);
}

extern "C" int ttlh_fp8_glu(const void* gate, int64_t gate_ld, const void* up, int64_t up_ld,
                            int dtype, int act, void* codes, int64_t codes_ld, void* scales,
                            int64_t scales_ld, int64_t rows, int64_t dim, void* stream) {
  clear_error();
  TTLH_REQUIRE(act == TTLH_GLU_SILU || act == TTLH_GLU_GELU, TTLH_EINVAL,
               "ttlh_fp8_glu: unknown activation");
  return run_units("ttlh_fp8_glu", gate, gate_ld, up, up_ld, dtype, act, codes, codes_ld, scales,
                   scales_ld, rows, dim, stream);
}

extern "C" int ttlh_fp8_rms_norm(const void* x, int64_t x_ld, const void* residual,
                                 int64_t residual_ld, void* total, int64_t total_ld, int dtype,
                                 const void* weight, int weight_dtype, float eps, void* codes,
                                 int64_t codes_ld, void* scales, int64_t scales_ld, int64_t rows,
                                 int64_t dim, void* stream) {
  clear_error();
  const char* fn = "ttlh_fp8_rms_norm";
  int st = check_rows(fn, rows, dim, dtype);
  if (st != TTLH_OK) return st;
  TTLH_REQUIRE(weight_dtype == TTLH_BF16 || weight_dtype == TTLH_F32, TTLH_EINVAL,
               "%s: bf16 or f32 weights", fn);
  TTLH_REQUIRE(eps >= 0.0f && std::isfinite(eps), TTLH_EINVAL, "%s: eps must be finite and not negative", fn);
  if (rows == 0) return TTLH_OK;
  NormArgs p;
  st = check_out(fn, rows, codes, codes_ld, scales, scales_ld, &p.o);
  if (st != TTLH_OK) return st;
  TTLH_REQUIRE(x && weight, TTLH_EINVAL, "%s: null pointer", fn);
  p.x = x;
  p.residual = residual;
  p.total = total;
  p.weight = weight;
  p.x_ld = x_ld;
  p.residual_ld = residual_ld;
  p.total_ld = total_ld;
  p.rows = static_cast<int32_t>(rows);
  p.dim = static_cast<int32_t>(dim);
  p.weight_f32 = weight_dtype == TTLH_F32;
  p.eps = eps;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto run = [&](auto kernel, int lanes) {
    const int per = kThreads / lanes;
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>((rows + per - 1) / per)), dim3(kThreads), 0, s, p);
  };
  const auto pick = [&](auto value) {
    typedef decltype(value) T;
    if (dim <= 512)
      run(fp8_norm_kernel<T, 64, 1>, 64);
    else if (dim <= 2048)
      run(fp8_norm_kernel<T, 256, 1>, 256);
    else if (dim <= 4096)
      run(fp8_norm_kernel<T, 256, 2>, 256);
    else if (dim <= 8192)
      run(fp8_norm_kernel<T, 256, 4>, 256);
    else
      run(fp8_norm_kernel<T, 256, 0>, 256);
  };
  dtype == TTLH_BF16 ? pick(uint16_t()) : pick(float());
  return check_launch("fp8_norm_kernel");
}
