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
// 10^5) is therefore decided in fp64.  So is a code whose value is within 2^-20 of the middle between
// two (one in 10^5; found where the codes of the value a little up and a little down differ, two
// instructions a value).  Scales and codes are those of the values in fp64 (to 2^-40; nearer to a border
// than that they may be those of its other side), but for magnitudes below 2^-126, of a value or of
// one on the way to it (a norm before its weight, a gate's exponential, its integral), of which fp32 has
// less than 24 bits.

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
  u32x4 w[sizeof(T) / 2];
  // n: how many of them there are.  All eight, or zeros; nothing waits for the values here, so that
  // loads of several operands are under way at once.
  __device__ __forceinline__ void load(const T* p, int n) {
#pragma unroll
    for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h) w[h] = u32x4{0u, 0u, 0u, 0u};
    if (n >= 8) {
#pragma unroll
      for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h)
        w[h] = *reinterpret_cast<const u32x4u*>(p + h * (16 / sizeof(T)));
    }
  }
  // the first n of fewer than eight: a row's end
  __device__ __forceinline__ void load_end(const T* p, int n) {
    if (n <= 0 || n >= 8) return;
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 2)
          w[0][i / 2] |= static_cast<uint32_t>(p[i]) << (16 * (i & 1));
        else
          w[i / 4][i % 4] = __float_as_uint(p[i]);
      }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 2)
      return __uint_as_float(i & 1 ? w[0][i / 2] & 0xffff0000u : w[0][i / 2] << 16);
    else
      return __uint_as_float(w[i / 4][i % 4]);
  }
};

template <typename T>
__device__ __forceinline__ void store_eight(T* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<u32x4u*>(p) = u32x4{cvt_pk_bf16x2(v[0], v[1]), cvt_pk_bf16x2(v[2], v[3]),
                                            cvt_pk_bf16x2(v[4], v[5]), cvt_pk_bf16x2(v[6], v[7])};
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<u32x4u*>(p + 4 * h) =
            u32x4{__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]),
                  __float_as_uint(v[4 * h + 3])};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}

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

__device__ __forceinline__ uint2 eight_codes(const float (&y)[8], float by) {
  return uint2{four_codes<TTLH_CACHE_E4M3>(y[0] * by, y[1] * by, y[2] * by, y[3] * by),
               four_codes<TTLH_CACHE_E4M3>(y[4] * by, y[5] * by, y[6] * by, y[7] * by)};
}

// The code of x, rounded once: to fp32 towards zero, with the last place odd where something was
// lost, then to the nearest code.
__device__ __forceinline__ uint32_t code_of(double x) {
  const float f = static_cast<float>(x);
  const double back = static_cast<double>(f);
  uint32_t b = __float_as_uint(f);
  if (back != x) b = (fabs(back) > fabs(x) ? b - 1u : b) | 1u;
  return four_codes<TTLH_CACHE_E4M3>(__uint_as_float(b), 0.0f, 0.0f, 0.0f) & 255u;
}

// No value that decides a code or a scale is off by more, relative to its size, less 2^-24 for the products
// below.  Measured for every fp32 gate (whose integral is 2^-126 or more), u = 1: silu 4.2 x 2^-24, gelu
// 7.6 x 2^-24 (6.3 x 2^-24 up to |g| = 12); u adds 2^-24.
constexpr float kNear = 0x1p-20f;

// The codes of a wave's 512 values (n of a lane's eight exist) and their scales, to
// `codes` (the lane's) and `word`.  exact(i): value i in fp64, where fp32 does not decide
// a scale or a code.
template <bool EXACT, typename F>
__device__ __forceinline__ void emit(const float (&y)[8], F exact, int n, uint8_t* codes,
                                     uint32_t* word) {
  // the largest magnitude's bits (NaN: the largest): of the positive values as signed numbers, of the
  // negative ones as unsigned, without clearing eight signs
  int positive = 0;
  uint32_t negative = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    positive = max(positive, static_cast<int>(__float_as_uint(y[i])));
    negative = max(negative, __float_as_uint(y[i]));
  }
  const uint32_t m = row_max(max(static_cast<uint32_t>(positive), negative & 0x7fffffffu));
  int s = scale_code(m);
  if constexpr (!EXACT) {
    const bool open = scale_open(m) && s != kScaleNan;
    if (__any(open)) {
      // The largest is among the values within the errors of two.  (Of an open group alone: in one of
      // zeros, past the row's end too, every value is that near.)
      uint32_t near = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        near |= open && (__float_as_uint(y[i]) & 0x7fffffffu) + 128u >= m ? 1u << i : 0u;
      double big = 0.0;
      for (; near; near &= near - 1) big = fmax(big, fabs(exact(__ffs(near) - 1)));
#pragma unroll
      for (int i = 8; i; i >>= 1) big = fmax(big, __shfl_xor(big, i));
      if (open)
        s = scale_code64(static_cast<uint64_t>(__double_as_longlong(big)));
    }
  }
  const float inv = __uint_as_float(inverse_scale_bits(s));
  uint2 w = eight_codes(y, EXACT ? inv : inv * (1.0f + kNear));
  if constexpr (!EXACT) {
    const uint2 v = eight_codes(y, inv * (1.0f - kNear));
    const uint2 differ = {w.x ^ v.x, w.y ^ v.y};
    // (zeros, past the row's end too, do not)
    if (__any((differ.x | differ.y) != 0)) {
      uint64_t open = s == kScaleNan ? 0u : static_cast<uint64_t>(differ.y) << 32 | differ.x;
      while (open) {
        const int i = __builtin_ctzll(open) >> 3, at = 8 * (i & 3);
        const uint32_t c = code_of(exact(i) * static_cast<double>(inv));
        if (i < 4) w.x = (w.x & ~(255u << at)) | c << at;
        else w.y = (w.y & ~(255u << at)) | c << at;
        open &= ~(uint64_t(255) << (8 * i));
      }
    }
  }
  if (s == kScaleNan) w = uint2{0u, 0u};
  if (n >= 8) {
    *reinterpret_cast<uint2u*>(codes) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) codes[i] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
  }
  // (a group past the row's end: what a norm makes of its zeros is NaN where the row holds one)
  if (!EXACT && n <= 0) s = kScaleLeast;
  const uint32_t four = static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 0)) |
                        static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 16)) << 8 |
                        static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 32)) << 16 |
                        static_cast<uint32_t>(__builtin_amdgcn_readlane(s, 48)) << 24;
  if ((threadIdx.x & 63) == 0) *word = four;
}

// --- as they are, and gated -----------------------------------------------------

constexpr int kActNone = -1;

// x, or lo or hi where it is past them; a NaN: lo.  (fminf and fmaxf take two instructions each, the
// first to make NaN quiet: gelu 4099 x 11008 62 -> 58 us without them)
__device__ __forceinline__ float within(float x, float lo, float hi) {
  return __builtin_amdgcn_fmed3f(x, lo, hi);
}

// exp(x) for x <= 0, to a unit in the last place: 2^n 2^f with n + f = x log2 e, f from -1/2 to 1/2;
// results below 2^-126 keep their last place too.  (-150: zero, and NaN; a caller's product with x
// is what says NaN)
__device__ __forceinline__ float exp_down(float x) {
  constexpr float kL2E = 1.44269502e+00f, kL2ELo = 1.92596299e-08f;
  x = within(x, -150.0f, 0.0f);
  const float n = rintf(x * kL2E);
  const float f = __builtin_fmaf(x, kL2ELo, __builtin_fmaf(x, kL2E, -n));
  return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(n));
}

// 1 / d for d from 1 to 2, to one unit in the last place
__device__ __forceinline__ float reciprocal(float d) {
  const float r = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
}

// silu: with e = exp(-|g|), g / (1 + e) or g e / (1 + e), so that nothing overflows.
// gelu: g times the normal distribution's integral up to g, which below 0 is exp(-g^2 / 2) times a
// function that falls from 1/2 like 1 / |g|: a polynomial in s = (|g| - 4) / (|g| + 4), the variable that
// Shepherd and Laframboise (1981) took for the scaled complementary error function, with coefficients
// fitted here (least relative error, up to |g| = 14.5: 2^-25.9; beyond that the exponential is zero).  The library's complementary error function took three times as long:
// 4099 x 11008 bf16 89 us.
template <int ACT, bool BF16>
__device__ __forceinline__ float gated(float g, float u) {
  const float x = fabsf(g);
  if constexpr (ACT == TTLH_GLU_SILU) {
    const float e = exp_down(-x);
    return (g < 0.0f ? g * e : g) * reciprocal(1.0f + e) * u;
  } else {
    const float z = within(x, 0.0f, 16.0f);  // (the exponential is zero there)
    const float s = (z - 4.0f) * __builtin_amdgcn_rcpf(z + 4.0f);
    float h = -6.528619269374758e-05f;
    h = __builtin_fmaf(h, s, -0.00016782732564024627f);
    h = __builtin_fmaf(h, s, 0.0006577639142051339f);
    h = __builtin_fmaf(h, s, 0.0005025526625104249f);
    h = __builtin_fmaf(h, s, -0.008497918024659157f);
    h = __builtin_fmaf(h, s, 0.030865497887134552f);
    h = __builtin_fmaf(h, s, -0.07170674204826355f);
    h = __builtin_fmaf(h, s, 0.12437920272350311f);
    h = __builtin_fmaf(h, s, -0.17039774358272552f);
    h = __builtin_fmaf(h, s, 0.09441064298152924f);
    // 2^(n + f) = exp(-z^2 / 2), with the square's rounding error (of bf16: none) and the constant's tail
    constexpr float kC = -0.7213475108146667f, kCLo = -9.6298149e-09f;  // -log2 e / 2
    const float q = z * z, n = rintf(q * kC);
    float f = __builtin_fmaf(q, kCLo, __builtin_fmaf(q, kC, -n));
    if constexpr (!BF16) f = __builtin_fmaf(__builtin_fmaf(z, z, -q), kC, f);
    h = __builtin_amdgcn_ldexpf(h * __builtin_amdgcn_exp2f(f), static_cast<int>(n));
    return __builtin_fmaf(-x, h, within(g, 0.0f, 3.4028235e38f)) * u;
  }
}
// The same in fp64, to 2^-40, in few registers (the rare path decides the kernel's number of them,
// and with it how many waves a SIMD has).  The integral of the normal distribution below -x: up to
// x = 3 one half less the series phi(x) (x + x^3 / 3 + x^5 / 15 ..), from there on the continued
// fraction phi(x) / (x + 1 / (x + 2 / (x + 3 / ..))), both as far as x asks for.  (4099 x 11008 bf16, all
// gates 8, so that one product in 16 lies between two codes: 147 us; with 49 and 60 steps always, 280)
template <int ACT>
__device__ __forceinline__ double gated64(double g, double u) {
  const double x = fabs(g);
  if constexpr (ACT == TTLH_GLU_SILU) {
    const double e = exp(-x);
    return (g < 0.0 ? g * e : g) / (1.0 + e) * u;
  } else {
    const double phi = 0.39894228040143267794 * exp(-0.5 * x * x);
    const auto over = [](double d) {
      const double r = __builtin_amdgcn_rcp(d);
      return fma(fma(-d, r, 1.0), r, r);
    };
    double h;
    if (x < 3.0) {
      double term = x, sum = x;
#pragma unroll 1
      for (int i = 3, end = 30 + static_cast<int>(20.0 * x); i < end; i += 2) {
        term *= x * x * over(i);
        sum += term;
      }
      h = 0.5 - phi * sum;
    } else {
      double f = x;
#pragma unroll 1
      for (int i = 6 + static_cast<int>(560.0 * over(x * x)); i > 0; --i) f = fma(static_cast<double>(i), over(f), x);
      h = phi / f;
    }
    return g * (g < 0.0 ? h : 1.0 - h) * u;
  }
}

struct UnitArgs {
  const void* a;
  const void* b;
  int64_t a_ld, b_ld;
  Out o;
  int32_t units, dim, words;  // a unit: a word of a row
};

template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void fp8_units_kernel(const UnitArgs p) {
  const int unit = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= p.units) return;
  const int row = unit / p.words, word = unit - row * p.words;
  const int at = word * kFp8Word + (threadIdx.x & 63) * 8, n = p.dim - at;
  const T* pa = static_cast<const T*>(p.a) + row * p.a_ld + at;
  const T* pb = static_cast<const T*>(p.b) + row * p.b_ld + at;
  uint8_t* codes = p.o.codes + row * p.o.codes_ld + at;
  uint32_t* to = p.o.scales + word * p.o.scales_ld + row;
  Eight<T> a, b;
  a.load(pa, n);
  if constexpr (ACT != kActNone) b.load(pb, n);
  a.load_end(pa, n);
  if constexpr (ACT != kActNone) b.load_end(pb, n);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    y[i] = ACT == kActNone ? a[i] : gated<ACT == kActNone ? 0 : ACT, sizeof(T) == 2>(a[i], b[i]);
  emit<ACT == kActNone>(y, [&](int i) {
    return gated64<ACT == kActNone ? 0 : ACT>(static_cast<double>(to_f32(pa[i])), static_cast<double>(to_f32(pb[i])));
  }, min(n, 8), codes, to);
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
  double by_dim;  // 1 / dim
};

// the sum of x over the LANES (64, or a whole workgroup) that have a row
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
// of squares (in fp64: a group near a scale's border needs the exact norm) and the codes.  SWEEPS 0:
// any length, read twice.  SUM: there is a residual (asked in the kernel, 4099 x 11008 bf16 without one
// took 48 us in place of 35).
template <typename T, bool SUM, int LANES, int SWEEPS>
__global__ __launch_bounds__(LANES > kThreads ? LANES : kThreads) void fp8_norm_kernel(const NormArgs p) {
  constexpr int kStep = LANES * 8, kKept = SWEEPS ? SWEEPS : 1;
  const int row = LANES > 64 ? blockIdx.x
                             : blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & (LANES - 1);
  if (row >= p.rows) return;  // (a whole wave of its own where LANES is 64)
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* r = SUM ? static_cast<const T*>(p.residual) + row * p.residual_ld : nullptr;
  T* total = p.total ? static_cast<T*>(p.total) + row * p.total_ld : nullptr;
  // the values of SWEEPS places from lane * 8 + at on
  Eight<T> v[kKept], more[SUM ? kKept : 1];
  const auto read = [&](int at) {
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      const int k = at + lane * 8 + i * kStep;
      v[i].load(x + k, p.dim - k);
      if constexpr (SUM) more[i].load(r + k, p.dim - k);
    }
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      const int k = at + lane * 8 + i * kStep;
      v[i].load_end(x + k, p.dim - k);
      if constexpr (SUM) more[i].load_end(r + k, p.dim - k);
    }
  };
  const auto value = [&](int i, int e) { return SUM ? v[i][e] + more[SUM ? i : 0][e] : v[i][e]; };
  double sum = 0.0;
  const auto add = [&]() {
#pragma unroll
    for (int i = 0; i < kKept; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        double d = v[i][e];
        if constexpr (SUM) d += static_cast<double>(more[i][e]);
        sum = fma(d, d, sum);
      }
  };
  if constexpr (SWEEPS > 0) {
    read(0);
    add();
  } else {
    for (int at = 0; at < p.dim; at += kStep) {
      read(at);
      add();
    }
  }
  // 1 / sqrt(mean + eps), the hardware's to 2^-14 and better, twice as many places a step
  const double a = row_sum<LANES>(sum) * p.by_dim + static_cast<double>(p.eps);
  double by = __builtin_amdgcn_rsq(a);
#pragma unroll
  for (int i = 0; i < 2; ++i) by = fma(by * 0.5, fma(-a * by, by, 1.0), by);
  if (a > 1.7e308) by = 0.0;  // (infinite: its values make their own groups NaN)
  const float by32 = static_cast<float>(by);
  const int from = __builtin_amdgcn_readfirstlane(lane >> 6) * kFp8Word;
  const auto write = [&](int i, int word) {  // (whole waves: one has a word of the row or is past it)
    const int at = word * kFp8Word + (lane & 63) * 8, n = p.dim - at;
    float t[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = value(i, e);
    const auto weigh = [&](auto type) {
      typedef decltype(type) W;
      Eight<W> w;
      w.load(static_cast<const W*>(p.weight) + at, n);
      w.load_end(static_cast<const W*>(p.weight) + at, n);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = t[e] * by32 * w[e];
    };
    p.weight_f32 ? weigh(float()) : weigh(uint16_t());
    emit<false>(y, [&](int e) {
      double d = to_f32(x[at + e]);
      if constexpr (SUM) d += static_cast<double>(to_f32(r[at + e]));
      const double g = p.weight_f32 ? static_cast<const float*>(p.weight)[at + e]
                                    : to_f32(static_cast<const uint16_t*>(p.weight)[at + e]);
      return d * by * g;
    }, min(n, 8), p.o.codes + row * p.o.codes_ld + at, p.o.scales + word * p.o.scales_ld + row);
    if (total) store_eight(total + at, n, t);  // (after the values are read: total may be x or residual)
  };
  if constexpr (SWEEPS > 0) {
#pragma unroll
    for (int i = 0; i < SWEEPS; ++i)
      if (from + i * kStep < p.dim) write(i, (from + i * kStep) / kFp8Word);
  } else {
    for (int at = 0; at + from < p.dim; at += kStep) {
      read(at);
      write(0, (at + from) / kFp8Word);
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

int check_out(const char* fn, int64_t rows, int64_t dim, void* codes, int64_t codes_ld, void* scales,
              int64_t scales_ld, Out* o) {
  TTLH_REQUIRE(codes && scales, TTLH_EINVAL, "%s: null pointer", fn);
  TTLH_REQUIRE((rows == 1 || codes_ld >= dim) && (dim <= kFp8Word || scales_ld >= rows), TTLH_EINVAL,
               "%s: rows of codes or words of scales lie on one another", fn);
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
  st = check_out(fn, rows, dim, codes, codes_ld, scales, scales_ld, &p.o);
  if (st != TTLH_OK) return st;
  TTLH_REQUIRE(a && b, TTLH_EINVAL, "%s: null pointer", fn);
  p.a = a;
  p.b = b;
  p.a_ld = a_ld;
  p.b_ld = b_ld;
  const int64_t words = (dim + kFp8Word - 1) / kFp8Word, units = rows * words;
  // (a launch has less than 2^32 threads)
  TTLH_REQUIRE(units <= (int64_t(1) << 26) - kThreads / 64, TTLH_EUNSUPPORTED, "%s: too many rows or values", fn);
  p.units = static_cast<int32_t>(units);
  p.dim = static_cast<int32_t>(dim);
  p.words = static_cast<int32_t>(words);
  const dim3 grid(static_cast<uint32_t>((units + kThreads / 64 - 1) / (kThreads / 64)));
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
  // (positive: 1 / sqrt of it is a number in fp32, whatever the row)
  TTLH_REQUIRE(eps > 0.0f && std::isfinite(eps), TTLH_EINVAL, "%s: eps must be positive and finite", fn);
  if (rows == 0) return TTLH_OK;
  NormArgs p;
  st = check_out(fn, rows, dim, codes, codes_ld, scales, scales_ld, &p.o);
  if (st != TTLH_OK) return st;
  TTLH_REQUIRE(x && weight, TTLH_EINVAL, "%s: null pointer", fn);
  TTLH_REQUIRE(!total || rows == 1 || total_ld >= dim, TTLH_EINVAL, "%s: rows of the sum lie on one another", fn);
  // (a launch has less than 2^32 threads: 64, 256 or 512 a row)
  TTLH_REQUIRE(rows < (int64_t(1) << (dim <= 2048 ? 26 : 23)), TTLH_EUNSUPPORTED, "%s: too many rows", fn);
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
  p.by_dim = 1.0 / static_cast<double>(dim);
  hipStream_t s = static_cast<hipStream_t>(stream);
  // a wave a row up to 2048 values (8192 x 1024 bf16: 9.4 us, a workgroup a row 13.0), then a workgroup
  const auto run = [&](auto kernel, int lanes) {
    const int per = lanes > 64 ? 1 : kThreads / 64;
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>((rows + per - 1) / per)),
                       dim3(lanes > kThreads ? lanes : kThreads), 0, s, p);
  };
  const auto pick = [&](auto value, auto sum) {
    typedef decltype(value) T;
    constexpr bool S = decltype(sum)::value;
    if (dim <= 512)
      run(fp8_norm_kernel<T, S, 64, 1>, 64);
    else if (dim <= 1024)
      run(fp8_norm_kernel<T, S, 64, 2>, 64);
    else if (dim <= 2048)
      run(fp8_norm_kernel<T, S, 64, 4>, 64);
    else if (dim <= 4096)
      run(fp8_norm_kernel<T, S, 256, 2>, 256);
    else if (dim <= 8192)
      run(fp8_norm_kernel<T, S, 256, 4>, 256);
    else if (dim <= 12288)
      run(fp8_norm_kernel<T, S, 512, 3>, 512);
    else if (dim <= 16384)
      run(fp8_norm_kernel<T, S, 512, 4>, 512);
    else
      run(fp8_norm_kernel<T, S, 256, 0>, 256);
  };
  const auto sums = [&](auto value) {
    residual ? pick(value, std::true_type()) : pick(value, std::false_type());
  };
  dtype == TTLH_BF16 ? sums(uint16_t()) : sums(float());
  return check_launch("fp8_norm_kernel");
}
