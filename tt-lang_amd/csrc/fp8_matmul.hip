// Products of e4m3 codes with a scale for each 128 of K, for gfx950:
//   C[m, n] = sum over groups g of 2^(ex[m, g] + ew[n / 128, g]) sum over k in g of x[m, k] w[n, k]
// with fp32 accumulation.  x [M, K] and w [N, K] are both contiguous along K.
//
// Scales are powers of two, so a scaled MFMA applies them to its operands: a group costs no
// instruction of its own, and one accumulator runs through all of K.
//
// The fp8 MFMA aligns the products of eight neighbouring k to 2^-13 of the largest of them
// before it adds them (measured; sums of such eights are right to fp32), which leaves an error of
// 2^-19 of the products' sizes on average, far below the rounding of a bf16 result.  Results in
// fp32 (WIDE) keep fp32's accuracy: codes become bf16, which holds them exactly times a power of two in
// bf16's range, and go through bf16 MFMAs, at half the rate.  The exponents of a group's two scales are divided
// between the operands so that both are in that range (wide_w, wide_x); where the sum of the two leaves no
// such division (x's values from some 2^104 on, of weights of ordinary size), the rows of x concerned are
// computed again at the end, group by group, with the scales applied to the sums (4096^3 with one such row
// 475 us in place of 123; with one NaN row, whose results the same code writes, 131).
//
// Three kernels (choose_form, at the end, has the rule).  All of them bring whole lines of 128
// codes, a group, to LDS by direct-to-LDS loads of eight lanes a row: lanes of one load that lie in
// different rows, or halves of lines at different times, cost up to four times the rate at which a CU
// takes them (64 bytes a clock), and that rate, not memory, bounds the middle sizes.  A chunk of 16
// codes lies at its place XOR row / 2, so that an MFMA operand's reads meet no bank twice.  Codes past
// K are loaded as zeros, from kZeros: no kernel has a case for the last group.  With all CUs loading, each
// gets about 65 KB a us from its XCD's L2 (32 bytes a clock), and middle sizes run at that: 512 x 4096 x
// 4096 in blocks of 64 x 128 takes 201 MB so, 12 us of its 15.  (Dividing K among workgroups too, their
// parts joined by the last to arrive, brought 32 x 4096 x 11008 from 16.7 to 16.3 us and nothing else.)
//  * fp8_direct_kernel: few results.  The waves of a workgroup divide K, each with LDS of its own and
//    no barrier, and their sums are added in wave order.  1 x 22016 x 4096 19.0 us (4.7 TB/s of
//    weights; one quarter of the lanes' rate, straight to registers: 19.2, but 32 x 4096 x 11008 26.0 ->
//    16.2), 64 x 4096 x 4096 6.9 us.
//  * fp8_block_kernel: a ring of three buffers and one barrier a group, 64 x 64 to 128 x 256 results.
//    512 x 4096 x 4096 15.0 us (halves of lines: 21), 2048 x 4096 x 4096 36.4 us.
//  * fp8_large_kernel: 256 x 256, bf16 results.  8192 x 22016 x 4096 555 to 595 us by the card (2.5 to
//    2.7 PFLOP/s; in stages of half lines and a ring of four 703), 8192^3 380 to 400 us (2.8 PFLOP/s):
//    the MFMAs are busy 78% of the cycles, at the clock that the power cap leaves (1.5 GHz).

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "ttlh_common.h"
#include "ttlh_fp8.h"

namespace ttlh {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;

// s_waitcnt: at most n vector loads outstanding; all LDS reads done
constexpr int vmcnt_imm(int n) { return 0x0F70 | (n & 0xF) | ((n >> 4) << 14); }
constexpr int kLdsDone = 0xC07F;

// until at most n (to 2) rounds of LOADS loads are outstanding
template <int LOADS>
__device__ __forceinline__ void wait_behind(int n) {
  static_assert(2 * LOADS < 64, "what the counter holds");
  if (n == 2) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * LOADS));
  else if (n == 1) __builtin_amdgcn_s_waitcnt(vmcnt_imm(LOADS));
  else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
}

// What is read in the place of codes past K.
__device__ __attribute__((aligned(16))) const uint32_t kZeros[4] = {0u, 0u, 0u, 0u};

// 16 bytes at src + k a lane, or zeros, to LDS: lane l's land at to + 16 l.
__device__ __forceinline__ void load_lds(const uint8_t* src, int k, bool there, uint8_t* to) {
  const uint8_t* from = there ? src + k : reinterpret_cast<const uint8_t*>(kZeros);
  __builtin_amdgcn_global_load_lds(from, (lds_void*)to, 16, 0, 0);
}

struct Fp8Args {
  const uint8_t* x;
  const uint8_t* w;
  const uint32_t* xs;  // [words, M] dwords of four scales, xs_ld dwords from word to word
  const uint32_t* ws;  // [words, ceil(N / 128)]
  void* c;
  int64_t x_ld, w_ld, xs_ld, ws_ld, c_ld;
  int32_t M, N, K;
  int32_t grid_m, grid_n;
  int32_t c_f32;
  int32_t c_vec;   // four neighbouring results are one aligned store
  int32_t c_vec8;  // eight (bf16) are
};

// 32 codes of a row: the 16-byte chunks q and q + 4 of a group's eight
struct Frag {
  u32x4 lo, hi;
};

__device__ __forceinline__ i32x8 all8(const Frag& f) {
  return i32x8{static_cast<int>(f.lo[0]), static_cast<int>(f.lo[1]), static_cast<int>(f.lo[2]),
               static_cast<int>(f.lo[3]), static_cast<int>(f.hi[0]), static_cast<int>(f.hi[1]),
               static_cast<int>(f.hi[2]), static_cast<int>(f.hi[3])};
}

// eight codes (dwords a, b) times 2^(s - 127) as bf16; NaN where s is 255, whatever the codes are
__device__ __forceinline__ bf16x8 widened(uint32_t a, uint32_t b, int s) {
  const float scale = __uint_as_float(static_cast<uint32_t>(s) << 23);
  const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false);
  const bf16x2 q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true);
  const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false);
  const bf16x2 t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true);
  return bf16x8{p[0], p[1], q[0], q[1], r[0], r[1], t[0], t[1]};
}

// byte J of a dword of scales
template <int J>
__device__ __forceinline__ int scale_byte(uint32_t s) {
  return static_cast<int>(s >> (8 * J) & 255);
}

// acc += A . B over one group; sa, sb: its scales (WIDE: those of the operands, of wide_w and wide_x)
template <bool WIDE>
__device__ __forceinline__ f32x4 mma16(const Frag& a, const Frag& b, f32x4 acc, uint32_t sa, uint32_t sb) {
  if constexpr (!WIDE) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(all8(a), all8(b), acc, 0, 0, 0, static_cast<int>(sa), 0,
                                                            static_cast<int>(sb));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 u = h ? a.hi : a.lo, v = h ? b.hi : b.lo;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(u[2 * i], u[2 * i + 1], sa),
                                                      widened(v[2 * i], v[2 * i + 1], sb), acc, 0, 0, 0);
    }
    return acc;
  }
}

// Workgroup i runs on XCD i % 8: each XCD takes a contiguous run of the block order, in which
// the row blocks of one column of blocks follow each other and share w through that XCD's L2.
__device__ __forceinline__ void block_of(const Fp8Args& p, int& bm, int& bn) {
  const int n = gridDim.x, id = blockIdx.x;
  const int per = n >> 3, rem = n & 7, x = id & 7;
  const int i = x * per + min(x, rem) + (id >> 3);
  bn = i / p.grid_m;
  bm = i - bn * p.grid_m;
}

// four neighbouring results of a row
__device__ __forceinline__ void store4(const Fp8Args& p, int row, int col, f32x4 v) {
  if (row >= p.M || col >= p.N) return;
  const int64_t at = row * p.c_ld + col;
  const int n = p.N - col;
  if (p.c_f32) {
    float* c = static_cast<float*>(p.c) + at;
    if (p.c_vec && n >= 4) {
      *reinterpret_cast<f32x4*>(c) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) c[i] = v[i];
    }
  } else {
    uint16_t* c = static_cast<uint16_t*>(p.c) + at;
    const u32x2 w = {cvt_pk_bf16x2(v[0], v[1]), cvt_pk_bf16x2(v[2], v[3])};
    if (p.c_vec && n >= 4) {
      *reinterpret_cast<u32x2*>(c) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) c[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// Rows of x whose scales leave bf16's range, into fp32: a lane's results of a tile of T x T (T 16: four,
// 32: sixteen), of x's row `row` and w's from `col` on, over the groups from `first` on in steps of `step`.
// The codes as they are, exact in bf16, make a group's sums, which the scales are then applied to.
template <int T>
struct FarTile {
  typedef float Sums __attribute__((ext_vector_type(T == 16 ? 4 : 16)));
  static constexpr int kK = T == 16 ? 32 : 16;  // of an MFMA: a lane has eight codes of it

  static __device__ __forceinline__ Sums of(const Fp8Args& p, int row, int col, int first, int step) {
    const int lane = threadIdx.x & 63, at = 8 * (lane / T);
    row = min(row, p.M - 1);
    const uint8_t* x = p.x + row * p.x_ld + at;
    const uint8_t* w = p.w + min(col + lane % T, p.N - 1) * p.w_ld + at;
    const uint32_t* xs = p.xs + row;
    const uint32_t* ws = p.ws + min(col, p.N - 1) / kFp8Group;
    Sums sum;
#pragma unroll
    for (int r = 0; r < T * T / 64; ++r) sum[r] = 0.0f;
    const int groups = (p.K + kFp8Group - 1) / kFp8Group;
#pragma unroll 1
    for (int g = first; g < groups; g += step) {
      Sums s;
#pragma unroll
      for (int r = 0; r < T * T / 64; ++r) s[r] = 0.0f;
#pragma unroll
      for (int k = g * kFp8Group, i = 0; i < kFp8Group / kK; ++i, k += kK) {
        u32x2 a = {0u, 0u}, b = {0u, 0u};
        if (k + at < p.K) {  // (K is a multiple of 16: all eight exist)
          a = *reinterpret_cast<const u32x2*>(w + k);
          b = *reinterpret_cast<const u32x2*>(x + k);
        }
        const bf16x8 u = widened(a[0], a[1], 127), v = widened(b[0], b[1], 127);
        if constexpr (T == 16)
          s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u, v, s, 0, 0, 0);
        else
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u, v, s, 0, 0, 0);
      }
      int ex, ew;
      scales(xs, ws, p, g, ex, ew);
#pragma unroll
      for (int r = 0; r < T * T / 64; ++r) sum[r] += __builtin_amdgcn_ldexpf(s[r], ex + ew - 254);
    }
    return sum;
  }

  // group g's
  static __device__ __forceinline__ void scales(const uint32_t* xs, const uint32_t* ws, const Fp8Args& p, int g,
                                                int& ex, int& ew) {
    const int64_t word = g >> 2;
    ex = static_cast<int>(xs[word * p.xs_ld] >> (8 * (g & 3)) & 255);
    ew = static_cast<int>(ws[word * p.ws_ld] >> (8 * (g & 3)) & 255);
  }

  // whether the row's results of those groups are NaN, and if not, whether they leave bf16's range
  static __device__ __forceinline__ void look(const Fp8Args& p, int row, int col, int first, int step, bool& far,
                                              bool& nan) {
    const uint32_t* xs = p.xs + min(row, p.M - 1);
    const uint32_t* ws = p.ws + min(col, p.N - 1) / kFp8Group;
    const int groups = (p.K + kFp8Group - 1) / kFp8Group;
    far = nan = false;
#pragma unroll 8
    for (int g = first; g < groups; g += step) {
      int ex, ew;
      scales(xs, ws, p, g, ex, ew);
      far |= wide_far(wide_rest(ex, ew));
      nan |= max(ex, ew) == kScaleNan;
    }
    far = far && !nan;
  }
};

// WIDE: the largest scales that a lane has seen of its rows of x, and of w's.
struct Seen {
  int rest = 0, ex = 0, ew = 0;
  // the scale of x's operand for a row's e and the wave's w
  __device__ __forceinline__ int take(int e, int w) {
    const int r = wide_rest(e, w);
    rest = max(rest, r);
    ex = max(ex, e);
    return wide_x(r);
  }
  // whether results of the wave have to be made anew
  __device__ __forceinline__ bool any() const { return __any(wide_far(rest) || max(ex, ew) == kScaleNan); }
};

// MT x 16 rows of x, NT x 16 of w a workgroup; wave v of WAVES takes the groups v, v + WAVES ..
// of K, two of them in flight.
template <int MT, int NT, int WAVES, bool WIDE>
__global__ __launch_bounds__(WAVES * 64) void fp8_direct_kernel(const Fp8Args p) {
  static_assert(WAVES % 4 == 0 && 128 % (NT * 16) == 0, "one byte of the scales a wave, one block of w's");
  constexpr int kRows = (MT + NT) * 16;  // of a wave's group: those of w, then those of x
  constexpr int kSlot = kRows * kFp8Group;
  __shared__ __attribute__((aligned(16))) uint8_t b0[WAVES * kSlot], b1[WAVES * kSlot];
  int bm, bn;
  block_of(p, bm, bn);
  // (uniform, and known to be: an MFMA behind a branch that the compiler takes for divergent
  // runs whether or not its lanes are masked)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto slot = [&](int a) -> uint8_t* { return (a ? b1 : b0) + wave * kSlot; };
  const int m0 = bm * MT * 16, n0 = bn * NT * 16;
  const int groups = (p.K + kFp8Group - 1) / kFp8Group;
  const int n = groups > wave ? (groups - wave + WAVES - 1) / WAVES : 0;  // of this wave

  // Loads: eight rows of 128 codes an instruction, eight lanes a row (a row's 16 bytes by lanes 16
  // apart, as the MFMA has them, are a quarter of the rate: 16 bytes a clock and CU).  Chunk c of
  // row r of a tile lies at c ^ (r / 2 & 7).  Rows past the last one are read as the last one:
  // they reach results that are not stored.
  const int chunk = 16 * ((lane & 7) ^ (lane >> 4));  // of a tile's rows 0 to 7; of 8 to 15: ^ 64
  const uint8_t* src[kRows / 8];
#pragma unroll
  for (int i = 0; i < kRows / 8; ++i) {
    const int row = 8 * i + (lane >> 3);
    src[i] = (i < 2 * NT ? p.w + min(n0 + row, p.N - 1) * p.w_ld
                         : p.x + min(m0 + row - 16 * NT, p.M - 1) * p.x_ld) + (i & 1 ? chunk ^ 64 : chunk);
  }
  const int r = lane & 15, q = lane >> 4;
  const uint8_t* ws = reinterpret_cast<const uint8_t*>(p.ws + n0 / kFp8Group) + (wave & 3);
  const uint8_t* xs[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    xs[i] = reinterpret_cast<const uint8_t*>(p.xs + min(m0 + 16 * i + r, p.M - 1)) + (wave & 3);
  uint32_t sw[2], sx[2][MT];
  const auto load = [&](int a, int i) {  // (past the wave's last group: zeros)
    const int g = wave + WAVES * i, k = g * kFp8Group, word = min(g, groups - 1) >> 2;
    const bool even = k + chunk < p.K, odd = k + (chunk ^ 64) < p.K;
#pragma unroll
    for (int j = 0; j < kRows / 8; ++j) load_lds(src[j], k, j & 1 ? odd : even, slot(a) + j * 1024);
    sw[a] = ws[4 * word * p.ws_ld];
#pragma unroll
    for (int j = 0; j < MT; ++j) sx[a][j] = xs[j][4 * word * p.xs_ld];
    __builtin_amdgcn_sched_barrier(0);
  };
  // of a group (the scales are bytes at any address, which no scalar load reads: vmcnt sees them all)
  constexpr int kLoads = kRows / 8 + 1 + MT;

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // A lane has row r of a tile, chunks q and q + 4.
  const int at_lo = r * kFp8Group + 16 * (q ^ (r >> 1)), at_hi = at_lo ^ 64;
  Seen seen;
  const auto multiply = [&](int a) {
    Frag w[NT], x[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
      w[j] = Frag{*reinterpret_cast<const u32x4*>(slot(a) + j * 2048 + at_lo),
                  *reinterpret_cast<const u32x4*>(slot(a) + j * 2048 + at_hi)};
#pragma unroll
    for (int i = 0; i < MT; ++i)
      x[i] = Frag{*reinterpret_cast<const u32x4*>(slot(a) + (NT + i) * 2048 + at_lo),
                  *reinterpret_cast<const u32x4*>(slot(a) + (NT + i) * 2048 + at_hi)};
    if constexpr (WIDE) {
      // (volatile: the compiler would move what depends on a scale alone in front of the wait above, right
      // behind the scale's load, and wait there: 100 x 4000 x 4096 12.3 us in place of 10.1)
      asm volatile("" : "+v"(sw[a]));
      const int ew = __builtin_amdgcn_readfirstlane(sw[a]);
      seen.ew = max(seen.ew, ew);
      sw[a] = wide_w(ew);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        asm volatile("" : "+v"(sx[a][i]));
        sx[a][i] = seen.take(sx[a][i], ew);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mma16<WIDE>(w[j], x[i], acc[i][j], sw[a], sx[a][i]);
    __builtin_amdgcn_sched_barrier(0);  // (the slot is read before it is loaded anew)
  };
#pragma unroll
  for (int a = 0; a < 2; ++a) load(a, a);
  int i = 0;
  for (; i + 2 < n; i += 2) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      wait_behind<kLoads>(1);
      multiply(a);
      load(a, i + a + 2);
    }
  }
#pragma unroll
  for (int a = 0; a < 2; ++a)
    if (i + a < n) {
      wait_behind<kLoads>(1 - a);
      multiply(a);
    }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (no load of a wave without groups is left to land)
  __syncthreads();
  // The waves' sums, where the codes were: a lane has four neighbouring results of row r, columns
  // 16 j + 4 q ..
  static_assert(MT * NT * 1024 <= kSlot, "a wave's sums fit its slot");
  f32x4* part = reinterpret_cast<f32x4*>(b0);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) part[(wave * MT * NT + i * NT + j) * 64 + lane] = acc[i][j];
  if constexpr (WIDE) {
    if (seen.any()) {
#pragma unroll 1
      for (int i = 0; i < MT; ++i) {
        const int row = m0 + 16 * i + r;
        bool far, nan;
        FarTile<16>::look(p, row, n0, wave, WAVES, far, nan);
        const bool some = __any(far);
#pragma unroll 1
        for (int j = 0; j < NT; ++j) {
          f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
          if (some) s = FarTile<16>::of(p, row, n0 + 16 * j, wave, WAVES);
          if (nan) s += __builtin_nanf("");
          if (far || nan) part[(wave * MT * NT + i * NT + j) * 64 + lane] = s;
        }
      }
    }
  }
  __syncthreads();
  for (int t = wave; t < MT * NT; t += WAVES) {
    f32x4 s = part[t * 64 + lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) s += part[(v * MT * NT + t) * 64 + lane];
    store4(p, m0 + 16 * (t / NT) + r, n0 + 16 * (t % NT) + 4 * q, s);
  }
}

// --- more results ---------------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));

// One k = 64 step of a 32 x 32 tile; E: the scales' byte (WIDE: as in mma16)
template <bool WIDE, int E>
__device__ __forceinline__ f32x16 mma32(const Frag& a, const Frag& b, f32x16 acc, uint32_t sa, uint32_t sb) {
  if constexpr (!WIDE) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(all8(a), all8(b), acc, 0, 0, E, static_cast<int>(sa), E,
                                                           static_cast<int>(sb));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 u = h ? a.hi : a.lo, v = h ? b.hi : b.lo;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widened(u[2 * i], u[2 * i + 1], sa),
                                                      widened(v[2 * i], v[2 * i + 1], sb), acc, 0, 0, 0);
    }
    return acc;
  }
}

// Blocks in bands of `band` rows of blocks; an XCD's blocks follow each other there.
__device__ __forceinline__ void banded_block(const Fp8Args& p, int band, int& bm, int& bn) {
  const int n = gridDim.x, id = blockIdx.x;
  const int per = n >> 3, rem = n & 7, x = id & 7;
  const int i = x * per + min(x, rem) + (id >> 3);
  const int size = band * p.grid_n, b = i / size, in = i - b * size;
  const int rows = min(band, p.grid_m - b * band);
  bn = in / rows;
  bm = b * band + in - bn * rows;
}

// A tile of 32 x 32 results from row, col: a lane has row lane % 32 and the columns 8 r + 4 h ..
// + 3 (r < 4, h = lane / 32).  WHOLE: bf16, all columns exist and eight are one aligned store; the
// halves of two r change places, so that a lane has eight neighbours.
template <bool WHOLE>
__device__ __forceinline__ void store_tile(const Fp8Args& p, int row, int col, const f32x16& v) {
  const int lane = threadIdx.x & 63, h = lane >> 5;
  row += lane & 31;
  if constexpr (!WHOLE) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      store4(p, row, col + 8 * r + 4 * h, f32x4{v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]});
  } else {
    u32x4* c = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.c) + row * p.c_ld + col + 8 * h);
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      const auto e = __builtin_amdgcn_permlane32_swap(cvt_pk_bf16x2(v[4 * r], v[4 * r + 1]),
                                                      cvt_pk_bf16x2(v[4 * r + 4], v[4 * r + 5]), false, false);
      const auto o = __builtin_amdgcn_permlane32_swap(cvt_pk_bf16x2(v[4 * r + 2], v[4 * r + 3]),
                                                      cvt_pk_bf16x2(v[4 * r + 6], v[4 * r + 7]), false, false);
      if (row < p.M) c[r] = u32x4{e[0], o[0], e[1], o[1]};
    }
  }
}

// Results of TX x TW tiles, acc[i][j] tile i of x's rows and j of w's.
template <int TX, int TW>
__device__ __forceinline__ void store_tiles(const Fp8Args& p, int m0, int n0, const f32x16 (&acc)[TX][TW]) {
  const bool whole = !p.c_f32 && p.c_vec8 && n0 + 32 * TW <= p.N;
  if (whole) {
#pragma unroll
    for (int i = 0; i < TX; ++i)
#pragma unroll
      for (int j = 0; j < TW; ++j) store_tile<true>(p, m0 + 32 * i, n0 + 32 * j, acc[i][j]);
  } else {
#pragma unroll
    for (int i = 0; i < TX; ++i)
#pragma unroll
      for (int j = 0; j < TW; ++j) store_tile<false>(p, m0 + 32 * i, n0 + 32 * j, acc[i][j]);
  }
}

// The scales of a wave's TX x 32 rows of x (a lane's in each tile) and of its rows of w, which are
// in one block: a word, four groups, at a time, one ahead.
template <int TX, bool WIDE>
struct Scales {
  const uint32_t* ws;
  const uint32_t* xs[TX];
  uint32_t lane0 = 0;
  uint32_t w, x[TX], next_w, next_x[TX];
  int words;
  uint32_t past;  // bytes of the last word that are of no group: those scales may be anything
  // What the waits below count: loads that are vector loads whatever the compiler does.  x's addresses are a
  // lane's own.  w's is the same for a wave, so its load may be a scalar one, which vmcnt does not see; but
  // for `lane0`, which the compiler does not know to be 0.  (WIDE: not counted, the waits one load stricter
  // than they may have to be, and w's scales in scalar registers.  2048 x 4096 x 4096 into f32 64.3 us, 67 the
  // other way; 250 x 4000 x 4096 into bf16 11.2 us so, 10.8 the other way.)
  static constexpr int kLoads = WIDE ? TX : TX + 1;

  __device__ __forceinline__ Scales(const Fp8Args& p, int m, int n) {
    words = (p.K + kFp8Word - 1) / kFp8Word;
    const int last = (p.K - 1) / kFp8Group & 3;
    past = last == 3 ? 0u : ~0u << (8 * last + 8);
    ws = p.ws + min(n, p.N - 1) / kFp8Group;
    if constexpr (!WIDE) asm volatile("" : "+v"(lane0));
#pragma unroll
    for (int i = 0; i < TX; ++i) xs[i] = p.xs + min(m + 32 * i + static_cast<int>(threadIdx.x & 31), p.M - 1);
    load(p, 0);
  }
  __device__ __forceinline__ void load(const Fp8Args& p, int word) {
    word = min(word, words - 1);
    next_w = (ws + word * p.ws_ld)[lane0];
#pragma unroll
    for (int i = 0; i < TX; ++i) next_x[i] = xs[i][word * p.xs_ld];
  }
  __device__ __forceinline__ void take(const Fp8Args& p, int word) {
    const uint32_t none = word == words - 1 ? past : 0u;  // (their codes are zeros, their scale 1 / 2^127)
    w = next_w & ~none;
    if constexpr (WIDE) w = __builtin_amdgcn_readfirstlane(w);  // (what is made of it is scalar, and free)
#pragma unroll
    for (int i = 0; i < TX; ++i) x[i] = next_x[i] & ~none;
    load(p, word + 1);
    __builtin_amdgcn_sched_barrier(0);  // (the waits below count these loads)
  }
};

template <typename F, int... I>
__device__ __forceinline__ void each_until(F f, std::integer_sequence<int, I...>) {
  (void)(f(std::integral_constant<int, I>()) && ...);
}

// A wave has TX x TW tiles of 32 x 32 (of x's rows, of w's), four waves a block of 64 TX x 64 TW; a
// ring of three buffers.  A group's fragments are read while the one before it is multiplied.
template <int TX, int TW, bool WIDE>
__global__ __launch_bounds__(256, TX * TW < 3 ? 2 : 1) void fp8_block_kernel(const Fp8Args p) {
  constexpr int kRing = 3;
  constexpr int kXBytes = 64 * TX * kFp8Group, kWBytes = 64 * TW * kFp8Group;
  __shared__ __attribute__((aligned(16))) uint8_t x0[kXBytes], x1[kXBytes], x2[kXBytes], w0[kWBytes], w1[kWBytes],
      w2[kWBytes];
  const auto xbuf = [&](auto q) -> uint8_t* {
    constexpr int Q = decltype(q)::value % kRing;
    return Q == 0 ? x0 : Q == 1 ? x1 : x2;
  };
  const auto wbuf = [&](auto q) -> uint8_t* {
    constexpr int Q = decltype(q)::value % kRing;
    return Q == 0 ? w0 : Q == 1 ? w1 : w2;
  };
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int bm, bn;
  banded_block(p, 4, bm, bn);
  const int wm = (wave & 1) * 32 * TX, wn = (wave >> 1) * 32 * TW;
  const int m0 = bm * 64 * TX, n0 = bn * 64 * TW;
  const int groups = (p.K + kFp8Group - 1) / kFp8Group;

  // a thread's loads of a group: rows 32 i + t / 8; chunk c of row r lies at c ^ (r / 2 & 7)
  const int chunk = 16 * ((t & 7) ^ (t >> 4 & 7));
  const uint8_t *xsrc[2 * TX], *wsrc[2 * TW];
  // (rows past the last one are read as the last one: they reach results that are not stored)
#pragma unroll
  for (int i = 0; i < 2 * TX; ++i)
    xsrc[i] = p.x + static_cast<int64_t>(min(m0 + 32 * i + (t >> 3), p.M - 1)) * p.x_ld + chunk;
#pragma unroll
  for (int i = 0; i < 2 * TW; ++i)
    wsrc[i] = p.w + static_cast<int64_t>(min(n0 + 32 * i + (t >> 3), p.N - 1)) * p.w_ld + chunk;
  const int base = wave * 1024;  // where a wave's lanes land
  constexpr int kLoads = 2 * (TX + TW);
  const auto load_piece = [&](auto q, int k, bool there, int i) {
    if (i < 2 * TX)
      load_lds(xsrc[i], k, there, xbuf(q) + i * 4096 + base);
    else
      load_lds(wsrc[i - 2 * TX], k, there, wbuf(q) + (i - 2 * TX) * 4096 + base);
  };

  // fragments: row lane % 32 of a tile, chunks 4 k + 2 h and 4 k + 2 h + 1 of 64 codes k, h = lane / 32
  const int l32 = lane & 31, h = lane >> 5;
  int at[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) at[c] = l32 * kFp8Group + ((4 * (c >> 1) + 2 * h + (c & 1)) ^ (l32 >> 1 & 7)) * 16;
  struct Frags {
    Frag w[TW][2], x[TX][2];
  };
  Frags f0, f1;
  constexpr int kReads = 4 * (TX + TW);
  const auto read_piece = [&](auto q, Frags& f, int y) {  // all of the first 64 codes, then the others
    const int k = y / (kReads / 2), z = y % (kReads / 2);
    const uint8_t* b = z < 2 * TW ? wbuf(q) + wn * kFp8Group : xbuf(q) + wm * kFp8Group;
    const int i = (z < 2 * TW ? z : z - 2 * TW) >> 1;
    const u32x4 v = *reinterpret_cast<const u32x4*>(b + i * 32 * kFp8Group + at[2 * k + (z & 1)]);
    Frag& g = z < 2 * TW ? f.w[i][k] : f.x[i][k];
    if (z & 1) g.hi = v;
    else g.lo = v;
  };

  f32x16 acc[TX][TW];
#pragma unroll
  for (int i = 0; i < TX; ++i)
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  Scales<TX, WIDE> scale(p, m0 + wm, n0 + wn);
  Seen seen;
  each_until([&](auto q) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_piece(q, decltype(q)::value * kFp8Group, decltype(q)::value * kFp8Group + chunk < p.K, i);
    return true;
  }, std::make_integer_sequence<int, kRing>());
  wait_behind<kLoads>(kRing - 1);
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int y = 0; y < kReads; ++y) read_piece(std::integral_constant<int, 0>(), f0, y);

  // Group s = U of a turn of the loop, whose fragments are in cur.  Behind the barrier every wave
  // has read its fragments of group s, so its buffers take group s + kRing (past the last one:
  // zeros), and group s + 1 has landed.
  const auto group = [&](auto uu, Frags& cur, Frags& nxt, int s) {
    constexpr int U = decltype(uu)::value, E = U % 4;
    using Next = std::integral_constant<int, U + 1>;
    if constexpr (E == 0) scale.take(p, s >> 2);
    uint32_t sw = scale.w, sx[TX];
#pragma unroll
    for (int i = 0; i < TX; ++i)
      sx[i] = WIDE ? seen.take(scale_byte<E>(scale.x[i]), scale_byte<E>(sw)) : scale.x[i];
    if constexpr (WIDE) {
      seen.ew = max(seen.ew, scale_byte<E>(sw));
      sw = wide_w(scale_byte<E>(sw));
    }
    if constexpr (WIDE) __builtin_amdgcn_sched_barrier(0);  // (in front of the barrier, where waves wait)
    const int k2 = (s + kRing) * kFp8Group;
    const bool there = k2 + chunk < p.K;
    __builtin_amdgcn_s_waitcnt(kLdsDone);
    // (are the scales' loads, at a word's first group, among those behind group s + 1's?)
    __builtin_amdgcn_s_waitcnt(vmcnt_imm((kRing - 2) * kLoads + (E <= kRing - 2 ? Scales<TX, WIDE>::kLoads : 0)));
    __builtin_amdgcn_s_barrier();
    constexpr int kMma = 2 * TX * TW;
#pragma unroll
    for (int v = 0; v < kMma; ++v) {
      const int k = v / (TX * TW), i = v / TW % TX, j = v % TW;
      acc[i][j] = mma32<WIDE, E>(cur.w[j][k], cur.x[i][k], acc[i][j], sw, sx[i]);
      // the reads in the first three quarters, so that they are done at the barrier
      const int r0 = min(kReads, v * kReads * 4 / (3 * kMma)), r1 = min(kReads, (v + 1) * kReads * 4 / (3 * kMma));
#pragma unroll
      for (int z = 0; z < kReads; ++z)
        if (z >= r0 && z < r1) read_piece(Next(), nxt, z);
      const int l0 = v * kLoads / kMma, l1 = (v + 1) * kLoads / kMma;
#pragma unroll
      for (int z = 0; z < kLoads; ++z)
        if (z >= l0 && z < l1) load_piece(uu, k2, there, z);
      __builtin_amdgcn_sched_barrier(0);
    }
    return s + 1 < groups;
  };
  constexpr int kTurn = 12;  // whole rings, words and pairs of fragments
  for (int s = 0; s < groups; s += kTurn)
    each_until([&](auto uu) {
      constexpr int U = decltype(uu)::value;
      return U % 2 ? group(uu, f1, f0, s + U) : group(uu, f0, f1, s + U);
    }, std::make_integer_sequence<int, kTurn>());
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (no load is left to land in LDS that another has by then)
  store_tiles(p, m0 + wm, n0 + wn, acc);
  if constexpr (WIDE) {
    if (seen.any()) {
#pragma unroll 1
      for (int i = 0; i < TX; ++i) {
        const int row = m0 + wm + 32 * i + l32;
        bool far, nan;
        FarTile<32>::look(p, row, n0 + wn, 0, 1, far, nan);
        const bool some = __any(far);
#pragma unroll 1
        for (int j = 0; j < TW; ++j) {
          const int col = n0 + wn + 32 * j;
          f32x16 v = {};
          if (some) v = FarTile<32>::of(p, row, col, 0, 1);
          if (nan) v += __builtin_nanf("");
          if (far || nan) {  // (the lane that has stored these results before)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              store4(p, row, col + 8 * r + 4 * h, f32x4{v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]});
          }
        }
      }
    }
  }
}

// 256 x 256 results a workgroup, 128 x 128 a wave.  Two buffers of a group are all that LDS holds, so
// a buffer is given back in parts.  A wave keeps all fragments of w of a group, and goes through
// x's four tiles in turn, one read ahead; while the last one is multiplied it reads the next
// group's of w and its first of x.  Two barriers a group s:
//  * behind tile 0: everyone has read w and x's tiles 0 and 1 of s, whose memory takes those of s + 2;
//    tiles 2 and 3 of s have landed;
//  * behind tile 2: everyone has read x's tiles 2 and 3; w and tiles 0 and 1 of s + 1 have landed.
// Loads are 32 to 48 MFMAs ahead of their use.  CUT: K ends inside a group.  Without that the loads need
// no choice between codes and zeros: two vector instructions a load fewer, and 1.3% less time, since
// what bounds this kernel is power (workgroups set apart in time by up to 6 us, so that their stores do
// not meet: no change).
template <bool CUT>
__global__ __launch_bounds__(256, 1) void fp8_large_kernel(const Fp8Args p) {
  constexpr int kBytes = 256 * kFp8Group;
  __shared__ __attribute__((aligned(16))) uint8_t xa0[kBytes / 2], xb0[kBytes / 2], xa1[kBytes / 2],
      xb1[kBytes / 2], w0[kBytes], w1[kBytes];  // xa: tiles 0 and 1 of both halves of the rows
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int bm, bn;
  banded_block(p, 4, bm, bn);
  const int wm = wave & 1, wn = wave >> 1;
  const int m0 = bm * 256, n0 = bn * 256;
  const int groups = (p.K + kFp8Group - 1) / kFp8Group;

  // a thread's loads: rows 32 i + t / 8; chunk c of row r lies at c ^ (r / 2 & 7).  Row 32 (4 m + i)
  // of x is tile i of half m: piece 2 m + (i & 1) of xa or xb.
  const int chunk = 16 * ((t & 7) ^ (t >> 4 & 7));
  const uint8_t *xsrc[8], *wsrc[8];
  // (rows past the last one are read as the last one: they reach results that are not stored)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    xsrc[i] = p.x + static_cast<int64_t>(min(m0 + 32 * i + (t >> 3), p.M - 1)) * p.x_ld + chunk;
    wsrc[i] = p.w + static_cast<int64_t>(min(n0 + 32 * i + (t >> 3), p.N - 1)) * p.w_ld + chunk;
  }
  const int base = wave * 1024;
  const auto load = [&](const uint8_t* src, int k, bool there, uint8_t* to) {
    if constexpr (CUT)
      load_lds(src, k, there, to);
    else
      __builtin_amdgcn_global_load_lds(src + k, (lds_void*)to, 16, 0, 0);
  };
  const auto load_xa = [&](auto q, int k, bool there, int z) {
    load(xsrc[4 * (z >> 1) + (z & 1)], k, there, (decltype(q)::value & 1 ? xa1 : xa0) + z * 4096 + base);
  };
  const auto load_xb = [&](auto q, int k, bool there, int z) {
    load(xsrc[4 * (z >> 1) + 2 + (z & 1)], k, there, (decltype(q)::value & 1 ? xb1 : xb0) + z * 4096 + base);
  };
  const auto load_w = [&](auto q, int k, bool there, int z) {
    load(wsrc[z], k, there, (decltype(q)::value & 1 ? w1 : w0) + z * 4096 + base);
  };
  // where group s begins; past the last one CUT: zeros, else the last one's codes again (their scales
  // are then 2^-127, and products of 2^-254 add nothing)
  const auto begin = [&](int s) { return (CUT ? s : min(s, groups - 1)) * kFp8Group; };

  const int l32 = lane & 31, h = lane >> 5;
  int at[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) at[c] = l32 * kFp8Group + ((4 * (c >> 1) + 2 * h + (c & 1)) ^ (l32 >> 1 & 7)) * 16;
  Frag fw[4][2], fx[2][2];
  // chunk y of four of x's tile i, of w's tile j
  const auto read_x = [&](auto q, int i, int y) {
    constexpr bool Q = decltype(q)::value & 1;
    const uint8_t* from = (i < 2 ? (Q ? xa1 : xa0) : (Q ? xb1 : xb0)) + (2 * wm + (i & 1)) * 4096;
    const u32x4 v = *reinterpret_cast<const u32x4*>(from + at[y]);
    Frag& g = fx[i & 1][y >> 1];
    if (y & 1) g.hi = v;
    else g.lo = v;
  };
  const auto read_w = [&](auto q, int j, int y) {
    constexpr bool Q = decltype(q)::value & 1;
    const u32x4 v = *reinterpret_cast<const u32x4*>((Q ? w1 : w0) + (4 * wn + j) * 4096 + at[y]);
    Frag& g = fw[j][y >> 1];
    if (y & 1) g.hi = v;
    else g.lo = v;
  };

  f32x16 acc[4][4];  // [x tile][w tile]
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  Scales<4, false> scale(p, m0 + 128 * wm, n0 + 128 * wn);
  // the first group, and of the second what the first one's turn does not load
  {
    const int second_k = begin(1);
    const bool first = chunk < p.K, second = second_k + chunk < p.K;
#pragma unroll
    for (int z = 0; z < 4; ++z) load_xa(I0(), 0, first, z);
#pragma unroll
    for (int z = 0; z < 8; ++z) load_w(I0(), 0, first, z);
#pragma unroll
    for (int z = 0; z < 4; ++z) load_xb(I0(), 0, first, z);
#pragma unroll
    for (int z = 0; z < 4; ++z) load_xa(I1(), second_k, second, z);
#pragma unroll
    for (int z = 0; z < 8; ++z) load_w(I1(), second_k, second, z);
#pragma unroll
    for (int z = 0; z < 2; ++z) load_xb(I1(), second_k, second, z);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(14));
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int y = 0; y < 4; ++y) read_x(I0(), 0, y);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int y = 0; y < 4; ++y) read_w(I0(), j, y);

  const auto group = [&](auto uu, int s) {  // group s = U of a word
    constexpr int U = decltype(uu)::value;
    using Next = std::integral_constant<int, U + 1>;
    if constexpr (U == 0) scale.take(p, s >> 2);
    const int k1 = begin(s + 1), k2 = begin(s + 2);
    const bool there1 = k1 + chunk < p.K, there2 = k2 + chunk < p.K;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const int j = v >> 1, k = v & 1;
        acc[i][j] = mma32<false, U>(fw[j][k], fx[i & 1][k], acc[i][j], scale.w, scale.x[i]);
        if (v < 4) {  // the next tile of x
          if (i < 3) read_x(uu, i + 1, v);
          else read_x(Next(), 0, v);
        }
        if (i == 3 && k == 1)  // w's tile j of this group has been multiplied
#pragma unroll
          for (int y = 0; y < 4; ++y) read_w(Next(), j, y);
        // behind the first barrier 12 loads in 16 MFMAs, behind the second 4 in 16
        if (i == 0 && (v & 3) == 3) load_xb(Next(), k1, there1, 2 + (v >> 2));
        if (i == 1 || i == 2) {
          const int u = 8 * (i - 1) + v, z = u * 3 / 4;
          if ((u + 1) * 3 / 4 > z) {
            if (z < 4) load_xa(uu, k2, there2, z);
            else load_w(uu, k2, there2, z - 4);
          }
        }
        if (i == 3 && (v & 3) == 3) load_xb(uu, k2, there2, v >> 2);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i == 0 || i == 2) {
        __builtin_amdgcn_s_waitcnt(kLdsDone);
        // Behind the loads that have to have landed there are 16 (12 of the group after the next,
        // four of the next one's tiles 2 and 3), and in a word's first group the scales' five.
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(16 + (U == 0 ? Scales<4, false>::kLoads : 0)));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // (whole words: groups past the last one are zeros, and an exit in the middle of the turn would cost
  // the registers that hold the sums)
  for (int s = 0; s < groups; s += 4) {
    group(I0(), s);
    group(I1(), s + 1);
    group(std::integral_constant<int, 2>(), s + 2);
    group(std::integral_constant<int, 3>(), s + 3);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (no load is left to land in LDS that another has by then)
  store_tiles(p, m0 + 128 * wm, n0 + 128 * wn, acc);
}

// --- which of them ------------------------------------------------------------------

// A kernel's block of results, and how long a group of K takes it, in us, measured with cold
// weights: with a few workgroups on the chip, with one on each of its CUs, and for each of several
// that share a CU (0: a CU has one at a time); for results in bf16 and in f32.
struct Form {
  int bm, bn, waves;
  struct {
    float few, full, each;
  } t[2];
};
constexpr Form kForms[] = {
    {16, 16, 8, {{0.08f, 0.085f, 0.07f}, {0.08f, 0.085f, 0.08f}}},
    {32, 16, 8, {{0.08f, 0.097f, 0.13f}, {0.08f, 0.097f, 0.13f}}},
    {32, 32, 4, {{0.14f, 0.156f, 0.11f}, {0.15f, 0.16f, 0.13f}}},
    {32, 32, 8, {{0.11f, 0.135f, 0.0f}, {0.12f, 0.138f, 0.0f}}},
    {32, 64, 4, {{0.178f, 0.206f, 0.0f}, {0.235f, 0.25f, 0.0f}}},
    {64, 64, 4, {{0.25f, 0.28f, 0.0f}, {0.345f, 0.385f, 0.0f}}},
    {64, 64, 4, {{0.25f, 0.275f, 0.23f}, {0.41f, 0.456f, 0.35f}}},
    {64, 128, 4, {{0.306f, 0.39f, 0.37f}, {0.565f, 0.675f, 0.59f}}},
    {128, 128, 4, {{0.4f, 0.61f, 0.0f}, {0.8f, 1.1f, 0.0f}}},
    {128, 256, 4, {{0.65f, 1.06f, 0.0f}, {1.37f, 1.97f, 0.0f}}},
    {256, 256, 4, {{1.0f, 1.65f, 0.0f}, {1e9f, 1e9f, 0.0f}}},
};
constexpr float kBytesPerUs = 5.15e6f;  // of a large copy

// The one that takes the least time a group of K: rounds of workgroups where a CU has one, their
// number and that of the fullest CU on average where it has several, and never less than the codes
// take from memory; the smaller blocks where that decides.  64 x 22016 x 4096: 25.6 us with 64 x 128
// (29 x 128 and 26.5 x 128 x 128, 31.5 of 32 x 32); 512 x 4096 x 4096: 15.0 (16.9 with 64 x 64, 21.7
// with 128 x 128); 2048 x 4096 x 4096: 36.4 with 128 x 256 (45 with 256 x 256, 47 with 128 x 128).
int choose_form(int64_t M, int64_t N, bool f32) {
  const float memory = 128.0f * (static_cast<float>(M) + static_cast<float>(N)) / kBytesPerUs;
  int best = 0;
  float least = 0.0f;
  for (int i = 0; i < static_cast<int>(sizeof(kForms) / sizeof(kForms[0])); ++i) {
    const Form& f = kForms[i];
    const auto& t = f.t[f32];
    const int64_t blocks = ((M + f.bm - 1) / f.bm) * ((N + f.bn - 1) / f.bn);
    const float n = static_cast<float>(blocks) / num_cus();
    float time;
    if (n <= 1.0f)
      time = t.few + (t.full - t.few) * n;
    else if (t.each == 0.0f)
      time = t.full * std::ceil(n);
    else
      time = std::max(t.full, t.each * 0.5f * (n + std::ceil(n)));
    time = std::max(time, memory);
    if (i == 0 || time < least) {
      best = i;
      least = time;
    }
  }
  return best;
}

}  // namespace
}  // namespace ttlh

using namespace ttlh;

extern "C" int ttlh_matmul_fp8(const void* x, int64_t x_ld, const void* x_scale, int64_t xs_ld,
                               const void* w, int64_t w_ld, const void* w_scale, int64_t ws_ld,
                               void* c, int c_dtype, int64_t c_ld, int64_t M, int64_t N, int64_t K,
                               void* stream) {
  clear_error();
  const char* fn = "ttlh_matmul_fp8";
  TTLH_REQUIRE(M >= 0 && N >= 0 && K > 0 && K % 16 == 0, TTLH_EINVAL,
               "%s: K must be a positive multiple of 16", fn);
  TTLH_REQUIRE(c_dtype == TTLH_BF16 || c_dtype == TTLH_F32, TTLH_EINVAL, "%s: C must be bf16 or f32", fn);
  TTLH_REQUIRE(M < (int64_t(1) << 28) && N < (int64_t(1) << 28) && K <= (int64_t(1) << 28),
               TTLH_EUNSUPPORTED, "%s: sizes are less than 2^28", fn);
  if (M == 0 || N == 0) return TTLH_OK;
  TTLH_REQUIRE(x && x_scale && w && w_scale && c, TTLH_EINVAL, "%s: null pointer", fn);
  TTLH_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0 &&
                   (x_ld % 16 == 0 || M == 1) && (w_ld % 16 == 0 || N == 1),
               TTLH_EINVAL, "%s: rows of codes must be 16-byte aligned", fn);
  TTLH_REQUIRE(((reinterpret_cast<uintptr_t>(x_scale) | reinterpret_cast<uintptr_t>(w_scale)) & 3) == 0,
               TTLH_EINVAL, "%s: the scales must be 4-byte aligned", fn);
  const int size = c_dtype == TTLH_BF16 ? 2 : 4;
  TTLH_REQUIRE(reinterpret_cast<uintptr_t>(c) % size == 0, TTLH_EINVAL, "%s: C is off its elements", fn);
  TTLH_REQUIRE(M == 1 || c_ld >= N, TTLH_EINVAL, "%s: rows of C lie on one another", fn);
  Fp8Args a;
  a.x = static_cast<const uint8_t*>(x);
  a.w = static_cast<const uint8_t*>(w);
  a.xs = static_cast<const uint32_t*>(x_scale);
  a.ws = static_cast<const uint32_t*>(w_scale);
  a.c = c;
  a.x_ld = x_ld;
  a.w_ld = w_ld;
  a.xs_ld = xs_ld;
  a.ws_ld = ws_ld;
  a.c_ld = c_ld;
  a.M = static_cast<int32_t>(M);
  a.N = static_cast<int32_t>(N);
  a.K = static_cast<int32_t>(K);
  a.c_f32 = c_dtype == TTLH_F32;
  a.c_vec = reinterpret_cast<uintptr_t>(c) % (4 * size) == 0 && c_ld % 4 == 0;
  a.c_vec8 = reinterpret_cast<uintptr_t>(c) % 16 == 0 && c_ld % 8 == 0;
  const int i = choose_form(M, N, a.c_f32);
  a.grid_m = static_cast<int32_t>((M + kForms[i].bm - 1) / kForms[i].bm);
  a.grid_n = static_cast<int32_t>((N + kForms[i].bn - 1) / kForms[i].bn);
  // (a launch has less than 2^32 threads)
  TTLH_REQUIRE(static_cast<int64_t>(a.grid_m) * a.grid_n < (int64_t(1) << 26) / kForms[i].waves,
               TTLH_EUNSUPPORTED, "%s: too many blocks of results", fn);
  const dim3 grid(static_cast<uint32_t>(a.grid_m) * a.grid_n);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto run = [&](auto narrow, auto wide) {
    hipLaunchKernelGGL(a.c_f32 ? wide : narrow, grid, dim3(64 * kForms[i].waves), 0, s, a);
    return check_launch("a kernel of ttlh_matmul_fp8");
  };
  switch (i) {
    case 0: return run(fp8_direct_kernel<1, 1, 8, false>, fp8_direct_kernel<1, 1, 8, true>);
    case 1: return run(fp8_direct_kernel<2, 1, 8, false>, fp8_direct_kernel<2, 1, 8, true>);
    case 2: return run(fp8_direct_kernel<2, 2, 4, false>, fp8_direct_kernel<2, 2, 4, true>);
    case 3: return run(fp8_direct_kernel<2, 2, 8, false>, fp8_direct_kernel<2, 2, 8, true>);
    case 4: return run(fp8_direct_kernel<2, 4, 4, false>, fp8_direct_kernel<2, 4, 4, true>);
    case 5: return run(fp8_direct_kernel<4, 4, 4, false>, fp8_direct_kernel<4, 4, 4, true>);
    case 6: return run(fp8_block_kernel<1, 1, false>, fp8_block_kernel<1, 1, true>);
    case 7: return run(fp8_block_kernel<1, 2, false>, fp8_block_kernel<1, 2, true>);
    case 8: return run(fp8_block_kernel<2, 2, false>, fp8_block_kernel<2, 2, true>);
    case 9: return run(fp8_block_kernel<2, 4, false>, fp8_block_kernel<2, 4, true>);
    default:  // (bf16 results alone)
      return K % kFp8Group ? run(fp8_large_kernel<true>, fp8_large_kernel<true>)
                           : run(fp8_large_kernel<false>, fp8_large_kernel<false>);
  }
}

extern "C" int ttlh_matmul_fp8_form(int64_t M, int64_t N, int c_dtype) {
  return M > 0 && N > 0 ? choose_form(M, N, c_dtype == TTLH_F32) : 0;
}
