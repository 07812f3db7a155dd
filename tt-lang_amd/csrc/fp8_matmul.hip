// Products of e4m3 codes with a scale for each 128 of K, for gfx950:
//   C[m, n] = sum over groups g of 2^(ex[m, g] + ew[n / 128, g]) sum over k in g of x[m, k] w[n, k]
// with fp32 accumulation.  x [M, K] and w [N, K] are both contiguous along K.
//
// Scales are powers of two, so a scaled MFMA applies them to its operands: a group costs no
// instruction of its own, and one accumulator runs through all of K.
//
// The fp8 MFMA aligns the products of eight neighbouring k to 2^-13 of the largest of them
// before it adds them (measured; sums of such eights are right to fp32): 2^-17 of a product's
// size on average, far below the rounding of a bf16 result.  Results in fp32 (WIDE) keep fp32's
// accuracy: codes times scale become bf16, which holds them exactly, and go through bf16 MFMAs,
// at half the rate.
//
// fp8_direct_kernel: few rows of x, HBM bound by w.  Operands go from memory straight into the
// MFMA registers; a workgroup has a block of outputs and its waves divide K in words of 512,
// each with all loads of a word in flight; their sums meet in LDS and are added in wave order.
//
// fp8_block_kernel: many rows, MFMA bound.  Stages of 64 codes of K reach LDS by direct-to-LDS
// loads, two to three stages ahead in a ring of four buffers, one barrier a stage; a wave has
// 128 x 128 (T = 4) or 64 x 64 results, and its fragments of a stage are read while the stage
// before it is multiplied.  8192 x 22016 x 4096: 703 us, 2.1 PFLOP/s (64 x 64: 950 us).

#include <algorithm>
#include <type_traits>

#include "ttlh_common.h"
#include "ttlh_fp8.h"

namespace ttlh {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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

// eight codes (dwords a, b) times 2^(s - 127) as bf16; NaN where s is
__device__ __forceinline__ bf16x8 widened(uint32_t a, uint32_t b, uint32_t s) {
  const float scale = __uint_as_float(s << 23);
  const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false);
  const bf16x2 q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true);
  const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false);
  const bf16x2 t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true);
  bf16x8 v = {p[0], p[1], q[0], q[1], r[0], r[1], t[0], t[1]};
  if (s == kScaleNan) v = __builtin_bit_cast(bf16x8, u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u});
  return v;
}

// acc += A . B over one group; sa, sb: dwords of scales, the group's in byte J
template <bool WIDE, int J>
__device__ __forceinline__ f32x4 mma16(const Frag& a, const Frag& b, f32x4 acc, uint32_t sa, uint32_t sb) {
  if constexpr (!WIDE) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(all8(a), all8(b), acc, 0, 0, J, static_cast<int>(sa), J,
                                                            static_cast<int>(sb));
  } else {
    const uint32_t ea = sa >> (8 * J) & 255, eb = sb >> (8 * J) & 255;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 u = h ? a.hi : a.lo, v = h ? b.hi : b.lo;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(u[2 * i], u[2 * i + 1], ea),
                                                      widened(v[2 * i], v[2 * i + 1], eb), acc, 0, 0, 0);
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

// eight neighbouring results of a row in bf16 (p.c_vec; c_vec8: as one store)
__device__ __forceinline__ void store8(const Fp8Args& p, int row, int col, u32x4 v) {
  if (row >= p.M || col >= p.N) return;
  uint16_t* c = static_cast<uint16_t*>(p.c) + row * p.c_ld + col;
  const int n = p.N - col;
  if (p.c_vec8 && n >= 8) {
    *reinterpret_cast<u32x4*>(c) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) c[i] = static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1)));
  }
}

// MT x 16 rows of x, NT x 16 of w a workgroup.
template <int MT, int NT, int WAVES, bool WIDE>
__global__ __launch_bounds__(WAVES * 64) void fp8_direct_kernel(const Fp8Args p) {
  int bm, bn;
  block_of(p, bm, bn);
  // (uniform, and known to be: an MFMA behind a branch that the compiler takes for divergent
  // runs whether or not its lanes are masked)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int m0 = bm * MT * 16, n0 = bn * NT * 16;
  const uint8_t *xp[MT], *wp[NT];
  const uint32_t *xs[MT], *ws[NT];
  // rows past the last one are read as the last one: they reach results that are not stored
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = min(m0 + 16 * i + r, p.M - 1);
    xp[i] = p.x + row * p.x_ld + 16 * q;
    xs[i] = p.xs + row;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int row = min(n0 + 16 * j + r, p.N - 1);
    wp[j] = p.w + row * p.w_ld + 16 * q;
    ws[j] = p.ws + row / kFp8Group;
  }
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // chunk (of 16 codes) k .. of a lane, zeros past K
  const auto chunk = [&](const uint8_t* base, int k) {
    return k + 16 * q < p.K ? *reinterpret_cast<const u32x4*>(base + k) : u32x4{0u, 0u, 0u, 0u};
  };
  const int words = (p.K + kFp8Word - 1) / kFp8Word;
  for (int word = wave; word < words; word += WAVES) {
    const int k0 = word * kFp8Word;
    uint32_t sx[MT], sw[NT];
    Frag a[NT][4], b[MT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) sw[j] = ws[j][word * p.ws_ld];
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i] = xs[i][word * p.xs_ld];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
        a[j][g] = Frag{chunk(wp[j], k0 + 128 * g), chunk(wp[j], k0 + 128 * g + 64)};
#pragma unroll
      for (int i = 0; i < MT; ++i)
        b[i][g] = Frag{chunk(xp[i], k0 + 128 * g), chunk(xp[i], k0 + 128 * g + 64)};
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        acc[i][j] = mma16<WIDE, 0>(a[j][0], b[i][0], acc[i][j], sw[j], sx[i]);
        // (a group past K has codes of zero, but its scale need not be a number)
        if (k0 + 128 < p.K) acc[i][j] = mma16<WIDE, 1>(a[j][1], b[i][1], acc[i][j], sw[j], sx[i]);
        if (k0 + 256 < p.K) acc[i][j] = mma16<WIDE, 2>(a[j][2], b[i][2], acc[i][j], sw[j], sx[i]);
        if (k0 + 384 < p.K) acc[i][j] = mma16<WIDE, 3>(a[j][3], b[i][3], acc[i][j], sw[j], sx[i]);
      }
  }
  // a lane has four neighbouring results of row r: columns 16 j + 4 q ..
  __shared__ f32x4 part[WAVES][MT * NT][64];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  for (int t = wave; t < MT * NT; t += WAVES) {
    f32x4 s = part[0][t][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) s += part[v][t][lane];
    store4(p, m0 + 16 * (t / NT) + r, n0 + 16 * (t % NT) + 4 * q, s);
  }
}

// --- many rows: through LDS ---------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kBlockThreads = 256;
constexpr int kStage = 64;  // codes of K a stage

// s_waitcnt: at most n vector loads outstanding; all LDS reads done
constexpr int vmcnt_imm(int n) { return 0x0F70 | (n & 0xF) | ((n >> 4) << 14); }
constexpr int kLdsDone = 0xC07F;

// One k = 64 step of a 32 x 32 tile; e: the scales' byte
template <bool WIDE, int E>
__device__ __forceinline__ f32x16 mma32(const Frag& a, const Frag& b, f32x16 acc, uint32_t sa, uint32_t sb) {
  if constexpr (!WIDE) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(all8(a), all8(b), acc, 0, 0, E, static_cast<int>(sa), E,
                                                           static_cast<int>(sb));
  } else {
    const uint32_t ea = sa >> (8 * E) & 255, eb = sb >> (8 * E) & 255;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 u = h ? a.hi : a.lo, v = h ? b.hi : b.lo;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widened(u[2 * i], u[2 * i + 1], ea),
                                                      widened(v[2 * i], v[2 * i + 1], eb), acc, 0, 0, 0);
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

// A wave has T x T tiles of 32 x 32, four waves a block of 64 T x 64 T.
template <int T, bool WIDE>
__device__ __forceinline__ void fp8_block(const Fp8Args& p) {
  constexpr int kRows = 64 * T;           // of x, and of w, a block
  constexpr int kLoads = kRows / 64;      // of 16 bytes a thread for one operand's stage
  __shared__ __attribute__((aligned(16))) uint8_t x0[kRows * kStage], x1[kRows * kStage],
      x2[kRows * kStage], x3[kRows * kStage], w0[kRows * kStage], w1[kRows * kStage],
      w2[kRows * kStage], w3[kRows * kStage];
  const auto xbuf = [&](auto q) -> uint8_t* {
    constexpr int Q = decltype(q)::value & 3;
    return Q == 0 ? x0 : Q == 1 ? x1 : Q == 2 ? x2 : x3;
  };
  const auto wbuf = [&](auto q) -> uint8_t* {
    constexpr int Q = decltype(q)::value & 3;
    return Q == 0 ? w0 : Q == 1 ? w1 : Q == 2 ? w2 : w3;
  };
  int bm, bn;
  banded_block(p, 4, bm, bn);
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = (wave & 1) * 32 * T, wn = (wave >> 1) * 32 * T;
  const int m0 = bm * kRows, n0 = bn * kRows;

  // a thread's loads of a stage: rows i 64 + t / 4; chunk c of row r lies at c ^ (r / 4 & 3)
  const int chunk = 16 * ((t & 3) ^ (t >> 4 & 3));
  const uint8_t *xsrc[kLoads], *wsrc[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    // (rows past the last one are read as the last one: they reach results that are not stored)
    xsrc[i] = p.x + static_cast<int64_t>(min(m0 + 64 * i + (t >> 2), p.M - 1)) * p.x_ld + chunk;
    wsrc[i] = p.w + static_cast<int64_t>(min(n0 + 64 * i + (t >> 2), p.N - 1)) * p.w_ld + chunk;
  }
  const int base = wave * 1024;  // where a wave's lanes land, 16 bytes each
  const auto load_piece = [&](auto q, int k0, int i) {
    if (i < kLoads)
      __builtin_amdgcn_global_load_lds(xsrc[i] + k0, (lds_void*)(xbuf(q) + i * 4096 + base), 16, 0, 0);
    else
      __builtin_amdgcn_global_load_lds(wsrc[i - kLoads] + k0,
                                       (lds_void*)(wbuf(q) + (i - kLoads) * 4096 + base), 16, 0, 0);
  };
  const int nk = (p.K + kStage - 1) / kStage, full = p.K / kStage;
  // any stage; chunks past K are read as the last one, and not used
  const auto load_stage = [&](auto q, int s) {
    const int k0 = min(s * kStage, p.K - 16 - chunk);
#pragma unroll
    for (int i = 0; i < 2 * kLoads; ++i) load_piece(q, k0, i);
  };

  // fragments: row lane % 32 of a tile, chunks 2 h and 2 h + 1 with h = lane / 32
  const int l32 = lane & 31, h = lane >> 5, xr = l32 >> 2 & 3;
  const int at_lo = l32 * kStage + ((2 * h) ^ xr) * 16, at_hi = l32 * kStage + ((2 * h + 1) ^ xr) * 16;
  struct Frags {
    Frag w[T], x[T];
  };
  Frags f0, f1;
  // piece y of the 4 T that read a stage's fragments
  const auto read_piece = [&](auto q, Frags& f, int y) {
    const uint8_t* b = y < 2 * T ? wbuf(q) + wn * kStage : xbuf(q) + wm * kStage;
    const int i = (y < 2 * T ? y : y - 2 * T) >> 1;
    const u32x4 v = *reinterpret_cast<const u32x4*>(b + i * 32 * kStage + (y & 1 ? at_hi : at_lo));
    Frag& g = y < 2 * T ? f.w[i] : f.x[i];
    if (y & 1) g.hi = v;
    else g.lo = v;
  };
  const auto read_stage = [&](auto q, Frags& f, int s) {
#pragma unroll
    for (int y = 0; y < 4 * T; ++y) read_piece(q, f, y);
    const int left = p.K - s * kStage;
    if (left < kStage) {  // zeros past K
      const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < T; ++i) {
        if (32 * h >= left) f.w[i].lo = f.x[i].lo = zero;
        if (32 * h + 16 >= left) f.w[i].hi = f.x[i].hi = zero;
      }
    }
  };

  f32x16 acc[T][T];  // [w tile][x tile]
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  // scales of four stages (two groups: half a word of four)
  const int words = (p.K + kFp8Word - 1) / kFp8Word;
  const uint32_t* ws = p.ws + min(n0 + wn, p.N - 1) / kFp8Group;  // (a wave's rows of w are in one block)
  const uint32_t* xs[T];
#pragma unroll
  for (int j = 0; j < T; ++j) xs[j] = p.xs + min(m0 + wm + 32 * j + l32, p.M - 1);
  uint32_t sw, sx[T], next_w, next_x[T];
  const auto load_scales = [&](int four) {  // stages 4 four ..
    const int word = min(four >> 1, words - 1);
    next_w = ws[word * p.ws_ld];
#pragma unroll
    for (int j = 0; j < T; ++j) next_x[j] = xs[j][word * p.xs_ld];
  };
  const auto take_scales = [&](int four) {
    const int by = 16 * (four & 1);
    sw = next_w >> by;
#pragma unroll
    for (int j = 0; j < T; ++j) sx[j] = next_x[j] >> by;
  };

  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  load_scales(0);
  load_stage(I0(), 0);
  if (1 < nk) load_stage(I1(), 1);
  if (2 < nk) load_stage(I2(), 2);
  if (3 < nk) load_stage(I3(), 3);
  constexpr int kStageLoads = 2 * kLoads;
  const auto wait_behind = [&](int stages) {  // at most so many stages' loads are outstanding
    if (stages >= 3) __builtin_amdgcn_s_waitcnt(vmcnt_imm(3 * kStageLoads));
    else if (stages == 2) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * kStageLoads));
    else if (stages == 1) __builtin_amdgcn_s_waitcnt(vmcnt_imm(kStageLoads));
    else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  };
  wait_behind(min(nk - 1, 3));
  __builtin_amdgcn_s_barrier();
  read_stage(I0(), f0, 0);

  // Stage s, in buffers Q = s % 4, whose fragments are in cur.  Behind the barrier every wave has
  // read its fragments of stage s, so the buffers take stage s + 4, and stage s + 1 has landed.
  // STEADY: stages up to s + 4 exist and are whole.
  const auto stage = [&](auto qq, auto steady, Frags& cur, Frags& nxt, int s) {
    constexpr int Q = decltype(qq)::value, E = Q >> 1;
    constexpr bool STEADY = decltype(steady)::value;
    using Next = std::integral_constant<int, (Q + 1) & 3>;
    __builtin_amdgcn_s_waitcnt(kLdsDone);
    if constexpr (STEADY) {
      // (the scales' loads lie behind those of stage s + 1 in the second and third of four)
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * kStageLoads + (Q == 1 || Q == 2 ? T + 1 : 0)));
      __builtin_amdgcn_s_barrier();
      constexpr int kMma = T * T, kReads = 4 * T;
      int y = 0;
#pragma unroll
      for (int v = 0; v < kMma; ++v) {
        const int i = v / T, j = v % T;
        acc[i][j] = mma32<WIDE, E>(cur.w[i], cur.x[j], acc[i][j], sw, sx[j]);
        // the reads in the first three quarters, so that they are done at the barrier
        const int upto = min(kReads, (v + 1) * kReads * 4 / (3 * kMma));
#pragma unroll
        for (int z = 0; z < kReads; ++z)
          if (z >= y && z < upto) read_piece(Next(), nxt, z);
        y = upto;
        // 2 T loads over T T steps
        const int l0 = v * kStageLoads / kMma, l1 = (v + 1) * kStageLoads / kMma;
#pragma unroll
        for (int z = 0; z < kStageLoads; ++z)
          if (z >= l0 && z < l1) load_piece(qq, (s + 4) * kStage, z);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      if (s + 1 < nk) wait_behind(min(nk - 2 - s, 2));
      __builtin_amdgcn_s_barrier();
      if (s + 1 < nk) read_stage(Next(), nxt, s + 1);
      if (s + 4 < nk) load_stage(qq, s + 4);
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < T; ++j) acc[i][j] = mma32<WIDE, E>(cur.w[i], cur.x[j], acc[i][j], sw, sx[j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int s = 0;
  for (; s + 8 <= full; s += 4) {
    take_scales(s >> 2);
    load_scales((s >> 2) + 1);
    __builtin_amdgcn_sched_barrier(0);
    stage(I0(), std::true_type(), f0, f1, s);
    stage(I1(), std::true_type(), f1, f0, s + 1);
    stage(I2(), std::true_type(), f0, f1, s + 2);
    stage(I3(), std::true_type(), f1, f0, s + 3);
  }
  for (; s < nk; s += 4) {
    take_scales(s >> 2);
    load_scales((s >> 2) + 1);
    stage(I0(), std::false_type(), f0, f1, s);
    if (s + 1 < nk) stage(I1(), std::false_type(), f1, f0, s + 1);
    if (s + 2 < nk) stage(I2(), std::false_type(), f0, f1, s + 2);
    if (s + 3 < nk) stage(I3(), std::false_type(), f1, f0, s + 3);
  }

  // A lane has row lane % 32 of x's tiles and, of w's, columns 8 r + 4 h .. + 3 (r < 4).  bf16:
  // the halves of two r change places, so that a lane has eight neighbours.
#pragma unroll
  for (int j = 0; j < T; ++j) {
    const int row = m0 + wm + 32 * j + l32;
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int col = n0 + wn + 32 * i;
      if (p.c_f32 || !p.c_vec) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          store4(p, row, col + 8 * r + 4 * h,
                 f32x4{acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]});
      } else {
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          uint32_t a0 = cvt_pk_bf16x2(acc[i][j][4 * r], acc[i][j][4 * r + 1]);
          uint32_t a1 = cvt_pk_bf16x2(acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]);
          uint32_t b0 = cvt_pk_bf16x2(acc[i][j][4 * r + 4], acc[i][j][4 * r + 5]);
          uint32_t b1 = cvt_pk_bf16x2(acc[i][j][4 * r + 6], acc[i][j][4 * r + 7]);
          const auto e = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
          const auto o = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
          store8(p, row, col + 8 * (r + h), u32x4{e[0], o[0], e[1], o[1]});
        }
      }
    }
  }
}

template <int T, bool WIDE>
__global__ __launch_bounds__(kBlockThreads, T == 4 ? 1 : 2) void fp8_block_kernel(const Fp8Args p) {
  fp8_block<T, WIDE>(p);
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto run = [&](auto kernel, int bm, int bn, int waves) {
    a.grid_m = static_cast<int32_t>((M + bm - 1) / bm);
    a.grid_n = static_cast<int32_t>((N + bn - 1) / bn);
    if (static_cast<int64_t>(a.grid_m) * a.grid_n >= (int64_t(1) << 31)) {
      set_error("%s: too many blocks of results", fn);
      return static_cast<int>(TTLH_EUNSUPPORTED);
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.grid_m) * a.grid_n), dim3(waves * 64), 0, s, a);
    return check_launch("fp8_direct_kernel");
  };
  if (M > 64) {
    if (a.c_f32) return run(fp8_block_kernel<2, true>, 128, 128, 4);
    if (M * N >= 192 * 65536) return run(fp8_block_kernel<4, false>, 256, 256, 4);
    return run(fp8_block_kernel<2, false>, 128, 128, 4);
  }
  if (a.c_f32) return M <= 16 ? run(fp8_direct_kernel<1, 1, 8, true>, 16, 16, 8) : run(fp8_direct_kernel<2, 2, 8, true>, 32, 32, 8);
  return M <= 16 ? run(fp8_direct_kernel<1, 1, 8, false>, 16, 16, 8) : run(fp8_direct_kernel<2, 2, 8, false>, 32, 32, 8);
}
