// Attention of new tokens over an 8-bit key/value cache (see ttlhip.h) for gfx950:
//   o = softmax(cap(scale q K^T)) V,  fp32 scores, statistics and sums.
//
// The q heads that share a cache head, for all new tokens of a sequence, are the
// rows of one problem: row r is token r / group, head r % group of the group.  The
// rows go in tiles, and K and V are read once for a tile.  Codes are whole numbers
// (or e4m3 values) that bf16 holds exactly, so the products run on the codes and the
// scales multiply what comes out: K's the scores, V's the probabilities before
// their rounding to bf16 for the second product.  Both kernels compute the
// transposes S^T = K Q^T and O^T += V^T P^T: a row's scores, its maximum and its part
// of O then lie in the same lanes, and P^T needs no exchange between the products
// (the order of the positions inside a product is free).
//
//  * cached_rows_kernel: up to 16 MT rows in a tile (answers token by token, drafts):
//    HBM bound.  Four waves take turns at 32 positions and meet in LDS at the end;
//    codes go from memory to registers, no LDS on the way.  One new token each, 8 x 128
//    heads, joined: 16 sequences of up to 65537 positions 239 us (5.7 TB/s), 32 of up
//    to 8192 72 us (4.8 TB/s), one of 501 9.4 us (the latency of its dependent reads).
//  * cached_tiles_kernel: tiles of 128 or 256 rows (prompts): bound by the vector ALU,
//    which works for the softmax and the decoding between MFMAs.  Blocks of 64 positions
//    are decoded once into LDS for four or eight waves of 32 rows.  2048 new tokens at
//    18000, 32 / 8 heads of 128: 570 us, 1.0 PFLOP/s; four prompts of up to 2049 tokens, 32 / 8
//    heads of 64 and capped scores (two more transcendentals for each): 101 us.
//
// Few tiles with many positions are divided into parts (see Plan), whose results
// meet in cached_join_kernel in the order of the parts.
//
// A page whose K or V scale is negative or not finite makes NaN of what sees it.  A NaN
// in V's scale is carried by the scores instead (Subtiles::finish): a row that does
// not see the page has a probability of 0 there, and 0 NaN would be NaN.

#include <cmath>
#include <type_traits>

#include "ttlh_common.h"
#include "ttlh_kvcache.h"
#include "ttlh_kvdev.h"

namespace ttlh {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr float kLog2e = 1.4426950408889634f;

struct CachedArgs {
  CacheArgs c;
  const uint16_t* q;
  uint16_t* o;
  int64_t q_token, q_head, o_token, o_head;
  int32_t group;
  int32_t window;     // 0: none
  int32_t target;     // parts of all sequences together, for one head, about; 0: undivided
  int32_t least;      // positions of a part, at least
  int32_t turns;      // 1: the workgroups with tiles are few enough to run at once
  float scale_log2;   // |scale| log2 e, or 2 |scale| log2 e / softcap
  uint32_t flip;      // sign bits of two bf16, if the scale is negative: Q's change
  float cap_log2;     // softcap log2 e, or 0
  float* part_o;      // [slot, head, rows of a tile, dim]
  float* part_ml;     // [slot, head, rows of a tile, 2]: maximum and sum
  int32_t* chunk;     // Division::chunk, for the join
};

// ---- which part of which tile of which sequence a workgroup has --------------
//
// Lengths are on the device, so the division is made there, by every workgroup for
// itself, from one pass over the sequences: with W the positions of all tiles
// together, a part has the fewest positions (at least `least`) with which there are no
// more than `target` parts, as many as the chip has places (for more than 64 sequences,
// or more tiles than that, W / (target - tiles / 2)), so the parts are alike whatever
// the lengths are.  There are at most (tiles + target) parts, and at most 2 target
// of them belong to tiles of several parts, which have `slots` for their results.
struct Plan {
  int b, first, n, len;      // the sequence, its new tokens and positions
  int row0, rows;            // the tile's first row, the sequence's rows
  int part, parts, slot;     // this part; the slot of the tile's part 0
};

template <int BM>
struct Division {
  const CachedArgs& p;
  int chunk;
  // Of sequence threadIdx.x % 64, where there are no more than 64: its new tokens and
  // positions, its tiles, the positions that its rows see between them.
  int first, n, len, tiles, range;

  __device__ __forceinline__ void extent(int b) {
    first = n = len = tiles = range = 0;
    if (b >= p.c.seqs) return;
    seq_tokens(p.c, b, first, n);
    len = p.c.lengths[b];
    if (n == 0) return;
    int lo, hi, x;
    tiles = (n * p.group + BM - 1) / BM;
    seen_by(p.c, len, n, 0, p.window, lo, x);
    seen_by(p.c, len, n, n - 1, p.window, x, hi);
    range = hi > lo ? hi - lo : 0;
  }
  __device__ __forceinline__ void divide() {
    const int lane = threadIdx.x & 63;
    extent(lane);
    chunk = 0x7fffffff;
    if (p.target == 0) return;
    // (in fp32: off by less than one part in 2 target, and the same in every wave)
    float sum = static_cast<float>(tiles) * range, all = tiles;
    for (int b = lane + 64; b < p.c.seqs; b += 64) {
      extent(b);
      sum += static_cast<float>(tiles) * range;
      all += tiles;
    }
    // (for up to 64 sequences: the parts of `least` positions)
    const float least = p.least;
    const float few = wave_total(tiles * fmaxf(ceilf(range * __builtin_amdgcn_rcpf(least)), 1.0f));
    all = wave_total(all);
    sum = wave_total(sum);
    float each;
    if (p.c.seqs > 64 || all > p.target) {
      // (a tile's last part is half a part too many on average: so many places are left)
      each = sum / fmaxf(p.target - 0.5f * all, 0.5f * p.target);
    } else {
      each = few <= p.target ? least : fill(sum, all, p.target);
      // Tiles of 128 rows have two workgroups on a CU, which take 1.7 times as long
      // then: where twice the parts are not that much shorter, one each.
      if (BM == 128 && 2 * all <= p.target && 2 * few > p.target) {
        const float alone = fill(sum, all, 0.5f * p.target);
        if (alone < 1.7f * each) each = alone;
      }
    }
    // (up: of a length below `each`, such as a multiple of 64 that it is a fraction above,
    // one sequence can have more parts than there are workgroups)
    chunk = max((static_cast<int>(ceilf(fminf(each, 1073741824.0f))) + 63) & ~63, p.least);
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.chunk = chunk;
    if (p.c.seqs > 64) tiles = range = 0;
  }
  // The positions of a part: with W = sum positions in `all` tiles, W / (target - all x)
  // for the first x of these with which there are no more than `target` parts (1 has
  // no more: a tile's last part is less than one part too many).  (The totals are
  // independent, so that their latencies overlap: searched one after the other, the
  // start of each workgroup took 0.5 us longer.)
  __device__ __forceinline__ float fill(float sum, float all, float target) const {
    const float w = __builtin_amdgcn_rcpf(fmaxf(sum, 1.0f));
    float inv[3], parts[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      inv[i] = (target - 0.25f * (i + 1) * all) * w;
      parts[i] = tiles * fmaxf(ceilf(range * inv[i] - 0x1p-10f), 1.0f);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) parts[i] = wave_total(parts[i]);
    float best = (target - all) * w;
#pragma unroll
    for (int i = 2; i >= 0; --i)
      if (parts[i] <= target) best = inv[i];
    return __builtin_amdgcn_rcpf(fmaxf(best, 0x1p-30f));
  }
  // the same division again (JOIN)
  __device__ __forceinline__ void divided(int chunk_) {
    extent(threadIdx.x & 63);
    chunk = chunk_;
    if (p.c.seqs > 64) tiles = range = 0;
  }
  // Tile `item` of all, those that see the most positions first (by 64 of them): with
  // prompts of several lengths the last workgroups to start are then the shortest.
  // For up to 64 sequences, none divided, without a window.
  __device__ __forceinline__ bool find_longest(int item, Plan& w) {
    // tiles whose last row sees at least 64 level positions
    const auto count = [&](int level) {
      if (level == 0) return tiles;
      const int64_t y = int64_t(level) * 64 - 1 - (int64_t(len) - n);  // needs token y or a later one
      if (level * 64 > capacity(p.c) || y >= n) return 0;
      return y <= 0 ? tiles : tiles - static_cast<int>(y * p.group / BM);
    };
    const auto total = [&](int x) { return __builtin_amdgcn_readlane(prefix_sum(x), 63); };
    int lo = 0, hi = (capacity(p.c) >> 6) + 1;  // total(count(lo)) > item >= total(count(hi))
    if (total(tiles) <= item) return false;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (total(count(mid)) > item)
        lo = mid;
      else
        hi = mid;
    }
    const int with = count(lo), more = count(hi), mine = with - more;
    const int left = item - total(more), end = prefix_sum(mine);
    const int l = __builtin_amdgcn_readfirstlane(__ffsll(__ballot(end > left)) - 1) & 63;
    const auto at = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
    w.b = l;
    w.first = at(first);
    w.n = at(n);
    w.len = at(len);
    w.row0 = (at(tiles) - at(with) + left - (at(end) - at(mine))) * BM;
    w.rows = w.n * p.group;
    w.part = w.slot = 0;
    w.parts = 1;
    return w.row0 >= 0 && w.row0 < w.rows;
  }
  // item `item` of the parts (JOIN: of the tiles of several parts), or false past the
  // last one
  template <bool JOIN>
  __device__ __forceinline__ bool find(int item, Plan& w) {
    const int lane = threadIdx.x & 63;
    int items = 0, slots = 0;
    for (int b0 = 0; b0 < p.c.seqs; b0 += 64) {
      if (p.c.seqs > 64) extent(b0 + lane);
      const int parts = range > chunk ? (range - 1) / chunk + 1 : 1;
      const int mine_slots = parts > 1 ? tiles * parts : 0;
      const int mine = !JOIN ? tiles * parts : parts > 1 ? tiles : 0;
      const int end = prefix_sum(mine), send = prefix_sum(mine_slots);
      const unsigned long long past = __ballot(items + end > item);
      if (past) {
        const int l = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
        const auto at = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
        const int local = item - items - (at(end) - at(mine)), nt = at(tiles);
        w.b = b0 + l;
        w.parts = at(parts);
        // (the last tile of a prompt sees the most: it goes first)
        const int before = JOIN ? local : local / w.parts, tile = nt - 1 - before;
        w.part = JOIN ? 0 : local - before * w.parts;
        w.slot = slots + at(send) - at(mine_slots) + before * w.parts;
        w.first = at(first);
        w.n = at(n);
        w.len = at(len);
        w.row0 = tile * BM;
        w.rows = w.n * p.group;
        // (always, unless starts overlap)
        return (w.parts == 1 || (w.slot >= 0 && w.slot + w.parts <= 2 * p.target)) &&
               w.row0 >= 0 && w.row0 < w.rows;
      }
      items += __builtin_amdgcn_readlane(end, 63);
      slots += __builtin_amdgcn_readlane(send, 63);
    }
    return false;
  }
};

// The positions of a part of a tile: those its rows see, [lo, hi) in all parts, of
// which this part has [begin, end), begin a multiple of ALIGN; and the positions
// [all_lo, all_hi) that every row sees.
struct Span {
  int lo, hi, all_lo, all_hi, begin, end;
};
template <int BM, int ALIGN>
__device__ __forceinline__ Span span_of(const CachedArgs& p, const Plan& w) {
  Span s;
  const int i0 = w.row0 / p.group, i1 = (min(w.row0 + BM, w.rows) - 1) / p.group;
  seen_by(p.c, w.len, w.n, i0, p.window, s.lo, s.all_hi);
  seen_by(p.c, w.len, w.n, i1, p.window, s.all_lo, s.hi);
  if (p.c.pages == 0) s.hi = 0;
  const int from = s.lo & ~(ALIGN - 1);
  const int units = s.hi > from ? (s.hi - from + ALIGN - 1) / ALIGN : 0;
  const int per = (units + w.parts - 1) / w.parts;
  s.begin = from + min(units, w.part * per) * ALIGN;
  s.end = min(s.hi, from + min(units, (w.part + 1) * per) * ALIGN);
  return s;
}

// ---- codes to bf16 -----------------------------------------------------------

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Byte J of w as a signed number, in one instruction.  (As asm: written in C++, the
// conversions of one dword's bytes become one vector conversion, whose four results
// then live until the last of them is used, and the registers do not suffice.)
template <int J>
__device__ __forceinline__ float int8_of(uint32_t w) {
  float f;
  if constexpr (J == 0)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0"
        : "=v"(f) : "v"(w));
  else if constexpr (J == 1)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1"
        : "=v"(f) : "v"(w));
  else if constexpr (J == 2)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2"
        : "=v"(f) : "v"(w));
  else
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3"
        : "=v"(f) : "v"(w));
  return f;
}

// bytes 2 i, 2 i + 1 of w
template <int FMT, int I>
__device__ __forceinline__ uint32_t pair_of(uint32_t w) {
  if constexpr (FMT == TTLH_CACHE_E4M3)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, I == 1));
  else
    return cvt_pk_bf16x2(int8_of<2 * I>(w), int8_of<2 * I + 1>(w));
}
template <int FMT>
__device__ __forceinline__ u32x4 eight_of(uint32_t a, uint32_t b) {
  if constexpr (FMT == TTLH_CACHE_INT8) {
    // (one block: between separate ones the compiler leaves wait states that these
    // instructions, which write whole registers, do not need)
    u32x4 w;
    uint32_t t[4];
    asm("v_cvt_f32_i32_sdwa %0, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
        "v_cvt_f32_i32_sdwa %4, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1\n\t"
        "v_cvt_f32_i32_sdwa %1, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
        "v_cvt_f32_i32_sdwa %5, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3\n\t"
        "v_cvt_f32_i32_sdwa %2, sext(%9) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
        "v_cvt_f32_i32_sdwa %6, sext(%9) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1\n\t"
        "v_cvt_f32_i32_sdwa %3, sext(%9) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
        "v_cvt_f32_i32_sdwa %7, sext(%9) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3\n\t"
        "v_cvt_pk_bf16_f32 %0, %0, %4\n\t"
        "v_cvt_pk_bf16_f32 %1, %1, %5\n\t"
        "v_cvt_pk_bf16_f32 %2, %2, %6\n\t"
        "v_cvt_pk_bf16_f32 %3, %3, %7\n\t"
        "s_nop 0"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]),
          "=&v"(t[3])
        : "v"(a), "v"(b));
    return w;
  }
  return u32x4{pair_of<FMT, 0>(a), pair_of<FMT, 1>(a), pair_of<FMT, 0>(b), pair_of<FMT, 1>(b)};
}
// byte J of a and of b
template <int FMT, int J>
__device__ __forceinline__ uint32_t pair_across(uint32_t a, uint32_t b) {
  if constexpr (FMT == TTLH_CACHE_E4M3) {
    // one permutation serves two neighbouring J
    constexpr uint32_t sel = J < 2 ? 0x05010400u : 0x07030602u;
    return pair_of<FMT, (J & 1)>(__builtin_amdgcn_perm(b, a, sel));
  } else {
    return cvt_pk_bf16x2(int8_of<J>(a), int8_of<J>(b));
  }
}

__device__ __forceinline__ float uniform(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

__device__ __forceinline__ bf16x8 query(const CachedArgs& p, const uint16_t* at) {
  u32x4 v = *reinterpret_cast<const u32x4*>(at);
  v ^= p.flip;
  return __builtin_bit_cast(bf16x8, v);
}

// What a wave knows about 64 subtiles of 16 positions, one in a lane: the page (or
// -1), where the codes are, counted in subtiles (page 0's where there is no page), the
// scores' factor and V's scale.
struct Subtiles {
  int page;
  uint32_t unit;
  float kscale, vscale;

  // In three steps, so that a wave with other work need not wait for a load: the
  // table's entry, the scales of its page, the factors.
  __device__ __forceinline__ void ask_page(const CachedArgs& p, int b, int pos) {
    page = pos >= 0 && pos < capacity(p.c) ? p.c.table[b * p.c.table_ld + (pos >> p.c.shift)] : -1;
  }
  __device__ __forceinline__ void ask_scales(const CachedArgs& p, int h, int pos) {
    if (page < 0 || page >= p.c.pages) page = -1;
    const int64_t at = static_cast<int64_t>(max(page, 0)) * p.c.heads + h;
    unit = static_cast<uint32_t>(at << (p.c.shift - 4)) + ((pos & ((1 << p.c.shift) - 1)) >> 4);
    kscale = p.c.k_scale[at];
    vscale = p.c.v_scale[at];
  }
  __device__ __forceinline__ void finish(float scale) {
    const bool fine = kscale >= 0.0f && kscale < INFINITY && vscale >= 0.0f && vscale < INFINITY;
    kscale = fine ? kscale * scale : __int_as_float(0x7fc00000);
    // (page 0's scale says nothing where there is no page: restage_v() would put page
    // 0's codes, which may be NaN, where clear_unseen() put zeros)
    vscale = fine && page >= 0 ? fmaxf(vscale, 0x1p-126f) : 1.0f;
  }
};

// C tanh(t) = C - 2 C / (1 + e^2t), from x = 2 t log2 e: off by 2^-22 C, whatever t is.
// Up to C = 128 that is 2^-15 of a score, 1/64 of what the rounding of p to bf16 is.
constexpr float kNearCap = 128.0f;
__device__ __forceinline__ float capped(float x, float cap) {
  return __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x)), cap);
}
// The same for larger C, off by 2^-21 of itself: up to |t| = 1/2 as t times a polynomial
// in t^2 (tanh(t) / t at Chebyshev's nodes, right to 2^-26), above as above.
__device__ __forceinline__ float capped_far(float x, float cap) {
  const float w = x * x;  // 4 log2(e)^2 t^2
  float q = __builtin_fmaf(w, 3.564945473e-6f, -9.181317000e-5f);
  q = __builtin_fmaf(w, q, 1.922384137e-3f);
  q = __builtin_fmaf(w, q, -4.003743082e-2f);
  q = __builtin_fmaf(w, q, 1.0f);
  const float y = x * (cap * 0.34657359028f) * q;  // (ln 2 / 2)
  return w < 2.0813689810f ? y : capped(x, cap);
}

__device__ __forceinline__ float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_add(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_add(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- few rows ----------------------------------------------------------------
//
// A wave's step: 32 positions (two subtiles of 16, each on one page) against 16 MT
// rows.  Lane (n = lane % 16, g = lane / 16).  S^T: 16x16x32 MFMAs, lane (n, g) has
// K's row n of a subtile, 16 bytes at 16 g (and at 64 + 16 g), which are two
// operands; S^T leaves it positions 4 g + i of each subtile for row n of the tile.
// O^T: operand k = 8 g + 4 s + i is position 16 s + 4 g + i, so those scores are
// the P^T operand as they stand, and lane (n, g) reads D / 16 bytes at n D / 16 of
// its 8 positions, byte j of which is the operand of tile j: O^T's row m of tile j
// is element m D / 16 + j.
constexpr int kRowWaves = 4;
constexpr int kStep = 32;

// workgroups on a CU, by their registers
constexpr int rows_per_cu(int dim, int mt) {
  return dim == 128 ? (mt == 1 ? 3 : 2) : (mt == 1 ? 4 : mt == 2 ? 3 : 2);
}

template <int D, int FMT, int MT>
struct Rows {
  static constexpr int NK = D / 64;   // 16-byte loads of a K row
  static constexpr int NC = D / 32;   // K operands of a subtile
  static constexpr int NV = D / 64;   // dwords of a V load
  static constexpr int NT = D / 16;   // tiles of O^T

  struct Codes {
    u32x4 k[2][NK];
    uint32_t v[2][4][NV];
  };

  const CachedArgs& p;
  const Plan& w;
  const Span& s;
  int h, n, g;
  // Q^T operands: with three row tiles in LDS, an operand's 64 lanes side by side
  // (in registers, 44 of them would spill)
  static constexpr bool kQinLds = MT > 2 && D == 128;
  bf16x8 q[kQinLds ? 1 : MT][kQinLds ? 1 : NC];
  const bf16x8* q_lds;
  f32x4 o[MT][NT];
  float m[MT], l[MT];
  uint32_t k_off, v_off;  // the lane's bytes in a subtile
  Subtiles sub;

  // step k's subtile t: its first byte in the cache
  __device__ __forceinline__ int64_t subtile_at(int k, int t) const {
    return static_cast<int64_t>(static_cast<uint32_t>(
               __builtin_amdgcn_readlane(sub.unit, (2 * k + t) & 63))) * (16 * D);
  }
  __device__ __forceinline__ void load_k(Codes& x, int k) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* kp = p.c.k + subtile_at(k, t);
#pragma unroll
      for (int i = 0; i < NK; ++i) x.k[t][i] = *reinterpret_cast<const u32x4*>(kp + 64 * i + k_off);
    }
  }
  __device__ __forceinline__ void load_v(Codes& x, int k) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* vp = p.c.v + subtile_at(k, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (NV == 2) {
          const u32x2 v = *reinterpret_cast<const u32x2*>(vp + i * D + v_off);
          x.v[t][i][0] = v[0];
          x.v[t][i][1] = v[1];
        } else {
          x.v[t][i][0] = *reinterpret_cast<const uint32_t*>(vp + i * D + v_off);
        }
      }
    }
  }
  __device__ __forceinline__ int wave() const {
    return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  }

  // step k; the codes of step k + 2, if `more`, follow it into the same registers
  __device__ __forceinline__ void step(Codes& x, int k, bool more) {
    const int pos = s.begin + (k * kRowWaves + wave()) * kStep;
    float ks[2], vs[2];
    bool there[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int l = (2 * k + t) & 63;
      ks[t] = uniform(sub.kscale, l);
      vs[t] = uniform(sub.vscale, l);
      there[t] = __builtin_amdgcn_readlane(sub.page, l) >= 0;
    }
    const bool mask = !there[0] || !there[1] || pos < s.all_lo || pos + kStep > s.all_hi;
    f32x4 sc[MT][2];
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
      for (int t = 0; t < 2; ++t) sc[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      bf16x8 kf[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4 raw = x.k[t][c >> 1];
        kf[t] = __builtin_bit_cast(
            bf16x8, (c & 1) ? eight_of<FMT>(raw[2], raw[3]) : eight_of<FMT>(raw[0], raw[1]));
      }
#pragma unroll
      for (int r = 0; r < MT; ++r) {
        const bf16x8 qf = kQinLds ? q_lds[(r * NC + c) * 64] : q[kQinLds ? 0 : r][kQinLds ? 0 : c];
#pragma unroll
        for (int t = 0; t < 2; ++t)
          sc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t], qf, sc[r][t], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (more) load_k(x, k + 2);
    if (mask) {
      // codes that no row sees may be anything: 0 times them has to be 0
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = pos + 16 * t + 4 * g + i;
          const bool seen = there[t] && j >= s.lo && j < s.hi;
#pragma unroll
          for (int d = 0; d < NV; ++d) x.v[t][i][d] = seen ? x.v[t][i][d] : 0u;
        }
    }
    bf16x8 pf[MT];
#pragma unroll
    for (int r = 0; r < MT; ++r) {
      float e[8];
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) e[4 * t + i] = sc[r][t][i] * ks[t];
      if (p.cap_log2 > kNearCap * kLog2e) {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = capped_far(e[i], p.cap_log2);
      } else if (p.cap_log2 != 0.0f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = capped(e[i], p.cap_log2);
      }
      if (mask) {
        int from, end;
        seen_by(p.c, w.len, w.n, min(w.row0 + 16 * r + n, w.rows - 1) / p.group, p.window, from, end);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = pos + 16 * t + 4 * g + i;
            if (!there[t] || j < from || j >= end) e[4 * t + i] = -INFINITY;
          }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, e[i]);
      if (__any(mx > m[r])) {  // (else the maximum stands, and so do the sums)
        const float to = fmaxf(m[r], xor32_max(xor16_max(mx)));
        const float alpha = to == m[r] ? 1.0f : __builtin_amdgcn_exp2f(m[r] - to);
        m[r] = to;
        l[r] *= alpha;
#pragma unroll
        for (int j = 0; j < NT; ++j) o[r][j] *= alpha;
      }
      const float mm = m[r] == -INFINITY ? 0.0f : m[r];
      float sum = 0.0f;
      u32x4 pk;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[4 * t + i] = __builtin_amdgcn_exp2f(e[4 * t + i] - mm);
          sum += e[4 * t + i];
        }
        pk[2 * t] = cvt_pk_bf16x2(e[4 * t] * vs[t], e[4 * t + 1] * vs[t]);
        pk[2 * t + 1] = cvt_pk_bf16x2(e[4 * t + 2] * vs[t], e[4 * t + 3] * vs[t]);
      }
      l[r] += sum;
      pf[r] = __builtin_bit_cast(bf16x8, pk);
    }
    products(x, pf);
    if (more) load_v(x, k + 2);
  }

  template <int J>
  __device__ __forceinline__ bf16x8 vfrag(const Codes& x) const {
    u32x4 f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f[2 * t] = pair_across<FMT, (J & 3)>(x.v[t][0][J / 4], x.v[t][1][J / 4]);
      f[2 * t + 1] = pair_across<FMT, (J & 3)>(x.v[t][2][J / 4], x.v[t][3][J / 4]);
    }
    return __builtin_bit_cast(bf16x8, f);
  }
  template <int J = 0>
  __device__ __forceinline__ void products(const Codes& x, const bf16x8 (&pf)[MT]) {
    const bf16x8 vf = vfrag<J>(x);
#pragma unroll
    for (int r = 0; r < MT; ++r)
      o[r][J] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[r], o[r][J], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (J + 1 < NT) products<J + 1>(x, pf);
  }
};

template <int D, int FMT, int MT>
__global__ __launch_bounds__(kRowWaves * 64, rows_per_cu(D, MT)) void cached_rows_kernel(
    const CachedArgs p) {
  constexpr int BM = 16 * MT;
  constexpr int LD = D + 4;  // LDS row: 16 rows' 16-byte writes spread over the banks
  typedef Rows<D, FMT, MT> R;
  __shared__ bf16x8 q_lds[R::kQinLds ? MT * (D / 32) * 64 : 1];
  __shared__ float part[kRowWaves][16][LD];
  __shared__ float ml[kRowWaves][BM][2];

  Division<BM> div{p};
  div.divide();
  const int h = blockIdx.x % p.c.heads;
  Plan w;
  if (!div.template find<false>(blockIdx.x / p.c.heads, w)) return;
  const Span s = span_of<BM, kStep>(p, w);
  R x{p, w, s, h};
  const int lane = threadIdx.x & 63, wave = x.wave();
  x.n = lane & 15;
  x.g = lane >> 4;
  x.k_off = x.n * D + 16 * x.g;
  x.v_off = 4 * x.g * D + x.n * (D / 16);
  // steps of this wave: k * 4 + wave of the part's
  const int total = s.end > s.begin ? (s.end - s.begin + kStep - 1) / kStep : 0;
  const int steps = total > wave ? (total - wave - 1) / kRowWaves + 1 : 0;
  typename R::Codes a, b;
  int kn;
  const auto refill = [&](int k) {  // steps k .. k + 31, two subtiles each
    const int pos = s.begin + ((k + (lane >> 1)) * kRowWaves + wave) * kStep + 16 * (lane & 1);
    x.sub.ask_page(p, w.b, pos < s.hi ? pos : -1);
    x.sub.ask_scales(p, h, pos);
    kn = min(steps, k + 32);
    x.load_k(a, k);
    x.load_v(a, k);
    if (k + 1 < kn) {
      x.load_k(b, k + 1);
      x.load_v(b, k + 1);
    }
    x.sub.finish(p.scale_log2);
  };
#pragma unroll
  for (int r = 0; r < MT; ++r) {
    const int row = min(w.row0 + 16 * r + x.n, w.rows - 1);
    const int i = row / p.group;
    const uint16_t* qp = p.q + static_cast<int64_t>(w.first + i) * p.q_token +
                         static_cast<int64_t>(h * p.group + row - i * p.group) * p.q_head;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const bf16x8 qf = query(p, qp + 64 * (c >> 1) + 16 * x.g + 8 * (c & 1));
      if constexpr (R::kQinLds) {
        if (wave == (r * (D / 32) + c) % kRowWaves) q_lds[(r * (D / 32) + c) * 64 + lane] = qf;
      } else {
        x.q[r][c] = qf;
      }
    }
    x.m[r] = -INFINITY;
    x.l[r] = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) x.o[r][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  if (steps > 0) refill(0);
  if constexpr (R::kQinLds) {
    x.q_lds = q_lds + lane;
    __syncthreads();
  }
  for (int k0 = 0; k0 < steps; k0 += 32) {
    if (k0 > 0) refill(k0);
    for (int k = k0; k < kn; k += 2) {
      x.step(a, k, k + 2 < kn);
      if (k + 1 < kn) x.step(b, k + 1, k + 3 < kn);
    }
  }

  // The waves meet: first their maxima, by which each scales its sums and O; then
  // O in LDS, 16 rows at a time, a thread adding four elements of a row in the
  // order of the waves.
  const int rows = min(BM, w.rows - w.row0);
#pragma unroll
  for (int r = 0; r < MT; ++r) {
    x.l[r] = xor32_add(xor16_add(x.l[r]));
    if (x.g == 0) ml[wave][16 * r + x.n][0] = x.m[r];
  }
  __syncthreads();
  const int64_t slot = (static_cast<int64_t>(w.slot + w.part) * p.c.heads + h) * BM;
#pragma unroll
  for (int r = 0; r < MT; ++r) {
    if (16 * r >= rows) break;  // (uniform)
    if (16 * r + x.n < rows) {
      float mt = -INFINITY;
#pragma unroll
      for (int v = 0; v < kRowWaves; ++v) mt = fmaxf(mt, ml[v][16 * r + x.n][0]);
      const float f = __builtin_amdgcn_exp2f(x.m[r] - (mt == -INFINITY ? 0.0f : mt));
      if (x.g == 0) ml[wave][16 * r + x.n][1] = x.l[r] * f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < D / 16; j += 4)
          *reinterpret_cast<f32x4*>(&part[wave][x.n][(4 * x.g + i) * (D / 16) + j]) =
              f32x4{x.o[r][j][i] * f, x.o[r][j + 1][i] * f, x.o[r][j + 2][i] * f,
                    x.o[r][j + 3][i] * f};
    }
    __syncthreads();
    for (int e = threadIdx.x; e < min(16, rows - 16 * r) * (D / 4); e += kRowWaves * 64) {
      const int row = e / (D / 4), d = (e % (D / 4)) * 4;
      float lt = 0.0f;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int v = 0; v < kRowWaves; ++v) {
        lt += ml[v][16 * r + row][1];
        acc += *reinterpret_cast<const f32x4*>(&part[v][row][d]);
      }
      const int at = w.row0 + 16 * r + row;
      if (w.parts > 1) {
        *reinterpret_cast<f32x4*>(p.part_o + (slot + 16 * r + row) * D + d) = acc;
        if (d == 0) {
          float mt = -INFINITY;
#pragma unroll
          for (int v = 0; v < kRowWaves; ++v) mt = fmaxf(mt, ml[v][16 * r + row][0]);
          p.part_ml[(slot + 16 * r + row) * 2] = mt;
          p.part_ml[(slot + 16 * r + row) * 2 + 1] = lt;
        }
      } else {
        const int i = at / p.group;
        const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
        uint16_t* op = p.o + static_cast<int64_t>(w.first + i) * p.o_token +
                       static_cast<int64_t>(h * p.group + at - i * p.group) * p.o_head + d;
        *reinterpret_cast<u32x2*>(op) = u32x2{cvt_pk_bf16x2(acc[0] * inv, acc[1] * inv),
                                              cvt_pk_bf16x2(acc[2] * inv, acc[3] * inv)};
      }
    }
    if (16 * (r + 1) < rows) __syncthreads();
  }
}

// ---- many rows ---------------------------------------------------------------
//
// 32 rows a wave; blocks of 64 positions in 32x32x16 MFMAs, K and V
// decoded to bf16 in LDS: K row-major, 16-byte chunk c of row r at c ^ (r & 15) (dim
// 64: c ^ ((r >> 1) & 7)); V row-major, read with ds_read_b64_tr_b16, chunk c of row r
// at c ^ 4 (r & 3) (dim 64: c ^ 4 ((r >> 1) & 1)).  Two buffers of each.
//
// A block has 32 MFMAs and, for each, about eight other vector instructions (for 32
// rows of 64 scores three each and the decoding), so these are laid between the
// MFMAs, which run meanwhile; two waves share a SIMD.  In order, with half t the
// block's positions 32 t .. 32 t + 31:
//     S of half 0            | the next block's K codes are decoded into LDS
//     S of half 1            | softmax of half 0
//     O += V P of half 0     | softmax of half 1
//     O += V P of half 1     | the next block's V codes are decoded into LDS
// The running maximum m moves only where a lane's sum shows that it lags (or where
// there is none yet): p is at most 2^8 then, which bf16 and fp32 hold as well as 1,
// and half a block needs no maximum before its exponentials.
// (Softmax, decoding and products one after the other took 700 us for 2048 new
// tokens at 18000, 32 / 8 heads of 128.)
//
// NW waves: four, two workgroups on a CU, or (dim 128) eight, which share the decoding,
// and one (see choose()).
constexpr int kBlock = 64;
// How scores are capped: not, as capped() does, as capped_far() does.
constexpr int kUncapped = 0, kCapped = 1, kCappedFar = 2;

template <int D, int FMT, int CAP, int NW>
struct Tiles {
  static constexpr int ND = D / 32, NDC = D / 16;
  static constexpr int kChunks = D / 8;                           // of eight codes in a row
  static constexpr int kSweep = NW * 64 / kChunks;                // rows of one load of all threads
  static constexpr int kUnits = kBlock / kSweep;                  // loads of a thread, for K and for V
  static_assert(kUnits >= 1 && kUnits <= NDC / 2, "each unit is staged behind an MFMA of its own");
  static constexpr int kProducts = 2 * NDC + 4 * ND;              // MFMAs of a block
  static constexpr int kAhead = 4;                                // operands read ahead
  static constexpr float kFar = 256.0f;

  const CachedArgs& p;
  const Plan& w;
  const Span& s;
  uint16_t (*Ks)[kBlock * D];
  uint16_t (*Vs)[kBlock * D];
  int hd, wave, lane, l32, h;
  int from, end;   // what the lane's row sees
  bf16x8 qop[NDC];
  f32x16 o[ND];
  f32x16 cur[2];   // scores of the two halves
  bf16x8 f[kAhead];
  u32x4 pw[4];     // P of the block's subtiles as bf16
  float m, l, rs, part;  // rs, part: sums of p over half a block, over a subtile
  Subtiles sub;    // of the sixteen blocks of the one that computes
  Subtiles next;   // of the next sixteen, from the middle of these on
  float lv, iv;    // sub's log2 and reciprocal of V's scales
  uint64_t paged, broken; // sub's subtiles with a page; with a scale that makes NaN
  uint64_t special;       // its subtiles that some row does not see, or with such scales
  u32x2 kraw[kUnits], vraw[kUnits];
  uint32_t load_unit;  // sub.unit, or next.unit, of the block whose codes are loaded
  int k_frag, v_frag[ND], k_to, v_to;
  uint32_t unit_off;

  static __device__ __forceinline__ int k_swz(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
  static __device__ __forceinline__ int v_swz(int r) {
    return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
  }

  __device__ __forceinline__ void setup() {
    k_frag = l32 * D + ((h ^ k_swz(l32)) << 3);
    const int vr = (lane & 15) >> 2;
#pragma unroll
    for (int j = 0; j < ND; ++j) {
      const int chunk = 4 * j + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      v_frag[j] = (4 * h + vr) * D + ((chunk ^ v_swz(vr)) << 3) + 4 * (lane & 1);
    }
    // the thread's chunk: row `row` of each sweep; 16 (or 8) lanes write a whole row
    const int row = threadIdx.x / kChunks, c = threadIdx.x % kChunks;
    k_to = row * D + ((c ^ k_swz(row)) << 3);
    v_to = row * D + ((c ^ v_swz(row)) << 3);
    unit_off = (row & 15) * D + c * 8;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[j][r] = 0.0f;
  }

  // ---- codes ----
  // the subtile of the thread's unit i (the 64 / kChunks rows of a wave's load are in one)
  __device__ __forceinline__ int unit_sub(int i) const {
    return (kSweep / 16) * i + wave / (16 * kChunks / 64);
  }
  __device__ __forceinline__ void ask_page(Subtiles& x, int kb) const {  // kb a multiple of 16
    const int pos = s.begin + kb * kBlock + lane * 16;
    x.ask_page(p, w.b, pos < s.hi ? pos : -1);
  }
  __device__ __forceinline__ void ask_scales(Subtiles& x, int kb) const {
    x.ask_scales(p, hd, s.begin + kb * kBlock + lane * 16);
  }
  __device__ __forceinline__ void finish(int kb) {  // kb a multiple of 16
    broken = __ballot(!(sub.kscale < INFINITY));
    if (!(sub.kscale < INFINITY)) sub.kscale = 1.0f;  // (hide() makes the NaN)
    sub.kscale = fmaxf(sub.kscale, 0x1p-126f);        // (0 times -inf would be NaN)
    const bool far = far_scale(sub.vscale);           // (restage_v() multiplies by the rest)
    const float by_p = far ? near_part(sub.vscale) : sub.vscale;
    lv = __builtin_amdgcn_logf(by_p);
    iv = __builtin_amdgcn_rcpf(by_p);
    paged = __ballot(sub.page >= 0);
    const int pos = s.begin + (kb * 4 + lane) * 16;
    special = __ballot(sub.page < 0 || far || pos < s.all_lo || pos + 16 > s.all_hi) | broken;
  }
  // whether block kb of the sixteen has such a subtile (the first of the next sixteen
  // is not known yet: it may)
  __device__ __forceinline__ bool is_special(int kb) const { return (special >> ((kb & 15) * 4)) & 15; }
  __device__ __forceinline__ bool may_be_special(int kb) const { return (kb & 15) == 0 || is_special(kb); }
  // Of V scales so small or large that p times them leaves the exponents' range, the
  // power of two 2^-60 or 2^60 goes to p and the rest into V itself: a code times the rest
  // is at most 448 * 2^68, where a code times the scale could be infinite, which makes NaN
  // of the rows that do not see it (0 times infinity).
  static __device__ __forceinline__ bool far_scale(float v) { return v < 0x1p-60f || v > 0x1p60f; }
  static __device__ __forceinline__ float near_part(float v) { return v < 1.0f ? 0x1p-60f : 0x1p60f; }
  __device__ __forceinline__ void restage_v(int kb) const {
    const bool later = (kb & 15) == 0 && kb > 0;
    const float scale = later ? next.vscale : sub.vscale;
    const uint32_t unit = later ? next.unit : sub.unit;
    const int at = (kb & 15) * 4;
    if (((__ballot(far_scale(scale)) >> at) & 15) == 0) return;
    for (int i = 0; i < kUnits; ++i) {
      float f = uniform(scale, at + unit_sub(i));
      const int j = s.begin + kb * kBlock + i * kSweep + static_cast<int>(threadIdx.x) / kChunks;
      if (!far_scale(f) || j < s.lo || j >= s.hi) continue;
      f *= f < 1.0f ? 0x1p60f : 0x1p-60f;
      const uint32_t u = __builtin_amdgcn_readlane(unit, at + unit_sub(i));
      const u32x2 raw = *reinterpret_cast<const u32x2*>(p.c.v + static_cast<uint64_t>(u) * (16 * D) +
                                                        unit_off);
      u32x4 v = eight_of<FMT>(raw[0], raw[1]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = cvt_pk_bf16x2(__uint_as_float(v[j] << 16) * f, __uint_as_float(v[j] & 0xffff0000u) * f);
      *reinterpret_cast<u32x4*>(Vs[kb & 1] + v_to + i * kSweep * D) = v;
    }
  }
  // unit I of block kb's codes into registers (any lane's load_unit is in the cache)
  template <int I>
  __device__ __forceinline__ void load(const uint8_t* codes, u32x2 (&raw)[kUnits], int kb) const {
    const uint32_t u = __builtin_amdgcn_readlane(load_unit, (kb & 15) * 4 + unit_sub(I));
    raw[I] = *reinterpret_cast<const u32x2*>(codes + static_cast<uint64_t>(u) * (16 * D) + unit_off);
  }
  template <int I = 0>
  __device__ __forceinline__ void load_all(int kb) {
    load<I>(p.c.k, kraw, kb);
    load<I>(p.c.v, vraw, kb);
    if constexpr (I + 1 < kUnits) load_all<I + 1>(kb);
  }
  template <int I>
  __device__ __forceinline__ void stage(uint16_t* to, const u32x2 (&raw)[kUnits]) const {
    *reinterpret_cast<u32x4*>(to + I * kSweep * D) = eight_of<FMT>(raw[I][0], raw[I][1]);
  }
  template <int I = 0>
  __device__ __forceinline__ void stage_all(int buf) {
    stage<I>(Ks[buf] + k_to, kraw);
    stage<I>(Vs[buf] + v_to, vraw);
    if constexpr (I + 1 < kUnits) stage_all<I + 1>(buf);
  }
  // bits: the subtiles of block kb (this one or the next) that have a page
  __device__ __forceinline__ int pages_of(int kb) const {
    const uint64_t all = (kb & 15) == 0 && kb > 0 ? __ballot(next.page >= 0) : paged;
    return (all >> ((kb & 15) * 4)) & 15;
  }
  // V codes of block kb that no row sees may be anything, and 0 times them has to be 0
  __device__ __forceinline__ void clear_unseen(int kb) {
    const int pos = s.begin + kb * kBlock, pages = pages_of(kb);
    if (pos >= s.lo && pos + kBlock <= s.hi && pages == 15) return;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int j = pos + i * kSweep + static_cast<int>(threadIdx.x) / kChunks;
      if (!((pages >> unit_sub(i)) & 1) || j < s.lo || j >= s.hi) vraw[i] = u32x2{0u, 0u};
    }
  }

  // ---- products ----
  // MFMA operand i of a block: K's, then V's: V^T operand i of lane (d = 32 j + l32,
  // h), j = i % ND, has positions {16 c + 4 h + u, 16 c + 4 h + 8 + u}, c = i / ND
  template <int I>
  __device__ __forceinline__ void read(const uint16_t* Kc, const uint16_t* Vc) {
    if constexpr (I < 2 * NDC) {
      f[I % kAhead] = *reinterpret_cast<const bf16x8*>(Kc + (k_frag ^ ((I % NDC) * 16)) +
                                                       (I / NDC) * 32 * D);
    } else if constexpr (I < kProducts) {
      constexpr int i = I - 2 * NDC;
      const uint16_t* at = Vc + v_frag[i % ND] + 16 * (i / ND) * D;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at);
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + 8 * D));
      const i16x8 x = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      f[I % kAhead] = __builtin_bit_cast(bf16x8, x);
    }
  }
  template <int I>
  __device__ __forceinline__ void product(const uint16_t* Kc, const uint16_t* Vc) {
    if constexpr (I < 2 * NDC) {
      constexpr int t = I / NDC;
      if constexpr (I % NDC == 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r) cur[t][r] = 0.0f;
      }
      cur[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[I % kAhead], qop[I % NDC], cur[t], 0, 0, 0);
    } else {
      constexpr int i = I - 2 * NDC;
      o[i % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[I % kAhead],
                                                          __builtin_bit_cast(bf16x8, pw[i / ND]),
                                                          o[i % ND], 0, 0, 0);
    }
    read<I + kAhead>(Kc, Vc);
  }

  // ---- softmax ----
  // Of a block's subtile c: the scores' factor, log2 and reciprocal of V's scale.
  struct Factors {
    float ks[4], lv[4], iv[4];
    int there, bad, pos;  // bits: subtiles with a page; with a scale that makes NaN
    bool edge;            // some row does not see all of it, or some scale is bad
  };
  static __device__ __forceinline__ float nan_value() { return __int_as_float(0x7fc00000); }
  // Half T of an edge block: scores that are not seen, and those of bad pages.
  // (Where scores are capped it takes what pair() left: capped scores, or, with C tanh t =
  // C - 2 C u, the u = 1 / (1 + e^2t), of which u = inf is not seen.)
  template <int T>
  __device__ __forceinline__ void hide(const Factors& k) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int c = 2 * T + (r >> 3), j = k.pos + 32 * T + 8 * (r >> 2) + 4 * h + (r & 3);
      if ((k.bad >> c) & 1) cur[T][r] = nan_value();
      if (!((k.there >> c) & 1) || j < from || j >= end) cur[T][r] = CAP == kCapped ? INFINITY : -INFINITY;
    }
  }
  // the factor of what settle() and again() find in cur, subtile c
  __device__ __forceinline__ float factor(const Factors& k, int c) const {
    return CAP == kCapped ? -2.0f * p.cap_log2 : CAP == kCappedFar ? 1.0f : k.ks[c];
  }
  // p times V's scale = 2^(x f + b) of scores 2 Q, 2 Q + 1 of half T: the K scale in f
  // (or, capped, in x) and V's in b.  (Accumulator r: position 32 T + 8 (r / 4) + 4 h +
  // r % 4 of the block, subtile 2 T + r / 8.)
  template <int T, int Q>
  __device__ __forceinline__ void pair(const Factors& k, float base) {
    constexpr int c = 2 * T + Q / 4;
    const float f = factor(k, c), b = base + k.lv[c];
    float e[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      float x = cur[T][2 * Q + z];
      if constexpr (CAP == kCapped) {
        x = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * k.ks[c]));
        cur[T][2 * Q + z] = x;
      } else if constexpr (CAP == kCappedFar) {
        x = capped_far(x * k.ks[c], p.cap_log2);
        cur[T][2 * Q + z] = x;
      }
      e[z] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, f, b));
    }
    sum<T, Q>(k, e[0] + e[1]);
    pw[c][Q % 4] = cvt_pk_bf16x2(e[0], e[1]);
  }
  // (a subtile's pairs first, then times its 1 / V scale)
  template <int T, int Q>
  __device__ __forceinline__ void sum(const Factors& k, float x) {
    constexpr int c = 2 * T + Q / 4;
    part = Q % 4 == 0 ? x : part + x;
    if constexpr (Q % 4 == 3) rs = Q == 3 ? part * k.iv[c] : __builtin_fmaf(part, k.iv[c], rs);
  }
  __device__ __forceinline__ float base() const {
    return (CAP == kCapped ? p.cap_log2 : 0.0f) - (m == -INFINITY ? 0.0f : m);
  }
  // The same for the whole of half T from what pair() left in cur.  (As asm, like the
  // products' rescaling below: in C++ a second set of P lives across the branch.)
  template <int T, int Q = 0>
  __device__ __forceinline__ void again(const Factors& k, float base) {
    constexpr int c = 2 * T + Q / 4;
    const float f = factor(k, c), b = base + k.lv[c];
    float e0, e1;
    asm volatile(
        "v_fma_f32 %1, %3, %5, %6\n\t"
        "v_fma_f32 %2, %4, %5, %6\n\t"
        "v_exp_f32 %1, %1\n\t"
        "v_exp_f32 %2, %2\n\t"
        "s_nop 1\n\t"
        "v_cvt_pk_bf16_f32 %0, %1, %2"
        : "+v"(pw[c][Q % 4]), "=&v"(e0), "=&v"(e1)
        : "v"(cur[T][2 * Q]), "v"(cur[T][2 * Q + 1]), "v"(f), "v"(b));
    sum<T, Q>(k, e0 + e1);
    if constexpr (Q < 7) again<T, Q + 1>(k, base);
  }
  template <int T>
  __device__ __forceinline__ void settle(const Factors& k) {
    if ((CAP && k.edge) || __any(rs > kFar || m == -INFINITY)) {
      if (CAP && k.edge) hide<T>(k);
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = cur[T][8 * c];
#pragma unroll
        for (int r = 1; r < 8; ++r)
          x = CAP == kCapped ? fminf(x, cur[T][8 * c + r]) : fmaxf(x, cur[T][8 * c + r]);
        mx = fmaxf(mx, __builtin_fmaf(x, factor(k, 2 * T + c), CAP == kCapped ? p.cap_log2 : 0.0f));
      }
      const float to = fmaxf(m, xor32_max(mx));
      const float alpha = to == m ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      l *= alpha;
      // (as asm: written in C++, the compiler keeps a second O across the branch, and
      // spills.  It does not see the asm read the MFMAs' results and write their
      // operands, so the wait states are explicit.)
      asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) asm volatile("v_mul_f32 %0, %1, %0" : "+v"(o[j][r]) : "v"(alpha));
      m = to;
      again<T>(k, base());
      asm volatile("s_nop 7");
    }
    l += rs;  // of this lane's positions: the two halves of a row meet at the end
  }

  // MFMA I and what is laid behind it; buf: kb & 1.  (A half's products are NDC MFMAs
  // too.  The first pair waits for the second MFMA: the scores of the half before it
  // are not there yet.)
  template <int Q, int N, int T>
  __device__ __forceinline__ void pairs(const Factors& k, float b) {
    if constexpr (N > 0) {
      pair<T, Q>(k, b);
      pairs<Q + 1, N - 1, T>(k, b);
    }
  }
  template <int buf, int I = 0>
  __device__ __forceinline__ void chain(const Factors& k, float b, int kb) {
    product<I>(Ks[buf], Vs[buf]);
    __builtin_amdgcn_sched_barrier(0);
    constexpr int g = I / NDC, i = I % NDC;
    if constexpr (g == 0 && (i & 1) && i / 2 < kUnits) stage<i / 2>(Ks[buf ^ 1] + k_to, kraw);
    if constexpr (g == 0 && !(i & 1) && i > 0 && i / 2 < kUnits) load<i / 2 - 1>(p.c.k, kraw, kb + 2);
    if constexpr (g == 1 && i == 0) load<kUnits - 1>(p.c.k, kraw, kb + 2);
    if constexpr (g == 1 || g == 2) {
      constexpr int kDone[5] = {0, 0, 2, 5, 8};  // (dim 64) pairs before MFMA i
      constexpr int from = D == 128 ? (i ? i - 1 : 0) : kDone[i % 4];
      constexpr int to = i == NDC - 1 ? 8 : D == 128 ? i : kDone[i % 4 + 1];
      pairs<from, to - from, g - 1>(k, b);
    }
    if constexpr (g == 3 && (i & 1) && i / 2 < kUnits) stage<i / 2>(Vs[buf ^ 1] + v_to, vraw);
    if constexpr (g == 3 && !(i & 1) && i > 0 && i / 2 < kUnits) load<i / 2 - 1>(p.c.v, vraw, kb + 2);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (g == 0 && i == NDC - 1) {
      if (!CAP && k.edge) hide<0>(k);
    }
    if constexpr (g == 1 && i == NDC - 1) {
      settle<0>(k);
      b = base();
      if (!CAP && k.edge) hide<1>(k);
    }
    if constexpr (g == 2 && i == NDC - 1) {
      settle<1>(k);
      if (may_be_special(kb + 1)) clear_unseen(kb + 1);
    }
    if constexpr (I + 1 < kProducts) chain<buf, I + 1>(k, b, kb);
  }

  // Block kb; the next one's codes (in registers) go to the other LDS buffers, and
  // those of the one after it follow into the registers.
  template <int buf>
  __device__ __forceinline__ void block(int kb) {
    const uint16_t *Kc = Ks[buf], *Vc = Vs[buf];
    read<0>(Kc, Vc);
    read<1>(Kc, Vc);
    read<2>(Kc, Vc);
    read<3>(Kc, Vc);
    __builtin_amdgcn_sched_barrier(0);
    Factors k;
    const int at = (kb & 15) * 4;
    k.pos = s.begin + kb * kBlock;
    k.there = (paged >> at) & 15;
    k.bad = (broken >> at) & 15;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      k.ks[t] = uniform(sub.kscale, at + t);
      k.lv[t] = uniform(lv, at + t);
      k.iv[t] = uniform(iv, at + t);
    }
    k.edge = is_special(kb);
    chain<buf>(k, base(), kb);
    load<kUnits - 1>(p.c.v, vraw, kb + 2);
    if (may_be_special(kb + 1)) restage_v(kb + 1);
  }
  // the same without the block itself
  __device__ __forceinline__ void skip(int kb) {
    clear_unseen(kb + 1);
    stage_all((kb & 1) ^ 1);
    restage_v(kb + 1);
    load_all(kb + 2);
  }
};

template <int D, int FMT, int CAP, int NW>
__global__ __launch_bounds__(NW * 64, D == 64 && !CAP ? 3 : 2) void cached_tiles_kernel(
    const CachedArgs p) {
  constexpr int kRows = 32 * NW;
  __shared__ __attribute__((aligned(256))) uint16_t KV[2][2][kBlock * D];
  Division<kRows> div{p};
  div.divide();
  Plan w;
  const int item = blockIdx.x / p.c.heads;
  const bool sorted = p.window == 0 && p.c.seqs > 1 && p.c.seqs <= 64 &&
                      !__any(div.range > div.chunk);
  if (!(sorted ? div.find_longest(item, w) : div.template find<false>(item, w))) return;
  const Span s = span_of<kRows, kBlock>(p, w);
  Tiles<D, FMT, CAP, NW> x{p, w, s, KV[0], KV[1]};
  x.hd = blockIdx.x % p.c.heads;
  x.lane = threadIdx.x & 63;
  x.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  x.l32 = x.lane & 31;
  x.h = x.lane >> 5;
  x.setup();
  const int nb = s.end > s.begin ? (s.end - s.begin + kBlock - 1) / kBlock : 0;
  if (nb > 0) {
    x.ask_page(x.sub, 0);
    x.ask_scales(x.sub, 0);
    x.load_unit = x.sub.unit;
    x.load_all(0);
    x.sub.finish(p.scale_log2);
    x.next = x.sub;
  }
  const int row = w.row0 + x.wave * 32 + x.l32, qrow = min(row, w.rows - 1);
  const int i = qrow / p.group;
  const int64_t head = x.hd * p.group + qrow - i * p.group;
  seen_by(p.c, w.len, w.n, i, p.window, x.from, x.end);
  const uint16_t* qp = p.q + static_cast<int64_t>(w.first + i) * p.q_token + head * p.q_head;
#pragma unroll
  for (int dc = 0; dc < D / 16; ++dc)
    x.qop[dc] = query(p, qp + dc * 16 + 8 * x.h);
  // the positions that some row of this wave sees
  const int i_lo = min(w.row0 + x.wave * 32, w.rows - 1) / p.group;
  const int i_hi = min(w.row0 + x.wave * 32 + 31, w.rows - 1) / p.group;
  int wave_lo, wave_hi, unused;
  seen_by(p.c, w.len, w.n, i_lo, p.window, wave_lo, unused);
  seen_by(p.c, w.len, w.n, i_hi, p.window, unused, wave_hi);
  if (w.row0 + x.wave * 32 >= w.rows) wave_hi = 0;
  if (nb > 0) {
    x.finish(0);
    x.clear_unseen(0);
    x.stage_all(0);
    x.restage_v(0);
    x.load_all(1);
  }
  __syncthreads();
  const auto step = [&](int kb, auto buf) {
    const int pos = s.begin + kb * kBlock;
    if (pos < wave_hi && pos + kBlock > wave_lo)
      x.template block<decltype(buf)::value>(kb);
    else
      x.skip(kb);
    __syncthreads();
  };
  for (int kb = 0; kb < nb; kb += 2) {
    if ((kb & 15) == 0 && kb > 0) {
      x.sub = x.next;
      x.finish(kb);
    }
    if ((kb & 15) == 8 && kb + 8 < nb) x.ask_page(x.next, kb + 8);
    if ((kb & 15) == 10 && kb + 6 < nb) x.ask_scales(x.next, kb + 6);
    if ((kb & 15) == 12 && kb + 4 < nb) x.next.finish(p.scale_log2);
    if ((kb & 15) == 14) x.load_unit = x.next.unit;
    // Of two waves on a SIMD the older one goes first all the time, and where all
    // workgroups run at once its CU is half empty when it has ended: so the two (as far
    // as their numbers tell them) go first in turns (628 -> 612 us for 512 workgroups).
    // Where others wait for a place, the older ones are the longer ones.
    if (p.turns) {
      if (((blockIdx.x >> 8) ^ (kb >> 1)) & 1)
        __builtin_amdgcn_s_setprio(1);
      else
        __builtin_amdgcn_s_setprio(0);
    }
    step(kb, std::integral_constant<int, 0>());
    if (kb + 1 < nb) step(kb + 1, std::integral_constant<int, 1>());
  }
  if (row >= w.rows) return;
  const float lt = xor32_add(x.l);
  if (w.parts > 1) {
    const int64_t at = (static_cast<int64_t>(w.slot + w.part) * p.c.heads + x.hd) * kRows +
                       (row - w.row0);
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<f32x4*>(p.part_o + at * D + 32 * j + 8 * u + 4 * x.h) =
            f32x4{x.o[j][4 * u], x.o[j][4 * u + 1], x.o[j][4 * u + 2], x.o[j][4 * u + 3]};
    if (x.h == 0) {
      p.part_ml[at * 2] = x.m;
      p.part_ml[at * 2 + 1] = lt;
    }
    return;
  }
  const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
  uint16_t* op = p.o + static_cast<int64_t>(w.first + i) * p.o_token + head * p.o_head;
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int u = 0; u < 4; ++u)
      *reinterpret_cast<u32x2*>(op + 32 * j + 8 * u + 4 * x.h) =
          u32x2{cvt_pk_bf16x2(x.o[j][4 * u] * inv, x.o[j][4 * u + 1] * inv),
                cvt_pk_bf16x2(x.o[j][4 * u + 2] * inv, x.o[j][4 * u + 3] * inv)};
}

// The parts of a tile, kRows rows at a time (blockIdx.y has every gridDim.y-th of them)
// by four waves, wave v taking parts v, v + 4, .., and the waves' results in their
// order: the same sum whenever the parts are the same.  A lane has four elements of
// a row.
template <int D, int BM>
__global__ __launch_bounds__(256) void cached_join_kernel(const CachedArgs p) {
  constexpr int kRows = 256 / D;  // 64 lanes, D / 4 a row
  __shared__ f32x4 acc_s[4][64];
  __shared__ float m_s[4][64], l_s[4][64];
  Division<BM> div{p};
  div.divided(__builtin_amdgcn_readfirstlane(*p.chunk));
  Plan w;
  if (!div.template find<true>(blockIdx.x / p.c.heads, w)) return;
  const int h = blockIdx.x % p.c.heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rows = min(BM, w.rows - w.row0);
  for (int r0 = blockIdx.y * kRows; r0 < rows; r0 += gridDim.y * kRows) {
    const int row = r0 + lane / (D / 4), d = (lane % (D / 4)) * 4;
    const bool mine = row < rows;
    const int64_t step = static_cast<int64_t>(p.c.heads) * BM;
    const int64_t at = (static_cast<int64_t>(w.slot) * p.c.heads + h) * BM + (mine ? row : 0);
    float m = -INFINITY, l = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kAhead = 4;
    for (int i0 = wave; i0 < w.parts; i0 += 4 * kAhead) {
      float pm[kAhead], pl[kAhead];
      f32x4 po[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const bool there = i0 + 4 * i < w.parts;
        const int64_t r = at + (there ? i0 + 4 * i : i0) * step;
        pm[i] = there ? p.part_ml[r * 2] : -INFINITY;
        pl[i] = p.part_ml[r * 2 + 1];
        po[i] = *reinterpret_cast<const f32x4*>(p.part_o + r * D + d);
      }
      float to = m;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) to = fmaxf(to, pm[i]);
      const float mm = to == -INFINITY ? 0.0f : to, f = __builtin_amdgcn_exp2f(m - mm);
      l *= f;
      acc *= f;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float e = __builtin_amdgcn_exp2f(pm[i] - mm);
        if (i0 + 4 * i < w.parts) {
          l += pl[i] * e;
          acc += po[i] * e;
        }
      }
      m = to;
    }
    m_s[wave][lane] = m;
    l_s[wave][lane] = l;
    acc_s[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && mine) {
      float mt = -INFINITY;
#pragma unroll
      for (int v = 0; v < 4; ++v) mt = fmaxf(mt, m_s[v][lane]);
      const float mm = mt == -INFINITY ? 0.0f : mt;
      float lt = 0.0f;
      acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float f = __builtin_amdgcn_exp2f(m_s[v][lane] - mm);
        lt += l_s[v][lane] * f;
        acc += acc_s[v][lane] * f;
      }
      const int i = (w.row0 + row) / p.group;
      const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
      uint16_t* op = p.o + static_cast<int64_t>(w.first + i) * p.o_token +
                     static_cast<int64_t>(h * p.group + w.row0 + row - i * p.group) * p.o_head + d;
      *reinterpret_cast<u32x2*>(op) = u32x2{cvt_pk_bf16x2(acc[0] * inv, acc[1] * inv),
                                            cvt_pk_bf16x2(acc[2] * inv, acc[3] * inv)};
    }
    __syncthreads();  // the next rows' results go over these
  }
}

// ---- the choice --------------------------------------------------------------

// Rows of a tile and about how many parts, by the sizes that the host knows.
struct Choice {
  int bm;
  int64_t tiles;   // at most
  int32_t target, least;
};
Choice choose(const ttlh_kv_cache* c, int64_t q_heads, int64_t window) {
  Choice x;
  const int64_t group = q_heads / c->heads;
  // rows of a sequence: on average, half as many again where they may differ
  const int64_t rows = c->tokens * group;
  const int64_t some = (c->starts ? rows + rows / 2 : rows) / (c->seqs > 0 ? c->seqs : 1);
  x.bm = some <= 16 ? 16 : some <= 32 ? 32 : some <= 48 ? 48 : 128;
  const int64_t most = c->width * c->page;  // positions that a sequence's tokens see
  // Eight waves of 32 rows decode a block once in place of twice, but their workgroup is
  // alone on its CU: its start and end are in nobody's shadow, and what it has less
  // to do than others is lost.  So they have dim 128 (dim 64: 389 us as four, 400 as
  // eight), long walks, and two rounds of tiles (4096 new tokens at 8192, 32 / 8 heads:
  // 430 -> 400 us; in one round, 8 sequences of 256 at 8192 lose, 234 -> 248) or one
  // chunk, whose tiles are alike (2048 at 18000 605 -> 570, 256 at 65536 307 -> 291).
  const int64_t wide = (c->starts ? rows / 256 : 0) * c->heads;
  const int64_t walk = window > 0 && window + 256 < most ? window + 256 : most;  // a tile's
  const bool alike = c->seqs == 1 && 4 * c->tokens <= walk && wide * walk >= 1500000;
  if (c->dim == 128 && rows >= 1024 * c->seqs && walk >= 4000 && (wide >= 512 || alike)) x.bm = 256;
  x.tiles = (c->starts ? rows / x.bm + c->seqs : c->seqs * ((group + x.bm - 1) / x.bm));
  const int64_t certain = (c->starts ? rows / x.bm : x.tiles) * c->heads;
  // As many parts as the chip has places (32 answers of up to 8192 positions 72 us;
  // with half as many 83, a tenth more 78, twice as many 72; 16 drafts 80, 99, 103, 86).
  // A part's start and end cost about as much as 512 positions; where there are two workgroups
  // for each CU undivided, parts of fewer than 2048 do not pay (768 tiles of 1024
  // positions: 25 us, halved 31), and where the tiles fill all places only those of
  // much longer sequences than the others are divided.
  const int64_t places = 256 * (x.bm == 256 ? 1 : x.bm == 128 ? 2 : rows_per_cu(c->dim, x.bm / 16));
  x.least = certain >= places ? 4096 : certain >= 512 ? 2048 : 512;
  const int64_t positions = window > 0 && window + c->tokens < most ? window + c->tokens : most;
  // The join costs a launch: one token of up to 896 positions 12.3 us, in two parts 12.9
  // (1024: 13.2, 12.7; dim 64, 1280: 11.5, 12.2); 32 tokens of 640 24.4 and 24.9, of 768
  // 27.0 and 26.4.
  const int64_t alone = x.bm > 16 ? 704 : c->dim == 64 ? 1280 : 960;
  x.target = positions <= (x.least > 512 ? x.least : alone)
                 ? 0
                 : static_cast<int32_t>((places + c->heads - 1) / c->heads);
  return x;
}

int64_t workspace_bytes(const ttlh_kv_cache* c, const Choice& x) {
  return x.target == 0 ? 0 : 2 * int64_t(x.target) * c->heads * x.bm * (c->dim + 2) * 4 + 16;
}

}  // namespace
}  // namespace ttlh

using namespace ttlh;

extern "C" int64_t ttlh_sdpa_cached_workspace_bytes(const ttlh_kv_cache* cache, int64_t q_heads) {
  CacheArgs a;
  if (check_cache("ttlh_sdpa_cached_workspace_bytes", cache, &a) != TTLH_OK || q_heads <= 0 ||
      q_heads % cache->heads)
    return 0;
  // No less than with a window: that only lowers the positions, and what it may change
  // the tiles to, 128 rows in place of 256, has twice the places, half the rows, and
  // where 256 rows have a `least` of 4096 the same one.
  return workspace_bytes(cache, choose(cache, q_heads, 0));
}

extern "C" int ttlh_sdpa_cached(const ttlh_kv_cache* cache, const void* Q, void* O, int64_t q_heads,
                                int64_t q_token, int64_t q_head, int64_t o_token, int64_t o_head,
                                float scale, int64_t window, float softcap, void* workspace,
                                int64_t workspace_size, void* stream) {
  clear_error();
  CachedArgs a;
  const int st = check_cache("ttlh_sdpa_cached", cache, &a.c);
  if (st != TTLH_OK) return st;
  TTLH_REQUIRE(q_heads > 0 && q_heads % cache->heads == 0, TTLH_EINVAL,
               "ttlh_sdpa_cached: q heads must be a multiple of the cache's");
  // (rows, rounded up to a tile, fit an int)
  TTLH_REQUIRE(q_heads < 65536 && cache->tokens * q_heads <= (int64_t(1) << 31) - 512, TTLH_EUNSUPPORTED,
               "ttlh_sdpa_cached: too many q heads or tokens");
  TTLH_REQUIRE(std::isfinite(scale), TTLH_EINVAL, "ttlh_sdpa_cached: scale must be finite");
  TTLH_REQUIRE(softcap == 0.0f || (softcap >= 0x1p-16f && softcap <= 0x1p16f), TTLH_EINVAL,
               "ttlh_sdpa_cached: softcap must be 0 or from 2^-16 to 2^16");
  TTLH_REQUIRE(std::fabs(scale) <= 1e30f, TTLH_EINVAL, "ttlh_sdpa_cached: scale is at most 1e30");
  TTLH_REQUIRE(window >= 0, TTLH_EINVAL, "ttlh_sdpa_cached: window must not be negative");
  if (cache->seqs == 0 || cache->tokens == 0) return TTLH_OK;
  TTLH_REQUIRE(Q && O, TTLH_EINVAL, "ttlh_sdpa_cached: null pointer");
  TTLH_REQUIRE(((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(O)) & 15) == 0 &&
                   ((q_token | q_head | o_token | o_head) & 7) == 0,
               TTLH_EINVAL, "ttlh_sdpa_cached: Q and O must be 16-byte aligned, strides multiples of 8");
  const Choice x = choose(cache, q_heads, window);
  const int64_t need = workspace_bytes(cache, x);
  TTLH_REQUIRE(need == 0 || (workspace && workspace_size >= need &&
                             (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
               TTLH_EINVAL, "ttlh_sdpa_cached: the workspace must have %lld bytes, 16-byte aligned",
               static_cast<long long>(need));
  a.q = static_cast<const uint16_t*>(Q);
  a.o = static_cast<uint16_t*>(O);
  a.q_token = q_token;
  a.q_head = q_head;
  a.o_token = o_token;
  a.o_head = o_head;
  a.group = static_cast<int32_t>(q_heads / cache->heads);
  a.window = static_cast<int32_t>(window < (int64_t(1) << 31) ? window : 0);
  a.target = x.target;
  a.least = x.least;
  a.turns = x.bm == 128 && x.tiles * cache->heads <= 768;
  a.scale_log2 = std::fabs(softcap > 0.0f ? scale / softcap * 2.0f * kLog2e : scale * kLog2e);
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  a.cap_log2 = softcap * kLog2e;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + 2 * int64_t(x.target) * cache->heads * x.bm * cache->dim;
  a.chunk = reinterpret_cast<int32_t*>(a.part_ml + 2 * int64_t(x.target) * cache->heads * x.bm * 2);
  const int64_t items = (x.tiles + x.target) * cache->heads;
  static_assert(kRowWaves == 4, "256 threads, but for tiles of 256 rows");
  const int threads = x.bm == 256 ? 512 : 256;  // (all workgroups' together fit 32 bits)
  TTLH_REQUIRE(items * threads < (int64_t(1) << 32), TTLH_EUNSUPPORTED,
               "ttlh_sdpa_cached: too many tiles");
  const dim3 grid(static_cast<uint32_t>(items));
  // (at most target tiles have several parts; rows of a tile: without starts no more
  // than the group.  Most workgroups of the join find nothing to do: few of them.)
  const int64_t rows = !cache->starts && a.group < x.bm ? a.group : x.bm;
  const int64_t rounds = (rows * cache->dim + 255) / 256;
  const dim3 joins(static_cast<uint32_t>((x.tiles < x.target ? x.tiles : x.target) * cache->heads),
                   static_cast<uint32_t>(rounds < 8 ? rounds : 8));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto run = [&](auto kernel, auto join) {
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, a);
    if (x.target) hipLaunchKernelGGL(join, joins, dim3(256), 0, s, a);
  };
  const auto pick = [&](auto dim, auto fmt) {
    constexpr int D = decltype(dim)::value, F = decltype(fmt)::value;
    if (x.bm == 16)
      run(cached_rows_kernel<D, F, 1>, cached_join_kernel<D, 16>);
    else if (x.bm == 32)
      run(cached_rows_kernel<D, F, 2>, cached_join_kernel<D, 32>);
    else if (x.bm == 48)
      run(cached_rows_kernel<D, F, 3>, cached_join_kernel<D, 48>);
    else {
      const auto tiles = [&](auto cap) {
        constexpr int C = decltype(cap)::value;
        if constexpr (D == 128) {
          if (x.bm == 256) run(cached_tiles_kernel<D, F, C, 8>, cached_join_kernel<D, 256>);
        }
        if (x.bm == 128) run(cached_tiles_kernel<D, F, C, 4>, cached_join_kernel<D, 128>);
      };
      if (softcap == 0.0f)
        tiles(std::integral_constant<int, kUncapped>());
      else if (softcap <= kNearCap)
        tiles(std::integral_constant<int, kCapped>());
      else
        tiles(std::integral_constant<int, kCappedFar>());
    }
  };
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  const std::integral_constant<int, TTLH_CACHE_INT8> i8;
  const std::integral_constant<int, TTLH_CACHE_E4M3> f8;
  if (cache->dim == 128)
    cache->format == TTLH_CACHE_INT8 ? pick(d128, i8) : pick(d128, f8);
  else
    cache->format == TTLH_CACHE_INT8 ? pick(d64, i8) : pick(d64, f8);
  return check_launch("ttlh_sdpa_cached");
}
