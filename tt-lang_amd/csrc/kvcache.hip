// Rotary positions and the writes of an 8-bit key/value cache for gfx950.
//
// rope: plane i of a head, (x_i, x_j), becomes scale (x_i cos a - x_j sin a,
// x_j cos a + x_i sin a) with a = position * freqs[i]; both directions are one
// rotation, so the gradient is the same kernel with -a.  HBM bound: x is read and
// written once.  The angles are the only arithmetic that matters: a far position
// times a frequency has to be right to 2^-24 of a turn after whole turns are taken
// off, which fp32 cannot hold from position 2^10 on, so a workgroup computes the
// angles of its tokens in fp64, once for all heads, into LDS.  8192 x 40 x 128 bf16:
// 36.4 us, 4.6 TB/s; one token's 2.7 us, less than a launch takes on the host.
//
// kv_cache_write: reads the tokens once and writes a byte for each value; HBM bound
// for prompts, latency bound for a token each.
//  * kv_write_kernel: a workgroup for each page that gets tokens and head, K and V.
//    The values stay in registers between the search for the largest one and their
//    rounding (22,552 tokens of prompts, 8 x 128 bf16: 31 us, 4.4 TB/s; read twice,
//    an element at a time, 121 us).
//  * kv_write_one_kernel (no starts: a token for each sequence): a thread for each
//    eight values, so that a page's head is a group of 8 or 16 lanes that needs no
//    barrier; earlier codes are touched where a scale grows (64 tokens, 8 x 128 bf16:
//    4.5 us, the latency of length, table, values and scale; 7.5 with the launch).

#include <cmath>
#include <type_traits>

#include "ttlh_common.h"
#include "ttlh_kvcache.h"
#include "ttlh_kvdev.h"

namespace ttlh {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeAngles = 512;  // cos, sin pairs that a workgroup keeps

struct RopeArgs {
  const void* x;
  void* out;
  const void* positions;
  const double* freqs;
  int64_t x_token, x_head, o_token, o_head;
  int32_t tokens, heads, dim, rot;
  int32_t tpb;       // tokens of a workgroup
  int32_t hpb;       // heads of a workgroup
  int32_t units;     // vectors (rotated: pairs of vectors) of a head
  int32_t turned;    // of them, rotated
  uint32_t by_units, by_heads;  // ceil(2^32 / units), ceil(2^32 / hpb); 0 for one
  int32_t pos_bytes;
  float scale;
  int32_t backward;
};

// cos and sin of `a` radians: whole quarter turns off in fp64, then the Taylor
// series on [-pi/4, pi/4] (next terms at most 1.0e-15, and 2.6e-14 of the sine's first).
__device__ __forceinline__ void cos_sin(double a, float& c, float& s) {
  const double q = rint(a * 0.63661977236758134308);  // 2 / pi
  // pi / 2 in two parts, so that q * pi / 2 is right for q up to 2^31
  double t = fma(q, -1.57079632679489655800, a);
  t = fma(q, -6.12323399573676603587e-17, t);
  const double z = t * t;
  double sn = fma(z, 1.0 / 6227020800.0, -1.0 / 39916800.0);
  sn = fma(z, sn, 1.0 / 362880.0);
  sn = fma(z, sn, -1.0 / 5040.0);
  sn = fma(z, sn, 1.0 / 120.0);
  sn = fma(z, sn, -1.0 / 6.0);
  sn = fma(t * z, sn, t);
  double cs = fma(z, -1.0 / 87178291200.0, 1.0 / 479001600.0);
  cs = fma(z, cs, -1.0 / 3628800.0);
  cs = fma(z, cs, 1.0 / 40320.0);
  cs = fma(z, cs, -1.0 / 720.0);
  cs = fma(z, cs, 1.0 / 24.0);
  cs = fma(z, cs, -0.5);
  cs = fma(z, cs, 1.0);
  const int n = static_cast<int>(static_cast<int64_t>(q) & 3);
  const double u = (n & 1) ? sn : cs, w = (n & 1) ? cs : sn;
  c = static_cast<float>((n == 1 || n == 2) ? -u : u);
  s = static_cast<float>((n & 2) ? -w : w);
}

// e / d with by = ceil(2^32 / d): exact while e d < 2^32
__device__ __forceinline__ uint32_t divided(uint32_t e, uint32_t by) {
  return by ? __umulhi(e, by) : e;
}

template <typename T, int V>
struct Vec {
  float v[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) {
      v[0] = to_f32(*p);
    } else if constexpr (sizeof(T) == 2) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const f32x4 w = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = w[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1) {
      *p = from_f32<T>(v[0]);
    } else if constexpr (sizeof(T) == 2) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = cvt_pk_bf16x2(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<u32x4*>(p) = w;
    } else {
      *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    }
  }
};

// A unit: vectors of the planes i .. (or one vector of neighbouring planes), or one
// that is copied.
template <typename T, int V, bool INTER>
struct Unit {
  Vec<T, V> a, b;
  T* o;
  int lo, hi, angle;  // elements of the vectors, the first angle
  bool there, turned;

  __device__ __forceinline__ void read(const RopeArgs& p, uint32_t e, int t0, int h0, int nh,
                                       int half) {
    const uint32_t th = divided(e, p.by_units), u = e - th * p.units;
    const uint32_t t = divided(th, p.by_heads), h = th - t * p.hpb;
    there = static_cast<int>(h) < nh;
    if (!there) return;
    const T* x = static_cast<const T*>(p.x) + (t0 + t) * p.x_token + (h0 + h) * p.x_head;
    o = static_cast<T*>(p.out) + (t0 + t) * p.o_token + (h0 + h) * p.o_head;
    turned = static_cast<int>(u) < p.turned;
    if (!turned) {
      lo = p.rot + (u - p.turned) * V;
    } else if constexpr (INTER && V > 1) {
      lo = u * V;
      angle = t * half + u * (V / 2);
    } else {
      lo = INTER ? 2 * u : u * V;
      hi = INTER ? lo + 1 : lo + half;
      angle = t * half + u * V;
      b.load(x + hi);
    }
    a.load(x + lo);
  }
  __device__ __forceinline__ void write(const RopeArgs& p, const float* cs, const float* sn) {
    if (!there) return;
    if (!turned) {
      a.store(o + lo);
    } else if constexpr (INTER && V > 1) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float c = cs[angle + i], s = sn[angle + i];
        b.v[2 * i] = a.v[2 * i] * c - a.v[2 * i + 1] * s;
        b.v[2 * i + 1] = a.v[2 * i + 1] * c + a.v[2 * i] * s;
      }
      b.store(o + lo);
    } else {
      Vec<T, V> y, z;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float c = cs[angle + i], s = sn[angle + i];
        y.v[i] = a.v[i] * c - b.v[i] * s;
        z.v[i] = b.v[i] * c + a.v[i] * s;
      }
      y.store(o + lo);
      z.store(o + hi);
    }
  }
};

// V: elements of a vector (16 bytes, or one element where sizes or addresses do
// not allow that).  INTER: planes of neighbouring elements; with V = 1 a rotated
// unit is one plane there.
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const RopeArgs p) {
  __shared__ float cs[kRopeAngles], sn[kRopeAngles];
  const int t0 = blockIdx.x * p.tpb, nt = min(p.tpb, p.tokens - t0);
  const int h0 = blockIdx.y * p.hpb, nh = min(p.hpb, p.heads - h0);
  const int half = p.rot >> 1;
  for (int i = threadIdx.x; i < nt * half; i += kRopeThreads) {
    const int t = i / half;
    const double pos = p.pos_bytes == 8
                           ? static_cast<double>(static_cast<const int64_t*>(p.positions)[t0 + t])
                           : static_cast<double>(static_cast<const int32_t*>(p.positions)[t0 + t]);
    float c, s;
    cos_sin(pos * p.freqs[i - t * half], c, s);
    cs[i] = c * p.scale;
    sn[i] = (p.backward ? -s : s) * p.scale;
  }
  __syncthreads();
  // Units of one vector go two at a time: both are read before either is written
  // (which the compiler could not do by itself, x may be out), so that a thread has
  // two loads in flight, as one unit of two vectors has (4099 x 33 x 96 f32 28 ->
  // 24.6 us; two units of two vectors: 8192 x 40 x 128 bf16 35 -> 41 us).
  constexpr uint32_t kAtOnce = INTER && V > 1 ? 2 : 1;
  const uint32_t n = static_cast<uint32_t>(nt) * p.hpb * p.units;
  for (uint32_t e0 = threadIdx.x; e0 < n; e0 += kAtOnce * kRopeThreads) {
    Unit<T, V, INTER> a, b;
    const bool two = kAtOnce == 2 && e0 + kRopeThreads < n;
    a.read(p, e0, t0, h0, nh, half);
    if (two) b.read(p, e0 + kRopeThreads, t0, h0, nh, half);
    a.write(p, cs, sn);
    if (two) b.write(p, cs, sn);
  }
}

// ---------------------------------------------------------------------------

struct WriteArgs {
  CacheArgs c;
  const void* x[2];
  int64_t token[2], head[2];
  bool vec;  // 16-byte loads
};

// pages that sequence b's new tokens reach
struct PagesOf {
  const CacheArgs& c;
  __device__ int operator()(int b) const {
    int first, n;
    seq_tokens(c, b, first, n);
    const int64_t len = c.lengths[b], begin = len - n;
    const int64_t end = len < capacity(c) ? len : capacity(c);
    const int64_t from = begin > 0 ? begin : 0;
    return end > from ? static_cast<int>(((end - 1) >> c.shift) - (from >> c.shift) + 1) : 0;
  }
};

// Eight neighbouring values.
template <typename T>
struct Eight {
  u32x4 w[sizeof(T) / 2];
  // vec: 16-byte loads; else element by element
  __device__ __forceinline__ void load(const T* x, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        w[i] = reinterpret_cast<const u32x4*>(x)[i];
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[0][i] = x[2 * i] | static_cast<uint32_t>(x[2 * i + 1]) << 16;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i / 4][i % 4] = __float_as_uint(x[i]);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = u32x4{0u, 0u, 0u, 0u};
  }
  __device__ __forceinline__ uint32_t bits(int i) const {  // of value i as fp32
    if constexpr (sizeof(T) == 2)
      return (i & 1) ? w[0][i / 2] & 0xffff0000u : w[0][i / 2] << 16;
    else
      return w[i / 4][i % 4];
  }
  // the largest magnitude by its bits: infinities and NaN are larger than any number
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, bits(i) & 0x7fffffffu);
    return m;
  }
  // the codes of value * inv (zeros where inv is NaN)
  template <int FMT>
  __device__ __forceinline__ uint2 codes(float inv) const {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = inv == inv ? __uint_as_float(bits(i)) * inv : 0.0f;
    return uint2{four_codes<FMT>(v[0], v[1], v[2], v[3]), four_codes<FMT>(v[4], v[5], v[6], v[7])};
  }
};

// codes whose scale grows: times `down` = old / new scale, and rounded again
template <int FMT>
__device__ __forceinline__ uint2 scaled_down(uint2 c, float down) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = from_code<FMT>(static_cast<uint8_t>((i < 4 ? c.x : c.y) >> (8 * (i & 3)))) * down;
  return uint2{four_codes<FMT>(v[0], v[1], v[2], v[3]), four_codes<FMT>(v[4], v[5], v[6], v[7])};
}

// SWEEPS: rounds of 256 threads with eight values each that cover a page's head.
template <typename T, int FMT, int D, int SWEEPS>
__global__ __launch_bounds__(256) void kv_write_kernel(const WriteArgs p) {
  constexpr int kPer = D / 8;              // threads of a token
  constexpr int kTokens = 256 / kPer;      // tokens of a sweep
  const CacheArgs& c = p.c;
  int b, j;
  if (!find_item(c.seqs, blockIdx.x, PagesOf{c}, b, j)) return;
  const int h = blockIdx.y;
  int first, n;
  seq_tokens(c, b, first, n);
  const int len = c.lengths[b];  // (>= 1 here)
  const int64_t begin = static_cast<int64_t>(len) - n;
  const int page0 = (static_cast<int>(begin > 0 ? begin >> c.shift : 0) + j) << c.shift;
  const int lo = begin > page0 ? static_cast<int>(begin) - page0 : 0;  // slots lo .. hi - 1
  const int hi = min(len - page0, 1 << c.shift);
  const int t0 = threadIdx.x / kPer, e = (threadIdx.x % kPer) * 8;
  Eight<T> x[2][SWEEPS];
  uint32_t big[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < SWEEPS; ++i) {
    const int t = t0 + i * kTokens;
#pragma unroll
    for (int z = 0; z < 2; ++z)
      if (t >= lo && t < hi)
        x[z][i].load(static_cast<const T*>(p.x[z]) + (first + page0 - begin + t) * p.token[z] +
                         h * p.head[z] + e, p.vec);
      else
        x[z][i].clear();
  }
  const int page = page_at(c, b, page0);  // (under the loads)
  if (page < 0) return;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
#pragma unroll
    for (int i = 0; i < SWEEPS; ++i) big[z] = max(big[z], x[z][i].largest());
    big[z] = wave_max(big[z]);
  }
  __shared__ uint32_t part[2][4];
  if ((threadIdx.x & 63) == 0) {
    part[0][threadIdx.x >> 6] = big[0];
    part[1][threadIdx.x >> 6] = big[1];
  }
  __syncthreads();
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    float* scale = (z ? c.v_scale : c.k_scale) + static_cast<int64_t>(page) * c.heads + h;
    uint8_t* codes = (z ? c.v : c.k) + slot_offset(c, page, h, 0) + e;
    const uint32_t m = max(max(part[z][0], part[z][1]), max(part[z][2], part[z][3]));
    float s = scale_for(__uint_as_float(m), FMT);
    if (lo > 0) {  // earlier tokens
      const float old = sound_scale(*scale);
      s = joined_scale(old, s);
      if (s > old)
        for (int t = t0; t < lo; t += kTokens) {
          uint2* at = reinterpret_cast<uint2*>(codes + t * D);
          *at = scaled_down<FMT>(*at, old / s);
        }
    }
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < SWEEPS; ++i) {
      const int t = t0 + i * kTokens;
      if (t >= lo && t < hi) *reinterpret_cast<uint2*>(codes + t * D) = x[z][i].template codes<FMT>(inv);
    }
    if (lo > 0) __syncthreads();  // (uniform) every thread has read the old scale
    if (threadIdx.x == 0) *scale = s;
  }
}

template <typename T, int FMT, int D>
__global__ __launch_bounds__(256) void kv_write_one_kernel(const WriteArgs p) {
  constexpr int kPer = D / 8;
  const CacheArgs& c = p.c;
  const int b = blockIdx.x;
  const int unit = blockIdx.y * (256 / kPer) + threadIdx.x / kPer;  // (head, K or V)
  const int h = unit >> 1, z = unit & 1, e = (threadIdx.x % kPer) * 8;
  const int pos = c.lengths[b] - 1, page = page_at(c, b, c.lengths[b] > 0 ? pos : -1);
  if (page < 0 || h >= c.heads) return;
  const int slot = pos & ((1 << c.shift) - 1);
  float* scale = (z ? c.v_scale : c.k_scale) + static_cast<int64_t>(page) * c.heads + h;
  uint8_t* codes = (z ? c.v : c.k) + slot_offset(c, page, h, 0) + e;
  Eight<T> x;
  x.load(static_cast<const T*>(z ? p.x[1] : p.x[0]) + b * (z ? p.token[1] : p.token[0]) +
             h * (z ? p.head[1] : p.head[0]) + e, p.vec);
  const float old = sound_scale(*scale);
  uint32_t m = x.largest();
#pragma unroll
  for (int i = kPer / 2; i; i >>= 1)
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), i)));
  float s = scale_for(__uint_as_float(m), FMT);
  if (slot > 0) {
    s = joined_scale(old, s);
    if (s > old)
      for (int t = 0; t < slot; ++t) {
        uint2* at = reinterpret_cast<uint2*>(codes + t * D);
        *at = scaled_down<FMT>(*at, old / s);
      }
  }
  *reinterpret_cast<uint2*>(codes + slot * D) = x.template codes<FMT>(1.0f / s);
  // (the group's lanes have all read the old scale: they run in one wave, and the
  // exchanges above need its value from no one)
  if (e == 0 && !(slot > 0 && s == old)) *scale = s;
}

}  // namespace
}  // namespace ttlh

using namespace ttlh;

extern "C" int ttlh_rope(const void* x, void* out, int dtype, const void* positions, int pos_bytes,
                         const double* freqs, int64_t tokens, int64_t heads, int64_t dim,
                         int64_t rot, int64_t x_token, int64_t x_head, int64_t o_token,
                         int64_t o_head, int interleaved, float scale, int backward,
                         void* stream) {
  clear_error();
  TTLH_REQUIRE(tokens >= 0 && heads >= 0 && dim > 0, TTLH_EINVAL, "ttlh_rope: bad sizes");
  TTLH_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= dim, TTLH_EINVAL,
               "ttlh_rope: rot must be even and at most the head's elements");
  TTLH_REQUIRE(rot <= 2 * kRopeAngles, TTLH_EUNSUPPORTED, "ttlh_rope: rot is at most %d",
               2 * kRopeAngles);
  TTLH_REQUIRE(dtype == TTLH_BF16 || dtype == TTLH_F32, TTLH_EINVAL, "ttlh_rope: bf16 or f32");
  TTLH_REQUIRE(pos_bytes == 4 || pos_bytes == 8, TTLH_EINVAL, "ttlh_rope: int32 or int64 positions");
  TTLH_REQUIRE(std::isfinite(scale), TTLH_EINVAL, "ttlh_rope: scale must be finite");
  if (tokens == 0 || heads == 0) return TTLH_OK;
  TTLH_REQUIRE(x && out && positions && (freqs || !rot), TTLH_EINVAL, "ttlh_rope: null pointer");
  TTLH_REQUIRE(tokens < (int64_t(1) << 31) && heads < (int64_t(1) << 20) && dim <= 32768,
               TTLH_EUNSUPPORTED, "ttlh_rope: too many tokens, heads or elements");
  RopeArgs a;
  a.x = x;
  a.out = out;
  a.positions = positions;
  a.freqs = freqs;
  a.x_token = x_token;
  a.x_head = x_head;
  a.o_token = o_token;
  a.o_head = o_head;
  a.tokens = static_cast<int32_t>(tokens);
  a.heads = static_cast<int32_t>(heads);
  a.dim = static_cast<int32_t>(dim);
  a.rot = static_cast<int32_t>(rot);
  a.pos_bytes = pos_bytes;
  a.scale = scale;
  a.backward = backward != 0;
  const int wide = dtype == TTLH_BF16 ? 8 : 4;
  const int64_t turned_in = interleaved ? rot : rot / 2;  // elements that vectors of a turn start in
  const bool vec = turned_in % wide == 0 && (dim - rot) % wide == 0 && x_token % wide == 0 &&
                   x_head % wide == 0 && o_token % wide == 0 && o_head % wide == 0 &&
                   ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const int V = vec ? wide : 1;
  a.turned = static_cast<int32_t>(vec ? turned_in / V : rot / 2);
  a.units = a.turned + static_cast<int32_t>((dim - rot) / V);
  // (magic divisions: exact while dividend x divisor < 2^32)
  a.hpb = static_cast<int32_t>(heads < 65536 / a.units ? heads : (a.units < 65536 ? 65536 / a.units : 1));
  if (a.hpb > 64) a.hpb = 64;
  const int half = a.rot > 0 ? a.rot / 2 : 1;
  a.tpb = kRopeAngles / half;
  if (a.tpb > 4) a.tpb = 4;
  while (a.tpb > 1 && (static_cast<int64_t>(a.tpb) * a.hpb * a.units >= 65536 ||
                       tokens / a.tpb < 2048))
    a.tpb >>= 1;
  a.by_units = static_cast<uint32_t>(((uint64_t(1) << 32) + a.units - 1) / a.units);
  a.by_heads = static_cast<uint32_t>(((uint64_t(1) << 32) + a.hpb - 1) / a.hpb);
  TTLH_REQUIRE((heads + a.hpb - 1) / a.hpb < 65536, TTLH_EUNSUPPORTED, "ttlh_rope: too many heads");
  const dim3 grid(static_cast<uint32_t>((tokens + a.tpb - 1) / a.tpb),
                  static_cast<uint32_t>((heads + a.hpb - 1) / a.hpb));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kRopeThreads), 0, s, a); };
  if (dtype == TTLH_BF16 && vec)
    interleaved ? run(rope_kernel<uint16_t, 8, true>) : run(rope_kernel<uint16_t, 8, false>);
  else if (dtype == TTLH_BF16)
    interleaved ? run(rope_kernel<uint16_t, 1, true>) : run(rope_kernel<uint16_t, 1, false>);
  else if (vec)
    interleaved ? run(rope_kernel<float, 4, true>) : run(rope_kernel<float, 4, false>);
  else
    interleaved ? run(rope_kernel<float, 1, true>) : run(rope_kernel<float, 1, false>);
  return check_launch("rope_kernel");
}

namespace ttlh {

int check_cache(const char* fn, const ttlh_kv_cache* c, CacheArgs* a) {
  TTLH_REQUIRE(c, TTLH_EINVAL, "%s: null cache", fn);
  TTLH_REQUIRE(c->page == 16 || c->page == 32 || c->page == 64 || c->page == 128, TTLH_EUNSUPPORTED,
               "%s: pages have 16, 32, 64 or 128 tokens", fn);
  TTLH_REQUIRE(c->dim == 64 || c->dim == 128, TTLH_EUNSUPPORTED, "%s: dim must be 64 or 128", fn);
  TTLH_REQUIRE(c->format == TTLH_CACHE_INT8 || c->format == TTLH_CACHE_E4M3, TTLH_EINVAL,
               "%s: unknown format of codes", fn);
  TTLH_REQUIRE(c->pages >= 0 && c->width >= 0 && c->heads > 0 && c->seqs >= 0 && c->tokens >= 0 &&
                   (c->table_ld >= c->width || c->seqs <= 1),
               TTLH_EINVAL, "%s: bad sizes", fn);
  TTLH_REQUIRE(c->pages < (int64_t(1) << 31) && c->heads < 65536 && c->seqs < (int64_t(1) << 24) &&
                   c->tokens < (int64_t(1) << 28) && c->width * c->page <= (int64_t(1) << 30),
               TTLH_EUNSUPPORTED, "%s: too many pages, positions, heads, sequences or tokens", fn);
  TTLH_REQUIRE(c->starts || c->tokens == c->seqs, TTLH_EINVAL,
               "%s: without starts there is one token for each sequence", fn);
  if (c->seqs == 0 || c->tokens == 0) return TTLH_OK;
  TTLH_REQUIRE(c->lengths && (c->table || !c->width), TTLH_EINVAL, "%s: null pointer", fn);
  TTLH_REQUIRE((c->k && c->v && c->k_scale && c->v_scale) || !c->pages, TTLH_EINVAL,
               "%s: null pointer", fn);
  TTLH_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) == 0,
               TTLH_EINVAL, "%s: the codes must be 16-byte aligned", fn);
  a->k = static_cast<uint8_t*>(c->k);
  a->v = static_cast<uint8_t*>(c->v);
  a->k_scale = c->k_scale;
  a->v_scale = c->v_scale;
  a->table = c->table;
  a->lengths = c->lengths;
  a->starts = c->starts;
  a->table_ld = c->table_ld;
  a->pages = static_cast<int32_t>(c->pages);
  a->width = static_cast<int32_t>(c->width);
  a->heads = static_cast<int32_t>(c->heads);
  a->seqs = static_cast<int32_t>(c->seqs);
  a->tokens = static_cast<int32_t>(c->tokens);
  a->shift = __builtin_ctz(c->page);
  a->dim = c->dim;
  return TTLH_OK;
}

}  // namespace ttlh

extern "C" int ttlh_kv_cache_write(const ttlh_kv_cache* cache, const void* k, const void* v,
                                   int dtype, int64_t k_token, int64_t k_head, int64_t v_token,
                                   int64_t v_head, void* stream) {
  clear_error();
  WriteArgs a;
  const int st = check_cache("ttlh_kv_cache_write", cache, &a.c);
  if (st != TTLH_OK) return st;
  TTLH_REQUIRE(dtype == TTLH_BF16 || dtype == TTLH_F32, TTLH_EINVAL,
               "ttlh_kv_cache_write: bf16 or f32 values");
  if (cache->seqs == 0 || cache->tokens == 0 || cache->width == 0) return TTLH_OK;
  TTLH_REQUIRE(k && v, TTLH_EINVAL, "ttlh_kv_cache_write: null pointer");
  a.x[0] = k;
  a.x[1] = v;
  a.token[0] = k_token;
  a.token[1] = v_token;
  a.head[0] = k_head;
  a.head[1] = v_head;
  const int wide = dtype == TTLH_BF16 ? 8 : 4;
  a.vec = (k_token | k_head | v_token | v_head) % wide == 0 &&
          ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto pick = [&](auto value, auto fmt, auto dim) {
    typedef decltype(value) T;
    constexpr int F = decltype(fmt)::value, D = decltype(dim)::value;
    if (!cache->starts) {
      const dim3 grid(static_cast<uint32_t>(cache->seqs),
                      static_cast<uint32_t>((2 * cache->heads * (D / 8) + 255) / 256));
      hipLaunchKernelGGL((kv_write_one_kernel<T, F, D>), grid, dim3(256), 0, s, a);
      return;
    }
    // n tokens reach at most (n - 2) / page + 2 pages
    const dim3 grid(static_cast<uint32_t>(cache->tokens / cache->page + 2 * cache->seqs),
                    static_cast<uint32_t>(cache->heads));
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    const int sweeps = cache->page * D / 2048;
    if (sweeps <= 1)
      run(kv_write_kernel<T, F, D, 1>);
    else if (sweeps == 2)
      run(kv_write_kernel<T, F, D, 2>);
    else if (sweeps == 4)
      run(kv_write_kernel<T, F, D, 4>);
    else if constexpr (D == 128)
      run(kv_write_kernel<T, F, D, 8>);
  };
  const std::integral_constant<int, TTLH_CACHE_INT8> i8;
  const std::integral_constant<int, TTLH_CACHE_E4M3> f8;
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  const auto dims = [&](auto value, auto fmt) {
    cache->dim == 128 ? pick(value, fmt, d128) : pick(value, fmt, d64);
  };
  const bool int8 = cache->format == TTLH_CACHE_INT8;
  if (dtype == TTLH_BF16)
    int8 ? dims(uint16_t(), i8) : dims(uint16_t(), f8);
  else
    int8 ? dims(float(), i8) : dims(float(), f8);
  return check_launch("kv_write_kernel");
}
