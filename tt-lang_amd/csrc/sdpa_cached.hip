// Attention of new tokens over an 8-bit key/value cache (see ttlhip.h) for gfx950.
// One wave for each (new token, q head): its positions one after the other, with
// the running maximum and sum of an online softmax, a lane for each 64th element.

#include <cmath>

#include "ttlh_common.h"
#include "ttlh_kvcache.h"
#include "ttlh_kvdev.h"

namespace ttlh {
namespace {

struct CachedArgs {
  CacheArgs c;
  const uint16_t* q;
  uint16_t* o;
  int64_t q_token, q_head, o_token, o_head;
  int32_t q_heads, group;
  int32_t window;  // 0: none
  float scale, softcap;
};

struct TokensOf {
  const CacheArgs& c;
  __device__ int operator()(int b) const {
    int first, n;
    seq_tokens(c, b, first, n);
    return n;
  }
};

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int i = 32; i; i >>= 1) x += __shfl_xor(x, i);
  return x;
}

template <int D, int FMT>
__global__ __launch_bounds__(64) void sdpa_cached_simple(const CachedArgs p) {
  const CacheArgs& c = p.c;
  int b, i, first, n;
  if (!find_item(c.seqs, blockIdx.x, TokensOf{c}, b, i)) return;
  seq_tokens(c, b, first, n);
  const int hq = blockIdx.y, h = hq / p.group, lane = threadIdx.x;
  float q[D / 64], o[D / 64], m = -INFINITY, l = 0.0f;
  const uint16_t* qr = p.q + (first + i) * p.q_token + hq * p.q_head;
  for (int d = 0; d < D / 64; ++d) {
    q[d] = bf16_to_f32(qr[d * 64 + lane]);
    o[d] = 0.0f;
  }
  int from, end;
  seen_by(c, c.lengths[b], n, i, p.window, from, end);
  for (int j = from; j < end; ++j) {
    const int page = page_at(c, b, j);
    if (page < 0) continue;
    const int64_t at = slot_offset(c, page, h, j & ((1 << c.shift) - 1));
    const int64_t sc = static_cast<int64_t>(page) * c.heads + h;
    float s = 0.0f;
    for (int d = 0; d < D / 64; ++d) s += q[d] * from_code<FMT>(c.k[at + d * 64 + lane]);
    s = wave_sum(s) * c.k_scale[sc] * p.scale;
    if (p.softcap > 0.0f) s = p.softcap * tanhf(s / p.softcap);
    const float mn = fmaxf(m, s), e = expf(s - (mn == -INFINITY ? 0.0f : mn));
    const float alpha = m == -INFINITY ? 0.0f : expf(m - mn);
    l = l * alpha + e;
    for (int d = 0; d < D / 64; ++d)
      o[d] = o[d] * alpha + e * (from_code<FMT>(c.v[at + d * 64 + lane]) * c.v_scale[sc]);
    m = mn;
  }
  uint16_t* orow = p.o + (first + i) * p.o_token + hq * p.o_head;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int d = 0; d < D / 64; ++d) orow[d * 64 + lane] = f32_to_bf16(o[d] * inv);
}

}  // namespace
}  // namespace ttlh

using namespace ttlh;

extern "C" int64_t ttlh_sdpa_cached_workspace_bytes(const ttlh_kv_cache* cache, int64_t q_heads) {
  return 0;
}

extern "C" int ttlh_sdpa_cached(const ttlh_kv_cache* cache, const void* Q, void* O, int64_t q_heads,
                                int64_t q_token, int64_t q_head, int64_t o_token, int64_t o_head,
                                float scale, int64_t window, float softcap, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  clear_error();
  CachedArgs a;
  const int st = check_cache("ttlh_sdpa_cached", cache, &a.c);
  if (st != TTLH_OK) return st;
  TTLH_REQUIRE(q_heads > 0 && q_heads % cache->heads == 0 && q_heads < 65536, TTLH_EINVAL,
               "ttlh_sdpa_cached: q heads must be a multiple of the cache's");
  TTLH_REQUIRE(std::isfinite(scale), TTLH_EINVAL, "ttlh_sdpa_cached: scale must be finite");
  TTLH_REQUIRE(softcap >= 0.0f && std::isfinite(softcap), TTLH_EINVAL,
               "ttlh_sdpa_cached: softcap must be finite and not negative");
  TTLH_REQUIRE(window >= 0, TTLH_EINVAL, "ttlh_sdpa_cached: window must not be negative");
  if (cache->seqs == 0 || cache->tokens == 0) return TTLH_OK;
  TTLH_REQUIRE(Q && O, TTLH_EINVAL, "ttlh_sdpa_cached: null pointer");
  TTLH_REQUIRE(((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(O)) & 15) == 0 &&
                   ((q_token | q_head | o_token | o_head) & 7) == 0,
               TTLH_EINVAL, "ttlh_sdpa_cached: Q and O must be 16-byte aligned, strides multiples of 8");
  a.q = static_cast<const uint16_t*>(Q);
  a.o = static_cast<uint16_t*>(O);
  a.q_token = q_token;
  a.q_head = q_head;
  a.o_token = o_token;
  a.o_head = o_head;
  a.q_heads = static_cast<int32_t>(q_heads);
  a.group = static_cast<int32_t>(q_heads / cache->heads);
  a.window = static_cast<int32_t>(window < (int64_t(1) << 31) ? window : 0);
  a.scale = scale;
  a.softcap = softcap;
  const dim3 grid(static_cast<uint32_t>(cache->tokens), static_cast<uint32_t>(q_heads));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64), 0, s, a); };
  const bool int8 = cache->format == TTLH_CACHE_INT8;
  if (cache->dim == 128)
    int8 ? run(sdpa_cached_simple<128, TTLH_CACHE_INT8>) : run(sdpa_cached_simple<128, TTLH_CACHE_E4M3>);
  else
    int8 ? run(sdpa_cached_simple<64, TTLH_CACHE_INT8>) : run(sdpa_cached_simple<64, TTLH_CACHE_E4M3>);
  return check_launch("sdpa_cached_simple");
}
