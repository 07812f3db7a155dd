// What the kernels of the 8-bit key/value cache share, and can run on the host:
// where a position of a sequence lies, and the scale of a page's codes.
//
// The cache is an array of pages [pages, heads, page, dim] of 8-bit codes, for K
// and for V, with one fp32 scale for each page and head.  table[b][i] names the
// page of positions i * page .. of sequence b.  lengths[b] counts its tokens, the
// new ones of the call among them: new token i of n is at position
// lengths[b] - n + i.  New tokens are packed: sequence b's are starts[b] ..
// starts[b + 1] (without starts: one each).
//
// Tables, lengths and starts are read by the kernels alone, so the kernels bound
// what they find there: a position has a place only where it is inside the table
// and its page inside the cache, tokens are inside the packed ones.
#pragma once

#include <stdint.h>
#include <string.h>

#include "../../include/ttlhip.h"

#if defined(__HIPCC__)
#define TTLH_HD __host__ __device__ inline
#else
#define TTLH_HD inline
#endif

namespace ttlh {

struct CacheArgs {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;  // null: one new token of each sequence
  int64_t table_ld;
  int32_t pages, width, heads, seqs, tokens;
  int32_t shift;  // log2 of the tokens in a page
  int32_t dim;
};

// sequence b's new tokens: the first packed one, and how many
TTLH_HD void seq_tokens(const CacheArgs& c, int b, int& first, int& n) {
  if (!c.starts) {
    first = b;
    n = 1;
    return;
  }
  const int lo = c.starts[b], hi = c.starts[b + 1];
  first = lo < 0 ? 0 : lo > c.tokens ? c.tokens : lo;
  const int end = hi > c.tokens ? c.tokens : hi;
  n = end > first ? end - first : 0;
}

// the positions that the table can name (the host checks that they fit an int)
TTLH_HD int capacity(const CacheArgs& c) { return c.width << c.shift; }

// the page of position pos of sequence b, or -1 where it has none
TTLH_HD int page_at(const CacheArgs& c, int b, int pos) {
  if (pos < 0 || pos >= capacity(c)) return -1;
  const int p = c.table[b * c.table_ld + (pos >> c.shift)];
  return p >= 0 && p < c.pages ? p : -1;
}

// the first element of slot `slot` of a page's head
TTLH_HD int64_t slot_offset(const CacheArgs& c, int page, int head, int slot) {
  return (((static_cast<int64_t>(page) * c.heads + head) << c.shift) + slot) * c.dim;
}

// the positions from .. end - 1 that new token i of n sees in a sequence of `len`
// tokens, as far as a table can name them
TTLH_HD void seen_by(const CacheArgs& c, int len, int n, int i, int window, int& from, int& end) {
  const int64_t past = static_cast<int64_t>(len) - n + i + 1, cap = capacity(c);
  const int64_t lo = window > 0 && past > window ? past - window : 0;
  end = static_cast<int>(past < 0 ? 0 : past > cap ? cap : past);
  from = static_cast<int>(lo > cap ? cap : lo);
}

TTLH_HD uint32_t float_bits(float f) {
  uint32_t u;
  memcpy(&u, &f, 4);
  return u;
}
TTLH_HD float bits_float(uint32_t u) {
  float f;
  memcpy(&f, &u, 4);
  return f;
}

// The scale of values of largest magnitude a: the smallest power of two s >= 2^-126
// with a <= top * s, top = 127 (int8) = 1.984375 x 2^6 or 448 (e4m3) = 1.75 x 2^8;
// NaN where a is not finite.  A power of two, so that x / s is exact, a code is one
// rounding of x, and codes whose page's scale grows are shifted, not measured anew.
TTLH_HD float scale_for(float a, int format) {
  const uint32_t u = float_bits(a) & 0x7fffffffu;
  const int e = static_cast<int>(u >> 23);
  if (e == 255) return bits_float(0x7fc00000u);
  const int top_exp = format == TTLH_CACHE_INT8 ? 6 : 8;
  const uint32_t top_mant = format == TTLH_CACHE_INT8 ? 0x7e0000u : 0x600000u;
  const int s = e - top_exp + ((u & 0x7fffffu) > top_mant ? 1 : 0);  // biased
  return bits_float(static_cast<uint32_t>(s < 1 ? 1 : s) << 23);
}

// A page's scale as its readers take it: one that is negative or not finite is NaN,
// and stays so while tokens are appended.  (Codes of a negative scale, scaled down, would
// be codes of a finite one, or leave their range.)
TTLH_HD float sound_scale(float s) {
  return s >= 0.0f && s < bits_float(0x7f800000u) ? s : bits_float(0x7fc00000u);
}

// the scale of a page that holds earlier tokens under `old`, a sound_scale(), and gets
// new ones that need `need`: the larger; NaN stays
TTLH_HD float joined_scale(float old, float need) {
  if (!(old < bits_float(0x7f800000u)) || need != need) return bits_float(0x7fc00000u);
  return old > need ? old : need;
}

}  // namespace ttlh
