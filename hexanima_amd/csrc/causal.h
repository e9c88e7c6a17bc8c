// What the kernels of the causal text model's attention path share: the two 16-bit types, their vectors and conversions, and
// the lookups of packed sequences and of the paged cache.
#pragma once
#include "hxa_common.h"

// rows and heads a call takes: grids of one wave a row and group of heads stay below 2^32 threads
constexpr int HXA_MAX_ROWS = 1 << 25, HXA_MAX_HEADS = 4096;
// sequences of a plan: wave_count_le's steps stay below 2^31
constexpr int HXA_MAX_SEQS = 1 << 30;

typedef __bf16 hxa_b;
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));

template <typename T>
struct HxaVec;
template <>
struct HxaVec<hxa_h> {
  typedef half2_t v2;
  typedef half4_t v4;
  typedef half8_t v8;
  static constexpr uint32_t EXP = 0x7c007c00u;  // the exponent bits of two values
};
template <>
struct HxaVec<hxa_b> {
  typedef bf2_t v2;
  typedef bf4_t v4;
  typedef bf8_t v8;
  static constexpr uint32_t EXP = 0x7f807f80u;
};

// Number of entries of the ascending list x[0 .. n) that are <= t, by the whole wave: 64 entries a step, and above 64 entries first
// their 64 (then 64 of 64, ...) subdivisions, so 4096 sequences take two dependent loads.
HXA_DEV int wave_count_le(const int *__restrict__ x, int n, int t, int lane) {
  int lo = 0;
  while (n > 64) {
    const int step = (n + 63) >> 6, at = (lane + 1) * step - 1;
    const bool le = at < n && x[lo + at] <= t;
    const int whole = __popcll(__ballot(le)) * step;  // these are all <= t
    lo += whole;
    n = min(n - whole, step);
  }
  return lo + __popcll(__ballot(lane < n && x[lo + lane] <= t));
}

// The page row (a row of hd values in the pools) of a cached token, or -1: entry e of a page table, head h, row r of the page
HXA_DEV long cache_row(int e, int npages, int H, int h, int page, int r) {
  return (unsigned)e < (unsigned)npages ? ((long)e * H + h) * page + r : -1;
}

// host side: hxa_kv_cache checks shared by the calls on it (HXA_OK or the error, with its message set)
int hxa_kv_check(const hxa_kv_cache *c, int T, const char *who);
int hxa_kv_check_q8(const hxa_kv_cache_q8 *c, int T, const char *who);
