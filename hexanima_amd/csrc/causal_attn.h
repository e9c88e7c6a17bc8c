// What the attention kernels of the causal text model share, over 16-bit keys (causal_attn.hip) and over a cache of int8 (cached_q8.hip): work
// items and their limits, tiles in LDS, the results' way out, the join of partial results, the launches.
#pragma once
#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>
#include <tuple>

#include "causal.h"
#include "causal_walk.h"
#include "kernels.h"

namespace {

constexpr float L2E = 1.4426950408889634f;
constexpr float RESCALE2 = 5.5f * L2E;  // growth of the maximum, in powers of two, that is left unscaled

HXA_DEV float16_t mma32(half8_t a, half8_t b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
HXA_DEV float16_t mma32(bf8_t a, bf8_t b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
HXA_DEV float4_t mma16(half8_t a, half8_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
HXA_DEV float4_t mma16(bf8_t a, bf8_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
typedef short short4_t __attribute__((ext_vector_type(4)));
HXA_DEV float4_t mma16h(half4_t a, half4_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
HXA_DEV float4_t mma16h(bf4_t a, bf4_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4_t, a), __builtin_bit_cast(short4_t, b), c, 0, 0, 0);
}
typedef __attribute__((address_space(3))) short4_t lds_short4_t;
template <typename V4>
HXA_DEV V4 read_tr(const uint8_t *p) {
  return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t *)(lds_void_t *)p));
}
HXA_DEV float sum2(half2_t h, float l) { return __builtin_amdgcn_fdot2(h, (half2_t){(hxa_h)1.0f, (hxa_h)1.0f}, l, false); }
HXA_DEV float sum2(bf2_t h, float l) { return __builtin_amdgcn_fdot2_f32_bf16(h, (bf2_t){(hxa_b)1.0f, (hxa_b)1.0f}, l, false); }
HXA_DEV float max16(float v) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48, which all get it
  const int x = __builtin_bit_cast(int, v);
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  v = fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1]));
  float lo, hi;
  halves(v, lo, hi);
  return fmaxf(lo, hi);
}
HXA_DEV float add16(float v) {
  const int x = __builtin_bit_cast(int, v);
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  v = __builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]);
  float lo, hi;
  halves(v, lo, hi);
  return lo + hi;
}

// the thread, opaque: what follows from it is computed again for each item, not kept in registers across them
HXA_DEV int this_thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// where the keys of a work item lie
template <typename T>
struct Keys {
  const T *k, *v;   // contiguous: row 0 of the sequence and key head; paged: the pools
  long ldk, ldv;    // contiguous: row strides
  const int *prefix, *table;  // paged: the prefix's pages, the sequence's own
  int P, page, npages, H, h;
  uint32_t pm;  // 2^32 / page, as Item's gm
  // place of token y in its table, and in the page
  HXA_DEV unsigned slot(unsigned y, unsigned &in_page) const {
    unsigned n = __umulhi(y, pm);
    in_page = y - n * page;
    const bool one = in_page >= (unsigned)page;
    in_page -= one ? page : 0;
    return n + one;
  }
};

// a work item: rows [r0, r0 + rows of the mode) of nrows rows that belong together, keys [x0, x1)
struct Item {
  int r0, nrows, G;
  uint32_t gm;  // 2^32 / G, rounded down (2^32 - 1 for G = 1)
  int tok0;  // row R is token tok0 + R / G of the call
  int x0, x1;
  // row R sees the keys x <= base + R / G (not causal: base), but none past cap, and those up to least in any case
  int base, cap, least;
  bool causal;
};
// R / G and the rest: the product with the rounded reciprocal is at most one too small
HXA_DEV int row_tok(const Item &it, int R, int &rest) {
  int t = (int)__umulhi((uint32_t)R, it.gm);
  rest = R - t * it.G;
  if (rest >= it.G) {
    rest -= it.G;
    t++;
  }
  return t;
}
HXA_DEV int tok_limit(const Item &it, int tok) { return max(min(it.causal ? it.base + tok : it.base, it.cap), it.least); }
HXA_DEV int row_limit(const Item &it, int R) {
  int rest;
  return tok_limit(it, row_tok(it, R, rest));
}

template <typename T, int HD>
struct Geo {
  static constexpr int RB = HD * 2;          // bytes of a row
  static constexpr int TB = KT * RB;         // of a tile
  static constexpr int CH = HD / 8;          // 16-byte chunks a row = lanes a row of a load
  static constexpr int RPL = 64 / CH;        // rows of one wave-wide load (1 KB)
  static constexpr int NLD = KT / RPL / 4;   // loads a wave and tile, for K and for V each, of rows 4 RPL apart
  static constexpr int NOFF = HD == 256 ? 2 : 1;  // of them different up to a whole number of 16 rows (permutation and swizzles repeat)
  static constexpr int FLAGS = 4 * TB;       // LDS past the tiles: the flags of fix_v
  static constexpr int LDS = 4 * TB + 64;
};

// The tile loader, for all modes: row i of LDS, of K and of V, holds key (PERM ? krow_key(i) : i) of the tile; chunk c of a row is at
// c ^ fk(row) in K, c ^ fv(row) in V. (One order for both, so a page row is looked up once for its key and its value.)
template <typename T, int HD, bool PERM>
struct Swz {
  static HXA_DEV int fk(int row) { return HD == 64 ? (row >> 1) & 7 : row & 15; }
  // PERM (rows modes): 32 lanes read 4 keys x 64 bytes; few rows: 8 keys x 32 bytes
  static HXA_DEV int fv(int row) {
    if (PERM) return HD == 64 ? (row & 2) << 1 : (row & 3) << 2;
    return HD == 64 ? (row & 6) : (row & 7) << 1;
  }
};

// what an item leaves: rows of o, or (part != nullptr) fp32 partials of slot `slot`: part[slot][row][hd] unscaled and
// ml[row][slot] = (maximum in powers of two, sum), row = token Hq + head
template <typename T>
struct Out {
  T *o;
  long ldo;
  float *part;
  float2_t *ml;
  long rows;  // T Hq
  int slot, nslots, Hq;
};

HXA_DEV bool is_minus_0(float x) { return __builtin_bit_cast(uint32_t, x) == 0x80000000u; }

// whether an accumulator of the lanes `mask`, which hold a row together, is NaN
template <typename A, int N>
HXA_DEV bool zero_times_bad(const A (&acc)[N], uint64_t mask) {
  bool bad = false;
#pragma unroll
  for (int d = 0; d < N; d++)
#pragma unroll
    for (int e = 0; e < (int)(sizeof(A) / 4); e++) bad |= acc[d][e] != acc[d][e];
  return (__ballot(bad) & mask) != 0;
}

// rows mode: the wave's accumulators to their rows
template <typename T, int HD, int W>
HXA_DEV void rows_out(const Out<T> &out, const Item &it, int head0, float c, uint8_t *lds, float16_t (&acc)[HD / 32], float m, float l) {
  typedef typename HxaVec<T>::v4 v4;
  typedef typename HxaVec<T>::v8 v8;
  const int tid = this_thread(), lane = tid & 63, wave = tid >> 6;
  const int rw = W == 4 ? wave : wave & 1;
  const bool second = W == 2 && wave >= 2;  // has handed its sums over
  const int g = lane >> 5, ql = lane & 31, r0 = it.r0 + rw * 32;
  if (out.part != nullptr) {
    const int R = r0 + ql;
    if (second || R >= it.nrows) return;
    int rest;
    const int tok = row_tok(it, R, rest);
    const long row = (long)(it.tok0 + tok) * out.Hq + head0 + rest;
    // a sum of 0: scores of -infinity alone (NaN scores give NaN). Their values weigh nothing, but 0 times one that is not finite is NaN: such
    // a partial is kept, under a sum of -0
    const bool kept = l == 0.0f && zero_times_bad(acc, 0x100000001ull << ql);
    if (g == 0) out.ml[row * out.nslots + out.slot] = (float2_t){m == -INFINITY ? m : m * c, kept ? -0.0f : l};
    if (l == 0.0f && !kept) return;
    float *p = out.part + (out.slot * out.rows + row) * HD;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
      for (int e4 = 0; e4 < 4; e4++)
        *(float4_t *)(p + 32 * d + 8 * e4 + 4 * g) =
            (float4_t){acc[d][4 * e4], acc[d][4 * e4 + 1], acc[d][4 * e4 + 2], acc[d][4 * e4 + 3]};
    return;
  }
  // whole rows: staged through LDS, 16-byte chunk c of row r at c ^ sw(r)
  reads_done_barrier();  // every wave is done with the tiles (and the join)
  if (second) return;
  constexpr int RB = HD * 2, CH = HD / 8;
  auto sw = [](int r) { return HD == 64 ? (r >> 1) & 7 : r & 15; };
  uint8_t *stage = lds + rw * 32 * RB;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (l == 0.0f) {  // no key, or scores of -infinity alone: zeros, whatever the values
#pragma unroll
    for (int d = 0; d < HD / 32; d++) acc[d] = (float16_t){};
  }
#pragma unroll
  for (int d = 0; d < HD / 32; d++)
#pragma unroll
    for (int e4 = 0; e4 < 4; e4++) {
      v4 x;
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = (T)(acc[d][4 * e4 + e] * inv);
      *(v4 *)(stage + ql * RB + (((4 * d + e4) ^ sw(ql)) << 4) + 8 * g) = x;
    }
  constexpr int RPP = 64 / CH, N = 32 / RPP;  // rows a pass, passes
  const int u = lane % CH, dt = RPP / it.G, dr = RPP - dt * it.G;  // from a lane's row to its next one
  const int r = lane / CH, left = it.nrows - r0;
  v8 x[N];
#pragma unroll
  for (int n = 0; n < N; n++) x[n] = *(const v8 *)(stage + (r + n * RPP) * RB + ((u ^ sw(r + n * RPP)) << 4));
  int rest;
  const int tok = row_tok(it, r0 + r, rest);
  T *p = out.o + (long)(it.tok0 + tok) * out.ldo + (long)(head0 + rest) * HD + 8 * u;
  const long step = dt * out.ldo + (long)dr * HD, wrap = out.ldo - (long)it.G * HD;
  auto store = [&](auto all) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      if (decltype(all)::value || r + n * RPP < left) *(v8 *)p = x[n];
      rest += dr;
      const bool w = rest >= it.G;
      rest -= w ? it.G : 0;
      p += step + (w ? wrap : 0);
    }
  };
  if (left >= 32) store(std::true_type{});
  else store(std::false_type{});
}

// ---- which rows a block of the grid takes ----
HXA_DEV int wave_scan_i(int v) {  // inclusive
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}
HXA_DEV int max_all(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(v, 63);
}
typedef int int4_t __attribute__((ext_vector_type(4)));
// causal_walk.h's wave: a lane's value is a register, its stash 16 bytes of LDS
struct Wave {
  typedef int I;
  typedef int4_t *Stash;
  static HXA_DEV int lanes(int base) { return base + (threadIdx.x & 63); }
  template <typename F, typename... A>
  static HXA_DEV int map(F f, A... a) { return f(a...); }
  template <typename F>
  static HXA_DEV uint64_t ballot(F f, int a) { return __ballot(f(a)); }
  static HXA_DEV int get(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
  static HXA_DEV int scan(int v) { return wave_scan_i(v); }
  static HXA_DEV int most(int v) { return max_all(v); }
  static HXA_DEV float rcp(float x) { return __builtin_amdgcn_rcpf(x); }
  static HXA_DEV void keep(int4_t *at, int a, int b, int c, int d) { *at = (int4_t){a, b, c, d}; }
  static HXA_DEV void kept(const int4_t *at, int &a, int &b, int &c, int &d) {
    const int4_t x = *at;
    a = x[0], b = x[1], c = x[2], d = x[3];
  }
};

// waves a SIMD: two workgroups a CU, so that one's softmax runs beside the other's matrix products; heads of 256 take the
// registers and LDS of a CU for one
#define HXA_CAUSAL_BOUNDS __launch_bounds__(256, HD == 256 ? 1 : 2)

struct CachedArgs : CachedWork {
  const void *q;
  void *o;
  long ldq, ldo;
  int Hq;
  uint32_t gm, pm;
  float cs;
  float *part;    // nullptr: nothing is split, straight to o
  float2_t *ml;
};
// The work of a workgroup over the cache, key head h: `run` computes each item (mode, item, where its result goes); the keys' places are left in s.
// LDS: bytes of the computation, behind which the stash lies.
template <typename T, int LDS, typename K, typename F>
HXA_DEV void walk_cache(const CachedArgs &p, int h, K &s, uint8_t *lds, F run) {
  const int q = blockIdx.x / p.c.H, P = p.c.prefix_len;
  Walk k{};
  Work w{};
  int4_t *stash = (int4_t *)(lds + LDS) + threadIdx.x;  // the lanes' sequences while a block is computed
  if (p.part == nullptr ? !find_block_of<Wave>(p, q, w) : !first_work<Wave>(p, q, stash, k, w)) return;
  for (;;) {
    s.prefix = p.c.prefix;
    s.table = p.c.table;
    s.P = P;
    s.page = p.c.page;
    s.pm = p.pm;
    s.npages = p.c.npages;
    s.H = p.c.H;
    s.h = h;
    Item it;
    it.G = p.G;
    it.gm = p.gm;
    int mode, slot_end;
    if (w.shared) {
      mode = p.p.np_mode;
      it.r0 = w.block * mode_rows(mode);
      it.nrows = p.T * p.G;
      it.tok0 = 0;
      it.x0 = w.t0 * KT;
      it.x1 = min(w.t1 * KT, P);
      it.base = it.cap = it.least = P - 1;
      it.causal = false;
      slot_end = p.p.sp_max;
    } else {
      const long len = w.len;
      const int held = (int)min(max(len, 0L), (long)p.c.ldt * p.c.page);
      s.table += (long)w.seq * p.c.ldt;
      it.r0 = w.block << p.p.rb_log;
      it.nrows = w.n * p.G;
      mode = rows_mode(min(it.nrows - it.r0, 1 << p.p.rb_log));
      it.tok0 = w.b;
      // own position of token j: len - n + j; a negative one sees the prefix alone
      it.causal = true;
      it.cap = P + held - 1;
      it.least = P - 1;
      const long base = (long)P + len - w.n;
      it.base = (int)max(min(base, (long)it.cap), (long)P - 1 - w.n);
      const int end = row_limit(it, min(it.r0 + mode_rows(mode), it.nrows) - 1) + 1;
      it.x0 = p.p.x_first + w.t0 * KT;
      it.x1 = (int)min((long)end, p.p.x_first + (long)w.t1 * KT);
      slot_end = p.p.sp_max + p.p.s_max;
    }
    const bool none = p.part != nullptr && !w.shared && it.x1 <= it.x0;  // a piece that ends before the block's first tile
    if (p.part != nullptr && (w.last || none)) {  // slots that no range fills: sums of nothing
      const int rows = min(mode_rows(mode), it.nrows - it.r0);
      const int from = none ? w.slot : w.slot + 1, free = (w.last ? slot_end : w.slot + 1) - from;
      for (int j = threadIdx.x; j < rows * free; j += 256) {
        int head;
        const int row = j / free, tok = row_tok(it, it.r0 + row, head);
        p.ml[((long)(it.tok0 + tok) * p.Hq + h * p.G + head) * (p.p.sp_max + p.p.s_max) + from + j - row * free] = (float2_t){-INFINITY, 0.0f};
      }
    }
    if (!none) run(mode, it, Out<T>{(T *)p.o, p.ldo, p.part, p.ml, (long)p.T * p.Hq, w.slot, p.p.sp_max + p.p.s_max, p.Hq});
    if (k.pos >= k.end) return;
    reads_done_barrier();  // every wave is done with the LDS
    if (!further_work<Wave>(p, k, stash, w)) return;
  }
}

// The partials of a row joined by a wave: lane s has the maximum and the sum of slot s (at most 64 of them), which give its weight
// 2^(m_s - m); then HD / 64 dims a lane over the slots that saw a key, eight of them in flight; one division, one rounding. A slot whose
// sum is +0 saw none and holds no values; one whose sum is -0 holds NaN where it has weights of 0 on values that are not finite. (64 tokens of 32 heads with 32 + 24 slots, a third of them used: 5 us; with the slots'
// sums strided by rows and shared by 8 groups of lanes 8.8.)
template <typename T, int HD>
__global__ __launch_bounds__(256) void cached_merge_kernel(CachedArgs p) {
  constexpr int E = HD / 64, N = 8;
  typedef float fe __attribute__((ext_vector_type(E)));
  const int lane = threadIdx.x & 63, nslots = p.p.sp_max + p.p.s_max;
  const uint32_t row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), rows = (uint32_t)p.T * p.Hq;
  if (row >= rows) return;
  const int tok = (int)(row / (uint32_t)p.Hq), head = (int)(row - (uint32_t)tok * p.Hq);
  if (tok < p.c.cu[0] || tok >= p.c.cu[p.c.nseq]) return;
  const float2_t x = lane < nslots ? p.ml[(long)row * nslots + lane] : (float2_t){-INFINITY, 0.0f};
  float m = x[0];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float w = x[1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x[0] - (m == -INFINITY ? 0.0f : m));
  const float l = wave_sum(x[1] * w);
  uint64_t left = __ballot(x[1] != 0.0f || is_minus_0(x[1]));
  fe o = {};
  while (left) {
    fe y[N];
    float a[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
      y[j] = (fe){};
      a[j] = 0.0f;
      if (left) {
        const int s = __builtin_ctzll(left);
        left &= left - 1;
        y[j] = *(const fe *)(p.part + ((long)s * rows + row) * HD + E * lane);
        a[j] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s));
      }
    }
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
      for (int e = 0; e < E; e++) o[e] += y[j][e] * a[j];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  typedef T te __attribute__((ext_vector_type(E)));
  te z;
#pragma unroll
  for (int e = 0; e < E; e++) z[e] = l == 0.0f ? (T)0.0f : (T)(o[e] * inv);
  *(te *)((T *)p.o + tok * p.ldo + (long)head * HD + E * lane) = z;
}

int causal_ncu() {
  static const int ncu = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
      return 256;
    return n;
  }();
  return ncu;
}

// kernels that take more than 64 KB of LDS: allowed once a device
int allow_lds(const void *f, int bytes, int id) {
  static std::mutex mu;
  static uint32_t done[HXA_MAX_DEVICES];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= HXA_MAX_DEVICES) return HXA_E_RESOURCE;
  std::lock_guard<std::mutex> lk(mu);
  if (done[dev] >> id & 1) return HXA_OK;
  if (hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return HXA_E_HIP;
  done[dev] |= 1u << id;
  return HXA_OK;
}
// runs f with the kernel's types: f.template operator()<T, HD>(an index below 6)
template <typename F>
int by_type(int dtype, int hd, F f) {
  if (dtype == HXA_DT_F16) {
    if (hd == 64) return f(hxa_h{}, std::integral_constant<int, 64>{}, 0);
    if (hd == 128) return f(hxa_h{}, std::integral_constant<int, 128>{}, 1);
    return f(hxa_h{}, std::integral_constant<int, 256>{}, 2);
  }
  if (hd == 64) return f(hxa_b{}, std::integral_constant<int, 64>{}, 3);
  if (hd == 128) return f(hxa_b{}, std::integral_constant<int, 128>{}, 4);
  return f(hxa_b{}, std::integral_constant<int, 256>{}, 5);
}
int launched(const char *who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HXA_OK : hxa_set_error(HXA_E_HIP, "%s: %s", who, hipGetErrorString(e));
}
bool rows_ok(const void *p, long ld, int H, int hd) { return p != nullptr && (uintptr_t)p % 16 == 0 && ld % 8 == 0 && ld >= (long)H * hd; }

uint32_t recip(int G) { return G == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / (uint32_t)G); }

// workgroups that run at once
int wg_slots(int hd) { return causal_ncu() * (hd == 256 ? 1 : 2); }

// ---- a call over the cache, host side ----
int cached_limits(const hxa_kv_cache &c, int T, int Hq, const char *who) {
  if (Hq <= 0 || Hq > HXA_MAX_HEADS || Hq % c.H || (long)T * Hq >= 1L << 30)
    return hxa_set_error(HXA_E_ARG, "%s: T=%d Hq=%d H=%d", who, T, Hq, c.H);
  // grids of fewer than 2^24 workgroups; the join's waves, one for each of T Hq rows, are fewer than 2^26 where there is one
  const long RT = (long)T * (Hq / c.H);
  if ((RT / 64 + c.nseq) * c.H >= 1L << 21)
    return hxa_set_error(HXA_E_ARG, "%s: T=%d nseq=%d H=%d are too many blocks", who, T, c.nseq, c.H);
  return HXA_OK;
}
// the call, after its checks of the cache; f gives the kernel of a type and head width, its bytes of LDS, and 0 or, for a second kernel of the same type
// and width, 6
template <typename A, typename F>
int cached_call(A &p, const hxa_kv_cache &c, const void *q, long ldq, void *o, long ldo, int T, int Hq, float scale, void *ws, long ws_bytes,
                hipStream_t st, const char *who, bool q8, F f) {
  if (!(scale > 0.0f) || !std::isfinite(scale)) return hxa_set_error(HXA_E_ARG, "%s: scale %g", who, (double)scale);
  if (T == 0 || c.nseq == 0) return HXA_OK;
  if (!rows_ok(q, ldq, Hq, c.hd) || !rows_ok(o, ldo, Hq, c.hd))
    return hxa_set_error(HXA_E_ARG, "%s: pointers null or not 16-byte aligned, or strides (%ld %ld)", who, ldq, ldo);
  if ((uintptr_t)ws % 16) return hxa_set_error(HXA_E_ARG, "%s: workspace not aligned", who);
  CachedPlan pl = cached_plan(c, T, Hq, true, wg_slots(c.hd), q8);
  const long need = cached_ws(pl, c, T, Hq);
  if (need > 0 && (ws == nullptr || ws_bytes < need)) pl = cached_plan(c, T, Hq, false, wg_slots(c.hd), q8);
  const int nslots = pl.sp_max + pl.s_max;
  static_cast<CachedArgs &>(p) = CachedArgs{{c, T, Hq / c.H, pl}, q, o, ldq, ldo, Hq, recip(Hq / c.H), recip(c.page), scale * L2E, nullptr, nullptr};
  if (nslots > 1) {
    p.part = (float *)ws;
    p.ml = (float2_t *)(p.part + (long)nslots * T * Hq * c.hd);
  }
  const long wgs = cached_items(pl) * c.H;
  return by_type(c.dtype, c.hd, [&](auto ty, auto hdc, int id) -> int {
    const auto [k, lds, more] = f(ty, hdc, pl, c);
    const int a = allow_lds((const void *)k, lds, 12 + id + more);
    if (a != HXA_OK) return hxa_set_error(a, "%s: %d bytes of LDS", who, lds);
    hxa_launch(k, dim3((unsigned)wgs), dim3(256), lds, st, p);
    if (nslots > 1)
      hxa_launch(cached_merge_kernel<decltype(ty), decltype(hdc)::value>, dim3((unsigned)ceil_div((long)T * Hq, 4)), dim3(256), 0, st,
                 static_cast<const CachedArgs &>(p));
    return launched(who);
  });
}

}  // namespace
