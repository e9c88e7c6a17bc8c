// Attention of new tokens over a paged cache of int8 with a scale for each page and head (hxa_attention_cached_q8): queries and results in fp16 / bf16,
// heads of 64, 128 or 256, grouped heads, a prefix that the batch shares. Rows, work items and modes are those of causal_attn.hip.
//
// With k = ks qk and v = vs qv (qk, qv the bytes, ks, vs the scales of their pages), in powers of two and with c = scale log2(e):
//   t_j = (q . qk_j) (c ks_j) + log2(vs_j),   w_j = 2^(t_j - m),   o = sum w_j qv_j / sum w_j / vs_j
// The values' scale is folded into the exponent, so that one running maximum m bounds what is rounded to fp16, the weight as it stands before its
// byte: a key whose page has small values loses no bits to one whose page has large ones, and the products take the bytes as they are. A byte is exact
// in fp16. q in bf16 is brought to fp16 by a power of two of its row, whose largest value it puts near 2^14: the row's values down to 2^-28 of that stay exact.
// t, m, both sums and O are held in fp32; the denominator adds the weights before they are rounded.
//
// Tiles of 64 keys go through registers: loaded while the tile before them is computed, then turned into fp16 rows in LDS once for all four
// waves. A byte is finite whatever it holds, so that a masked key needs nothing but a weight of 0.
#include "causal_attn.h"
#include "int8_rows.h"

namespace {

struct KeysQ8 : Keys<int8_t> {
  const float *ks, *vs;
};

template <int HD>
struct GeoQ8 {
  static constexpr int RB = HD * 2, TB = KT * RB;     // bytes of an fp16 row, of a tile
  static constexpr int CST = 2 * TB;                  // c ks, log2 vs and 1 / vs of the tile's keys
  static constexpr int LDS = 2 * TB + 2048;
  static constexpr int CH = HD / 16, N = KT * CH / 256;  // 16-byte chunks of a row of bytes; loads a thread, for K and for V each
};

// four bytes to fp16: u = q + 128 under the exponent of 1024 is 1024 + u
HXA_DEV uint2_t q8_halves(uint32_t d) {
  const uint32_t x = d ^ 0x80808080u;
  const half2_t c = {(hxa_h)1152.0f, (hxa_h)1152.0f};
  return (uint2_t){__builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - c),
                   __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - c)};
}

// The tiles of a work item: row (PERM ? krow_key(j) : j) of LDS holds key j, in the orders of Swz
template <int HD, bool PERM>
struct LoaderQ8 {
  typedef GeoQ8<HD> G_;
  typedef Swz<hxa_h, HD, PERM> S_;
  const KeysQ8 &s;
  const Item &it;
  uint8_t *lds;
  const float c;
  int tid, lane;
  int ent;
  unsigned in_page;
  uint4_t raw[2][G_::N];
  float ks, vs;  // of this lane's key
  HXA_DEV LoaderQ8(const KeysQ8 &s_, const Item &it_, uint8_t *lds_, float c_, int tid_)
      : s(s_), it(it_), lds(lds_), c(c_), tid(tid_), lane(tid_ & 63), ent(-1), in_page(0) {
    entry(0);
  }
  HXA_DEV void entry(int i) {  // the page of this lane's key of tile i
    const int x = it.x0 + i * KT + lane;
    ent = -1;
    if (x < it.x1) {
      const bool pre = x < s.P;
      const unsigned y = pre ? x : x - s.P;
      ent = (pre ? s.prefix : s.table)[s.slot(y, in_page)];
    }
  }
  // begins the loads of tile i; the mask of its keys that are there
  HXA_DEV uint64_t open(int i) {
    const bool ok = (unsigned)ent < (unsigned)s.npages;  // (-1 past x1)
    const uint32_t ph = ok ? (uint32_t)ent * s.H + s.h : 0;
    const uint32_t at = ok ? ph * s.page + in_page : 0;  // < 2^32: checked on the host
    const uint64_t mask = __ballot(ok);
    ks = ok ? s.ks[ph] : 0.0f;
    vs = ok ? s.vs[ph] : 0.0f;
    if (it.x0 + i * KT + KT < it.x1) entry(i + 1);
#pragma unroll
    for (int n = 0; n < G_::N; n++) {
      const int u = n * 256 + tid, key = u / G_::CH, ch = u % G_::CH;
      const uint64_t row = (uint64_t)(uint32_t)__shfl((int)at, key) * HD + ch * 16;
      raw[0][n] = *(const uint4_t *)(s.k + row);
      raw[1][n] = *(const uint4_t *)(s.v + row);
    }
    return mask;
  }
  // the tile opened last into LDS
  HXA_DEV void store() {
    const uint64_t zero = __ballot(!(vs > HXA_Q8_LEAST && vs < INFINITY));
    if (zero) {  // keys without a scale (or without a page): values of 0, whatever the bytes
#pragma unroll
      for (int n = 0; n < G_::N; n++)
        if ((zero >> ((n * 256 + tid) / G_::CH)) & 1) raw[1][n] = (uint4_t){0, 0, 0, 0};
    }
#pragma unroll
    for (int n = 0; n < G_::N; n++) {
      const int u = n * 256 + tid, key = u / G_::CH, ch = u % G_::CH;
      const int row = PERM ? krow_key(key) : key;  // (krow_key is its own inverse)
#pragma unroll
      for (int V = 0; V < 2; V++) {
        uint8_t *to = lds + V * G_::TB + row * G_::RB;
        const int f = V ? S_::fv(row) : S_::fk(row);
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint2_t a = q8_halves(raw[V][n][2 * e]), b = q8_halves(raw[V][n][2 * e + 1]);
          *(uint4_t *)(to + (((2 * ch + e) ^ f) << 4)) = (uint4_t){a.x, a.y, b.x, b.y};
        }
      }
    }
    if (tid < 64) {
      float *cst = (float *)(lds + G_::CST);
      const float a = ks > 0.0f && ks < INFINITY ? ks : 0.0f;
      const float b = vs > HXA_Q8_LEAST && vs < INFINITY ? vs : HXA_Q8_LEAST;
      cst[lane] = a * c;
      cst[64 + lane] = __builtin_amdgcn_logf(b);
      cst[128 + lane] = 1.0f / b;
    }
  }
};

// q's eight values as fp16; bf16: times a power of two, whose inverse the caller keeps
HXA_DEV half8_t q_halves(half8_t q, float) { return q; }
HXA_DEV half8_t q_halves(bf8_t q, float f) {
  half8_t r;
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = (hxa_h)((float)q[e] * f);
  return r;
}
// 2^(14 - e) for a row whose largest magnitude is 2^e .. 2^(e + 1); 1 for one of zeros, and where it is not finite
HXA_DEV float row_factor(float top) {
  const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
  return top >= 0x1p-100f && top < INFINITY ? __builtin_bit_cast(float, (uint32_t)(127 + 14 - e) << 23) : 1.0f;
}
template <typename V, int N>
HXA_DEV float most_of(const V (&q)[N]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf((float)q[i][e]));
  return m;
}

// ---- rows modes: as causal_attn.hip's rows_item; m and the sums in powers of two ----
template <typename T, int HD, int W>
HXA_DEV void rows_item_q8(const KeysQ8 &s, const Item &it, const T *q, long ldq, int head0, float c, uint8_t *lds, float16_t (&acc)[HD / 32],
                          float &mrun, float &lsum) {
  typedef GeoQ8<HD> G_;
  typedef typename HxaVec<T>::v8 v8;
  typedef Swz<hxa_h, HD, true> S_;
  constexpr bool BF = std::is_same<T, hxa_b>::value;
  constexpr int NB = W == 4 ? 2 : 1;
  constexpr int ND = HD / 32, AK = 2, AV = 3;
  const int tid = this_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = W == 4 ? wave : wave & 1, kh = W == 4 ? 0 : wave >> 1;
  const int g = lane >> 5, ql = lane & 31;

  const int R = it.r0 + rw * 32 + ql;
  const bool qok = R < it.nrows;
  const int Rc = qok ? R : it.nrows - 1;
  int rest;
  const int tok = row_tok(it, Rc, rest);
  const T *qp = q + (long)(it.tok0 + tok) * ldq + (long)(head0 + rest) * HD;
  half8_t qf[HD / 16];
  float back = 1.0f;  // what q was divided by
  {
    v8 raw[HD / 16];
#pragma unroll
    for (int i = 0; i < HD / 16; i++) raw[i] = *(const v8 *)(qp + i * 16 + 8 * g);
    float f = 1.0f;
    if (BF) {
      float lo, hi;
      halves(most_of(raw), lo, hi);
      f = row_factor(fmaxf(lo, hi));
      back = 1.0f / f;
    }
#pragma unroll
    for (int i = 0; i < HD / 16; i++) qf[i] = q_halves(raw[i], f);
  }
  const int lim = tok_limit(it, tok);
  const int last = it.nrows - 1;
  const int lim_min = row_limit(it, it.r0);
  const int wave_max = it.r0 + rw * 32 <= last ? row_limit(it, min(it.r0 + rw * 32 + 31, last)) : -1;

#pragma unroll
  for (int d = 0; d < ND; d++) acc[d] = (float16_t){};
  mrun = -INFINITY;
  lsum = 0.0f;
  const int nt = (it.x1 - it.x0 + KT - 1) / KT;
  if (nt <= 0) return;
  LoaderQ8<HD, true> ld(s, it, lds, c, tid);
  uint64_t km_next = ld.open(0);

  const int vrow = 4 * g + ((lane & 15) >> 2);
  const int vlow = ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) << 4) + (lane & 1) * 8;
  uint32_t vat[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) vat[d] = vrow * G_::RB + (((d << 2) ^ S_::fv(vrow)) << 4) + vlow;
  const uint8_t *kb = lds, *vb = lds + G_::TB;
  const float *cst = (const float *)(lds + G_::CST) + 32 * kh + 8 * g;
  auto kfrag = [&](int ds, int b) {
    const int row = (b + kh) * 32 + ql, ch = 2 * ds + g;
    return *(const half8_t *)(kb + row * G_::RB + ((ch ^ S_::fk(row)) << 4));
  };
  auto vfrag = [&](int n) {
    const uint8_t *at = vb + vat[n % ND] + (kh * 32 + n / ND * 16) * G_::RB;
    return __builtin_shufflevector(read_tr<half4_t>(at), read_tr<half4_t>(at + 8 * G_::RB), 0, 1, 2, 3, 4, 5, 6, 7);
  };

  for (int i = 0; i < nt; i++) {
    reads_done_barrier();  // every wave is done with tile i - 1
    ld.store();
    const uint64_t km = km_next;
    const int key0 = it.x0 + i * KT;
    if (i + 1 < nt) km_next = ld.open(i + 1);
    reads_done_barrier();  // tile i is in LDS
    if (key0 + 32 * kh > wave_max) continue;  // no row of this wave sees it
    const bool cut = km != ~0ull || key0 + KT - 1 > lim_min;
    float16_t S[NB];
    half8_t kf[AK + 1][NB];
#pragma unroll
    for (int ds = 0; ds < AK; ds++)
#pragma unroll
      for (int b = 0; b < NB; b++) kf[ds][b] = kfrag(ds, b);
#pragma unroll
    for (int ds = 0; ds < HD / 16; ds++) {
      __builtin_amdgcn_sched_barrier(0);
      if (ds + AK < HD / 16) {
#pragma unroll
        for (int b = 0; b < NB; b++) kf[(ds + AK) % (AK + 1)][b] = kfrag(ds + AK, b);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < NB; b++) S[b] = mma32(kf[ds % (AK + 1)][b], qf[ds], ds == 0 ? (float16_t){} : S[b]);
    }
    __builtin_amdgcn_sched_barrier(0);
    half8_t vf[AV + 1];
#pragma unroll
    for (int n = 0; n < AV; n++) vf[n] = vfrag(n);
    // scores to exponents: 8 keys of a lane lie side by side
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const float *at = cst + 32 * b + 16 * (r >> 3) + (r & 7);
        const float4_t k = *(const float4_t *)at, lv = *(const float4_t *)(at + 64);
#pragma unroll
        for (int e = 0; e < 4; e++) S[b][r + e] = fmaf(BF ? S[b][r + e] * back : S[b][r + e], k[e], lv[e]);
      }
    if (cut) {
      const int n = lim - key0 - 32 * kh - 8 * g;
      const uint64_t see = km >> (32 * kh + 8 * g);
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int k = 32 * b + 16 * (r >> 3) + (r & 7);
          if (k > n || !((see >> k) & 1)) S[b][r] = -INFINITY;
        }
    }
    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int r = 0; r < 16; r++) m4[r & 3] = fmaxf(m4[r & 3], S[b][r]);
    float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
    {
      float lo, hi;
      halves(mt, lo, hi);
      mt = fmaxf(lo, hi);
    }
    const bool need = mt - mrun > RESCALE2;  // also when mrun is still -inf
    if (__any(need)) {
      const float alpha = need ? __builtin_amdgcn_exp2f(mrun - mt) : 1.0f;
      if (need) mrun = mt;
      lsum *= alpha;
#pragma unroll
      for (int d = 0; d < ND; d++) acc[d] *= alpha;
    }
    const float mb = mrun == -INFINITY ? 0.0f : mrun;
    half8_t pf[NB][2];
    float ls[2] = {0.0f, 0.0f};
    auto expo2 = [&](int n) {
      const float2_t inv = *(const float2_t *)(cst + 128 + 32 * (n >> 4) + 16 * ((n >> 3) & 1) + (n & 7));
      const float p0 = __builtin_amdgcn_exp2f(S[n >> 4][n & 15] - mb);
      const float p1 = __builtin_amdgcn_exp2f(S[n >> 4][(n & 15) + 1] - mb);
      pf[n >> 4][(n >> 3) & 1][n & 7] = (hxa_h)p0;
      pf[n >> 4][(n >> 3) & 1][(n & 7) + 1] = (hxa_h)p1;
      ls[(n >> 1) & 1] = fmaf(p1, inv[1], fmaf(p0, inv[0], ls[(n >> 1) & 1]));
    };
#pragma unroll
    for (int n = 0; n < 16; n += 2) expo2(n);
#pragma unroll
    for (int n = 0; n < 2 * NB * ND; n++) {
      if (n + AV < 2 * NB * ND) vf[(n + AV) % (AV + 1)] = vfrag(n + AV);
      acc[n % ND] = mma32(vf[n % (AV + 1)], pf[n / (2 * ND)][n / ND & 1], acc[n % ND]);
      if (NB == 2 && n < 2 * ND && (ND < 8 || n % 2 == 0)) {
#pragma unroll
        for (int e = 0; e < (ND < 8 ? 8 / ND : 2); e += 2) expo2(16 + n * 8 / ND + e);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    lsum += ls[0] + ls[1];
  }
  {
    float lo, hi;
    halves(lsum, lo, hi);
    lsum = lo + hi;
  }
  if constexpr (W == 2) {  // join the halves of the keys
    constexpr int PART = HD / 8 * 64;
    reads_done_barrier();
    float4_t *ox = (float4_t *)lds + rw * PART;
    float *ml = (float *)((float4_t *)lds + W * PART) + rw * 128;
    if (kh == 1) {
#pragma unroll
      for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++)
          ox[(d * 4 + e4) * 64 + lane] = (float4_t){acc[d][4 * e4], acc[d][4 * e4 + 1], acc[d][4 * e4 + 2], acc[d][4 * e4 + 3]};
      ml[lane] = mrun;
      ml[64 + lane] = lsum;
    }
    reads_done_barrier();
    if (kh == 0) {
      const float m1 = ml[lane], l1 = ml[64 + lane], m = fmaxf(mrun, m1);
      const float mz = m == -INFINITY ? 0.0f : m;
      const float a0 = __builtin_amdgcn_exp2f(mrun - mz), a1 = __builtin_amdgcn_exp2f(m1 - mz);
      lsum = lsum * a0 + l1 * a1;
      mrun = m;
#pragma unroll
      for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++) {
          const float4_t o = ox[(d * 4 + e4) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; e++) acc[d][4 * e4 + e] = acc[d][4 * e4 + e] * a0 + o[e] * a1;
        }
    }
  }
}

// ---- few rows: 16 rows, each wave 16 keys of every tile ----
// Bound by reading the cache, so the tiles stay bytes until a wave needs its part of one: they go from memory straight into a ring of NS of them in LDS
// (global_load_lds), NS - 1 ahead, one barrier a tile, and a wave turns its own 16 keys into fp16 fragments. What the addresses need, a page's place and its scales, is in LDS as well, for 512 pages at a time: a load of it inside the loop would
// be waited for with all those behind it.
//
// LDS row 4 b + a of a wave's 16 holds key 4 a + b. K: a lane takes 16 bytes of its key, two slices of 8 dims; q's dims follow that order. V: dword u of
// keys 4 gi .. + 3 is dims 4 u .. + 3 of four keys, transposed by byte permutations: product j of a 64-dim group has dims 4 u + j. Chunks are swizzled
// so that the lanes of either read spread over the banks.
template <int HD>
struct FewQ8 {
  static constexpr int NS = HD == 64 ? 6 : 4, TB = KT * HD;  // tiles in the ring; bytes of a tile of K, or of V
  static constexpr int CH = HD / 16, RPL = 64 / CH;           // 16-byte chunks a row, rows of one wave-wide load
  static constexpr int NLD = HD / 64;                         // loads a wave and tile, for K and for V each
  static constexpr int PAGES = 512, TABLE = NS * 2 * TB;      // the pages' table, past the ring
  static constexpr int LDS = TABLE + PAGES * 16 + 16;
  static HXA_DEV int fk(int row) { return HD == 64 ? (row >> 2) & 3 : HD == 128 ? (row >> 1) & 7 : row & 15; }
  static HXA_DEV int fv(int row) { return HD == 64 ? 0 : HD == 128 ? (row << 1) & 4 : (row & 3) << 2; }
};
// row of LDS <-> key, within 16 (its own inverse)
HXA_DEV int few_row(int key) { return (key & ~15) | (key & 3) << 2 | (key >> 2 & 3); }

// The pages of keys x from `x0` on, PAGES of them: place in the pools (npages H page rows; ~0: not there) and scales
template <int HD>
struct PagesQ8 {
  const KeysQ8 &s;
  uint32_t *ph;
  float *ks, *lv, *iv;
  int first, own;  // entry of page slot n of the prefix: n - first, of the sequence: n + own
  HXA_DEV PagesQ8(const KeysQ8 &s_, uint8_t *lds) : s(s_), first(0), own(0) {
    ph = (uint32_t *)(lds + FewQ8<HD>::TABLE);
    ks = (float *)(ph + FewQ8<HD>::PAGES);
    lv = ks + FewQ8<HD>::PAGES;
    iv = lv + FewQ8<HD>::PAGES;
  }
  HXA_DEV int entry(int x, unsigned &in_page) const {
    const bool pre = x < s.P;
    return (int)s.slot(pre ? x : x - s.P, in_page) + (pre ? -first : own);
  }
  // whole workgroup, between barriers; whether a page of [x0, x1) is not there (in the words behind the table, once the workgroup has met)
  HXA_DEV void fill(int x0, int x1, float c, int tid) {
    constexpr int N = FewQ8<HD>::PAGES;
    unsigned in;
    int npre = 0;
    if (x0 < s.P) {
      first = (int)s.slot(x0, in);
      npre = (int)s.slot(s.P - 1, in) - first + 1;
      own = npre;
    } else {
      own = -(int)s.slot(x0 - s.P, in);
    }
    const int own_end = x1 > s.P ? (int)s.slot(x1 - 1 - s.P, in) + 1 + own : npre;  // entries of the sequence's pages end here
    const int pre_end = x1 > s.P ? npre : x1 > x0 ? (int)s.slot(x1 - 1, in) - first + 1 : 0;
    bool hole = false;
#pragma unroll
    for (int k = 0; k < N / 256; k++) {
      const int j = k * 256 + tid;
      const bool pre = j < npre, there = j < (pre ? pre_end : own_end);
      const int e = there ? (pre ? s.prefix[first + j] : s.table[j - own]) : -1;
      const bool ok = (unsigned)e < (unsigned)s.npages;
      hole |= there && !ok;
      const uint32_t at = ok ? (uint32_t)e * s.H + s.h : 0;
      const float a = ok ? s.ks[at] : 0.0f, b = ok ? s.vs[at] : 0.0f;
      const bool vok = b > HXA_Q8_LEAST && b < INFINITY;
      ph[j] = ok ? at : ~0u;
      ks[j] = a > 0.0f && a < INFINITY ? a * c : 0.0f;
      lv[j] = vok ? __builtin_amdgcn_logf(b) : -64.0f;
      iv[j] = vok ? 1.0f / b : 1.0f / HXA_Q8_LEAST;
    }
    int *flag = (int *)(iv + N);
    const bool any = __any(hole);
    if ((tid & 63) == 0) flag[tid >> 6] = any;
  }
  HXA_DEV bool holes() const {
    const int *flag = (const int *)(iv + FewQ8<HD>::PAGES);
    return (flag[0] | flag[1] | flag[2] | flag[3]) != 0;
  }
};

template <typename T, int HD>
HXA_DEV void few_item_q8(const KeysQ8 &s, const Item &it, const T *q, long ldq, int head0, float c, uint8_t *lds, const Out<T> &out) {
  typedef FewQ8<HD> F;
  typedef typename HxaVec<T>::v8 v8;
  typedef typename HxaVec<T>::v4 v4;
  constexpr bool BF = std::is_same<T, hxa_b>::value;
  constexpr int NG = HD / 64, NS = F::NS;  // groups of 64 dims
  const int tid = this_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int gi = lane >> 4, ql = lane & 15;
  const int R = it.r0 + ql, last = it.nrows - 1, Rc = min(R, last);
  float4_t acc[NG][4];
#pragma unroll
  for (int g = 0; g < NG; g++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[g][j] = (float4_t){};
  float mrun = -INFINITY, lsum = 0.0f;
  const int nt = (it.x1 - it.x0 + KT - 1) / KT;
  if (nt > 0) {
    PagesQ8<HD> pages(s, lds);
    // q: dims 16 (4 d + gi) + 8 e .. + 7 in qf[d][e]
    int rest;
    const int tok = row_tok(it, Rc, rest);
    const T *qp = q + (long)(it.tok0 + tok) * ldq + (long)(head0 + rest) * HD;
    half8_t qf[NG][2];
    float back = 1.0f;
    {
      v8 raw[2 * NG];
#pragma unroll
      for (int i = 0; i < 2 * NG; i++) raw[i] = *(const v8 *)(qp + 16 * (4 * (i >> 1) + gi) + 8 * (i & 1));
      float f = 1.0f;
      if (BF) {
        f = row_factor(max16(most_of(raw)));
        back = 1.0f / f;
      }
#pragma unroll
      for (int i = 0; i < 2 * NG; i++) qf[i >> 1][i & 1] = q_halves(raw[i], f);
    }
    const int lim = tok_limit(it, tok), lim_min = row_limit(it, it.r0);
    const bool four = ((s.page | s.P) & 3) == 0;  // keys 4 gi .. + 3 lie on one page
    uint32_t koff[F::NLD], voff[F::NLD], key_of[F::NLD];
#pragma unroll
    for (int n = 0; n < F::NLD; n++) {
      const int row = (n * 4 + wave) * F::RPL + lane / F::CH, ch = lane % F::CH;
      key_of[n] = few_row(row);
      koff[n] = (uint32_t)((ch ^ F::fk(row)) << 4);
      voff[n] = (uint32_t)((ch ^ F::fv(row)) << 4);
    }
    const int krow = 16 * wave + few_row(ql);
    const uint8_t *kat = lds + krow * HD, *vat = lds + F::TB + (16 * wave + gi) * HD;  // keys 4 gi + e: rows 16 w + 4 e + gi
    uint32_t vch[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) vch[g] = (uint32_t)((((4 * g + (ql >> 2)) ^ F::fv(gi)) << 4) + (ql & 3) * 4);
    const int kstep = it.x0 + 16 * wave + 4 * gi;

    // loads of tile i into its place of the ring
    auto load = [&](int i) {
      const int x = it.x0 + i * KT + lane;
      uint32_t at = 0;
      if (x < it.x1) {
        unsigned in;
        const uint32_t p = pages.ph[pages.entry(x, in)];
        at = p == ~0u ? 0 : p * s.page + in;  // < 2^32: checked on the host
      }
      uint8_t *to = lds + (i % NS) * 2 * F::TB + wave * 1024;
#pragma unroll
      for (int n = 0; n < F::NLD; n++) {
        const uint64_t row = (uint64_t)(uint32_t)__shfl((int)at, (int)key_of[n]) * HD;
        g2l16_opaque((const uint8_t *)s.k + row + koff[n], to + n * 4096);
        g2l16_opaque((const uint8_t *)s.v + row + voff[n], to + F::TB + n * 4096);
      }
    };
    for (int t0 = 0; t0 < nt;) {
      // the pages from tile t0 on, and how many tiles they reach
      if (t0 > 0) reads_done_barrier();
      pages.fill(it.x0 + t0 * KT, it.x1, c, tid);
      reads_done_barrier();
      const bool holes = pages.holes();
      int t1 = nt;
      {
        unsigned in;
        // (an entry is a page of one key at least)
        while (pages.entry(min(it.x0 + t1 * KT, it.x1) - 1, in) >= F::PAGES) {
          const int over = pages.entry(min(it.x0 + t1 * KT, it.x1) - 1, in) - F::PAGES + 1;
          t1 -= max(1, (int)min((long)(over - 1) * s.page / KT, (long)t1 - t0 - 1));
        }
      }
#pragma unroll
      for (int i = 0; i < NS - 1; i++)
        if (t0 + i < t1) load(t0 + i);
      for (int i = t0; i < t1; i++) {
        // tile i has landed: the loads of the `newer` tiles behind it may still fly
        const int newer = min(NS - 2, t1 - 1 - i);
        constexpr int L = 2 * F::NLD;
        if (newer >= NS - 2) wait_vm<(NS - 2) * L>();
        else if (newer == 3) wait_vm<(NS > 5 ? 3 * L : 0)>();
        else if (newer == 2) wait_vm<(NS > 4 ? 2 * L : 0)>();
        else if (newer == 1) wait_vm<L>();
        else wait_vm<0>();
        reads_done_barrier();  // for every wave; and every wave is done with tile i - 1
        if (i + NS - 1 < t1) load(i + NS - 1);
        const int at = (i % NS) * 2 * F::TB;
        float4_t S = {};
#pragma unroll
        for (int d = 0; d < NG; d++) {
          const uint4_t w = *(const uint4_t *)(kat + at + (((4 * d + gi) ^ F::fk(krow)) << 4));
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint2_t a = q8_halves(w[2 * e]), b = q8_halves(w[2 * e + 1]);
            S = mma16(__builtin_bit_cast(half8_t, (uint4_t){a.x, a.y, b.x, b.y}), qf[d][e], S);
          }
        }
        const int x = kstep + i * KT;
        float4_t k, lv, iv;
        unsigned in;
        if (four) {
          const int p = min(pages.entry(min(x, it.x1 - 1), in), F::PAGES - 1);
          k = pages.ks[p];
          lv = pages.lv[p];
          iv = pages.iv[p];
        } else {
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const int p = min(pages.entry(min(x + r, it.x1 - 1), in), F::PAGES - 1);
            k[r] = pages.ks[p];
            lv[r] = pages.lv[p];
            iv[r] = pages.iv[p];
          }
        }
#pragma unroll
        for (int r = 0; r < 4; r++) S[r] = fmaf(BF ? S[r] * back : S[r], k[r], lv[r]);
        if (it.x0 + i * KT + KT - 1 > lim_min) {  // (a row's limit hides what lies past x1 too)
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (x + r > lim || x + r >= it.x1) S[r] = -INFINITY;
        }
        if (holes) {
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (pages.ph[min(pages.entry(min(x + r, it.x1 - 1), in), F::PAGES - 1)] == ~0u) S[r] = -INFINITY;
        }
        const float mt = max16(fmaxf(fmaxf(S[0], S[1]), fmaxf(S[2], S[3])));
        const bool need = mt - mrun > RESCALE2;
        if (__any(need)) {
          const float alpha = need ? __builtin_amdgcn_exp2f(mrun - mt) : 1.0f;
          if (need) mrun = mt;
          lsum *= alpha;
#pragma unroll
          for (int g = 0; g < NG; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[g][j] *= alpha;
        }
        const float mb = mrun == -INFINITY ? 0.0f : mrun;
        half4_t pf;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float p = __builtin_amdgcn_exp2f(S[r] - mb);
          pf[r] = (hxa_h)(iv[r] < 1.0f / HXA_Q8_LEAST ? p : p == p ? 0.0f : p);  // a page without a scale: values of 0, whatever the bytes
          lsum = fmaf(p, iv[r], lsum);
        }
#pragma unroll
        for (int g = 0; g < NG; g++) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = *(const uint32_t *)(vat + at + 4 * e * HD + vch[g]) ^ 0x80808080u;
          // bytes of two keys side by side, dims 0, 1 and 2, 3
          const uint32_t a0 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), a1 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
          const uint32_t b0 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), b1 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint32_t sel = j & 1 ? 0x04030402u : 0x04010400u;
            const half2_t bias = {(hxa_h)1152.0f, (hxa_h)1152.0f};
            const half2_t lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, j < 2 ? a0 : a1, sel)) - bias;
            const half2_t hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, j < 2 ? b0 : b1, sel)) - bias;
            acc[g][j] = mma16h(__builtin_shufflevector(lo, hi, 0, 1, 2, 3), pf, acc[g][j]);
          }
        }
      }
      t0 = t1;
    }
    lsum = add16(lsum);
  }
  // join the four waves: dims 64 g + 16 gi + 4 r .. + 3 of a lane are element r of its four products of group g. Wave w takes every fourth of them.
  constexpr int ND = 4 * NG;
  reads_done_barrier();
  float4_t *ox = (float4_t *)lds;                     // [wave][g 4 + r][lane]
  float2_t *mlx = (float2_t *)(lds + ND * 4 * 1024);  // [wave][row]
#pragma unroll
  for (int d = 0; d < ND; d++)
    ox[(wave * ND + d) * 64 + lane] = (float4_t){acc[d >> 2][0][d & 3], acc[d >> 2][1][d & 3], acc[d >> 2][2][d & 3], acc[d >> 2][3][d & 3]};
  if (gi == 0) mlx[wave * 16 + ql] = (float2_t){mrun, lsum};
  reads_done_barrier();
  float m = -INFINITY, l = 0.0f, a[4];
#pragma unroll
  for (int w = 0; w < 4; w++) m = fmaxf(m, mlx[w * 16 + ql][0]);
  const float mz = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const float2_t x = mlx[w * 16 + ql];
    a[w] = __builtin_amdgcn_exp2f(x[0] - mz);
    l += x[1] * a[w];
  }
  if (R >= it.nrows) return;
  int rest;
  const long tok = it.tok0 + row_tok(it, R, rest);
  const int head = head0 + rest;
  const long row = tok * out.Hq + head, at = out.slot * out.rows + row;
  if (out.part != nullptr) {
    if (wave == 0 && gi == 0) out.ml[row * out.nslots + out.slot] = (float2_t){m, l};
    if (l == 0.0f) return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int g = 0; g < NG; g++) {
    const int dim = 64 * g + 16 * gi + 4 * wave;
    float4_t o = {};
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float4_t x = ox[(w * ND + 4 * g + wave) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] += x[e] * a[w];
    }
    if (out.part != nullptr) {
      *(float4_t *)(out.part + at * HD + dim) = o;
    } else {
      v4 x;
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = (T)(o[e] * inv);
      *(v4 *)(out.o + tok * out.ldo + (long)head * HD + dim) = x;
    }
  }
}

template <int HD>
constexpr int lds_q8() { return std::max(GeoQ8<HD>::LDS, FewQ8<HD>::LDS); }
struct CachedQ8Args : CachedArgs {
  const float *ks, *vs;
};
template <typename T, int HD>
HXA_DEV void any_item_q8(int mode, const KeysQ8 &s, const Item &it, const CachedQ8Args &p, int head0, uint8_t *lds, const Out<T> &out) {
  if (mode == 1) {
    few_item_q8<T, HD>(s, it, (const T *)p.q, p.ldq, head0, p.cs, lds, out);
    return;
  }
  float16_t acc[HD / 32];
  float m, l;
  if (mode == 2) {
    rows_item_q8<T, HD, 2>(s, it, (const T *)p.q, p.ldq, head0, p.cs, lds, acc, m, l);
    rows_out<T, HD, 2>(out, it, head0, 1.0f, lds, acc, m, l);
  } else {
    rows_item_q8<T, HD, 4>(s, it, (const T *)p.q, p.ldq, head0, p.cs, lds, acc, m, l);
    rows_out<T, HD, 4>(out, it, head0, 1.0f, lds, acc, m, l);
  }
}
template <typename T, int HD>
__global__ HXA_CAUSAL_BOUNDS void cached_q8_kernel(CachedQ8Args p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int h = blockIdx.x % p.c.H;
  KeysQ8 s{};
  s.k = (const int8_t *)p.c.k;
  s.v = (const int8_t *)p.c.v;
  s.ks = p.ks;
  s.vs = p.vs;
  walk_cache<T, lds_q8<HD>()>(p, h, s, lds, [&](int mode, const Item &it, const Out<T> &out) { any_item_q8<T, HD>(mode, s, it, p, h * p.G, lds, out); });
}

int q8_check(const hxa_kv_cache_q8 *c, int T, int Hq) {
  const int r = hxa_kv_check_q8(c, T, "attention_cached_q8");
  return r != HXA_OK ? r : cached_limits(c->c, T, Hq, "attention_cached_q8");
}

}  // namespace

extern "C" long hxa_attention_cached_q8_ws_bytes(const hxa_kv_cache_q8 *c, int T, int Hq) {
  if (q8_check(c, T, Hq) != HXA_OK || T == 0 || c->c.nseq == 0) return 0;
  return cached_ws(cached_plan(c->c, T, Hq, true, wg_slots(c->c.hd)), c->c, T, Hq);
}

extern "C" int hxa_attention_cached_q8(const hxa_kv_cache_q8 *cache, const void *q, long ldq, void *o, long ldo, int T, int Hq, float scale,
                                       void *ws, long ws_bytes, void *stream) {
  const int r = q8_check(cache, T, Hq);
  if (r != HXA_OK) return r;
  CachedQ8Args p{};
  p.ks = cache->kscale;
  p.vs = cache->vscale;
  return cached_call(
      p, cache->c, q, ldq, o, ldo, T, Hq, scale, ws, ws_bytes, (hipStream_t)stream, "attention_cached_q8",
      [](auto ty, auto hdc) {
        constexpr int HD = decltype(hdc)::value;
        return std::make_pair(cached_q8_kernel<decltype(ty), HD>, lds_q8<HD>() + 4096);
      });
}
