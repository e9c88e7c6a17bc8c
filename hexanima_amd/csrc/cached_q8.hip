// Attention of new tokens over a paged cache of int8 with a scale for each page and head (hxa_attention_cached_q8): queries and results in fp16 / bf16,
// heads of 64, 128 or 256, grouped heads, a prefix that the batch shares. Rows, work items and modes are those of causal_attn.hip.
//
// With k = ks qk and v = vs qv (qk, qv the bytes, ks, vs the scales of their pages), in powers of two and with c = scale log2(e):
//   t_j = (q . qk_j) (c ks_j) + log2(vs_j),   w_j = 2^(t_j - m + 7),   o = sum w_j qv_j / sum w_j / vs_j
// The values' scale is folded into the exponent, so that one running maximum m bounds what is rounded to fp16, the weight as it stands before its
// byte: a key whose page has small values loses no bits to one whose page has large ones, and the products take the bytes as they are. A byte is exact
// in fp16. q in bf16 becomes fp16 as it is where its row's largest magnitude is 1 .. 2^15, otherwise times the power of two that puts the largest near
// 2^14: what is then 2^-17 or more stays exact, anything smaller is off by 2^-25 at most.
// t, m, both sums and O are held in fp32; the denominator adds the weights before they are rounded.
//
// A byte is finite whatever it holds, so that a masked key needs nothing but a weight of 0.
#include "causal_attn.h"
#include "int8_rows.h"

namespace {

// A row's weights are 2^7 times 2^(t - m), so up to 2^15 before their bytes: what fp16 keeps below 2^-14 in multiples of 2^-24 are weights below 2^-21 of
// the largest one, in multiples of 2^-31 of it (without it 5000 keys of 2^-27 the largest one's weight are nothing).
constexpr float LIFT = 7.0f;

struct KeysQ8 : Keys<int8_t> {
  const float *ks, *vs;
};

template <int HD>
struct GeoQ8 {
  static constexpr int RB = HD * 2, TB = KT * RB;    // bytes of an fp16 row, of a tile
  static constexpr int CH = HD / 16, RPL = 64 / CH;  // 16-byte chunks of a row of bytes, rows of one wave-wide load
  static constexpr int NLD = HD / 64;                // loads of a wave's keys of a tile, and of its values
  static constexpr int WB = 16 * HD;                 // bytes of a wave's keys of a tile, and of its values
  static constexpr int RAW = 2 * TB;                 // past K and V in fp16: each wave's bytes of two tiles
  static constexpr int CST = RAW + 4 * 4 * WB;       // c ks, log2 vs and 1 / vs of the tile's keys
  static constexpr int TABLE = CST + 768;            // the pages' table
  static constexpr int LDS = TABLE + 512 * 16 + 16;
};

// the least factor of a score, and what stands for a key scale of 0: scores are as good as 0, and -infinity stays what it is
constexpr float NO_SCALE = 0x1p-110f;
// the least key scale in the pages' table: a bf16 row's factor, up to 2^113, comes to it first, so there it is 0, which that factor leaves 0
template <bool BF>
constexpr float LEAST_KS = BF ? 0.0f : NO_SCALE;

// four bytes to fp16: u = q + 128 under the exponent of 1024 is 1024 + u
HXA_DEV uint2_t q8_halves(uint32_t d) {
  const uint32_t x = d ^ 0x80808080u;
  const half2_t c = {(hxa_h)1152.0f, (hxa_h)1152.0f};
  return (uint2_t){__builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - c),
                   __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - c)};
}

// q's eight values as fp16; bf16: times a power of two, whose inverse the caller keeps
HXA_DEV half8_t q_halves(half8_t q, float) { return q; }
HXA_DEV half8_t q_halves(bf8_t q, float f) {
  half8_t r;
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = (hxa_h)((float)q[e] * f);
  return r;
}
// 1 for a row whose largest magnitude is 1 .. 2^15, 0 or not finite, else 2^(14 - e) where it is 2^e .. 2^(e + 1)
HXA_DEV float row_factor(float top) {
  const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
  return top >= 0x1p-100f && top < INFINITY && !(top >= 1.0f && top < 0x1p15f) ? __builtin_bit_cast(float, (uint32_t)(127 + 14 - e) << 23) : 1.0f;
}
// a key's scale times what its row's queries were divided by, not below NO_SCALE
template <bool BF>
HXA_DEV float with_back(float k, float back) { return BF ? fmaxf(k * back, NO_SCALE) : k; }
// An exponent t - m is one fma of the score with the key's scale and log2(vs) - m: t is not rounded by itself, as m, the largest rounded t, was. Below 2^18 the two
// differ by less than 2^-5. Whether some row of the wave has a (finite) maximum farther out: then t is rounded first, so that no exponent passes
// what the running maximum leaves unscaled, at 64 steps and single ones 1% at most.
HXA_DEV bool far_scores(float mt) {
  constexpr uint32_t FAR = 0x48800000u;  // 2^18
  return __any((__builtin_bit_cast(uint32_t, mt) & 0x7fffffffu) - FAR < 0x7f800000u - FAR);
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

// The pages of keys x from a first one on, 512 of them: place in the pools (npages H page rows; ~0: not there) and scales
struct PagesQ8 {
  static constexpr int N = 512;
  const KeysQ8 &s;
  uint32_t *ph;
  float *ks, *lv, *iv;
  int *flag;
  int first, own;        // entry of page slot n of the prefix: n - first, of the sequence: n + own
  int npre, pre_end, own_end;
  HXA_DEV PagesQ8(const KeysQ8 &s_, uint8_t *table) : s(s_), first(0), own(0) {
    ph = (uint32_t *)table;
    ks = (float *)(ph + N);
    lv = ks + N;
    iv = lv + N;
    flag = (int *)(iv + N);
  }
  HXA_DEV int entry(int x, unsigned &in_page) const {
    const bool pre = x < s.P;
    return (int)s.slot(pre ? x : x - s.P, in_page) + (pre ? -first : own);
  }
  // the entries from key x0 on, of keys below x1
  HXA_DEV void start(int x0, int x1) {
    unsigned in;
    npre = 0;
    if (x0 < s.P) {
      first = (int)s.slot(x0, in);
      npre = (int)s.slot(s.P - 1, in) - first + 1;
      own = npre;
    } else {
      own = -(int)s.slot(x0 - s.P, in);
    }
    own_end = x1 > s.P ? (int)s.slot(x1 - 1 - s.P, in) + 1 + own : npre;
    pre_end = x1 > s.P ? npre : (int)s.slot(x1 - 1, in) - first + 1;
  }
  HXA_DEV bool there(int j) const { return j < (j < npre ? pre_end : own_end); }
  HXA_DEV int page_of(int j) const { return there(j) ? (j < npre ? s.prefix[first + j] : s.table[j - own]) : -1; }
  // the workgroup's threads take two pages each, e[k] of entry 256 k + tid; least: of a key scale
  HXA_DEV void fill(const int (&e)[2], float c, float least, int tid) {
    bool hole = false, bare = false;
    float a[2], b[2];
    uint32_t at[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const bool ok = (unsigned)e[k] < (unsigned)s.npages;
      hole |= !ok && there(k * 256 + tid);
      at[k] = ok ? (uint32_t)e[k] * s.H + s.h : ~0u;
      a[k] = ok ? s.ks[at[k]] : 0.0f;
      b[k] = ok ? s.vs[at[k]] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int j = k * 256 + tid;
      const bool vok = b[k] > HXA_Q8_LEAST && b[k] < INFINITY;
      bare |= at[k] != ~0u && !vok;
      ph[j] = at[k];
      ks[j] = a[k] > 0.0f && a[k] < INFINITY ? fmaxf(a[k] * c, least) : least;
      lv[j] = vok ? __builtin_amdgcn_logf(b[k]) : -64.0f;
      iv[j] = vok ? 1.0f / b[k] : 1.0f / HXA_Q8_LEAST;
    }
    const int any = (__any(hole) ? 1 : 0) | (__any(bare) ? 2 : 0);
    if ((tid & 63) == 0) flag[tid >> 6] = any;
  }
  // once the workgroup has met: 1: a page is not there; 2: one is without a value scale
  HXA_DEV int flags() const { return __builtin_amdgcn_readfirstlane(flag[0] | flag[1] | flag[2] | flag[3]); }
  HXA_DEV bool holes() const { return flags() & 1; }
  // where the steps [s0, s1) of `span` keys from x0 on, below x1, that the table reaches end
  HXA_DEV int reach(int s0, int s1, int span, int x0, int x1) const {
    for (;;) {
      unsigned in;
      const int over = entry(min(x0 + s1 * span, x1) - 1, in) - N + 1;
      if (over <= 0) return s1;
      s1 -= max(1, (int)min((long)(over - 1) * s.page / span, (long)s1 - s0 - 1));
    }
  }
};

// ---- rows modes: as causal_attn.hip's rows_item; m and the sums in powers of two ----
// A tile's bytes go straight into LDS two tiles ahead (each wave its 16 keys), from there through registers, where they become fp16 once for all four
// waves, into the tile that the products read. Pages' places and scales come from the table in LDS, as a load of them would be waited for with the keys'.
// Bound by the conversions, which the other workgroup's products hide in part. 64 decoding tokens with 470 keys each behind a prefix of 4096 36.1 us and 32 prompts of 75
// 57.1 (both 1% more since far scores are looked for); with the tile ahead held in registers and converted beside K's products 37.4 and 56.7 (128 tokens behind 200 keys each 29.0, here 27.3); with
// V converted beside K's products and K beside V's 40.1 and 68.3.
//
// G8: eight keys of a lane (8 g + 0 .. 7 of every 16) lie on one page, so that they share its scales: the maximum is taken of the scores, the
// scales go into one fma a score. (With constants for each key, 24 more 16-byte reads of LDS a tile: 32 prompts of 75 behind 4000 186 us against 168.)
template <typename T, int HD, int W, bool G8>
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
  const int lim = tok_limit(it, tok), lim_min = row_limit(it, it.r0);
#pragma unroll
  for (int d = 0; d < ND; d++) acc[d] = (float16_t){};
  mrun = -INFINITY;
  lsum = 0.0f;
  const int nt = (it.x1 - it.x0 + KT - 1) / KT;
  if (nt <= 0) return;

  // the wave's part of a tile: keys 16 wave .. + 15, as they come into one of two places, then as fp16 rows for all waves
  PagesQ8 pages(s, lds + G_::TABLE);
  constexpr int L = 2 * G_::NLD;  // loads a tile
  uint8_t *const raw = lds + G_::RAW + wave * (4 * G_::WB);
  const int xlane = it.x0 + 16 * wave + (lane & 15), ch = lane % G_::CH;
  auto pool_row = [&](uint32_t p, unsigned in) { return p == ~0u ? 0u : p * s.page + in; };  // < 2^32: checked on the host
  auto row_of = [&](int i) {
    const int x = xlane + i * KT;
    unsigned in;
    if (x >= it.x1) return 0u;
    const uint32_t p = pages.ph[pages.entry(x, in)];
    return pool_row(p, in);
  };
  auto load = [&](int i, uint32_t at) {
    uint8_t *to = raw + (i & 1) * 2 * G_::WB;
#pragma unroll
    for (int n = 0; n < G_::NLD; n++) {
      const uint64_t from = (uint64_t)(uint32_t)__shfl((int)at, n * G_::RPL + lane / G_::CH) * HD + ch * 16;
      g2l16_opaque((const uint8_t *)s.k + from, to + n * 1024);
      g2l16_opaque((const uint8_t *)s.v + from, to + G_::WB + n * 1024);
    }
  };
  // the first tiles' places and the table's pages from memory side by side, then the keys and the scales
  pages.start(it.x0, it.x1);
  int e0[2], e1[2];
  unsigned in0[2];
#pragma unroll
  for (int i = 0; i < 2; i++) e0[i] = xlane + i * KT < it.x1 ? pages.page_of(pages.entry(xlane + i * KT, in0[i])) : -1;
#pragma unroll
  for (int k = 0; k < 2; k++) e1[k] = pages.page_of(k * 256 + tid);
  half8_t qf[HD / 16];
  float back = 1.0f;  // what q was divided by
  {
    v8 x[HD / 16];
#pragma unroll
    for (int i = 0; i < HD / 16; i++) x[i] = *(const v8 *)(qp + i * 16 + 8 * g);
    uint32_t at0[2];
#pragma unroll
    for (int i = 0; i < 2; i++) at0[i] = (unsigned)e0[i] < (unsigned)s.npages ? pool_row((uint32_t)e0[i] * s.H + s.h, in0[i]) : 0u;
    load(0, at0[0]);
    if (nt > 1) load(1, at0[1]);
    pages.fill(e1, c, LEAST_KS<BF>, tid);
    float f = 1.0f;
    if (BF) {
      float lo, hi;
      halves(most_of(x), lo, hi);
      f = row_factor(fmaxf(lo, hi));
      back = 1.0f / f;
    }
#pragma unroll
    for (int i = 0; i < HD / 16; i++) qf[i] = q_halves(x[i], f);
  }

  const int vrow = 4 * g + ((lane & 15) >> 2);
  const int vlow = ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) << 4) + (lane & 1) * 8;
  uint32_t vat[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) vat[d] = vrow * G_::RB + (((d << 2) ^ S_::fv(vrow)) << 4) + vlow;
  const uint8_t *const kb = lds, *const vb = lds + G_::TB;
  const float *const cst = (const float *)(lds + G_::CST) + 32 * kh + 8 * g;

  for (int s0 = 0; s0 < nt;) {
    if (s0 > 0) {  // the next 512 pages
      reads_done_barrier();
      pages.start(it.x0 + s0 * KT, it.x1);
#pragma unroll
      for (int k = 0; k < 2; k++) e1[k] = pages.page_of(k * 256 + tid);
      pages.fill(e1, c, LEAST_KS<BF>, tid);
    }
    reads_done_barrier();
    const int flags = pages.flags();
    const int s1 = pages.reach(s0, nt, KT, it.x0, it.x1);  // the tiles whose pages are in the table
    if (s0 > 0) {
      load(s0, row_of(s0));
      if (s0 + 1 < s1) load(s0 + 1, row_of(s0 + 1));
    }
    uint32_t at_next = s0 + 2 < s1 ? row_of(s0 + 2) : 0;
    for (int i = s0; i < s1; i++) {
      const int key0 = it.x0 + i * KT;
      __builtin_amdgcn_s_setprio(0);
      if (i + 1 < s1) wait_vm<L>();  // the wave's part of tile i has landed
      else wait_vm<0>();
      asm volatile("" ::: "memory");
      uint4_t w[2][G_::NLD];
      {
        const uint8_t *from = raw + (i & 1) * 2 * G_::WB + lane * 16;
#pragma unroll
        for (int n = 0; n < G_::NLD; n++) {
          w[0][n] = *(const uint4_t *)(from + n * 1024);
          w[1][n] = *(const uint4_t *)(from + G_::WB + n * 1024);
        }
      }
      reads_done_barrier();  // it is in registers; every wave is done with tile i - 1
      if (i + 2 < s1) {
        load(i + 2, at_next);
        if (i + 3 < s1) at_next = row_of(i + 3);
      }
      if (flags & 2) {  // pages without a value scale: values of 0, whatever the bytes
#pragma unroll
        for (int n = 0; n < G_::NLD; n++) {
          unsigned in;
          const int x = min(key0 + 16 * wave + n * G_::RPL + lane / G_::CH, it.x1 - 1);
          if (pages.iv[pages.entry(x, in)] >= 1.0f / HXA_Q8_LEAST) w[1][n] = (uint4_t){0, 0, 0, 0};
        }
      }
      uint64_t km = ~0ull;
      {
        int ln = lane;
        asm volatile("" : "+v"(ln));  // opaque: the loop keeps none of these addresses in registers
#pragma unroll
        for (int n = 0; n < G_::NLD; n++) {
          const int row = krow_key(16 * wave + n * G_::RPL + ln / G_::CH), c2 = 2 * (ln % G_::CH);  // (its own inverse)
#pragma unroll
          for (int V = 0; V < 2; V++) {
            uint8_t *to = lds + V * G_::TB + row * G_::RB;
            const int f = V ? S_::fv(row) : S_::fk(row);
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const uint2_t a = q8_halves(w[V][n][2 * e]), b = q8_halves(w[V][n][2 * e + 1]);
              *(uint4_t *)(to + (((c2 + e) ^ f) << 4)) = (uint4_t){a.x, a.y, b.x, b.y};
            }
          }
        }
        if (wave == 0 || (flags & 1)) {
          unsigned in;
          const int x = key0 + ln, e = pages.entry(min(x, it.x1 - 1), in);
          if (flags & 1) km = __ballot(x < it.x1 && pages.ph[e] != ~0u);
          if (wave == 0) {
            float *to = (float *)(lds + G_::CST) + ln;
            to[0] = pages.ks[e];
            to[64] = pages.lv[e];
            to[128] = pages.iv[e];
          }
        }
      }
      reads_done_barrier();  // tile i is in LDS
      __builtin_amdgcn_s_setprio(1);  // products before the other workgroup's conversions (32 prompts 57.1 us against 60.3)
      auto kfrag = [&](int ds, int b) {
        const int row = (b + kh) * 32 + ql, ch = 2 * ds + g;
        return *(const half8_t *)(kb + row * G_::RB + ((ch ^ S_::fk(row)) << 4));
      };
      auto vfrag = [&](int n) {
        const uint8_t *at = vb + vat[n % ND] + (kh * 32 + n / ND * 16) * G_::RB;
        return __builtin_shufflevector(read_tr<half4_t>(at), read_tr<half4_t>(at + 8 * G_::RB), 0, 1, 2, 3, 4, 5, 6, 7);
      };
      const bool cut = km != ~0ull || key0 + KT - 1 > min(lim_min, it.x1 - 1);
      float16_t S[NB];
      half8_t kf[AK + 1][NB];
#pragma unroll
      for (int ds = 0; ds < AK; ds++)
#pragma unroll
        for (int b = 0; b < NB; b++) kf[ds][b] = kfrag(ds, b);
      float kg[2 * NB], lg[2 * NB], ig[2 * NB], lm[2 * NB];  // G8: of keys 16 u + 8 g .. + 7
      if constexpr (G8) {
#pragma unroll
        for (int u = 0; u < 2 * NB; u++) kg[u] = with_back<BF>(cst[16 * u], back), lg[u] = cst[16 * u + 64], ig[u] = cst[16 * u + 128];
      }
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
      if constexpr (!G8) {
        // scores to exponents, four keys at a time (their constants two reads ahead: all of them at once are more registers than there are)
        auto at = [&](int u) { return cst + 16 * (u >> 1) + 4 * (u & 1); };
        float4_t k[2], lv[2];
        k[0] = *(const float4_t *)at(0), lv[0] = *(const float4_t *)(at(0) + 64);
#pragma unroll
        for (int u = 0; u < 4 * NB; u++) {
          if (u + 1 < 4 * NB) k[(u + 1) & 1] = *(const float4_t *)at(u + 1), lv[(u + 1) & 1] = *(const float4_t *)(at(u + 1) + 64);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float x = S[u >> 2][4 * (u & 3) + e];
            S[u >> 2][4 * (u & 3) + e] = fmaf(x, BF ? k[u & 1][e] * back : k[u & 1][e], lv[u & 1][e]);
          }
        }
      }
      if (cut) {
        // a row's limit hides the keys past x1 too (a range that ends before it ends with a tile); pages that are not there need the mask
        const int n = lim - key0 - 32 * kh - 8 * g, left = it.x1 - key0;
        if (km == ~0ull || km == (left >= KT ? ~0ull : (1ull << left) - 1)) {
#pragma unroll
          for (int b = 0; b < NB; b++)
#pragma unroll
            for (int r = 0; r < 16; r++)
              if (32 * b + 16 * (r >> 3) + (r & 7) > n) S[b][r] = -INFINITY;
        } else {
          const uint64_t see = km >> (32 * kh + 8 * g);
#pragma unroll
          for (int b = 0; b < NB; b++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
              const int k = 32 * b + 16 * (r >> 3) + (r & 7);
              if (k > n || !((see >> k) & 1)) S[b][r] = -INFINITY;
            }
        }
      }
      float mt = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2 * NB; u++) {
        float m8 = S[u >> 1][8 * (u & 1)];
#pragma unroll
        for (int r = 1; r < 8; r++) m8 = fmaxf(m8, S[u >> 1][8 * (u & 1) + r]);
        mt = fmaxf(mt, G8 ? fmaf(m8, kg[u], lg[u]) : m8);
      }
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
      float mb = mrun == -INFINITY ? 0.0f : mrun;
      if constexpr (G8) {
#pragma unroll
        for (int u = 0; u < 2 * NB; u++) lm[u] = lg[u] - (mb - LIFT);
      }
      if (far_scores(mt)) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int r = 0; r < 16; r++) S[b][r] = (G8 ? fmaf(S[b][r], kg[2 * b + (r >> 3)], lg[2 * b + (r >> 3)]) : S[b][r]) - mb;
#pragma unroll
        for (int u = 0; u < 2 * NB; u++) kg[u] = 1.0f, lm[u] = LIFT;
        mb = 0.0f;
      }
      half8_t pf[NB][2];
      float ls[2 * NB] = {};
      auto expo2 = [&](int n) {
        const int u = n >> 3;
        float p0 = S[n >> 4][n & 15], p1 = S[n >> 4][(n & 15) + 1];
        if constexpr (G8) {
          p0 = __builtin_amdgcn_exp2f(fmaf(p0, kg[u], lm[u]));
          p1 = __builtin_amdgcn_exp2f(fmaf(p1, kg[u], lm[u]));
          ls[u] += p0;
          ls[u] += p1;
        } else {
          const float2_t inv = *(const float2_t *)(cst + 128 + 16 * u + (n & 7));
          p0 = __builtin_amdgcn_exp2f(p0 - (mb - LIFT));
          p1 = __builtin_amdgcn_exp2f(p1 - (mb - LIFT));
          ls[u] = fmaf(p1, inv[1], fmaf(p0, inv[0], ls[u]));
        }
        pf[n >> 4][u & 1][n & 7] = (hxa_h)p0;
        pf[n >> 4][u & 1][(n & 7) + 1] = (hxa_h)p1;
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
#pragma unroll
      for (int u = 0; u < 2 * NB; u++) lsum = G8 ? fmaf(ls[u], ig[u], lsum) : lsum + ls[u];
    }
    s0 = s1;
    __builtin_amdgcn_s_setprio(0);
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
// Bound by reading the cache, and in short items by what follows one after the other. So the tiles stay bytes until a wave needs its part of one, and
// a wave fetches its own keys and waits for nobody: 16 keys of two tiles a step go from memory straight into its ring of RS steps in LDS
// (global_load_lds), are read into registers and their place is loaded again before the step is computed. What addresses and exponents need of
// the pages, their places and scales, is in LDS as well, for 512 pages at a time (a load of it inside the loop would be waited for with all
// those behind it); the first steps take their places from the tables themselves.
//
// Row 4 b + a of a wave's 16 holds key 4 a + b. K: a lane takes 16 bytes of its key, two slices of 8 dims; q's dims follow that order. V: dword u of
// keys 4 gi .. + 3 is dims 4 u .. + 3 of four keys, transposed by byte permutations: product j of a 64-dim group has dims 4 u + j. Chunks are swizzled
// so that the lanes of either read spread over the banks.
template <int HD>
struct FewQ8 {
  static constexpr int RS = HD == 64 ? 4 : 2;          // steps in a wave's ring
  static constexpr int TB = 16 * HD;                   // bytes of a wave's keys of a tile, and of its values
  static constexpr int CH = HD / 16, RPL = 64 / CH;    // 16-byte chunks a row, rows of one wave-wide load
  static constexpr int NLD = HD / 64;                  // loads of a tile's keys, and of its values
  static constexpr int TABLE = 4 * RS * 4 * TB;         // the pages' table, past the four rings
  static constexpr int LDS = TABLE + 512 * 16 + 16;
  static HXA_DEV int fk(int row) { return HD == 64 ? (row >> 2) & 3 : HD == 128 ? (row >> 1) & 7 : row & 15; }
  static HXA_DEV int fv(int row) { return HD == 64 ? 0 : HD == 128 ? (row << 1) & 4 : (row & 3) << 2; }
};
// row of LDS <-> key, within 16 (its own inverse)
HXA_DEV int few_row(int key) { return (key & 3) << 2 | (key >> 2 & 3); }

template <typename T, int HD, bool G8>
HXA_DEV void few_item_q8(const KeysQ8 &s, const Item &it, const T *q, long ldq, int head0, float c, uint8_t *lds, const Out<T> &out) {
  typedef FewQ8<HD> F;
  typedef typename HxaVec<T>::v8 v8;
  typedef typename HxaVec<T>::v4 v4;
  constexpr bool BF = std::is_same<T, hxa_b>::value;
  constexpr int NG = HD / 64, RS = F::RS;  // groups of 64 dims
  constexpr int L = 4 * F::NLD;            // loads a step
  const int tid = this_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int gi = lane >> 4, ql = lane & 15;
  const int R = it.r0 + ql, last = it.nrows - 1, Rc = min(R, last);
  float4_t acc[NG][4];
#pragma unroll
  for (int g = 0; g < NG; g++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[g][j] = (float4_t){};
  float mrun = -INFINITY, lsum = 0.0f;
  const int ns = (it.x1 - it.x0 + 2 * KT - 1) / (2 * KT);  // steps of two tiles
  if (ns > 0) {
    PagesQ8 pages(s, lds + F::TABLE);
    uint8_t *const ring = lds + wave * (RS * 4 * F::TB);
    uint32_t koff[F::NLD], voff[F::NLD];
    int from[F::NLD];  // the lane that knows the row of this lane's part of load n
#pragma unroll
    for (int n = 0; n < F::NLD; n++) {
      const int row = n * F::RPL + lane / F::CH, ch = lane % F::CH;
      from[n] = few_row(row);
      koff[n] = (uint32_t)((ch ^ F::fk(row)) << 4);
      voff[n] = (uint32_t)((ch ^ F::fv(row)) << 4);
    }
    // lane (h, key) of the first 32: the key of a step
    const int xlane = it.x0 + (lane >> 4 & 1) * KT + 16 * wave + ql;
    auto pool_row = [&](uint32_t p, unsigned in) { return p == ~0u ? 0u : p * s.page + in; };  // < 2^32: checked on the host
    auto row_of = [&](int st) {
      const int x = xlane + st * 2 * KT;
      unsigned in;
      if (x >= it.x1) return 0u;
      const uint32_t p = pages.ph[pages.entry(x, in)];
      return pool_row(p, in);
    };
    // loads of a step, whose keys' rows `at` has, into its place of the ring
    auto load = [&](int st, uint32_t at) {
      uint8_t *to = ring + (st % RS) * 4 * F::TB;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int n = 0; n < F::NLD; n++) {
          const uint64_t row = (uint64_t)(uint32_t)__shfl((int)at, 16 * h + from[n]) * HD;
          g2l16_opaque((const uint8_t *)s.k + row + koff[n], to + h * 2 * F::TB + n * 1024);
          g2l16_opaque((const uint8_t *)s.v + row + voff[n], to + h * 2 * F::TB + F::TB + n * 1024);
        }
    };
    // the first steps' places and the table's pages from memory side by side, then the keys and the scales
    pages.start(it.x0, it.x1);
    int e0[RS], e1[2];
    unsigned in0[RS];
#pragma unroll
    for (int i = 0; i < RS; i++) {
      const int x = xlane + i * 2 * KT;
      e0[i] = x < it.x1 ? pages.page_of(pages.entry(x, in0[i])) : -1;
    }
#pragma unroll
    for (int k = 0; k < 2; k++) e1[k] = pages.page_of(k * 256 + tid);
    // q: dims 16 (4 d + gi) + 8 e .. + 7 in qf[d][e]
    int rest;
    const int tok = row_tok(it, Rc, rest);
    const T *qp = q + (long)(it.tok0 + tok) * ldq + (long)(head0 + rest) * HD;
    v8 raw[2 * NG];
#pragma unroll
    for (int i = 0; i < 2 * NG; i++) raw[i] = *(const v8 *)(qp + 16 * (4 * (i >> 1) + gi) + 8 * (i & 1));
    uint32_t at0[RS];
#pragma unroll
    for (int i = 0; i < RS; i++) at0[i] = (unsigned)e0[i] < (unsigned)s.npages ? pool_row((uint32_t)e0[i] * s.H + s.h, in0[i]) : 0u;
#pragma unroll
    for (int i = 0; i < RS; i++)
      if (i < ns) load(i, at0[i]);
    pages.fill(e1, c, LEAST_KS<BF>, tid);
    half8_t qf[NG][2];
    float back = 1.0f;
    {
      float f = 1.0f;
      if (BF) {
        f = row_factor(max16(most_of(raw)));
        back = 1.0f / f;
      }
#pragma unroll
      for (int i = 0; i < 2 * NG; i++) qf[i >> 1][i & 1] = q_halves(raw[i], f);
    }
    const int lim = tok_limit(it, tok), lim_min = row_limit(it, it.r0);
    const int krow = few_row(ql);
    const uint8_t *kat = ring + krow * HD, *vat = ring + F::TB + gi * HD;  // values of key 4 gi + e: row 4 e + gi
    uint32_t vch[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) vch[g] = (uint32_t)((((4 * g + (ql >> 2)) ^ F::fv(gi)) << 4) + (ql & 3) * 4);

    for (int s0 = 0; s0 < ns;) {
      if (s0 > 0) {  // the next 512 pages
        reads_done_barrier();
        pages.start(it.x0 + s0 * 2 * KT, it.x1);
#pragma unroll
        for (int k = 0; k < 2; k++) e1[k] = pages.page_of(k * 256 + tid);
        pages.fill(e1, c, LEAST_KS<BF>, tid);
      }
      reads_done_barrier();
      const bool holes = pages.holes();
      const int s1 = pages.reach(s0, ns, 2 * KT, it.x0, it.x1);  // the steps whose pages are in the table
      if (s0 > 0) {
#pragma unroll
        for (int i = 0; i < RS; i++)
          if (s0 + i < s1) load(s0 + i, row_of(s0 + i));
      }
      // (the first table holds the first RS steps: fewer than 512 pages of a key each)
      uint32_t at_next = s0 + RS < s1 ? row_of(s0 + RS) : 0;
      for (int st = s0; st < s1; st++) {
        // this step has landed: the loads of the steps behind it may still fly
        const int newer = min(RS, s1 - st) - 1;
        if (newer == 0) wait_vm<0>();
        else if (newer == 1) wait_vm<L>();
        else if (newer == 2) wait_vm<(RS > 2 ? 2 * L : 0)>();
        else wait_vm<(RS > 3 ? 3 * L : 0)>();
        asm volatile("" ::: "memory");
        const int at = (st % RS) * 4 * F::TB;
        uint4_t kr[2][NG];
        uint32_t vr[2][NG][4];
        float k4[2][G8 ? 1 : 4], l4[2][G8 ? 1 : 4], i4[2][G8 ? 1 : 4];  // G8: keys 4 gi .. + 3 lie on one page
        const int x = it.x0 + st * 2 * KT + 16 * wave + 4 * gi;
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int d = 0; d < NG; d++) kr[h][d] = *(const uint4_t *)(kat + at + h * 2 * F::TB + (((4 * d + gi) ^ F::fk(krow)) << 4));
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          unsigned in;
#pragma unroll
          for (int r = 0; r < (G8 ? 1 : 4); r++) {
            const int p = pages.entry(min(x + h * KT + r, it.x1 - 1), in);
            k4[h][r] = with_back<BF>(pages.ks[p], back), l4[h][r] = pages.lv[p], i4[h][r] = pages.iv[p];
          }
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int g = 0; g < NG; g++)
#pragma unroll
            for (int e = 0; e < 4; e++) vr[h][g][e] = *(const uint32_t *)(vat + at + h * 2 * F::TB + 4 * e * HD + vch[g]);
        if (st + RS < s1) {
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the step is in registers, its place is free
          asm volatile("" ::: "memory");
          load(st + RS, at_next);
          if (st + RS + 1 < s1) at_next = row_of(st + RS + 1);
        }
        float4_t S[2] = {};
#pragma unroll
        for (int d = 0; d < NG; d++)
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const uint2_t a = q8_halves(kr[h][d][2 * e]), b = q8_halves(kr[h][d][2 * e + 1]);
              S[h] = mma16(__builtin_bit_cast(half8_t, (uint4_t){a.x, a.y, b.x, b.y}), qf[d][e], S[h]);
            }
        if (it.x0 + (st + 1) * 2 * KT - 1 > min(lim_min, it.x1 - 1)) {
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 4; r++)
              if (x + h * KT + r > lim || x + h * KT + r >= it.x1) S[h][r] = -INFINITY;
        }
        if (holes) {
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              unsigned in;
              if (pages.ph[pages.entry(min(x + h * KT + r, it.x1 - 1), in)] == ~0u) S[h][r] = -INFINITY;
            }
        }
        float mt;
        if constexpr (G8) {
          mt = fmaxf(fmaf(fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3])), k4[0][0], l4[0][0]),
                     fmaf(fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3])), k4[1][0], l4[1][0]));
        } else {
          mt = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 4; r++) mt = fmaxf(mt, fmaf(S[h][r], k4[h][r], l4[h][r]));
        }
        mt = max16(mt);
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
        float lm[2][G8 ? 1 : 4];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int r = 0; r < (G8 ? 1 : 4); r++) lm[h][r] = l4[h][r] - (mb - LIFT);
        if (far_scores(mt)) {
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              constexpr int one = G8 ? 0 : ~0;
              S[h][r] = fmaf(S[h][r], k4[h][r & one], l4[h][r & one]) - mb;
            }
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < (G8 ? 1 : 4); r++) k4[h][r] = 1.0f, lm[h][r] = LIFT;
        }
        half8_t pf;
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float l = 0.0f;
#pragma unroll
          for (int r = 0; r < 4; r++) {
            constexpr int one = G8 ? 0 : ~0;
            const float iv = i4[h][r & one], p = __builtin_amdgcn_exp2f(fmaf(S[h][r], k4[h][r & one], lm[h][r & one]));
            pf[4 * h + r] = (hxa_h)(iv < 1.0f / HXA_Q8_LEAST ? p : p == p ? 0.0f : p);  // a page without a scale: values of 0, whatever the bytes
            l = G8 ? l + p : fmaf(p, iv, l);
          }
          lsum = G8 ? fmaf(l, i4[h][0], lsum) : lsum + l;
        }
#pragma unroll
        for (int g = 0; g < NG; g++) {
          // bytes of two keys side by side, dims 0, 1 (w[..][0]) and 2, 3
          uint32_t w[4][2];
#pragma unroll
          for (int y = 0; y < 4; y++) {
            const uint32_t lo = vr[y >> 1][g][2 * (y & 1)] ^ 0x80808080u, hi = vr[y >> 1][g][2 * (y & 1) + 1] ^ 0x80808080u;
            w[y][0] = __builtin_amdgcn_perm(hi, lo, 0x05010400u);
            w[y][1] = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
          }
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const half2_t bias = {(hxa_h)1152.0f, (hxa_h)1152.0f};
            half8_t v;
#pragma unroll
            for (int y = 0; y < 4; y++) {
              const half2_t z = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w[y][j >> 1], j & 1 ? 0x04030402u : 0x04010400u)) - bias;
              v[2 * y] = z[0];
              v[2 * y + 1] = z[1];
            }
            acc[g][j] = mma16(v, pf, acc[g][j]);
          }
        }
      }
      s0 = s1;
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
template <typename T, int HD, bool G8>
HXA_DEV void any_item_q8(int mode, const KeysQ8 &s, const Item &it, const CachedQ8Args &p, int head0, uint8_t *lds, const Out<T> &out) {
  if (mode == 1) {
    few_item_q8<T, HD, G8>(s, it, (const T *)p.q, p.ldq, head0, p.cs, lds, out);
    return;
  }
  float16_t acc[HD / 32];
  float m, l;
  if (mode == 2) {
    rows_item_q8<T, HD, 2, G8>(s, it, (const T *)p.q, p.ldq, head0, p.cs, lds, acc, m, l);
    rows_out<T, HD, 2>(out, it, head0, 1.0f, lds, acc, m, l);
  } else {
    rows_item_q8<T, HD, 4, G8>(s, it, (const T *)p.q, p.ldq, head0, p.cs, lds, acc, m, l);
    rows_out<T, HD, 4>(out, it, head0, 1.0f, lds, acc, m, l);
  }
}
template <typename T, int HD, bool G8>
__global__ HXA_CAUSAL_BOUNDS void cached_q8_kernel(CachedQ8Args p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int h = blockIdx.x % p.c.H;
  KeysQ8 s{};
  s.k = (const int8_t *)p.c.k;
  s.v = (const int8_t *)p.c.v;
  s.ks = p.ks;
  s.vs = p.vs;
  walk_cache<T, lds_q8<HD>()>(p, h, s, lds, [&](int mode, const Item &it, const Out<T> &out) { any_item_q8<T, HD, G8>(mode, s, it, p, h * p.G, lds, out); });
}

int q8_check(const hxa_kv_cache_q8 *c, int T, int Hq) {
  const int r = hxa_kv_check_q8(c, T, "attention_cached_q8");
  return r != HXA_OK ? r : cached_limits(c->c, T, Hq, "attention_cached_q8");
}

}  // namespace

extern "C" long hxa_attention_cached_q8_ws_bytes(const hxa_kv_cache_q8 *c, int T, int Hq) {
  if (q8_check(c, T, Hq) != HXA_OK || T == 0 || c->c.nseq == 0) return 0;
  return cached_ws(cached_plan(c->c, T, Hq, true, wg_slots(c->c.hd), true), c->c, T, Hq);
}

extern "C" int hxa_attention_cached_q8(const hxa_kv_cache_q8 *cache, const void *q, long ldq, void *o, long ldo, int T, int Hq, float scale,
                                       void *ws, long ws_bytes, void *stream) {
  const int r = q8_check(cache, T, Hq);
  if (r != HXA_OK) return r;
  CachedQ8Args p{};
  p.ks = cache->kscale;
  p.vs = cache->vscale;
  return cached_call(
      p, cache->c, q, ldq, o, ldo, T, Hq, scale, ws, ws_bytes, (hipStream_t)stream, "attention_cached_q8", true,
      [](auto ty, auto hdc, const CachedPlan &pl, const hxa_kv_cache &d) {
        constexpr int HD = decltype(hdc)::value;
        // pages hold whole groups of eight keys, counted from where a range may begin
        const bool g8 = d.page % 8 == 0 && (d.prefix_len % 8 == 0 || pl.x_first == d.prefix_len);
        return std::make_tuple(g8 ? cached_q8_kernel<decltype(ty), HD, true> : cached_q8_kernel<decltype(ty), HD, false>, lds_q8<HD>() + 4096, g8 ? 6 : 0);
      });
}
