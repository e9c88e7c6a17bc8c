// Causal attention with grouped heads: over packed prompts (hxa_attention_causal) and over a paged cache with a shared prefix
// (hxa_attention_cached). fp16 / bf16 in and out, heads of 64, 128 or 256, fp32 softmax.
//
// Rows. The G = Hq / Hk query heads that read one key head are rows of one problem: row R of a sequence is token R / G, head
// h G + R % G. A workgroup of 4 waves takes consecutive rows of one sequence and one key head, so a key tile is loaded once for all G
// heads, and the rows of a tile span few tokens: less of the diagonal is computed to be masked.
//
// Online softmax: over 64-key tiles S = K Q^T, p = 2^(c S - c m) with c = scale log2(e) and the running maximum m, l += p,
// O^T = V^T P^T. O and l are rescaled only when m grows by more than 5.5 nats (p <= e^5.5 otherwise, well within fp16).
// p is rounded to the input type, as the matrix product takes it, and l adds it as rounded: equal values come out as they are, and a
// weight's rounding costs at most half a step of it on |v - o|. S, m, l and O stay in fp32.
//
// Tiles move global -> LDS directly, rows of K and V as they lie in memory, double buffered, one barrier a tile. V is transposed
// on its way out of LDS (ds_read_b64_tr_b16: 16 lanes that read 4 keys x 16 dims get 4 keys of one dim each), so no
// caller has to keep V transposed. K row order and chunk swizzles are chosen so that the scores in the accumulators
// are the B operand of the P V product and that the reads of 16 (32) lanes spread over the 64 LDS banks.
//
// Modes of a workgroup:
//   rows (W = 4): 128 rows, 32 a wave, every wave all 64 keys of a tile (32x32x16 MFMAs)
//   rows (W = 2): 64 rows, the two halves of the tile's keys to two waves each, joined at the end
//   few rows:     16 rows, 16 keys of the tile to each wave (16x16 MFMAs), joined at the end; bound by reading the cache
//
// Bound, and measured (32 query heads on 8 key heads of 128, bf16):
//   prompts: the matrix instructions, at the board's power limit from ~8000 tokens on (16384 tokens 1.89 - 1.97 ms on five cards, 1.12 - 1.16 PFLOP/s, 2.19
//            on a sixth); a shorter batch by its
//            longest block, whose tiles follow each other (a tile of 128 rows 2300 cycles alone, 3050 with two workgroups a CU, of them 1024 MFMAs)
//   single tokens: reading the keys (16 tokens over 90000 keys behind 32768 shared ones 99 us, 5.1 TB/s; 64 over 30000 behind 4096 40 us)
// Two workgroups a CU, one's softmax beside the other's matrix products, did better than one that interleaves the tiles' phases itself.
//
// What a mask hides has no part in a result: hidden scores become -inf before the maximum; values of keys that no row of the workgroup sees are
// zeroed in LDS (0 x NaN would be NaN), and values of keys that only some rows see are, where they are not finite, taken out of the
// matrix product and added, key by key, by the rows that see them at the end.
#include "causal_attn.h"

namespace {

template <typename T, int HD, bool PERM, bool PAGED>
struct Loader {
  typedef Geo<T, HD> G_;
  typedef Swz<T, HD, PERM> S_;
  const Keys<T> &s;
  const Item &it;
  uint8_t *lds;
  int lane, wave;
  uint32_t koff[G_::NOFF], voff[G_::NOFF];  // contiguous: byte offsets within a whole tile; paged: chunk offsets within a row
  int ent;           // paged: the page entry of this lane's key in the tile that is opened next
  unsigned in_page;  // and the key's place in that page
  uint32_t row[PAGED ? G_::NLD : 1];  // paged: page rows that this lane's loads of the tile opened last read
  HXA_DEV Loader(const Keys<T> &s_, const Item &it_, uint8_t *lds_, int lane_, int wave_) : s(s_), it(it_), lds(lds_), lane(lane_), wave(wave_) {
    ent = -1;
    in_page = 0;
#pragma unroll
    for (int j = 0; j < G_::NOFF; j++) {
      const int r = (j * 4 + wave) * G_::RPL + lane / G_::CH, c = lane % G_::CH;
      const int kr = PERM ? krow_key(r) : r;
      const int ck = c ^ S_::fk(r), cv = c ^ S_::fv(r);
      koff[j] = PAGED ? ck * 16u : ((uint32_t)kr * (uint32_t)s.ldk + ck * 8) * 2u;
      voff[j] = PAGED ? cv * 16u : ((uint32_t)kr * (uint32_t)s.ldv + cv * 8) * 2u;
    }
    if (PAGED) entry(0);
  }
  HXA_DEV uint8_t *kbuf(int i) const { return lds + (i & 1) * G_::TB; }
  HXA_DEV uint8_t *vbuf(int i) const { return lds + (2 + (i & 1)) * G_::TB; }
  HXA_DEV void entry(int i) {  // look up the page of this lane's key of tile i
    const int x = it.x0 + i * KT + lane;
    ent = -1;
    if (x < it.x1) {
      const bool pre = x < s.P;
      const unsigned y = pre ? x : x - s.P;
      ent = (pre ? s.prefix : s.table)[s.slot(y, in_page)];
    }
  }
  // tile i: where its keys lie, and the mask of those that are there; its loads follow
  HXA_DEV uint64_t open(int i) {
    const int key0 = it.x0 + i * KT;
    if constexpr (PAGED) {
      const bool ok = (unsigned)ent < (unsigned)s.npages;  // (-1 past x1)
      const uint32_t at = ok ? ((uint32_t)ent * s.H + s.h) * s.page + in_page : 0;  // < 2^32: checked on the host
      const uint64_t mask = __ballot(ok);
      if (key0 + KT < it.x1) entry(i + 1);
#pragma unroll
      for (int j = 0; j < G_::NLD; j++) {
        const int r = (j * 4 + wave) * G_::RPL + lane / G_::CH;
        row[j] = __shfl((int)at, PERM ? krow_key(r) : r);
      }
      return mask;
    } else {
      const int n = it.x1 - key0;
      return n >= KT ? ~0ull : (1ull << n) - 1;
    }
  }
  // whether tile i lies below x1, so that its loads need no clamp (paged: never one)
  HXA_DEV bool whole(int i) const { return PAGED || it.x0 + (i + 1) * KT <= it.x1; }
  // load n of the 2 NLD of this wave for tile i, the one opened last: K's, then V's. WHOLE: whole(i)
  template <bool WHOLE>
  HXA_DEV void load(int i, int n) {
    const bool V = n >= G_::NLD;
    const int j = V ? n - G_::NLD : n, blk = j * 4 + wave;
    uint8_t *to = (V ? vbuf(i) : kbuf(i)) + blk * 1024;
    const uint32_t off = V ? voff[j % G_::NOFF] : koff[j % G_::NOFF];
    if constexpr (PAGED) {
      g2l16_opaque((const uint8_t *)(V ? s.v : s.k) + (uint64_t)row[j] * G_::RB + off, to);
    } else {
      const int key0 = it.x0 + i * KT;
      const long ld = V ? s.ldv : s.ldk;
      const T *t = (V ? s.v : s.k) + (long)key0 * ld;
      if (WHOLE) {
        g2l16_sbase(t + (long)(j / G_::NOFF * G_::NOFF * 4 * G_::RPL) * ld, off, to);
      } else {  // rows past the keys read the last one
        int ln = lane;
        asm volatile("" : "+v"(ln));  // opaque: the loop keeps none of these addresses in registers
        const int r = blk * G_::RPL + ln / G_::CH, c = ln % G_::CH;
        const int from = min(PERM ? krow_key(r) : r, it.x1 - 1 - key0), ch = c ^ (V ? S_::fv(r) : S_::fk(r));
        g2l16_sbase(t, ((uint32_t)from * (uint32_t)ld + ch * 8) * 2u, to);
      }
    }
  }
  HXA_DEV void load_all(int i) {
    if (whole(i)) {
#pragma unroll
      for (int n = 0; n < 2 * G_::NLD; n++) load<true>(i, n);
    } else {
#pragma unroll
      for (int n = 0; n < 2 * G_::NLD; n++) load<false>(i, n);
    }
  }
  // the rows of key x, which is there
  HXA_DEV void rows(int x, const T *&kr, const T *&vr) const {
    if constexpr (PAGED) {
      const unsigned y = x < s.P ? x : x - s.P;
      unsigned in;
      const uint32_t e = (x < s.P ? s.prefix : s.table)[s.slot(y, in)];
      const uint64_t r = (uint64_t)((e * s.H + s.h) * s.page + in) * HD;
      kr = s.k + r;
      vr = s.v + r;
    } else {
      kr = s.k + (long)x * s.ldk;
      vr = s.v + (long)x * s.ldv;
    }
  }
};

// The values of tile i where the mask cuts it: rows of keys that are not there (km) become zeros; so do rows that only some rows of
// the workgroup see (keys past lim_min) and that hold an infinity or NaN: their mask is returned. Whole workgroup, ends with a barrier.
template <typename T, int HD, bool PERM>
HXA_DEV uint64_t fix_v(uint8_t *vb, uint8_t *flags, int key0, uint64_t km, int lim_min, int tid) {
  constexpr int RB = HD * 2, N = RB / 4 / 16;
  const int key = tid >> 2, lane = tid & 63;
  uint8_t *p = vb + (PERM ? krow_key(key) : key) * RB + (tid & 3) * (RB / 4);  // (krow_key is its own inverse)
  const bool dead = !((km >> key) & 1);
  bool bad = false;
  if (!dead && key0 + key > lim_min) {
    // a magnitude of at least the exponent's ones carries into the sign's place
    uint32_t carry = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const uint4_t x = *(const uint4_t *)(p + 16 * i);
#pragma unroll
      for (int e = 0; e < 4; e++) carry |= (x[e] & 0x7fff7fffu) + (0x80008000u - HxaVec<T>::EXP);
    }
    bad = (carry & 0x80008000u) != 0;
  }
  const uint64_t b = __ballot(bad);
  if (dead || ((b >> (lane & 60)) & 15)) {
#pragma unroll
    for (int i = 0; i < N; i++) *(uint4_t *)(p + 16 * i) = (uint4_t){0, 0, 0, 0};
  }
  const uint64_t rows = __ballot(lane < 16 && ((b >> (4 * (lane & 15))) & 15)) & 0xffff;
  if (lane == 0) ((uint16_t *)flags)[tid >> 6] = (uint16_t)rows;
  reads_done_barrier();
  const uint64_t f = *(const uint64_t *)flags;
  return ((uint64_t)__builtin_amdgcn_readfirstlane((int)(f >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)f);
}

// ---- rows modes ----
// One workgroup's rows against keys [x0, x1): the wave's O^T (lane (g, ql): row 32 rw + ql, dims 32 d + 8 i + 4 g .. + 3 in
// acc[d][4 i ..]), its maximum m and its row sum l (of both halves of the lanes).
template <typename T, int HD, int W, bool PAGED>
HXA_DEV void rows_item(const Keys<T> &s, const Item &it, const T *q, long ldq, int head0, float c, uint8_t *lds, float16_t (&acc)[HD / 32],
                       float &mrun, float &lsum) {
  typedef Geo<T, HD> G_;
  typedef typename HxaVec<T>::v8 v8;
  typedef typename HxaVec<T>::v4 v4;
  typedef Swz<T, HD, true> S_;
  constexpr int NB = W == 4 ? 2 : 1;       // 32-key blocks of a tile for each wave
  constexpr int ND = HD / 32, AK = 2, AV = 3;  // dim blocks; fragments of K (V) read ahead
  const int tid = this_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = W == 4 ? wave : wave & 1, kh = W == 4 ? 0 : wave >> 1;
  const int g = lane >> 5, ql = lane & 31;

  const int R = it.r0 + rw * 32 + ql;
  const bool qok = R < it.nrows;
  const int Rc = qok ? R : it.nrows - 1;
  int rest;
  const int tok = row_tok(it, Rc, rest);
  const T *qp = q + (long)(it.tok0 + tok) * ldq + (long)(head0 + rest) * HD;
  v8 qf[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; i++) qf[i] = *(const v8 *)(qp + i * 16 + 8 * g);
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
  Loader<T, HD, true, PAGED> ld(s, it, lds, lane, wave);
  uint64_t km = ld.open(0);
  ld.load_all(0);

  // V^T fragment of 32 dims d, keys kb .. kb + 15 (kb a multiple of 16): lane (g, ql) dim 32 d + ql, keys kb + 8 g .. + 7; 16 lanes read
  // 4 keys x 16 dims at a time: rows 4 g .. + 3 and 4 g + 8 .. + 3
  const int vrow = 4 * g + ((lane & 15) >> 2);
  const int vlow = ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) << 4) + (lane & 1) * 8;  // within 64 bytes
  uint32_t vat[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) vat[d] = vrow * G_::RB + (((d << 2) ^ S_::fv(vrow)) << 4) + vlow;  // fv(vrow + 8) is the same

  // One tile for this wave. MAIN: every row sees all of it, and the next tile is whole: its loads are issued one beside each
  // product of K (64 bytes a clock and CU: eight in a row hold a wave for 600 cycles). Fragments are read AK (AV) products ahead: without
  // the fences each is read right before its use, a LDS latency a product.
  auto tile = [&](int i, uint64_t kmi, bool cut, auto main) {
    constexpr bool MAIN = decltype(main)::value;
    const int key0 = it.x0 + i * KT;
    const uint8_t *kb = ld.kbuf(i), *vb = ld.vbuf(i);
    auto kfrag = [&](int ds, int b) {
      const int row = (b + kh) * 32 + ql, ch = 2 * ds + g;
      return *(const v8 *)(kb + row * G_::RB + ((ch ^ S_::fk(row)) << 4));
    };
    auto vfrag = [&](int n) {  // n = (16-key slice) ND + dims
      const uint8_t *at = vb + vat[n % ND] + (kh * 32 + n / ND * 16) * G_::RB;
      return __builtin_shufflevector(read_tr<v4>(at), read_tr<v4>(at + 8 * G_::RB), 0, 1, 2, 3, 4, 5, 6, 7);
    };
    float16_t S[NB];
    v8 kf[AK + 1][NB];
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
      if constexpr (MAIN) ld.template load<true>(i + 1, ds);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < NB; b++) S[b] = mma32(kf[ds % (AK + 1)][b], qf[ds], ds == 0 ? (float16_t){} : S[b]);
    }
    __builtin_amdgcn_sched_barrier(0);
    v8 vf[AV + 1];
#pragma unroll
    for (int n = 0; n < AV; n++) vf[n] = vfrag(n);
    __builtin_amdgcn_sched_barrier(0);
    if (!MAIN && cut) {
      // a row's limit hides the keys past x1 too (a range that ends before it ends with a tile); pages that are not there need the mask
      const int n = lim - key0 - 32 * kh - 8 * g, left = it.x1 - key0;
      if (!PAGED || kmi == (left >= KT ? ~0ull : (1ull << left) - 1)) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int r = 0; r < 16; r++)
            if (32 * b + 16 * (r >> 3) + (r & 7) > n) S[b][r] = -INFINITY;
      } else {
        const uint64_t see = kmi >> (32 * kh + 8 * g);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int k = 32 * b + 16 * (r >> 3) + (r & 7);
            if (k > n || !((see >> k) & 1)) S[b][r] = -INFINITY;
          }
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
    const bool need = (mt - mrun) * c > RESCALE2;  // also when mrun is still -inf
    if (__any(need)) {
      const float alpha = need ? __builtin_amdgcn_exp2f((mrun - mt) * c) : 1.0f;
      if (need) mrun = mt;
      lsum *= alpha;
#pragma unroll
      for (int d = 0; d < ND; d++) acc[d] *= alpha;
    }
    const float mb = mrun == -INFINITY ? 0.0f : mrun * c;
    v8 pf[NB][2];
    float ls[2] = {0.0f, 0.0f};
    // two probabilities: rounded to the type, and their sum as rounded
    auto expo2 = [&](int n) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(S[n >> 4][n & 15], c, -mb));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(S[n >> 4][(n & 15) + 1], c, -mb));
      const typename HxaVec<T>::v2 h = {(T)p0, (T)p1};
      pf[n >> 4][(n >> 3) & 1][n & 7] = h[0];
      pf[n >> 4][(n >> 3) & 1][(n & 7) + 1] = h[1];
      ls[(n >> 1) & 1] = sum2(h, ls[(n >> 1) & 1]);
    };
    // P V of a 32-key block beside the exponentials of the next one (in the compiler's order: fences as above change nothing, and cost 5%
    // with heads of 64)
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
  };

  int i = 0;
  const int nmain = PAGED ? min((lim_min + 1 - it.x0) / KT, nt - 1) : min(lim_min + 1 - it.x0, it.x1 - it.x0 - KT) / KT;
  while (i < nmain && km == ~0ull) {
    wait_vm<0>();
    reads_done_barrier();  // tile i has landed; every wave is done with tile i - 1
    km = ld.open(i + 1);
    tile(i, ~0ull, false, std::true_type{});
    i++;
  }
  // flags of the tiles whose values fix_v took out: only the last three can hold keys that some rows see and some do not
  uint64_t apart[3] = {0, 0, 0};
  for (; i < nt; i++) {
    wait_vm<0>();
    reads_done_barrier();
    const int key0 = it.x0 + i * KT;
    const uint64_t kmi = km;
    if (i + 1 < nt) {
      km = ld.open(i + 1);
      ld.load_all(i + 1);
    }
    const bool cut = kmi != ~0ull || key0 + KT - 1 > lim_min;
    if (cut) {
      const uint64_t f = fix_v<T, HD, true>(ld.vbuf(i), lds + G_::FLAGS, key0, kmi, lim_min, tid);
      if (i == nt - 1) apart[0] = f;
      if (i == nt - 2) apart[1] = f;
      if (i == nt - 3) apart[2] = f;
    }
    if (wave_max >= key0 + 32 * kh) tile(i, kmi, cut, std::false_type{});
  }
  float lo, hi;
  halves(lsum, lo, hi);
  lsum = lo + hi;
  if (apart[0] | apart[1] | apart[2]) {  // the values taken out, key by key, to the rows that see them
    const float mb = mrun == -INFINITY ? 0.0f : mrun * c;
#pragma unroll 1
    for (int k = 0; k < 3; k++) {
      uint64_t left = k == 0 ? apart[0] : k == 1 ? apart[1] : apart[2];
      for (; left; left &= left - 1) {
        const int f = __builtin_ctzll(left), x = it.x0 + (nt - 1 - k) * KT + f;
        if (W == 2 && f >> 5 != kh) continue;
        const T *kr, *vr;
        ld.rows(x, kr, vr);
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 16; j++) {
          const v8 kk = *(const v8 *)(kr + 16 * j + 8 * g);
#pragma unroll
          for (int e = 0; e < 8; e++) dot = fmaf((float)kk[e], (float)qf[j][e], dot);
        }
        halves(dot, lo, hi);
        const float p = __builtin_amdgcn_exp2f(fmaf(lo + hi, c, -mb));
        if (lim >= x) {
#pragma unroll
          for (int d = 0; d < HD / 32; d++)
#pragma unroll
            for (int e4 = 0; e4 < 4; e4++) {
              const v4 v = *(const v4 *)(vr + 32 * d + 8 * e4 + 4 * g);
#pragma unroll
              for (int e = 0; e < 4; e++) acc[d][4 * e4 + e] += p * (float)v[e];
            }
        }
      }
    }
  }
  if constexpr (W == 2) {  // join the halves of the keys: the second half's waves hand theirs to the first's
    constexpr int PART = HD / 8 * 64;  // float4 of a wave's accumulators
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
      const float a0 = __builtin_amdgcn_exp2f((mrun - mz) * c), a1 = __builtin_amdgcn_exp2f((m1 - mz) * c);
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

// ---- few rows ----
// 16 rows against keys [x0, x1), each wave 16 keys of every tile, and the result out
template <typename T, int HD, bool PAGED>
HXA_DEV void few_item(const Keys<T> &s, const Item &it, const T *q, long ldq, int head0, float c, uint8_t *lds, const Out<T> &out) {
  typedef Geo<T, HD> G_;
  typedef typename HxaVec<T>::v8 v8;
  typedef typename HxaVec<T>::v4 v4;
  typedef Swz<T, HD, false> S_;
  constexpr int ND = HD / 16;
  const int tid = this_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int gi = lane >> 4, ql = lane & 15;
  const int R = it.r0 + ql, last = it.nrows - 1, Rc = min(R, last);
  float4_t acc[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) acc[d] = (float4_t){};
  float mrun = -INFINITY, lsum = 0.0f;
  const int nt = (it.x1 - it.x0 + KT - 1) / KT;
  if (nt > 0) {
    Loader<T, HD, false, PAGED> ld(s, it, lds, lane, wave);
    uint64_t km_next = ld.open(0);
    ld.load_all(0);
    int rest;
    const int tok = row_tok(it, Rc, rest);
    const T *qp = q + (long)(it.tok0 + tok) * ldq + (long)(head0 + rest) * HD;
    v8 qf[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; i++) qf[i] = *(const v8 *)(qp + i * 32 + 8 * gi);
    const int lim = tok_limit(it, tok), lim_min = row_limit(it, it.r0);
    const int vkey = 16 * wave + 4 * gi + (ql >> 2);
    const int krow = 16 * wave + ql;
    uint64_t apart[2] = {0, 0};  // flags of the tiles whose values fix_v took out
    for (int i = 0; i < nt; i++) {
      wait_vm<0>();
      reads_done_barrier();
      const uint64_t km = km_next;
      const int key0 = it.x0 + i * KT;
      const bool more = i + 1 < nt;
      if (more) {
        km_next = ld.open(i + 1);
        ld.load_all(i + 1);
      }
      const bool cut = km != ~0ull || key0 + KT - 1 > lim_min;
      if (cut) {
        const uint64_t f = fix_v<T, HD, false>(ld.vbuf(i), lds + G_::FLAGS, key0, km, lim_min, tid);
        if (i == nt - 1) apart[0] = f;
        if (i == nt - 2) apart[1] = f;
      }
      const uint8_t *kb = ld.kbuf(i) + krow * G_::RB, *vb = ld.vbuf(i) + vkey * G_::RB;
      float4_t S = {};
#pragma unroll
      for (int ds = 0; ds < HD / 32; ds++) S = mma16(*(const v8 *)(kb + (((4 * ds + gi) ^ S_::fk(krow)) << 4)), qf[ds], S);
      if (cut) {
        const int n = lim - key0;
        const uint64_t see = (km & (n >= 63 ? ~0ull : n < 0 ? 0ull : (2ull << n) - 1)) >> (16 * wave + 4 * gi);
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (!((see >> r) & 1)) S[r] = -INFINITY;
      }
      const float mt = max16(fmaxf(fmaxf(S[0], S[1]), fmaxf(S[2], S[3])));
      const bool need = (mt - mrun) * c > RESCALE2;
      if (__any(need)) {
        const float alpha = need ? __builtin_amdgcn_exp2f((mrun - mt) * c) : 1.0f;
        if (need) mrun = mt;
        lsum *= alpha;
#pragma unroll
        for (int d = 0; d < ND; d++) acc[d] *= alpha;
      }
      const float mb = mrun == -INFINITY ? 0.0f : mrun * c;
      v4 pf;
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const typename HxaVec<T>::v2 h = {(T)__builtin_amdgcn_exp2f(fmaf(S[r], c, -mb)), (T)__builtin_amdgcn_exp2f(fmaf(S[r + 1], c, -mb))};
        pf[r] = h[0];
        pf[r + 1] = h[1];
        lsum = sum2(h, lsum);
      }
#pragma unroll
      for (int d = 0; d < ND; d++) {
        const int ch = 2 * d + ((ql & 3) >> 1);
        acc[d] = mma16h(read_tr<v4>(vb + ((ch ^ S_::fv(vkey)) << 4) + (ql & 1) * 8), pf, acc[d]);
      }
    }
    lsum = add16(lsum);
    if (apart[0] | apart[1]) {  // (16 rows span at most 16 tokens)
      const float mb = mrun == -INFINITY ? 0.0f : mrun * c;
#pragma unroll 1
      for (int k = 0; k < 2; k++) {
        uint64_t left = k == 0 ? apart[0] : apart[1];
        for (; left; left &= left - 1) {
          const int f = __builtin_ctzll(left), x = it.x0 + (nt - 1 - k) * KT + f;
          if (f >> 4 != wave) continue;
          const T *kr, *vr;
          ld.rows(x, kr, vr);
          float dot = 0.0f;
#pragma unroll
          for (int j = 0; j < HD / 32; j++) {
            const v8 kk = *(const v8 *)(kr + 32 * j + 8 * gi);
#pragma unroll
            for (int e = 0; e < 8; e++) dot = fmaf((float)kk[e], (float)qf[j][e], dot);
          }
          const float p = __builtin_amdgcn_exp2f(fmaf(add16(dot), c, -mb));
          if (lim >= x) {
#pragma unroll
            for (int d = 0; d < ND; d++) {
              const v4 v = *(const v4 *)(vr + 16 * d + 4 * gi);
#pragma unroll
              for (int e = 0; e < 4; e++) acc[d][e] += p * (float)v[e];
            }
          }
        }
      }
    }
  }
  // join the four waves: wave w takes the dims [w HD / 4, (w + 1) HD / 4)
  reads_done_barrier();
  float4_t *ox = (float4_t *)lds;                    // [wave][d][lane]
  float2_t *mlx = (float2_t *)(lds + ND * 4 * 1024);  // [wave][row]
#pragma unroll
  for (int d = 0; d < ND; d++) ox[(wave * ND + d) * 64 + lane] = acc[d];
  // a sum of -0: as in rows_out
  const bool bad = lsum == 0.0f && zero_times_bad(acc, 0x1000100010001ull << ql);
  if (gi == 0) mlx[wave * 16 + ql] = (float2_t){mrun, bad ? -0.0f : lsum};
  reads_done_barrier();
  float m = -INFINITY, l = 0.0f, a[4];
#pragma unroll
  for (int w = 0; w < 4; w++) m = fmaxf(m, mlx[w * 16 + ql][0]);
  const float mz = m == -INFINITY ? 0.0f : m;
  bool kept = false;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const float2_t x = mlx[w * 16 + ql];
    a[w] = __builtin_amdgcn_exp2f((x[0] - mz) * c);
    l += x[1] * a[w];
    kept |= is_minus_0(x[1]);
  }
  if (R >= it.nrows) return;
  int rest;
  const long tok = it.tok0 + row_tok(it, R, rest);
  const int head = head0 + rest;
  const long row = tok * out.Hq + head, at = out.slot * out.rows + row;
  if (out.part != nullptr) {
    if (wave == 0 && gi == 0) out.ml[row * out.nslots + out.slot] = (float2_t){m == -INFINITY ? m : m * c, l == 0.0f && kept ? -0.0f : l};
    if (l == 0.0f && !kept) return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int d4 = 0; d4 < ND / 4; d4++) {
    const int d = wave * (ND / 4) + d4;
    float4_t o = {};
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float4_t x = ox[(w * ND + d) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] += x[e] * a[w];
    }
    if (out.part != nullptr) {
      *(float4_t *)(out.part + at * HD + 16 * d + 4 * gi) = o;
    } else {
      v4 x;
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = l == 0.0f ? (T)0.0f : (T)(o[e] * inv);
      *(v4 *)(out.o + tok * out.ldo + (long)head * HD + 16 * d + 4 * gi) = x;
    }
  }
}

struct CausalArgs {
  const void *q, *k, *v;
  void *o;
  long ldq, ldk, ldv, ldo;
  const int *cu;
  int T, nseq, G, Hk, first;
  uint32_t gm;
  float c;
};

template <typename T, int HD, int W>
__global__ HXA_CAUSAL_BOUNDS void causal_kernel(CausalArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int h = blockIdx.x % p.Hk, blk = blockIdx.x / p.Hk;  // key heads innermost: with 8 of them each XCD keeps its own head's keys
  const Block b = find_block<Wave>(p.cu, p.nseq, p.T, p.G, 32 * W, blk, p.first);
  if (b.first < 0) return;
  const long row0 = b.b;
  Keys<T> s{};
  s.k = (const T *)p.k + row0 * p.ldk + (long)h * HD;
  s.v = (const T *)p.v + row0 * p.ldv + (long)h * HD;
  s.ldk = p.ldk;
  s.ldv = p.ldv;
  Item it;
  it.r0 = b.first;
  it.nrows = b.n * p.G;
  it.G = p.G;
  it.gm = p.gm;
  it.tok0 = b.b;
  it.base = 0;
  it.cap = b.n - 1;
  it.least = -1;
  it.causal = true;
  it.x0 = 0;
  it.x1 = row_limit(it, min(it.r0 + 32 * W, it.nrows) - 1) + 1;
  float16_t acc[HD / 32];
  float m, l;
  rows_item<T, HD, W, false>(s, it, (const T *)p.q, p.ldq, h * p.G, p.c, lds, acc, m, l);
  const Out<T> out{(T *)p.o, p.ldo, nullptr, nullptr, 0, 0, 0, 0};
  rows_out<T, HD, W>(out, it, h * p.G, p.c, lds, acc, m, l);
}

// ---- over the cache ----
template <typename T, int HD>
HXA_DEV void any_item(int mode, const Keys<T> &s, const Item &it, const CachedArgs &p, int head0, uint8_t *lds, const Out<T> &out) {
  if (mode == 1) {
    few_item<T, HD, true>(s, it, (const T *)p.q, p.ldq, head0, p.cs, lds, out);
    return;
  }
  float16_t acc[HD / 32];
  float m, l;
  if (mode == 2) {
    rows_item<T, HD, 2, true>(s, it, (const T *)p.q, p.ldq, head0, p.cs, lds, acc, m, l);
    rows_out<T, HD, 2>(out, it, head0, p.cs, lds, acc, m, l);
  } else {
    rows_item<T, HD, 4, true>(s, it, (const T *)p.q, p.ldq, head0, p.cs, lds, acc, m, l);
    rows_out<T, HD, 4>(out, it, head0, p.cs, lds, acc, m, l);
  }
}
template <typename T, int HD>
__global__ HXA_CAUSAL_BOUNDS void cached_kernel(CachedArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int h = blockIdx.x % p.c.H;
  Keys<T> s{};
  s.k = (const T *)p.c.k;
  s.v = (const T *)p.c.v;
  walk_cache<T, Geo<T, HD>::LDS>(p, h, s, lds, [&](int mode, const Item &it, const Out<T> &out) { any_item<T, HD>(mode, s, it, p, h * p.G, lds, out); });
}

}  // namespace

extern "C" int hxa_attention_causal(int dtype, const void *q, long ldq, const void *k, long ldk, const void *v, long ldv, void *o, long ldo,
                                    int T, const int *cu, int nseq, int Hq, int Hk, int hd, float scale, void *stream) {
  if (dtype != HXA_DT_F16 && dtype != HXA_DT_BF16) return hxa_set_error(HXA_E_MODE, "attention_causal: dtype %d", dtype);
  if (hd != 64 && hd != 128 && hd != 256) return hxa_set_error(HXA_E_MODE, "attention_causal: heads of %d", hd);
  if (T < 0 || T > HXA_MAX_ROWS || nseq < 0 || Hq <= 0 || Hk <= 0 || Hq > HXA_MAX_HEADS || Hq % Hk || (long)T * Hq >= 1L << 30)
    return hxa_set_error(HXA_E_ARG, "attention_causal: T=%d nseq=%d Hq=%d Hk=%d", T, nseq, Hq, Hk);
  if (!(scale > 0.0f) || !std::isfinite(scale)) return hxa_set_error(HXA_E_ARG, "attention_causal: scale %g", (double)scale);
  if (T == 0 || nseq == 0) return HXA_OK;
  if (!rows_ok(q, ldq, Hq, hd) || !rows_ok(k, ldk, Hk, hd) || !rows_ok(v, ldv, Hk, hd) || !rows_ok(o, ldo, Hq, hd))
    return hxa_set_error(HXA_E_ARG, "attention_causal: pointers null or not 16-byte aligned, or strides (%ld %ld %ld %ld)", ldq, ldk, ldv, ldo);
  if (ldk >= 1 << 24 || ldv >= 1 << 24) return hxa_set_error(HXA_E_ARG, "attention_causal: strides of %ld, %ld", ldk, ldv);
  if (!cu || (uintptr_t)cu % 4) return hxa_set_error(HXA_E_ARG, "attention_causal: cu");
  const int G = Hq / Hk;
  const long RT = (long)T * G;
  CausalArgs p{q, k, v, o, ldq, ldk, ldv, ldo, cu, T, nseq, G, Hk, second_layer(hd, causal_ncu(), Hk), recip(G), scale * L2E};
  // 64 rows a workgroup while 128 would leave workgroup places free
  const int mode = (RT / 128 + nseq) * Hk < wg_slots(hd) ? 2 : 4;
  const int rb = mode == 2 ? 64 : 128;
  const long wgs = (RT / rb + nseq) * Hk;
  if (wgs >= 1L << 24) return hxa_set_error(HXA_E_ARG, "attention_causal: T=%d nseq=%d Hq=%d are too many blocks", T, nseq, Hq);
  return by_type(dtype, hd, [&](auto ty, auto hdc, int id) -> int {
    typedef decltype(ty) T_;
    constexpr int HD = decltype(hdc)::value;
    const auto f = mode == 2 ? causal_kernel<T_, HD, 2> : causal_kernel<T_, HD, 4>;
    const int r = allow_lds((const void *)f, Geo<T_, HD>::LDS, 2 * id + (mode == 2));
    if (r != HXA_OK) return hxa_set_error(r, "attention_causal: %d bytes of LDS", Geo<T_, HD>::LDS);
    hxa_launch(f, dim3((unsigned)wgs), dim3(256), Geo<T_, HD>::LDS, (hipStream_t)stream, p);
    return launched("attention_causal");
  });
}

static int cached_check(const hxa_kv_cache *c, int T, int Hq) {
  const int r = hxa_kv_check(c, T, "attention_cached");
  return r != HXA_OK ? r : cached_limits(*c, T, Hq, "attention_cached");
}

extern "C" long hxa_attention_cached_ws_bytes(const hxa_kv_cache *c, int T, int Hq) {
  if (cached_check(c, T, Hq) != HXA_OK || T == 0 || c->nseq == 0) return 0;
  return cached_ws(cached_plan(*c, T, Hq, true, wg_slots(c->hd)), *c, T, Hq);
}

extern "C" int hxa_attention_cached(const hxa_kv_cache *c, const void *q, long ldq, void *o, long ldo, int T, int Hq, float scale, void *ws,
                                    long ws_bytes, void *stream) {
  const int r = cached_check(c, T, Hq);
  if (r != HXA_OK) return r;
  CachedArgs p{};
  return cached_call(p, *c, q, ldq, o, ldo, T, Hq, scale, ws, ws_bytes, (hipStream_t)stream, "attention_cached", false, [](auto ty, auto hdc, const CachedPlan &, const hxa_kv_cache &) {
    typedef decltype(ty) T_;
    constexpr int HD = decltype(hdc)::value;
    return std::make_tuple(cached_kernel<T_, HD>, Geo<T_, HD>::LDS + 4096, 0);
  });
}
