// Which rows and keys a workgroup of the causal attention kernels takes: the block of a batch of prompts, and the work over the cache.
// Index arithmetic only, by a whole wave: lanes hold sequences. What differs between lanes goes through the wave W (a value a lane, W::I;
// map, ballot, scan, get), everything else is the same in all lanes. The kernels run it on the wave's instructions; the CPU tests run the
// same source with 64 values in an array, and count that every row and tile is taken once.
#pragma once
#include <stdint.h>

#include "../../include/hexanima_hip.h"

#ifdef __HIP__
#define HXA_ANY __host__ __device__ __forceinline__
#else
#define HXA_ANY inline
#endif

namespace {

HXA_ANY int imin(int a, int b) { return a < b ? a : b; }
HXA_ANY int imax(int a, int b) { return a > b ? a : b; }
HXA_ANY long ceil_div(long a, long b) { return (a + b - 1) / b; }

constexpr int KT = 64;  // keys a tile

// ---- prompts ----
struct Block {
  int seq, b, n;  // the sequence, its first row in the call and its tokens
  int first;      // first row (token x G + head) of the block within the sequence; -1: none
};
// Block `blk` of the grid: sequence i has ceil(n_i G / RB) blocks, and a block's keys grow with its place in the sequence. Up to 16
// sequences, places are dealt from the highest down over all of them (the longest first); of blocks first .. 2 first - 1 the order is
// reversed (second_layer below). More sequences: in their order, each from its end. cu's entries are clamped into [0, T].
template <class W>
HXA_ANY Block find_block(const int *__restrict__ cu, int nseq, int T, int G, int RB, int blk, int first) {
  typedef typename W::I I;
  int seen = 0;  // blocks of the sequences before `base`
  for (int base = 0; base < nseq; base += 64) {
    const I b = W::map([&](int i) { return i < nseq ? imin(imax(cu[i], 0), T) : 0; }, W::lanes(base));
    const I e = W::map([&](int i, int b0) { return i < nseq ? imin(imax(cu[i + 1], b0), T) : 0; }, W::lanes(base), b);
    const I nb = W::map([&](int b0, int e0) { return ((e0 - b0) * G + RB - 1) / RB; }, b, e);  // (T G < 2^31 - RB: checked on the host)
    const I inc = W::scan(nb);
    const int total = W::get(inc, 63);
    Block r{0, 0, 0, -1};
    int w, j;
    if (nseq <= 16) {
      if (blk >= total) return r;
      if (blk >= first && blk < 2 * first) blk = imin(2 * first, total) - 1 - (blk - first);
      w = 0;
      j = total - 1 - blk;
      if (nseq > 1) {
        // S(L) = number of blocks at places >= L, 64 values of L a step; the block's place j has S(j + 1) <= blk < S(j). Throughout
        // S(lo) > blk >= S(hi) = s_hi; the last step of a round may reach past hi, whose S then stays.
        int lo = 0, hi = total, s_hi = 0;
        while (hi - lo > 1) {
          const int step = (hi - lo + 63) >> 6;
          const I L = W::map([&](int l) { return lo + (l + 1) * step; }, W::lanes(0));
          I s = W::map([](int) { return 0; }, L);
          for (int q = 0; q < nseq; q++) {
            const int n = W::get(nb, q);
            s = W::map([&](int x, int at) { return x + imax(n - at, 0); }, s, L);
          }
          const int k = __builtin_popcountll(W::ballot([&](int x) { return x > blk; }, s));
          lo += k * step;
          if (lo + step <= hi) {  // (so k < 64: the last L is hi at least, where S <= blk)
            hi = lo + step;
            s_hi = W::get(s, k);
          }
        }
        j = lo;
        uint64_t at = W::ballot([&](int n) { return n > j; }, nb);
        for (int k = blk - s_hi; k > 0; k--) at &= at - 1;
        w = __builtin_ctzll(at);
      }
    } else {
      const uint64_t hit = W::ballot([&](int x) { return seen + x > blk; }, inc);
      if (!hit) {
        seen += total;
        continue;
      }
      w = __builtin_ctzll(hit);
      j = seen + W::get(inc, w) - 1 - blk;  // blocks of the sequence behind this one
    }
    r.seq = base + w;
    r.b = W::get(b, w);
    r.n = W::get(e, w) - r.b;
    r.first = j * RB;
    return r;
  }
  return Block{0, 0, 0, -1};
}

// The first block of those that share the CUs with the first ones, of the same number. Where two workgroups run on a CU (heads of 64 and 128) it has
// the shortest of them beside its longest block (heads of 128, 4096 tokens, 32 / 8 heads: 149 -> 143 us). Heads of 256 take a CU for one:
// their second layer follows the first, longest first as well (2048 tokens, 32 / 8 heads: 95 -> 81 us against
// the reversed order; 6500, 10 / 2: 252 -> 218; 8192, 16 / 4, five layers: 526, 530), so none of its blocks is reversed.
inline int second_layer(int hd, int ncu, int Hk) { return hd == 256 ? 1 << 29 : imax(1, ncu / Hk); }

// ---- over the cache ----
// The keys of a sequence are one list: the prefix (P keys), then its own. The work of a key head, in grid order:
//   shared: np_blocks blocks of all T G rows x ranges of the prefix, without a mask (rows of unused tokens are computed and
//           never read); partial slots [0, sp_max)
//   own:    the blocks of rb of the sequences' rows, the last one in the mode that its rows need, over their keys
//           [x_first, P + own), slots from sp_max on
// Split (with a workspace), the own blocks' tiles are one list that is cut into as many equal pieces as run at once beside the shared
// ranges, wherever the cuts fall: a workgroup's piece may end one block, take others whole and begin another. A block counts SEG tiles
// more than it has, for its setup and its result. With few blocks every piece begins in its own block instead, where that costs fewer than
// SEG tiles: the second setup of a piece takes longer than they do. The cuts follow from the lengths as they are on the device, so
// neither one long sequence among short ones nor a few items more than places decide the time (128 sequences, 32 / 8 heads, 500 keys behind 300:
// 71 -> 65 us against pieces in their own blocks, 1024 of 300 behind 600: 458 -> 315; 16 of 1000: 18.8 us so, 20.2 cut anywhere).
// Not split, an item is a block.
// Over a cache of int8 a tile of few rows takes half the time or less, its setup and result as long as over 16 bits, and a tile of the prefix, which goes through fp16,
// longer: counted as 6 and 2 (64 sequences of 1900 behind 4096, 32 / 8 heads: 74 -> 67 us; 16 of 5600 behind 32768: 72 -> 66).
constexpr int SEG = 2, PRE4 = 5, Q8_SEG = 6, Q8_PRE4 = 8;
// tiles up to which nothing is split: any batch, blocks that fill a quarter of the places
constexpr int WHOLE = 6, WHOLE_MANY = 16, Q8_WHOLE = 10, Q8_WHOLE_MANY = 32;
// what the host decides, from sizes that it knows
struct CachedPlan {
  int np_mode, np_blocks, sp_max;  // sp_max 0: nothing is shared
  int rb_log, s_max;  // rows a block of a sequence: 64 or 128
  int x_first;    // 0: own blocks take the prefix too
  int budget;     // items a key head that run at once
  int least;      // tiles an item is worth
  int n_blocks;   // at most, of a key head
  int seg, pre4;  // what a block counts beside its tiles, and four tiles of the prefix, in tiles of few rows
};
struct CachedWork {
  hxa_kv_cache c;
  int T, G;
  CachedPlan p;
};
// modes: 1 few rows (16), 2 rows (64), 4 rows (128); the one for `rows` rows that belong together, or for the first of more than 128
HXA_ANY int mode_rows(int mode) { return mode == 1 ? 16 : 32 * mode; }
HXA_ANY int rows_mode(long rows) { return rows <= 16 ? 1 : rows <= 64 ? 2 : 4; }

// x / d rounded up; below 2^24 the product with the reciprocal is off by one at most
template <class W>
HXA_ANY uint32_t ceil_of(uint32_t x, uint32_t d) {
  if (x >= 1u << 24) return (x - 1) / d + 1;
  uint32_t y = (uint32_t)((float)x * W::rcp((float)d));
  const int left = (int)(x - y * d);
  if (left > 0) y += left > (int)d ? 2 : 1;
  if (left < 0 && left <= -(int)d) y--;
  return y;
}
template <class W>
HXA_ANY int floor_of(uint32_t x, uint32_t d) {
  if (x >= 1u << 24) return (int)(x / d);
  int y = (int)((float)x * W::rcp((float)d));
  const int left = (int)(x - (uint32_t)y * d);
  return left < 0 ? y - 1 : left >= (int)d ? y + 1 : y;
}
HXA_ANY uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// 64 sequences of the batch, one a lane: first row in the call, tokens, length, blocks, and tiles of a block (0 without rows)
template <class W>
struct Lanes {
  typename W::I b, n, len, nb, tiles;
  HXA_ANY void sizes(const CachedWork &p) {
    const int cap = p.c.ldt * p.c.page, before = p.c.prefix_len - p.p.x_first + KT - 1;  // (their sum is below 2^31)
    nb = W::map([&](int t) { return (t * p.G + (1 << p.p.rb_log) - 1) >> p.p.rb_log; }, n);
    tiles = W::map([&](int blocks, int l) { return blocks ? (int)((unsigned)(imin(imax(l, 0), cap) + before) / KT) : 0; }, nb, len);
  }
  HXA_ANY void load(const CachedWork &p, int base) {
    b = W::map([&](int i) { return i < p.c.nseq ? imin(imax(p.c.cu[i], 0), p.T) : 0; }, W::lanes(base));
    n = W::map([&](int i, int b0) { return i < p.c.nseq ? imin(imax(p.c.cu[i + 1], b0), p.T) - b0 : 0; }, W::lanes(base), b);
    len = W::map([&](int i) { return i < p.c.nseq ? p.c.len[i] : 0; }, W::lanes(base));
    sizes(p);
  }
};
// what a workgroup does next: a range of the prefix for all rows, or tiles [t0, t1) of a block of a sequence
struct Work {
  bool shared;
  int slot, t0, t1;
  bool last;                 // the block's last range: it fills the slots behind its own
  int block;
  int seq, b, n, len;        // own: the sequence, its rows in the call, its length
};
// the walk of a workgroup over its piece [pos, end) of the list; the lanes' sequences, and the list's end behind each (inc, from `seen` on), wait
// in the wave's stash while a block is computed
struct Walk {
  int pos, end, chunk, base, seen;
  bool own_pieces;  // a block is a whole number of pieces in the list
};
template <class W>
HXA_ANY typename W::I list_tiles(const Walk &k, const Lanes<W> &s, int seg) {
  return W::map([&](int t) { return k.own_pieces ? (int)ceil_of<W>(imax(t, 1), k.chunk) * k.chunk : t + seg; }, s.tiles);
}
template <class W>
HXA_ANY typename W::I list_ends(const Lanes<W> &s, const typename W::I &each) {
  return W::scan(W::map([](int nb, int x) { return nb * x; }, s.nb, each));
}
template <class W>
HXA_ANY void take(Work &w, const Lanes<W> &s, int l, int base) {
  w.seq = base + l;
  w.b = W::get(s.b, l);
  w.n = W::get(s.n, l);
  w.len = W::get(s.len, l);
}
// item `q` of a key head, not split: the whole blocks of all sequences, then what is left of each: the short items even the end of the launch
// out (32 prompts of 300 rows behind 1000 keys, 768 blocks on 512 places: 66 -> 61 us). More than 64 sequences keep their order: a second
// pass over their lengths costs each of 201 x 8 items more (109 -> 118 us).
template <class W>
HXA_ANY bool find_block_of(const CachedWork &p, int q, Work &w) {
  typedef typename W::I I;
  const int rb = 1 << p.p.rb_log;
  Lanes<W> s;
  s.load(p, 0);
  const bool whole = p.c.nseq <= 64 && W::ballot([&](int n) { return n * p.G >= rb; }, s.n) != 0;
  int seen = 0;
  for (int rest = whole ? 0 : 1; rest < 2; rest++) {
    for (int base = 0; base < p.c.nseq; base += 64) {
      if (base > 0) s.load(p, base);
      const I full = W::map([&](int nb, int n) { return whole ? nb - ((n * p.G & (rb - 1)) != 0) : 0; }, s.nb, s.n);
      const I cnt = W::map([&](int nb, int f) { return rest ? nb - f : f; }, s.nb, full);
      const I inc = W::scan(cnt);
      const uint64_t hit = W::ballot([&](int x) { return seen + x > q; }, inc);
      if (!hit) {
        seen += W::get(inc, 63);
        continue;
      }
      const int l = __builtin_ctzll(hit);
      take(w, s, l, base);
      w.block = q - seen - W::get(inc, l) + W::get(cnt, l) + (rest ? W::get(full, l) : 0);
      w.t0 = 0;
      w.t1 = 1 << 24;
      return true;
    }
  }
  return false;
}
// the work at the walk's place; pos < end
template <class W>
HXA_ANY bool next_work(const CachedWork &p, Walk &k, Lanes<W> &s, typename W::I each, typename W::I inc, typename W::Stash stash, Work &w) {
  uint64_t hit;
  while (!(hit = W::ballot([&](int x) { return k.seen + x > k.pos; }, inc))) {
    k.seen += W::get(inc, 63);
    k.base += 64;
    if (k.base >= p.c.nseq) return false;
    s.load(p, k.base);
    each = list_tiles<W>(k, s, p.p.seg);
    inc = list_ends<W>(s, each);
  }
  W::keep(stash, s.b, s.n, s.len, inc);
  const int l = __builtin_ctzll(hit), seg = k.own_pieces ? 0 : p.p.seg;
  take(w, s, l, k.base);
  const int eff = W::get(each, l), nb = W::get(s.nb, l);
  int at = k.pos - (k.seen + W::get(inc, l) - nb * eff);
  w.block = at < eff ? 0 : floor_of<W>(at, eff);
  at -= w.block * eff;  // the walk's place in the block: 0, or the first of a piece
  const int stop = k.pos - at + eff;
  w.slot = p.p.sp_max + (at == 0 ? 0 : (int)ceil_of<W>(at, k.chunk));
  w.t0 = imax(at - seg, 0);
  w.t1 = imax(imin(k.end, stop) - k.pos + at - seg, 0);
  w.last = stop <= k.end;
  k.pos = imin(k.end, stop);
  return true;
}
// the work behind the one that the walk has just done; pos < end
template <class W>
HXA_ANY bool further_work(const CachedWork &p, Walk &k, typename W::Stash stash, Work &w) {
  Lanes<W> s;
  typename W::I inc;
  W::kept(stash, s.b, s.n, s.len, inc);
  s.sizes(p);
  return next_work<W>(p, k, s, list_tiles<W>(k, s, p.p.seg), inc, stash, w);
}
// the first work of item `q` of a key head, split
template <class W>
HXA_ANY bool first_work(const CachedWork &p, int q, typename W::Stash stash, Walk &k, Work &w) {
  const CachedPlan &a = p.p;
  const int pt = a.sp_max ? (p.c.prefix_len + KT - 1) / KT : 0;
  Lanes<W> s;
  int own = 0, blocks = 0, longest = 0;
  for (int base = (p.c.nseq - 1) & ~63; base >= 0; base -= 64) {  // sums below 2^30: checked on the host
    s.load(p, base);
    own += W::get(list_ends<W>(s, s.tiles), 63);
    blocks += W::ballot([](int nb) { return nb > 1; }, s.nb) ? W::get(W::scan(s.nb), 63)
                                                             : __builtin_popcountll(W::ballot([](int nb) { return nb > 0; }, s.nb));
    longest = imax(longest, W::most(s.tiles));
  }
  // (16-bit keys: a tile of 128 rows takes about 5/4 of one of 16, 4600 cycles, 3800)
  const uint32_t pre = (uint32_t)a.np_blocks * pt * a.pre4 / 4;
  uint32_t chunk = umax(ceil_of<W>(own + a.seg * blocks + pre, a.budget), (uint32_t)a.least);
  // no more pieces of a block than slots
  if (longest + a.seg - 1 > (long)chunk * (a.s_max - 1)) chunk = ceil_of<W>(longest + a.seg - 1, a.s_max - 1);
  k.own_pieces = false;
  const int taken = blocks + a.np_blocks;  // every block has one piece that is not full
  if (2 * taken <= a.budget) {
    uint32_t whole = umax(ceil_of<W>(own + pre, a.budget - taken), (uint32_t)a.least);
    if (longest > (long)whole * a.s_max) whole = ceil_of<W>(longest, a.s_max);
    k.own_pieces = whole < chunk + a.seg;
    if (k.own_pieces) chunk = whole;
  }
  if (a.sp_max) {
    const uint32_t cp = umax((chunk * 4 + a.pre4 - 1) / a.pre4, ceil_of<W>(pt, a.sp_max));
    const int ns = (int)ceil_of<W>(pt, cp);
    if (q < ns * a.np_blocks) {
      w.shared = true;
      w.slot = q / a.np_blocks;
      w.block = q - w.slot * a.np_blocks;
      w.t0 = w.slot * (int)cp;
      w.t1 = w.t0 + (int)cp;
      w.last = w.slot == ns - 1;
      k.pos = k.end = 0;
      return true;
    }
    q -= ns * a.np_blocks;
  }
  const int total = k.own_pieces ? 1 << 30 : own + a.seg * blocks;
  if ((uint64_t)q * chunk >= (uint32_t)total) return false;
  k.chunk = (int)chunk;
  k.pos = q * (int)chunk;
  k.end = imin(k.pos + (int)chunk, total);
  k.base = k.seen = 0;
  w.shared = false;
  const typename W::I each = list_tiles<W>(k, s, p.p.seg);
  return next_work<W>(p, k, s, each, list_ends<W>(s, each), stash, w);
}

// The launch of a call over the cache, from sizes that the host knows (T, the table's width, the prefix): how the lengths on
// the device turn out does not change it, so a captured launch stays right.
//   Rows a workgroup: 64 where the average sequence has no more, else 128 (at 65 .. 96 rows one workgroup of 128 takes 0.97 us a
//   tile, two of 64 take 1.26); for what is left of a sequence 16 or 64 where that is enough, which is found on the device (a prompt of 1000
//   tokens and 63 single ones over 800 each behind 500, 32 / 8 heads: 89 -> 60 us against 128 rows for all).
//   Shared prefix: where sequences bring at most 16 rows on average, there are at least two of them and the prefix is worth four tiles (prompts
//   read it block by block). No more slots than ranges first_work's chunk can make.
//   Not split where the table and the prefix hold at most 6 tiles of keys, or 16 where the blocks fill a quarter of the places: a second
//   launch and what the ranges set up take longer than the tiles one after the other (single tokens, 16 / 8 heads of 128, us split, whole: one
//   sequence of 4 tiles 8.9, 7.4, of 8 9.2, 10.0; 16 of 4 9.6, 7.7, of 8 13.6, 11.1, of 16 19.5, 18.4; 64 of 4 18.2, 14.9, of 16 48.5, 43.1). int8: 10 tiles, 32 where the blocks are many (16 of 5: 13.1, 11.3; one of 13: 11.7, 14.0; 128 of 11, 32 / 8 heads: 33.7, 28.8; 16 of 20: 13.1, 16.4).
//   Ranges of keys: with few rows as many as run at once; where the partials would pass 1 GB fewer, down to two of the own keys beside two of the
//   prefix (four times T Hq rows in fp32). With more rows a partial
//   result is as wide as a row's output is in fp32, so keys are split only where the blocks fill less than 5/8 of the places (32 prompts of
//   75 tokens behind 1000, 16 / 8 heads, 456 blocks of 512 places: split in two 65 us, whole 51).
inline long cached_ws(const CachedPlan &p, const hxa_kv_cache &c, int T, int Hq) {
  const long slots = p.sp_max + p.s_max;
  return slots == 1 ? 0 : slots * T * Hq * (c.hd * 4L + 8);
}
// places: workgroups that run at once
inline CachedPlan cached_plan(const hxa_kv_cache &c, int T, int Hq, bool ws, long places, bool q8 = false) {
  const auto least = [](long a, long b) { return a < b ? a : b; };
  const int G = Hq / c.H;
  const long RT = (long)T * G, P = c.prefix_len, cap = (long)c.ldt * c.page;
  CachedPlan p{};
  p.seg = q8 ? Q8_SEG : SEG;
  p.pre4 = q8 ? Q8_PRE4 : PRE4;
  const int mode = rows_mode(ceil_div(RT, c.nseq));
  p.rb_log = mode == 4 ? 7 : 6;
  p.n_blocks = (int)((RT >> p.rb_log) + c.nseq);
  p.budget = imax(1, (int)(places / c.H));
  p.least = mode == 1 ? 1 : 4;
  p.s_max = 1;
  const long blocks = ceil_div(RT, mode_rows(mode)) + c.nseq / 2, most = ceil_div(cap + P, KT);
  if (!ws || most <= (q8 ? Q8_WHOLE : WHOLE)) return p;
  if (mode == 1 && c.nseq >= 2 && P >= 4 * KT) {
    p.np_mode = rows_mode(RT);
    p.np_blocks = (int)ceil_div(RT, mode_rows(p.np_mode));
    p.sp_max = (int)least(32, least(ceil_div(P, KT), ceil_div(p.budget, p.np_blocks) + 1));
    p.x_first = (int)P;
  }
  // int8, while the prefix's blocks are less than half the places: ranges and pieces, roundings included, are no more than places, as one that begins when the
  // first have ended ends last. More blocks are whole ranges, beside which the pieces need all places (us, places kept for the blocks / not, 32 / 8 heads of
  // 128: 64 sequences behind 4096 35.6, 40.9; 512 212, 258; 1024 504, 433; 2048, where the blocks are as many as the places, 20400, 830)
  if (q8 && 2 * (p.np_blocks + 1) <= p.budget) p.budget -= p.np_blocks + 1;
  // a list that is cut anywhere: a block of so many ranges touches one workgroup more
  const long tiles = ceil_div(cap + P - p.x_first, KT);
  if (mode == 1) p.s_max = most <= (q8 ? Q8_WHOLE_MANY : WHOLE_MANY) && blocks * c.H * 4 >= places && p.sp_max == 0 ? 1 : (int)least(31, tiles);
  else if (blocks * c.H * 8 < places * 5) p.s_max = (int)least(8, least(tiles / p.least, ceil_div(places, blocks * c.H)));
  p.s_max = imax(1, p.s_max);
  if (p.s_max > 1 || p.sp_max > 0) p.s_max++;
  while (p.s_max > 2 && cached_ws(p, c, T, Hq) > 1L << 30) p.s_max = p.s_max / 2 + 1;
  // a piece stays below 2^24 tiles (all tiles / half the budget at the most), so that its keys are counted in 31 bits, and the list below 2^29
  const long list = p.n_blocks * (tiles + p.seg) + ceil_div(P, KT) * p.np_blocks * (q8 ? 4 : 2);
  if (list >= least(1L << 29, (long)p.budget << 23)) p.sp_max = p.np_blocks = p.x_first = 0, p.s_max = 1;
  return p;
}
// workgroups a key head. Split: a range of the prefix for each of its blocks and pieces of the rest, as many as run at once (first_work's
// chunk is at least all tiles / budget), and two roundings up
inline long cached_items(const CachedPlan &p) { return p.sp_max + p.s_max > 1 ? (long)p.np_blocks + p.budget + 2 : p.n_blocks; }

}  // namespace
