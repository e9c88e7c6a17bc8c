// csrc/causal_walk.h on the CPU: the wave is an array of 64 values, and every row block and tile of a plan is counted. The functions return
// the number of mistakes (the first few on stderr).
#include <cstdio>
#include <cstdlib>
#include <cmath>
#include <vector>

#include "../hexanima_amd/csrc/causal_walk.h"

static int g_rcp;  // the last place of a reciprocal: rounded, one less, one more
static long g_bad;
#define EXPECT(ok, ...)                                   \
  do {                                                    \
    if (!(ok) && ++g_bad <= 3) {                          \
      fprintf(stderr, __VA_ARGS__);                       \
      fputc('\n', stderr);                                \
    }                                                     \
  } while (0)

struct HostWave {
  struct I {
    int v[64];
  };
  struct Kept {
    I x[4];
  };
  typedef Kept *Stash;
  static I lanes(int base) {
    I r;
    for (int l = 0; l < 64; l++) r.v[l] = base + l;
    return r;
  }
  template <typename F, typename... A>
  static I map(F f, const A &...a) {
    I r;
    for (int l = 0; l < 64; l++) r.v[l] = f(a.v[l]...);
    return r;
  }
  template <typename F>
  static uint64_t ballot(F f, const I &a) {
    uint64_t r = 0;
    for (int l = 0; l < 64; l++) r |= (uint64_t)(bool)f(a.v[l]) << l;
    return r;
  }
  static int get(const I &a, int lane) {
    EXPECT(lane >= 0 && lane < 64, "lane %d", lane);
    return a.v[lane & 63];
  }
  static I scan(const I &a) {
    I r;
    long s = 0;
    for (int l = 0; l < 64; l++) {
      s += a.v[l];
      EXPECT(s == (int)s, "a sum of %ld", s);
      r.v[l] = (int)s;
    }
    return r;
  }
  static int most(const I &a) {
    int m = a.v[0];
    for (int x : a.v) m = x > m ? x : m;
    return m;
  }
  static float rcp(float x) {
    const float r = 1.0f / x;
    return g_rcp == 0 ? r : std::nextafter(r, g_rcp < 0 ? 0.0f : 2.0f);
  }
  static void keep(Stash s, const I &a, const I &b, const I &c, const I &d) { *s = Kept{{a, b, c, d}}; }
  static void kept(Stash s, I &a, I &b, I &c, I &d) { a = s->x[0], b = s->x[1], c = s->x[2], d = s->x[3]; }
};

static int clampi(long x, long lo, long hi) { return (int)(x < lo ? lo : x > hi ? hi : x); }

// Blocks 0 .. grid - 1 of a batch of prompts: each block of each sequence once. order (grid entries): the place of block b in its sequence
extern "C" long host_find_block(const int *cu, int nseq, int T, int G, int RB, int first, long grid, int *order) {
  g_bad = 0;
  std::vector<std::vector<int>> hit(nseq);
  long want = 0, got = 0;
  for (int i = 0; i < nseq; i++) {
    const int b = clampi(cu[i], 0, T), n = clampi(cu[i + 1], b, T) - b;
    hit[i].assign(((long)n * G + RB - 1) / RB, 0);
    want += hit[i].size();
  }
  EXPECT(want <= grid, "%ld blocks, a grid of %ld", want, grid);
  for (long blk = 0; blk < grid; blk++) {
    const Block r = find_block<HostWave>(cu, nseq, T, G, RB, (int)blk, first);
    if (order) order[blk] = r.first < 0 ? -1 : r.first / RB;
    if (r.first < 0) continue;
    got++;
    const bool in = r.seq >= 0 && r.seq < nseq && r.first % RB == 0 && (size_t)(r.first / RB) < hit[r.seq].size();
    EXPECT(in, "block %ld: sequence %d, row %d of %d tokens", blk, r.seq, r.first, r.n);
    if (!in) continue;
    const int b = clampi(cu[r.seq], 0, T);
    EXPECT(r.b == b && r.n == clampi(cu[r.seq + 1], b, T) - b, "block %ld: sequence %d's rows %d + %d", blk, r.seq, r.b, r.n);
    EXPECT(++hit[r.seq][r.first / RB] == 1, "block %ld: place %d of sequence %d again", blk, r.first / RB, r.seq);
  }
  EXPECT(got == want, "%ld of %ld blocks", got, want);
  return g_bad;
}

extern "C" int host_second_layer(int hd, int ncu, int Hk) { return second_layer(hd, ncu, Hk); }

// The items of a key head over the cache, as the library plans them: every tile of every block in one piece, its pieces in slots of their own,
// the slots behind the last one filled, the prefix likewise; no work behind the grid. plan (if not null): the host's plan
extern "C" long host_cached(int hd, int Hq, int H, int T, int nseq, const int *cu, const int *len, int page, int ldt, int prefix_len,
                            int ws, long places, int rcp, int *plan) {
  g_bad = 0;
  g_rcp = rcp;
  CachedWork p{};
  p.c.H = H, p.c.hd = hd, p.c.page = page, p.c.ldt = ldt, p.c.prefix_len = prefix_len, p.c.nseq = nseq, p.c.cu = cu, p.c.len = len;
  p.T = T, p.G = Hq / H;
  p.p = cached_plan(p.c, T, Hq, ws != 0, places);
  const CachedPlan &a = p.p;
  if (plan) {
    const int x[] = {a.np_mode, a.np_blocks, a.sp_max, a.rb_log, a.s_max, a.x_first, a.budget, a.least, a.n_blocks};
    for (int i = 0; i < 9; i++) plan[i] = x[i];
  }
  const int nslots = a.sp_max + a.s_max, RB = 1 << a.rb_log;
  EXPECT(nslots <= 64, "%d slots", nslots);
  const long grid = cached_items(a);
  struct Own {
    int tiles, t = 0, slot = 0;
    bool last = false;
  };
  std::vector<std::vector<Own>> own(nseq);
  long want = 0, got = 0;
  for (int i = 0; i < nseq; i++) {
    const int b = clampi(cu[i], 0, T), n = clampi(cu[i + 1], b, T) - b;
    const long held = clampi(len[i], 0, (long)ldt * page);
    own[i].assign(((long)n * p.G + RB - 1) / RB, Own{(int)((held + prefix_len - a.x_first + KT - 1) / KT)});
    want += own[i].size();
  }
  const int pt = (prefix_len + KT - 1) / KT;
  std::vector<Own> shared(a.np_blocks, Own{pt});
  HostWave::Kept stash;
  auto piece = [&](Own &o, const Work &w, int slot0, int slots, const char *what) {
    EXPECT(!o.last, "%s block %d: work behind its last", what, w.block);
    EXPECT(w.slot == slot0 + o.slot && o.slot < slots, "%s block %d: slot %d, %d before", what, w.block, w.slot, o.slot);
    EXPECT((long)w.t1 * KT <= 0x7fffffff, "%s block %d: %d tiles", what, w.block, w.t1);
    EXPECT(w.t0 == o.t && w.t1 >= w.t0, "%s block %d: tiles %d .. %d behind %d", what, w.block, w.t0, w.t1, o.t);
    o.slot++;
    o.t = w.t1;
    o.last = w.last;
  };
  for (long q = 0; q < grid + 3; q++) {
    Walk k{};
    Work w{};
    if (nslots == 1) {
      if (!find_block_of<HostWave>(p, (int)q, w)) continue;
      EXPECT(q < grid, "item %ld of %ld", q, grid);
      const bool in = w.seq >= 0 && w.seq < nseq && w.block >= 0 && (size_t)w.block < own[w.seq].size();
      EXPECT(in, "item %ld: block %d of sequence %d", q, w.block, w.seq);
      if (!in) continue;
      Own &o = own[w.seq][w.block];
      EXPECT(!o.last && w.t0 == 0 && w.t1 >= o.tiles, "item %ld: block %d of sequence %d again, or not whole", q, w.block, w.seq);
      o.last = true;
      o.t = o.tiles;
      got++;
      continue;
    }
    if (!first_work<HostWave>(p, (int)q, &stash, k, w)) continue;
    EXPECT(q < grid, "item %ld of %ld", q, grid);
    if (w.shared) {
      EXPECT(w.block >= 0 && w.block < a.np_blocks, "item %ld: shared block %d of %d", q, w.block, a.np_blocks);
      if (w.block >= 0 && w.block < a.np_blocks) piece(shared[w.block], w, 0, a.sp_max, "shared");
      continue;
    }
    for (;;) {
      const bool in = w.seq >= 0 && w.seq < nseq && w.block >= 0 && (size_t)w.block < own[w.seq].size();
      EXPECT(in, "item %ld: block %d of sequence %d", q, w.block, w.seq);
      if (!in) break;
      EXPECT(w.b == clampi(cu[w.seq], 0, T) && w.len == len[w.seq], "item %ld: sequence %d's rows or length", q, w.seq);
      piece(own[w.seq][w.block], w, a.sp_max, a.s_max, "own");
      if (w.last) got++;
      if (k.pos >= k.end || !further_work<HostWave>(p, k, &stash, w)) break;
    }
  }
  EXPECT(got == want, "%ld of %ld blocks", got, want);
  for (auto &s : own)
    for (auto &o : s) EXPECT(o.last && o.t >= o.tiles, "a block of %d tiles: %d taken", o.tiles, o.t);
  for (auto &o : shared) EXPECT(o.last && o.t >= o.tiles, "a prefix of %d tiles: %d taken", o.tiles, o.t);
  return g_bad;
}
