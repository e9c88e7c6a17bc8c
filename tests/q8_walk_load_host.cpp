// The load of the items over a cache of int8: what the longest one of a key head and all of them together count.
#include "q8_walk_host.cpp"

// A key head's items as the kernels take them, in tiles of few rows: load[0] of the longest item, [1] of all of them, [2] of the longest block, [3] slots of a
// block, [4] places counted on, [5] slots of the prefix; all 0 where nothing is split
extern "C" void host_load(int hd, int Hq, int H, int T, int nseq, const int *cu, const int *len, int page, int ldt, int prefix_len, long places,
                          double *load) {
  CachedWork p{};
  p.c.H = H, p.c.hd = hd, p.c.page = page, p.c.ldt = ldt, p.c.prefix_len = prefix_len, p.c.nseq = nseq, p.c.cu = cu, p.c.len = len;
  p.T = T, p.G = Hq / H;
  p.p = cached_plan(p.c, T, Hq, true, places);
  const CachedPlan &a = p.p;
  for (int i = 0; i < 6; i++) load[i] = 0;
  if (a.sp_max + a.s_max == 1) return;
  const int pt = (prefix_len + KT - 1) / KT;
  HostWave::Kept stash;
  double most = 0, sum = 0, block = 0;
  for (int i = 0; i < nseq; i++)
    block = std::fmax(block, (double)a.seg + (clampi(len[i], 0, (long)ldt * page) + prefix_len - a.x_first + KT - 1) / KT);
  for (long q = 0; q < cached_items(a); q++) {
    Walk k{};
    Work w{};
    if (!first_work<HostWave>(p, (int)q, &stash, k, w)) continue;
    double c = 0;
    if (w.shared) {
      c = (imin(w.t1, pt) - w.t0) * a.pre4 / 4.0;
    } else {
      for (;;) {
        const int held = clampi(len[w.seq], 0, (long)ldt * page), tiles = (held + prefix_len - a.x_first + KT - 1) / KT;
        c += imax(0, imin(w.t1, tiles) - w.t0) + (w.t0 == 0 ? a.seg : 0);
        if (k.pos >= k.end || !further_work<HostWave>(p, k, &stash, w)) break;
      }
    }
    most = std::fmax(most, c);
    sum += c;
  }
  const double x[] = {most, sum, block, (double)a.s_max, (double)a.budget, (double)a.sp_max};
  for (int i = 0; i < 6; i++) load[i] = x[i];
}
