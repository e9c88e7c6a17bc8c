// New keys (normed and rotated on the way) and values into a paged cache of int8 with a scale for each page and head (hxa_kv_append_q8).
//
// A page and head that starts with the call's first row takes the scale s = max |x| / 127 of its new rows. One that holds earlier rows keeps its scale
// where the new rows fit, |x| <= 127 s; else it takes the least s 2^j that they fit, and the earlier rows become round(q 2^-j). So a value is
// rounded once with the scale of its time and at most once for each doubling: it is off by less than s (1/2 + 1/4 + ...) of the page's present
// scale, however many calls fill the page. (With s = max / 127 at every growth each of them, small ones too, would cost half a step.)
//
// A workgroup takes one page of one sequence and one head: its rows' maxima come first, so that the page is written once, and a page is nobody else's.
// hd / 16 lanes hold a row (causal_heads.h).
//
// Bound by HBM: 4 bytes read and 2 written per value of k and v, and for prompts by a workgroup's chain (lengths, rows, angles, maxima, bytes) with four of them a CU: 9001 tokens
// of 8 heads of 128 into pages of 64 21 us (2.6 TB/s; 26 with the library's sine and cosine; with an angle for a few heads at a time, in registers, 30: two workgroups
// a CU; for two heads, in LDS, 20, and 64 single tokens 8.7 for 7.1), 64000 tokens 109 us (3.6 TB/s; a large copy 5.1). Few tokens take the launch and three dependent loads: lengths, then pages beside the rows, then scales.
#include <algorithm>
#include <type_traits>

#include "causal_heads.h"
#include "int8_rows.h"

namespace {

constexpr int HELD = 2;

struct AppendQ8Args {
  hxa_kv_cache_q8 q;
  const void *k, *v;
  long ldk, ldv;
  int T;
  const float *gk;
  float eps;
  HeadRot r;
};

// Cosine and sine of 2 pi turns, |turns| <= 1/2: the nearest quarter taken off, Taylor's sums up to the 9th and 10th power on the +-pi / 4 that are left (their rest
// is below 2e-9), and the quarter's signs and exchange.
HXA_DEV void turn(float turns, float &c, float &s) {
  const float q = rintf(4.0f * turns);
  const float x = 6.283185307179586477f * fmaf(-0.25f, q, turns), y = x * x;
  float sn = fmaf(y, 2.7557319e-6f, -1.9841270e-4f), cs = fmaf(y, -2.7557319e-7f, 2.4801587e-5f);
  sn = fmaf(y, sn, 8.3333333e-3f), cs = fmaf(y, cs, -1.3888889e-3f);
  sn = fmaf(y, sn, -1.6666667e-1f), cs = fmaf(y, cs, 4.1666667e-2f);
  sn = fmaf(x * y, sn, x), cs = fmaf(y, cs, -0.5f);
  cs = fmaf(y, cs, 1.0f);
  const int n = (int)q;
  const bool odd = n & 1;
  const float a = odd ? sn : cs, b = odd ? cs : sn;
  c = (n + 1) & 2 ? -a : a;
  s = n & 2 ? -b : b;
}
// as head_angles
HXA_DEV void head_turns(const HeadRot &r, int j, double pos, float (&cs)[8], float (&sn)[8]) {
  if (j >= r.rot >> 4) return;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    double turns = pos * (double)r.freq[8 * j + e] * 0.15915494309189533577;
    turns -= rint(turns);
    float c, s;
    turn((float)turns, c, s);
    cs[e] = c * r.mscale;
    sn[e] = s * r.mscale;
  }
}

// The units of the grid: sequence i has those from cu[i] / page + 2 i on, one for each page that its new rows may touch (n rows touch at
// most n / page + 2). Finds the last sequence whose units begin at or below u (-1: none), its row range and length, and u's place among its units, by the
// whole wave: 64 entries a step.
struct Unit {
  int i, b, e, len;
  long at;
};
HXA_DEV Unit find_unit(const hxa_kv_cache &c, int T, long u, int lane) {
  int lo = 0, n = c.nseq;
  auto starts = [&](int i, int b) { return (long)(min(max(b, 0), T) / c.page) + 2L * i; };
  while (n > 64) {
    const int step = (n + 63) >> 6, at = lane * step;
    const int k = __popcll(__ballot(at < n && starts(lo + at, c.cu[lo + min(at, n - 1)]) <= u));
    if (k == 0) return Unit{-1, 0, 0, 0, 0};
    lo += (k - 1) * step;
    n = min(n - (k - 1) * step, step);
  }
  const int i = lo + min(lane, n - 1), b = c.cu[i], e = c.cu[i + 1], len = c.len[i];
  const int k = __popcll(__ballot(lane < n && starts(i, b) <= u)) - 1;
  if (k < 0) return Unit{-1, 0, 0, 0, 0};
  Unit r;
  r.i = lo + k;
  r.b = min(max(__builtin_amdgcn_readlane(b, k), 0), T);
  r.e = min(__builtin_amdgcn_readlane(e, k), T);  // past T: cut there, as in the attention
  r.len = __builtin_amdgcn_readlane(len, k);
  r.at = u - starts(r.i, r.b);
  return r;
}

// the scale of a page that had `old` (0: no earlier value) and whose new rows need `need`: `shift` doublings
HXA_DEV float grown(float old, float need, int &shift) {
  shift = 0;
  if (!(old > 0.0f)) return need;
  if (need <= old) return old;
  const float r = need / old;  // >= 1; 2^j <= r: the exponent, and one more where r is no power of two
  const uint32_t b = __builtin_bit_cast(uint32_t, r);
  shift = (int)(b >> 23) - 127 + ((b & 0x7fffff) != 0);
  if (shift > 64) return need;  // nothing is left of the earlier rows
  return old * __builtin_bit_cast(float, (uint32_t)(127 + shift) << 23);
}
// the earlier rows of a page, n bytes from p on: q -> round(q 2^-shift)
template <int NT>
HXA_DEV void shift_rows(int8_t *p, int n, int shift, int tid) {
  const float f = shift > 64 ? 0.0f : __builtin_bit_cast(float, (uint32_t)(127 - shift) << 23);
  for (int i = tid * 16; i < n; i += NT * 16) {
    uint4_t w = *(const uint4_t *)(p + i);
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = (float)(int8_t)(w[j + e / 4] >> (8 * (e & 3)));
      const uint2_t y = q8_pack(x, f);
      w[j] = y.x;
      w[j + 1] = y.y;
    }
    *(uint4_t *)(p + i) = w;
  }
}

// NT threads: the keys of HELD passes of NT / LPH rows stay in registers between their maxima and their bytes; further ones, and the values, are read again
template <typename T, int HD, int NT>
__global__ __launch_bounds__(NT, 4) void kv_append_q8_kernel(AppendQ8Args p) {
  typedef typename HxaVec<T>::v8 v8;
  constexpr int LPH = HD / 16, ROWS = NT / LPH;  // lanes a row, rows a pass
  const hxa_kv_cache &c = p.q.c;
  const int tid = threadIdx.x, lane = tid & 63, j = tid % LPH, sub = tid / LPH;
  const int h = blockIdx.x % c.H;
  const Unit w = find_unit(c, p.T, blockIdx.x / c.H, lane);
  if (w.i < 0) return;
  const long p0 = w.len - ((long)w.e - w.b);  // own position of row b
  const long pb = p0 > 0 ? p0 : 0, pe = min((long)w.len, (long)c.ldt * c.page);
  if (w.b >= w.e || pb >= pe) return;
  const long slot = pb / c.page + w.at;
  const long first = max(pb, slot * c.page), last = min(pe, (slot + 1) * c.page);
  if (first >= last) return;
  const int pg = c.table[(long)w.i * c.ldt + slot];
  const int r0 = (int)(first - slot * c.page), n = (int)(last - first);
  const long t0 = w.b + (first - p0);  // the row of the call at `first`

  int c0, c1;
  head_chunks(p.r, j, c0, c1);
  const T *ks0 = (const T *)p.k + t0 * p.ldk + (long)h * HD, *vs0 = (const T *)p.v + t0 * p.ldv + (long)h * HD + 16 * j;
  auto load = [&](int row, float (&a)[8], float (&z)[8], v8 (&y)[2]) {
    const T *v = vs0 + row * p.ldv;
    y[0] = *(const v8 *)v;
    y[1] = *(const v8 *)(v + 8);
    head_load(ks0 + row * p.ldk, c0, c1, a, z);
    float cs[8], sn[8];
    head_turns(p.r, j, (double)(c.prefix_len + first + row), cs, sn);
    head_turn<LPH>(a, z, p.gk, p.eps, p.r, j, c0, c1, cs, sn);
  };
  float ka[HELD][8], kz[HELD][8], kt = 0.0f, vt = 0.0f;
  auto most = [&](const float (&a)[8], const float (&z)[8], const v8 (&y)[2]) {
#pragma unroll
    for (int x = 0; x < 8; x++) {
      kt = fmaxf(kt, fmaxf(finite_abs(a[x]), finite_abs(z[x])));
      vt = fmaxf(vt, fmaxf(finite_abs((float)y[0][x]), finite_abs((float)y[1][x])));
    }
  };
#pragma unroll
  for (int d = 0; d < HELD; d++) {
    if (d * ROWS + sub < n) {
      v8 y[2];
      load(d * ROWS + sub, ka[d], kz[d], y);
      most(ka[d], kz[d], y);
    }
  }
  if ((unsigned)pg >= (unsigned)c.npages) return;
  const long ph = (long)pg * c.H + h;
  int8_t *kp = (int8_t *)c.k + ph * c.page * HD, *vp = (int8_t *)c.v + ph * c.page * HD;
  float ks = r0 > 0 ? p.q.kscale[ph] : 0.0f, vs = r0 > 0 ? p.q.vscale[ph] : 0.0f;
  ks = ks < INFINITY ? ks : 0.0f;
  vs = vs < INFINITY ? vs : 0.0f;
  for (int row = HELD * ROWS + sub; row < n; row += ROWS) {
    float a[8], z[8];
    v8 y[2];
    load(row, a, z, y);
    most(a, z, y);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    kt = fmaxf(kt, __shfl_xor(kt, d));
    vt = fmaxf(vt, __shfl_xor(vt, d));
  }
  if constexpr (NT > 64) {
    __shared__ float tops[2][NT / 64];
    if (lane == 0) {
      tops[0][tid >> 6] = kt;
      tops[1][tid >> 6] = vt;
    }
    __syncthreads();  // (and every thread has read the page's scales)
#pragma unroll
    for (int x = 0; x < NT / 64; x++) {
      kt = fmaxf(kt, tops[0][x]);
      vt = fmaxf(vt, tops[1][x]);
    }
  }
  int kshift, vshift;
  const float kn = grown(ks, q8_scale(kt), kshift), vn = grown(vs, q8_scale(vt), vshift);
  if (tid == 0) {
    p.q.kscale[ph] = kn;
    p.q.vscale[ph] = vn;
  }
  if (kshift) shift_rows<NT>(kp, r0 * HD, kshift, tid);
  if (vshift) shift_rows<NT>(vp, r0 * HD, vshift, tid);
  const float ki = kn > 0.0f ? 1.0f / kn : 0.0f, vi = vn > 0.0f ? 1.0f / vn : 0.0f;
  auto store = [&](int row, const float (&a)[8], const float (&z)[8], const v8 (&y)[2]) {
    int8_t *kr = kp + (long)(r0 + row) * HD, *vr = vp + (long)(r0 + row) * HD + 16 * j;
    *(uint2_t *)(kr + 8 * c0) = q8_pack(a, ki);
    *(uint2_t *)(kr + 8 * c1) = q8_pack(z, ki);
    float f[2][8];
#pragma unroll
    for (int x = 0; x < 8; x++) {
      f[0][x] = (float)y[0][x];
      f[1][x] = (float)y[1][x];
    }
    const uint2_t lo = q8_pack(f[0], vi), hi = q8_pack(f[1], vi);
    *(uint4_t *)vr = (uint4_t){lo.x, lo.y, hi.x, hi.y};
  };
#pragma unroll
  for (int d = 0; d < HELD; d++)
    if (d * ROWS + sub < n) {
      const T *v = vs0 + (d * ROWS + sub) * p.ldv;
      const v8 y[2] = {*(const v8 *)v, *(const v8 *)(v + 8)};
      store(d * ROWS + sub, ka[d], kz[d], y);
    }
  for (int row = HELD * ROWS + sub; row < n; row += ROWS) {
    float a[8], z[8];
    v8 y[2];
    load(row, a, z, y);
    store(row, a, z, y);
  }
}

}  // namespace

int hxa_kv_check_q8(const hxa_kv_cache_q8 *c, int T, const char *who) {
  if (!c) return hxa_set_error(HXA_E_ARG, "%s: no cache", who);
  const int r = hxa_kv_check(&c->c, T, who);
  if (r != HXA_OK || T == 0 || c->c.nseq == 0) return r;
  if (!c->kscale || !c->vscale || ((uintptr_t)c->kscale | (uintptr_t)c->vscale) % 4)
    return hxa_set_error(HXA_E_ARG, "%s: scales null or not aligned", who);
  return HXA_OK;
}

extern "C" int hxa_kv_append_q8(const hxa_kv_cache_q8 *c, const void *k, long ldk, const void *v, long ldv, int T, const float *gk, float eps,
                                const hxa_rope *rope, void *stream) {
  int r = hxa_kv_check_q8(c, T, "kv_append_q8");
  if (r != HXA_OK) return r;
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return hxa_set_error(HXA_E_ARG, "kv_append_q8: eps=%g", (double)eps);
  AppendQ8Args p{*c, k, v, ldk, ldv, T, gk, eps, {}};
  const hxa_kv_cache &d = c->c;
  r = rot_of(rope, d.hd, p.r, "kv_append_q8");
  if (r != HXA_OK) return r;
  if (T == 0 || d.nseq == 0 || d.ldt == 0) return HXA_OK;
  if (!row_ok(k, ldk, d.H, d.hd) || !row_ok(v, ldv, d.H, d.hd) || (uintptr_t)gk % 16)
    return hxa_set_error(HXA_E_ARG, "kv_append_q8: pointers null or not 16-byte aligned, or strides (%ld %ld)", ldk, ldv);
  const long wgs = ((long)T / d.page + 2L * d.nseq) * d.H;
  if (wgs >= 1L << 24) return hxa_set_error(HXA_E_ARG, "kv_append_q8: T=%d nseq=%d H=%d are too many pages", T, d.nseq, d.H);
  // as many threads as hold a page's rows on average (us with 256 threads, with these: 9001 tokens in pages of 16 43, 20; of 1 330, 110; 64 single
  // tokens 7.6, 6.3)
  const long rows = std::min<long>(d.page, std::max(1, T / d.nseq)) * (d.hd / 16);
  const int nt = rows <= 64 * HELD ? 64 : rows <= 128 * HELD ? 128 : 256;
  const hipStream_t st = (hipStream_t)stream;
  auto run = [&](auto ty, auto hdc) {
    typedef decltype(ty) T_;
    constexpr int HD = decltype(hdc)::value;
    const auto f = nt == 64 ? kv_append_q8_kernel<T_, HD, 64> : nt == 128 ? kv_append_q8_kernel<T_, HD, 128> : kv_append_q8_kernel<T_, HD, 256>;
    hxa_launch(f, dim3((unsigned)wgs), dim3(nt), 0, st, p);
  };
  auto heads = [&](auto ty) {
    if (d.hd == 64) run(ty, std::integral_constant<int, 64>{});
    else if (d.hd == 128) run(ty, std::integral_constant<int, 128>{});
    else run(ty, std::integral_constant<int, 256>{});
  };
  if (d.dtype == HXA_DT_F16) heads(hxa_h{});
  else heads(hxa_b{});
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HXA_OK : hxa_set_error(HXA_E_HIP, "kv_append_q8: %s", hipGetErrorString(e));
}
