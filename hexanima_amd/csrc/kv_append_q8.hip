// New keys (normed and rotated on the way) and values into a paged cache of int8 with a scale for each page and head (hxa_kv_append_q8).
//
// A page and head that starts with the call's first row takes the scale s = max |x| / 127 of its new rows. One that holds earlier rows keeps its scale
// where the new rows fit, |x| <= 127 s; else it takes the least s 2^j that they fit, and the earlier rows become round(q 2^-j). So a value is
// rounded once with the scale of its time and at most once for each doubling: it is off by less than s (1/2 + 1/4 + ...) of the page's present
// scale, however many calls fill the page. (With s = max / 127 at every growth each of them, small ones too, would cost half a step.)
//
// A workgroup takes one page of one sequence and one head: its rows' maxima come first, so that the page is written once, and a page is nobody else's.
// hd / 16 lanes hold a row (causal_heads.h). Bound by HBM: 4 bytes read and 2 written per value of k and v.
#include "causal_heads.h"
#include "int8_rows.h"

namespace {

struct AppendQ8Args {
  hxa_kv_cache_q8 q;
  const void *k, *v;
  long ldk, ldv;
  int T;
  const float *gk;
  float eps;
  HeadRot r;
};

// The units of the grid: sequence i has those from cu[i] / page + 2 i on, one for each page that its new rows may touch (n rows touch at
// most n / page + 2). Returns the last sequence whose units begin at or below u, by the whole wave: 64 entries a step.
HXA_DEV int unit_seq(const int *__restrict__ cu, int nseq, int T, int page, long u, int lane) {
  int lo = 0, n = nseq;
  auto starts = [&](int i) { return (long)(min(max(cu[i], 0), T) / page) + 2L * i; };
  while (n > 64) {
    const int step = (n + 63) >> 6, at = lane * step;
    const int k = __popcll(__ballot(at < n && starts(lo + at) <= u));
    if (k == 0) return -1;
    lo += (k - 1) * step;
    n = min(n - (k - 1) * step, step);
  }
  return lo + __popcll(__ballot(lane < n && starts(lo + lane) <= u)) - 1;
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
HXA_DEV void shift_rows(int8_t *p, int n, int shift, int tid) {
  const float f = shift > 64 ? 0.0f : __builtin_bit_cast(float, (uint32_t)(127 - shift) << 23);
  for (int i = tid * 16; i < n; i += 256 * 16) {
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

template <typename T, int HD>
__global__ __launch_bounds__(256) void kv_append_q8_kernel(AppendQ8Args p) {
  typedef typename HxaVec<T>::v8 v8;
  constexpr int LPH = HD / 16, ROWS = 256 / LPH, HELD = 2;  // rows a pass, passes whose rows stay in registers
  const hxa_kv_cache &c = p.q.c;
  const int tid = threadIdx.x, lane = tid & 63, j = tid % LPH, sub = tid / LPH;
  const int h = blockIdx.x % c.H;
  const long u = blockIdx.x / c.H;
  const int i = unit_seq(c.cu, c.nseq, p.T, c.page, u, lane);
  if (i < 0) return;
  const int b = min(max(c.cu[i], 0), p.T), e = min(c.cu[i + 1], p.T);  // past T: cut there, as in the attention
  const long len = c.len[i], p0 = len - ((long)e - b);                 // own position of row b
  const long pb = p0 > 0 ? p0 : 0, pe = min(len, (long)c.ldt * c.page);
  if (b >= e || pb >= pe) return;
  const long slot = pb / c.page + (u - (b / c.page + 2L * i));
  const long first = max(pb, slot * c.page), last = min(pe, (slot + 1) * c.page);
  if (first >= last) return;
  const int pg = c.table[(long)i * c.ldt + slot];
  if ((unsigned)pg >= (unsigned)c.npages) return;
  const int r0 = (int)(first - slot * c.page), n = (int)(last - first);
  const long t0 = b + (first - p0);  // the row of the call at `first`
  const long ph = (long)pg * c.H + h;
  int8_t *kp = (int8_t *)c.k + ph * c.page * HD, *vp = (int8_t *)c.v + ph * c.page * HD;
  float ks = r0 > 0 ? p.q.kscale[ph] : 0.0f, vs = r0 > 0 ? p.q.vscale[ph] : 0.0f;
  ks = ks < INFINITY ? ks : 0.0f;
  vs = vs < INFINITY ? vs : 0.0f;

  int c0, c1;
  head_chunks(p.r, j, c0, c1);
  auto load = [&](int row, float (&a)[8], float (&z)[8], v8 (&y)[2]) {
    const long t = t0 + row;
    const T *src = (const T *)p.v + t * p.ldv + (long)h * HD + 16 * j;
    y[0] = *(const v8 *)src;
    y[1] = *(const v8 *)(src + 8);
    head_load((const T *)p.k + t * p.ldk + (long)h * HD, c0, c1, a, z);
    float cs[8], sn[8];
    head_angles(p.r, j, (double)(c.prefix_len + first + row), cs, sn);
    head_turn<LPH>(a, z, p.gk, p.eps, p.r, j, c0, c1, cs, sn);
  };
  float ka[HELD][8], kz[HELD][8], kt = 0.0f, vt = 0.0f;
  v8 vv[HELD][2];
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
      load(d * ROWS + sub, ka[d], kz[d], vv[d]);
      most(ka[d], kz[d], vv[d]);
    }
  }
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
  __shared__ float tops[8];
  if (lane == 0) {
    tops[tid >> 6] = kt;
    tops[4 + (tid >> 6)] = vt;
  }
  __syncthreads();  // (and every thread has read the page's scales)
  kt = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  vt = fmaxf(fmaxf(tops[4], tops[5]), fmaxf(tops[6], tops[7]));
  int kshift, vshift;
  const float kn = grown(ks, q8_scale(kt), kshift), vn = grown(vs, q8_scale(vt), vshift);
  if (tid == 0) {
    p.q.kscale[ph] = kn;
    p.q.vscale[ph] = vn;
  }
  if (kshift) shift_rows(kp, r0 * HD, kshift, tid);
  if (vshift) shift_rows(vp, r0 * HD, vshift, tid);
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
    if (d * ROWS + sub < n) store(d * ROWS + sub, ka[d], kz[d], vv[d]);
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
  const hipStream_t st = (hipStream_t)stream;
#define HXA_AP(TY, HD) hxa_launch(kv_append_q8_kernel<TY, HD>, dim3((unsigned)wgs), dim3(256), 0, st, p)
  if (d.dtype == HXA_DT_F16) {
    if (d.hd == 64) HXA_AP(hxa_h, 64);
    if (d.hd == 128) HXA_AP(hxa_h, 128);
    if (d.hd == 256) HXA_AP(hxa_h, 256);
  } else {
    if (d.hd == 64) HXA_AP(hxa_b, 64);
    if (d.hd == 128) HXA_AP(hxa_b, 128);
    if (d.hd == 256) HXA_AP(hxa_b, 256);
  }
#undef HXA_AP
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HXA_OK : hxa_set_error(HXA_E_HIP, "kv_append_q8: %s", hipGetErrorString(e));
}
