// Per-head RMSNorm with the rotary positions in the same pass, for the queries and keys of a causal text model, and the same on
// the way into a paged cache.
//
// u = x rsqrt(mean x^2 + eps) gain; the pair (a, b) of frequency f at position p becomes (a cos - b sin, a sin + b cos) with the
// angle p f. The angle's turns p f / (2 pi) are formed in 64 bits and reduced there to [-1/2, 1/2] before sine and cosine
// are taken in 32: at position 70000 a 32-bit product would be off by 4e-3 radians.
//
// Bound by HBM: 2 bytes read and 2 written per value (kv_append: the same for k and v). hd / 16 lanes hold a head, 16 values
// each as two 16-byte loads; a lane's two chunks are partners of the rotation in either layout, so it needs no exchange, and the 8 angles a
// lane needs are the same for every head of the token: a wave takes one token and forms them once. 8192 tokens of 32 + 8 heads of 128: 37.0 us,
// 4.5 TB/s; 9001 tokens of 8 heads appended: 16.1 us, 4.6 TB/s (a large copy 4.8). Few tokens take the launch and three or four
// dependent loads, 3 .. 4 us.
#include "causal_heads.h"

namespace {

struct QkArgs {
  const void *q, *k;
  void *qo, *ko;
  long ldq, ldk, ldqo, ldko;
  int Hq, Hk, T;
  const float *gq, *gk;
  float eps;
  const int *pos;
  HeadRot r;
  int parts, per;  // waves a token, groups of heads each of them takes
};

// In place is allowed, so q / qo and k / ko carry no restrict: a lane reads its 16 values before it writes them.
template <typename T, int HD>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkArgs p) {
  constexpr int LPH = HD / 16, HPW = 64 / LPH;
  const int lane = threadIdx.x & 63, j = lane % LPH, sub = lane / LPH;
  const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const uint32_t tu = unit / (uint32_t)p.parts;
  const int part = (int)(unit - tu * p.parts);
  if (tu >= (uint32_t)p.T) return;
  const int t = (int)tu;
  int c0, c1;
  head_chunks(p.r, j, c0, c1);
  float cs[8], sn[8];
  head_angles(p.r, j, p.pos ? (double)p.pos[t] : (double)t, cs, sn);
  const int H = p.Hq + p.Hk;
  for (int g = 0; g < p.per; g++) {
    const int h = (part * p.per + g) * HPW + sub;
    if (h < H) {
      const bool isq = h < p.Hq;
      const T *src = isq ? (const T *)p.q + t * p.ldq + (long)h * HD : (const T *)p.k + t * p.ldk + (long)(h - p.Hq) * HD;
      T *dst = isq ? (T *)p.qo + t * p.ldqo + (long)h * HD : (T *)p.ko + t * p.ldko + (long)(h - p.Hq) * HD;
      float a[8], b[8];
      head_load(src, c0, c1, a, b);
      head_turn<LPH>(a, b, isq ? p.gq : p.gk, p.eps, p.r, j, c0, c1, cs, sn);
      head_store(dst, c0, c1, a, b);
    }
  }
}

struct AppendArgs {
  hxa_kv_cache c;
  const void *k, *v;
  long ldk, ldv;
  int T;
  const float *gk;
  float eps;
  HeadRot r;
};

// One wave a token: its sequence (a search of cu), its page row, then k's heads and v's. A pool's rows of one token are H pieces of
// 2 hd bytes a page apart, whole cache lines each, so their order costs nothing.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs p) {
  constexpr int LPH = HD / 16, HPW = 64 / LPH;
  const int lane = threadIdx.x & 63, j = lane % LPH, sub = lane / LPH;
  const int t = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  if (t >= p.T) return;
  const hxa_kv_cache &c = p.c;
  const int i = wave_count_le(c.cu + 1, c.nseq, t, lane);
  if (i >= c.nseq) return;
  const int b = c.cu[i], e = min(c.cu[i + 1], p.T);  // past T: cut there, as in the attention
  const long at = (long)c.len[i] - (e - (long)t);
  if (t < b || at < 0 || at >= (long)c.ldt * c.page) return;
  const int own = (int)at, slot = own / c.page, row = own - slot * c.page;
  const int pg = c.table[(long)i * c.ldt + slot];
  if (cache_row(pg, c.npages, c.H, 0, c.page, row) < 0) return;
  int c0, c1;
  head_chunks(p.r, j, c0, c1);
  float cs[8], sn[8];
  head_angles(p.r, j, (double)((long)c.prefix_len + own), cs, sn);
  for (int h = sub; h < c.H; h += HPW) {
    const long dst = cache_row(pg, c.npages, c.H, h, c.page, row) * HD;
    typedef typename HxaVec<T>::v8 v8;
    const T *vs = (const T *)p.v + t * p.ldv + (long)h * HD;
    const v8 v0 = *(const v8 *)(vs + 16 * j), v1 = *(const v8 *)(vs + 16 * j + 8);
    float a[8], b8[8];
    head_load((const T *)p.k + t * p.ldk + (long)h * HD, c0, c1, a, b8);
    *(v8 *)((T *)c.v + dst + 16 * j) = v0;
    *(v8 *)((T *)c.v + dst + 16 * j + 8) = v1;
    head_turn<LPH>(a, b8, p.gk, p.eps, p.r, j, c0, c1, cs, sn);
    head_store((T *)c.k + dst, c0, c1, a, b8);
  }
}

}  // namespace

int hxa_kv_check(const hxa_kv_cache *c, int T, const char *who) {
  if (!c) return hxa_set_error(HXA_E_ARG, "%s: no cache", who);
  if (c->dtype != HXA_DT_F16 && c->dtype != HXA_DT_BF16) return hxa_set_error(HXA_E_MODE, "%s: dtype %d", who, c->dtype);
  if (c->hd != 64 && c->hd != 128 && c->hd != 256) return hxa_set_error(HXA_E_MODE, "%s: heads of %d", who, c->hd);
  if (c->H <= 0 || c->H > HXA_MAX_HEADS || T > HXA_MAX_ROWS || c->page <= 0 || c->page > 65536 || c->npages <= 0 || T < 0 || c->nseq < 0 ||
      c->nseq > HXA_MAX_SEQS || c->ldt < 0 || c->prefix_len < 0)
    return hxa_set_error(HXA_E_ARG, "%s: H=%d page=%d npages=%d T=%d nseq=%d ldt=%d prefix_len=%d", who, c->H, c->page, c->npages, T,
                         c->nseq, c->ldt, c->prefix_len);
  if ((__int128)c->npages * c->H * c->page >= (__int128)1 << 32)
    return hxa_set_error(HXA_E_ARG, "%s: a pool of %d x %d x %d rows", who, c->npages, c->H, c->page);
  if ((long)c->ldt * c->page + c->prefix_len >= 1L << 30)
    return hxa_set_error(HXA_E_ARG, "%s: %d pages of %d and a prefix of %d", who, c->ldt, c->page, c->prefix_len);
  if (T > 0 && c->nseq == 0) return HXA_OK;  // no row of a sequence: nothing is done
  if (T == 0) return HXA_OK;
  if (!c->k || !c->v || ((uintptr_t)c->k | (uintptr_t)c->v) % 16) return hxa_set_error(HXA_E_ARG, "%s: pools null or not aligned", who);
  if (!c->cu || !c->len || ((uintptr_t)c->cu | (uintptr_t)c->len | (uintptr_t)c->table | (uintptr_t)c->prefix) % 4 ||
      (c->ldt > 0 && !c->table) || (c->prefix_len > 0 && !c->prefix))
    return hxa_set_error(HXA_E_ARG, "%s: plan pointers", who);
  return HXA_OK;
}

extern "C" int hxa_rope_freqs(int rot, double base, int scaling, double factor, double orig_len, double beta_fast, double beta_slow,
                              float *freq, float *mscale) {
  if (!freq || rot < 2 || rot % 2 || !(base > 1.0) || !std::isfinite(base) || !(factor >= 1.0) || !std::isfinite(factor))
    return hxa_set_error(HXA_E_ARG, "rope_freqs: rot=%d base=%g factor=%g", rot, base, factor);
  if (scaling < HXA_ROPE_PLAIN || scaling > HXA_ROPE_PARTS) return hxa_set_error(HXA_E_MODE, "rope_freqs: scaling %d", scaling);
  if (scaling == HXA_ROPE_BASE && rot < 4) return hxa_set_error(HXA_E_ARG, "rope_freqs: rot=%d has no slower pair", rot);
  if (scaling == HXA_ROPE_PARTS && (!(orig_len > 0.0) || !std::isfinite(orig_len) || !(beta_slow > 0.0) || !(beta_fast > beta_slow) ||
                                    !std::isfinite(beta_fast)))
    return hxa_set_error(HXA_E_ARG, "rope_freqs: orig_len=%g beta_fast=%g beta_slow=%g", orig_len, beta_fast, beta_slow);
  const double b = scaling == HXA_ROPE_BASE ? base * std::pow(factor, rot / (rot - 2.0)) : base;
  for (int i = 0; i < rot / 2; i++) {
    double f = std::pow(b, -2.0 * i / rot);
    if (scaling == HXA_ROPE_LINEAR) f /= factor;
    if (scaling == HXA_ROPE_PARTS) {
      // log of the turns falls linearly with i, so the share of the pair index between the two borders is the share of log(turns)
      const double turns = orig_len * f / 6.283185307179586477;
      const double keep = std::fmin(1.0, std::fmax(0.0, std::log(turns / beta_slow) / std::log(beta_fast / beta_slow)));
      f = f * keep + f / factor * (1.0 - keep);
    }
    freq[i] = (float)f;
  }
  if (mscale) *mscale = scaling == HXA_ROPE_PARTS ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  return HXA_OK;
}

extern "C" int hxa_qk_norm_rope(int dtype, const void *q, long ldq, int Hq, const void *k, long ldk, int Hk, int T, int hd,
                                const float *gq, const float *gk, float eps, const int *pos, const hxa_rope *rope, void *qo,
                                long ldqo, void *ko, long ldko, void *stream) {
  if (dtype != HXA_DT_F16 && dtype != HXA_DT_BF16) return hxa_set_error(HXA_E_MODE, "qk_norm_rope: dtype %d", dtype);
  if (hd != 64 && hd != 128 && hd != 256) return hxa_set_error(HXA_E_MODE, "qk_norm_rope: heads of %d", hd);
  if (T < 0 || T > HXA_MAX_ROWS || Hq < 0 || Hk < 0 || (long)Hq + Hk > HXA_MAX_HEADS || !(eps >= 0.0f) || !std::isfinite(eps))
    return hxa_set_error(HXA_E_ARG, "qk_norm_rope: T=%d Hq=%d Hk=%d eps=%g", T, Hq, Hk, (double)eps);
  QkArgs p{q, k, qo, ko, ldq, ldk, ldqo, ldko, Hq, Hk, T, gq, gk, eps, pos, {}, 1, 1};
  const int r = rot_of(rope, hd, p.r, "qk_norm_rope");
  if (r != HXA_OK) return r;
  if (T == 0 || Hq + Hk == 0) return HXA_OK;
  if ((Hq && (!row_ok(q, ldq, Hq, hd) || !row_ok(qo, ldqo, Hq, hd) || (q == qo && ldq != ldqo))) ||
      (Hk && (!row_ok(k, ldk, Hk, hd) || !row_ok(ko, ldko, Hk, hd) || (k == ko && ldk != ldko))))
    return hxa_set_error(HXA_E_ARG, "qk_norm_rope: pointers null or not 16-byte aligned, or strides (%ld %ld %ld %ld)", ldq, ldqo, ldk,
                         ldko);
  if (((uintptr_t)gq | (uintptr_t)gk) % 16 || (uintptr_t)pos % 4)
    return hxa_set_error(HXA_E_ARG, "qk_norm_rope: gains or positions not aligned");
  const int groups = (Hq + Hk + 1024 / hd - 1) / (1024 / hd);
  // one wave a token forms the angles once; few tokens are spread over more waves instead, a wave a group of heads (kernel us, one wave a token /
  // a wave a group: 32 + 8 heads of 128, 256 tokens 6.0 / 4.4, 1024 8.5 / 8.2, 2048 10.9 / 12.2; 10 + 2 of 256, 256 5.0 / 4.1, 1024 6.5 / 6.0, 1031
  // 6.2 / 6.5, 2048 8.2 / 9.0; two waves a token are within 10% of the better one from 1024 tokens on)
  p.parts = T < 1024 ? groups : 1;
  p.per = (groups + p.parts - 1) / p.parts;
  const long wgs = ((long)T * p.parts + 3) / 4;
  const hipStream_t st = (hipStream_t)stream;
#define HXA_QK(TY, HD) hxa_launch(qk_norm_rope_kernel<TY, HD>, dim3((unsigned)wgs), dim3(256), 0, st, p)
  if (dtype == HXA_DT_F16) {
    if (hd == 64) HXA_QK(hxa_h, 64);
    if (hd == 128) HXA_QK(hxa_h, 128);
    if (hd == 256) HXA_QK(hxa_h, 256);
  } else {
    if (hd == 64) HXA_QK(hxa_b, 64);
    if (hd == 128) HXA_QK(hxa_b, 128);
    if (hd == 256) HXA_QK(hxa_b, 256);
  }
#undef HXA_QK
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HXA_OK : hxa_set_error(HXA_E_HIP, "qk_norm_rope: %s", hipGetErrorString(e));
}

extern "C" int hxa_kv_append(const hxa_kv_cache *c, const void *k, long ldk, const void *v, long ldv, int T, const float *gk, float eps,
                             const hxa_rope *rope, void *stream) {
  int r = hxa_kv_check(c, T, "kv_append");
  if (r != HXA_OK) return r;
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return hxa_set_error(HXA_E_ARG, "kv_append: eps=%g", (double)eps);
  AppendArgs p{*c, k, v, ldk, ldv, T, gk, eps, {}};
  r = rot_of(rope, c->hd, p.r, "kv_append");
  if (r != HXA_OK) return r;
  if (T == 0 || c->nseq == 0 || c->ldt == 0) return HXA_OK;
  if (!row_ok(k, ldk, c->H, c->hd) || !row_ok(v, ldv, c->H, c->hd) || (uintptr_t)gk % 16)
    return hxa_set_error(HXA_E_ARG, "kv_append: pointers null or not 16-byte aligned, or strides (%ld %ld)", ldk, ldv);
  const unsigned wgs = (unsigned)(((long)T + 3) / 4);
  const hipStream_t st = (hipStream_t)stream;
#define HXA_AP(TY, HD) hxa_launch(kv_append_kernel<TY, HD>, dim3(wgs), dim3(256), 0, st, p)
  if (c->dtype == HXA_DT_F16) {
    if (c->hd == 64) HXA_AP(hxa_h, 64);
    if (c->hd == 128) HXA_AP(hxa_h, 128);
    if (c->hd == 256) HXA_AP(hxa_h, 256);
  } else {
    if (c->hd == 64) HXA_AP(hxa_b, 64);
    if (c->hd == 128) HXA_AP(hxa_b, 128);
    if (c->hd == 256) HXA_AP(hxa_b, 256);
  }
#undef HXA_AP
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HXA_OK : hxa_set_error(HXA_E_HIP, "kv_append: %s", hipGetErrorString(e));
}
