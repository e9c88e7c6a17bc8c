// A head's norm and rotation on hd / 16 lanes, for the kernels that bring queries and keys to their places (causal_heads.hip, kv_append_q8.hip; the
// mathematics and the lanes' shares are described in the first).
#pragma once
#include <cmath>

#include "causal.h"
#include "kernels.h"

namespace {

struct HeadRot {
  const float *freq;
  int rot, layout;
  float mscale;
};

// chunk indices (of 8 values) of lane j of a head
HXA_DEV void head_chunks(const HeadRot &r, int j, int &c0, int &c1) {
  const int nr = r.rot >> 4;  // lanes with rotated chunks
  if (j < nr && r.layout == HXA_ROPE_HALF) {
    c0 = j;
    c1 = j + nr;
  } else {  // the pairs of one chunk, or what passes (from chunk rot / 8 = 2 nr on)
    c0 = 2 * j;
    c1 = 2 * j + 1;
  }
}
// cosines and sines of lane j's 8 frequencies (8 j .. 8 j + 7 in either layout) at a position
HXA_DEV void head_angles(const HeadRot &r, int j, double pos, float (&cs)[8], float (&sn)[8]) {
  if (j >= r.rot >> 4) return;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    double turns = pos * (double)r.freq[8 * j + e] * 0.15915494309189533577;
    turns -= rint(turns);
    float s, c;
    sincospif((float)(2.0 * turns), &s, &c);
    cs[e] = c * r.mscale;
    sn[e] = s * r.mscale;
  }
}
// norm and rotation of the 16 values lane j holds (a: chunk c0, b: chunk c1)
template <int LPH>
HXA_DEV void head_turn(float (&a)[8], float (&b)[8], const float *__restrict__ gain, float eps, const HeadRot &r, int j, int c0, int c1,
                       const float (&cs)[8], const float (&sn)[8]) {
  if (gain != nullptr) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) ss = fmaf(a[e], a[e], ss);
#pragma unroll
    for (int e = 0; e < 8; e++) ss = fmaf(b[e], b[e], ss);
    ss += dpp_f<0xB1>(ss);
    ss += dpp_f<0x4E>(ss);
    if (LPH >= 8) ss += dpp_f<0x141>(ss);
    if (LPH >= 16) ss += dpp_f<0x140>(ss);
    const float k = rsqrtf(fmaf(ss, 1.0f / (16.0f * LPH), eps));
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const float4_t g0 = *(const float4_t *)(gain + 8 * c0 + e), g1 = *(const float4_t *)(gain + 8 * c1 + e);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        a[e + i] = a[e + i] * k * g0[i];
        b[e + i] = b[e + i] * k * g1[i];
      }
    }
  }
  if (j >= r.rot >> 4) return;
  if (r.layout == HXA_ROPE_HALF) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float x = a[e], y = b[e];
      a[e] = fmaf(x, cs[e], -(y * sn[e]));
      b[e] = fmaf(x, sn[e], y * cs[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float x = a[e], y = a[e + 1], z = b[e], w = b[e + 1];
      a[e] = fmaf(x, cs[e / 2], -(y * sn[e / 2]));
      a[e + 1] = fmaf(x, sn[e / 2], y * cs[e / 2]);
      b[e] = fmaf(z, cs[4 + e / 2], -(w * sn[4 + e / 2]));
      b[e + 1] = fmaf(z, sn[4 + e / 2], w * cs[4 + e / 2]);
    }
  }
}
template <typename T>
HXA_DEV void head_load(const T *__restrict__ p, int c0, int c1, float (&a)[8], float (&b)[8]) {
  typedef typename HxaVec<T>::v8 v8;
  const v8 x = *(const v8 *)(p + 8 * c0), y = *(const v8 *)(p + 8 * c1);
#pragma unroll
  for (int e = 0; e < 8; e++) {
    a[e] = (float)x[e];
    b[e] = (float)y[e];
  }
}
template <typename T>
HXA_DEV void head_store(T *__restrict__ p, int c0, int c1, const float (&a)[8], const float (&b)[8]) {
  typedef typename HxaVec<T>::v8 v8;
  v8 x, y;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    x[e] = (T)a[e];
    y[e] = (T)b[e];
  }
  *(v8 *)(p + 8 * c0) = x;
  *(v8 *)(p + 8 * c1) = y;
}

bool row_ok(const void *p, long ld, int H, int hd) { return p != nullptr && (uintptr_t)p % 16 == 0 && ld % 8 == 0 && ld >= (long)H * hd; }

int rot_of(const hxa_rope *rope, int hd, HeadRot &r, const char *who) {
  r = HeadRot{nullptr, 0, HXA_ROPE_HALF, 1.0f};
  if (rope == nullptr || rope->rot == 0) return HXA_OK;
  if (rope->rot < 0 || rope->rot > hd || rope->rot % 16)
    return hxa_set_error(HXA_E_ARG, "%s: %d rotated dims of heads of %d", who, rope->rot, hd);
  if (rope->layout != HXA_ROPE_HALF && rope->layout != HXA_ROPE_PAIRS)
    return hxa_set_error(HXA_E_MODE, "%s: rotary layout %d", who, rope->layout);
  if (rope->freq == nullptr || (uintptr_t)rope->freq % 4 || !std::isfinite(rope->mscale))
    return hxa_set_error(HXA_E_ARG, "%s: rotary frequencies or mscale", who);
  r = HeadRot{rope->freq, rope->rot, rope->layout, rope->mscale};
  return HXA_OK;
}

}  // namespace
