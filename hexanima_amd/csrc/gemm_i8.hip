// Products of int8 activations and int8 weights with a scale for each token and each channel (hxa_linear_i8):
// out[m][n] = sa[m] sw[n] sum_k a[m][k] w[n][k] + bias[n], the sum in int32 (exact), scales and bias in fp32, one rounding to 16 bits.
//
// The loops are gemm_kernel.h's and gemm_skinny.hip's (format HXG_I8): what moves is the same bytes a stage as with fp16 operands, 128 of each
// row, and a stage holds 128 k. v_mfma_i32_16x16x64_i8 takes the same 16 bytes a lane and operand as the fp16 instruction, in the same cycles.
// Bound by the matrix cores from about a thousand rows on: 6500 x 2048 -> 16384 228 us (1.92 POP/s in 6.5 rounds of 256 x 256 tiles), 8192 cubed
// 2.22 - 2.28 POP/s; below by the weights' bytes and a tile's chain of stages (64 x 8192 -> 2048 7.7 us, 1000 x 8192 -> 2048 24.8).
#define HXG_INSTANTIATE
#include "gemm_kernel.h"

namespace hxg {
template hipError_t launch_fmt<HXG_I8, false>(int, int, const GemmParamsI8 &, int, hipStream_t);
}
using namespace hxg;

namespace {

int ncu_i8() {
  static const int n = [] {
    int dev = 0, c = 0;
    if (hipGetDevice(&dev) != hipSuccess) dev = 0;
    return hipDeviceGetAttribute(&c, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && c > 0 ? c : 256;
  }();
  return n;
}

// K slices' int32 sums p[z][m][n] added and scaled: eight columns of a row a thread
__global__ __launch_bounds__(256) void sum_i8_kernel(GemmParamsI8 p, const int *__restrict__ part, int S) {
  const int c8 = p.N / 8;
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  if (c >= (long)p.M * c8) return;
  const int m = (int)(c / c8), n = (int)(c % c8) * 8;
  int4_t a0 = {}, a1 = {};
  for (int z = 0; z < S; z++) {
    const int *q = part + ((long)z * p.M + m) * p.N + n;
    a0 += *(const int4_t *)q;
    a1 += *(const int4_t *)(q + 4);
  }
  const float sa = p.sa[m];
  const float4_t w0 = *(const float4_t *)(p.sw + n), w1 = *(const float4_t *)(p.sw + n + 4);
  const float4_t b0 = p.bias ? *(const float4_t *)(p.bias + n) : (float4_t){}, b1 = p.bias ? *(const float4_t *)(p.bias + n + 4) : (float4_t){};
  const uint2_t x = p.dtype == HXA_DT_F16 ? scale_i8<hxa_h>(a0, sa, w0, b0) : scale_i8<__bf16>(a0, sa, w0, b0);
  const uint2_t y = p.dtype == HXA_DT_F16 ? scale_i8<hxa_h>(a1, sa, w1, b1) : scale_i8<__bf16>(a1, sa, w1, b1);
  *(uint4_t *)(p.out + (long)m * p.ldo + n) = (uint4_t){x.x, x.y, y.x, y.y};
}

// Cost of a form, as gemm.hip's: rounds of workgroups over the CUs x (a BM BN K + b) + c us, and for K slices the sum's launch and its bytes. bn 32, 16: gemm_skinny.hip's
// tiles (2048 x 8192 weights, one token: 16 x 16 over 8 waves 6.5, 32 x 32 over 4 9.6; 64 tokens: 32 x 16 9.4, 32 x 32 11.8, 64 x 64 in four slices 12.3).
// Fitted to every tile timed, weights from HBM, on 174 (M, N, K) of 1 - 6500 rows x 10 weights of 1 - 34 MB, in one to eight slices; the
// choice is 1.0% above the fastest form (geometric mean).
struct Cost {
  int bm, bn;
  float a, b, c;  // a per 2^20 BM BN K
};
constexpr Cost kCost[] = {
    {256, 256, 0.1647f, 9.89f, 3.83f}, {256, 192, 0.1936f, 7.32f, 3.54f}, {192, 256, 0.1934f, 7.97f, 2.80f}, {192, 192, 0.1765f, 8.45f, 1.19f},
    {256, 128, 0.1776f, 7.63f, 1.56f}, {128, 256, 0.1922f, 7.32f, 1.94f}, {192, 128, 0.1991f, 6.88f, 0.76f}, {128, 128, 0.2513f, 5.51f, 0.47f},
    {64, 128, 0.3865f, 1.03f, 3.17f}, {128, 64, 0.3898f, 0.26f, 4.05f}, {64, 64, 0.4510f, 1.20f, 2.92f}, {64, 32, 0.5902f, 2.01f, 1.97f},
    {32, 32, 0.8709f, 1.43f, 2.45f}, {32, 16, 0.9046f, 1.10f, 3.31f}, {16, 16, 1.3548f, 0.47f, 4.06f},
};
constexpr double kSumUs = 3.0, kSumBytesPerUs = 12.0e6;
struct Form {
  int bm, bn, ksplit;
};
bool built(int bm, int bn) {
  for (const Cost &c : kCost)
    if (c.bm == bm && c.bn == bn) return true;
  return false;
}
long tiles_of(int n, int b) { return ((long)n + b - 1) / b; }
int padded(int K) { return (K + 127) / 128 * 128; }
double cost_of(const Cost &c, int M, int N, int K, int S) {
  const long ncu = ncu_i8(), tiles = tiles_of(M, c.bm) * tiles_of(N, c.bn) * S;
  return (double)((tiles + ncu - 1) / ncu) * (c.a / 1048576.0 * c.bm * c.bn * (K / S) + c.b) + c.c;
}
Form form_of(int M, int N, int K, bool split) {
  K = padded(K);
  Form f{64, 64, 1};
  double best = 1e30;
  for (int S = 1; S <= (split ? 8 : 1); S *= 2) {
    if (K % (128 * S) || (S > 1 && K / S < 512)) continue;
    const double sum = S == 1 ? 0.0 : kSumUs + (8.0 * S + 2.0) * M * (double)N / kSumBytesPerUs;
    for (const Cost &c : kCost) {
      if (c.bn <= 32 && S > 1) continue;
      const double t = cost_of(c, M, N, K, S) + sum;
      if (t < best) best = t, f = Form{c.bm, c.bn, S};
    }
  }
  return f;
}

int prepare(GemmParamsI8 &p, int dtype, const void *a, long lda, const float *sa, int M, const void *w, long ldw, const float *sw, int N, int K,
            const float *bias, void *out, long ldo, const char *who) {
  if (dtype != HXA_DT_F16 && dtype != HXA_DT_BF16) return hxa_set_error(HXA_E_MODE, "%s: dtype %d", who, dtype);
  if (M < 0 || N < 0 || N % 8 || K < 1 || K > HXA_I8_MAX_K)
    return hxa_set_error(HXA_E_ARG, "%s: M=%d N=%d K=%d", who, M, N, K);
  if (M == 0 || N == 0) return HXA_OK;
  const int Kp = padded(K);
  if (!a || !w || !out || !sa || !sw || ((uintptr_t)a | (uintptr_t)w | (uintptr_t)out | (uintptr_t)sw | (uintptr_t)bias) % 16 || (uintptr_t)sa % 4)
    return hxa_set_error(HXA_E_ARG, "%s: pointers null or not aligned", who);
  if (lda % 16 || ldw % 16 || lda < Kp || ldw < Kp || lda >= 1L << 23 || ldw >= 1L << 23 || ldo % 8 || ldo < N)
    return hxa_set_error(HXA_E_ARG, "%s: strides (%ld %ld %ld) for N=%d K=%d", who, lda, ldw, ldo, N, K);
  p.A = (const hxa_h *)a;
  p.lda = lda / 2;
  p.W = w;
  p.w_rs = ldw / 2;
  p.w_gs = 32;
  p.M = M;
  p.N = N;
  p.Ktot = Kp / 2;
  p.out = (hxa_h *)out;
  p.ldo = ldo;
  p.sa = sa;
  p.sw = sw;
  p.bias = bias;
  p.dtype = dtype;
  p.clk = g_hxa_clk_gemm;
  return HXA_OK;
}

int launch(GemmParamsI8 &p, const Form &f, void *ws, hipStream_t st, const char *who) {
  const bool split = f.ksplit > 1;
  p.Kslice = p.Ktot / f.ksplit;
  p.epi = split ? HXA_EPI_PARTIAL_F32 : HXA_EPI_STORE;
  p.tiles_m = (int)tiles_of(p.M, f.bm);
  p.tiles_n = (int)tiles_of(p.N, f.bn);
  const int waves = f.bn <= 32 ? f.bn == 16 ? 8 : 4 : tile_nw(f.bm, f.bn, HXG_I8);
  if ((long)p.tiles_m * p.tiles_n * 64 * waves >= 1L << 32) return hxa_set_error(HXA_E_ARG, "%s: M=%d N=%d are too many tiles", who, p.M, p.N);
  // 8 XCD rectangles of the fewest A + W bytes, as gemm_prepare's
  long best = -1;
  for (int gm = 1; gm <= 8; gm *= 2) {
    if (p.tiles_m % gm || p.tiles_n % (8 / gm)) continue;
    const long bytes = (long)(p.tiles_m / gm) * f.bm + (long)(p.tiles_n / (8 / gm)) * f.bn;
    if (best < 0 || bytes < best) best = bytes, p.xcd_gm = gm;
  }
  hipError_t e;
  if (f.bn <= 32) {
    e = launch_skinny_i8(f.bm, f.bn, p, st);
  } else if (!split) {
    e = launch_fmt<HXG_I8, false>(f.bm, f.bn, p, 1, st);
  } else {
    GemmParamsI8 q = p;
    q.out32 = (float *)ws;
    q.ldo = p.N;
    q.out_zstride = (long)p.M * p.N;
    e = launch_fmt<HXG_I8, false>(f.bm, f.bn, q, f.ksplit, st);
    if (e == hipSuccess) {
      const long chunks = (long)p.M * (p.N / 8);
      hxa_launch(sum_i8_kernel, dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, st, p, (const int *)ws, f.ksplit);
      e = hipGetLastError();
    }
  }
  return e == hipSuccess ? HXA_OK : hxa_set_error(HXA_E_HIP, "%s: %s", who, hipGetErrorString(e));
}

long ws_of(const Form &f, int M, int N) { return f.ksplit > 1 ? (long)f.ksplit * M * N * 4 : 0; }

}  // namespace

extern "C" long hxa_linear_i8_ws_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || N % 8 || K < 1 || K > HXA_I8_MAX_K) return 0;
  return ws_of(form_of(M, N, K, true), M, N);
}

extern "C" int hxa_linear_i8(int dtype, const void *a, long lda, const float *sa, int M, const void *w, long ldw, const float *sw, int N, int K,
                             const float *bias, void *out, long ldo, void *ws, long ws_bytes, void *stream) {
  GemmParamsI8 p{};
  const int r = prepare(p, dtype, a, lda, sa, M, w, ldw, sw, N, K, bias, out, ldo, "linear_i8");
  if (r != HXA_OK || M == 0 || N == 0) return r;
  if ((uintptr_t)ws % 16) return hxa_set_error(HXA_E_ARG, "linear_i8: workspace not aligned");
  Form f = form_of(M, N, K, true);
  if (f.ksplit > 1 && (ws == nullptr || ws_bytes < ws_of(f, M, N))) f = form_of(M, N, K, false);
  return launch(p, f, ws, (hipStream_t)stream, "linear_i8");
}

extern "C" int hxa_linear_i8_tile(int dtype, const void *a, long lda, const float *sa, int M, const void *w, long ldw, const float *sw, int N, int K,
                                  const float *bias, void *out, long ldo, int bm, int bn, int ksplit, void *ws, long ws_bytes, void *stream) {
  GemmParamsI8 p{};
  const int r = prepare(p, dtype, a, lda, sa, M, w, ldw, sw, N, K, bias, out, ldo, "linear_i8_tile");
  if (r != HXA_OK || M == 0 || N == 0) return r;
  const Form f{bm, bn, ksplit};
  if (!built(bm, bn) || ksplit < 1 || ksplit > 64 || padded(K) % (128 * ksplit) || (bn <= 32 && ksplit > 1))
    return hxa_set_error(HXA_E_ARG, "linear_i8_tile: tile %d x %d, %d slices of K=%d", bm, bn, ksplit, K);
  if (ksplit > 1 && (ws == nullptr || (uintptr_t)ws % 16 || ws_bytes < ws_of(f, M, N)))
    return hxa_set_error(HXA_E_ARG, "linear_i8_tile: workspace");
  return launch(p, f, ws, (hipStream_t)stream, "linear_i8_tile");
}
