// Rows of 16-bit values to int8 with a scale each (hxa_quantize_rows): s = max |x| / 127, q = x (1 / max |x| * 127) rounded to the nearest integer.
//
// Bound by HBM: 2 bytes read and 1 written per value. A row is held in registers between its maximum and its rounding, so it is read once: by one
// wave where rows are short and many (no barrier), else by the four waves of a workgroup; rows of more than 16384 values are read a second time. 6500 rows
// of 8192 33.7 us (4.7 TB/s; a large copy 5.1), one row of 2048 2.1 us, a launch's time.
#include <algorithm>

#include "causal.h"
#include "int8_rows.h"
#include "kernels.h"

namespace {

struct QuantArgs {
  const void *x;
  long ldx, ldq;
  int M, K;
  int8_t *q;
  float *s;
};

// W waves a row, N chunks of 8 values a thread at a time
template <typename T, int W, int N>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantArgs p) {
  typedef typename HxaVec<T>::v8 v8 __attribute__((aligned(2)));  // rows begin anywhere (a contiguous matrix of an odd number of columns)
  constexpr int TPR = 64 * W;
  const int t = threadIdx.x % TPR;
  const long m = (long)blockIdx.x * (4 / W) + threadIdx.x / TPR;
  if (W == 1 && m >= p.M) return;
  const T *x = (const T *)p.x + m * p.ldx;
  int8_t *q = p.q + m * p.ldq;
  const int whole = p.K / 8, chunks = (p.K + 127) / 128 * 16;  // chunks of values alone, chunks written
  float v[N][8];
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int c = base + i * TPR + t;
      if (c < whole) {
        const v8 y = *(const v8 *)(x + 8 * c);
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = (float)y[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = 8 * c + e < p.K ? (float)x[8 * c + e] : 0.0f;
      }
    }
  };
  float top = 0.0f;
  for (int base = 0; base < chunks; base += N * TPR) {
    load(base);
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) top = fmaxf(top, finite_abs(v[i][e]));
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if constexpr (W == 4) {
    __shared__ float tops[4];
    if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  }
  const float least = fmaxf(top, 127.0f * HXA_Q8_LEAST);
  const float inv = top > 0.0f ? 1.0f / least * 127.0f : 0.0f;
  if (t == 0) p.s[m] = q8_scale(top);
  const bool again = chunks > N * TPR;
  for (int base = 0; base < chunks; base += N * TPR) {
    if (again) load(base);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int c = base + i * TPR + t;
      if (c < chunks) *(uint2_t *)(q + 8 * c) = q8_pack(v[i], inv);
    }
  }
}

}  // namespace

extern "C" int hxa_quantize_rows(int dtype, const void *x, long ldx, int M, int K, void *q, long ldq, float *scale, void *stream) {
  if (dtype != HXA_DT_F16 && dtype != HXA_DT_BF16) return hxa_set_error(HXA_E_MODE, "quantize_rows: dtype %d", dtype);
  if (M < 0 || M > HXA_MAX_ROWS || K < 1 || K > HXA_I8_MAX_K) return hxa_set_error(HXA_E_ARG, "quantize_rows: M=%d K=%d", M, K);
  if (M == 0) return HXA_OK;
  if (!x || (uintptr_t)x % 2 || !q || (uintptr_t)q % 16) return hxa_set_error(HXA_E_ARG, "quantize_rows: pointers null or not aligned");
  if (!scale || (uintptr_t)scale % 4) return hxa_set_error(HXA_E_ARG, "quantize_rows: scales null or not aligned");
  if (ldx < K || ldq % 16 || ldq < (K + 127) / 128 * 128)
    return hxa_set_error(HXA_E_ARG, "quantize_rows: strides (%ld %ld) for K=%d", ldx, ldq, K);
  const hipStream_t st = (hipStream_t)stream;
  const bool one = M >= 1024 && K <= 2048;
  constexpr int MOST = 1 << 23;  // rows a launch: a grid has fewer than 2^32 threads
  auto run = [&](auto ty) {
    typedef decltype(ty) T;
    for (long m0 = 0; m0 < M; m0 += MOST) {
      const int n = (int)std::min<long>(M - m0, MOST);
      const QuantArgs p{(const T *)x + m0 * ldx, ldx, ldq, n, K, (int8_t *)q + m0 * ldq, scale + m0};
      if (one) hxa_launch(quant_rows_kernel<T, 1, 4>, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, p);
      else if (K <= 2048) hxa_launch(quant_rows_kernel<T, 4, 1>, dim3((unsigned)n), dim3(256), 0, st, p);
      else if (K <= 8192) hxa_launch(quant_rows_kernel<T, 4, 4>, dim3((unsigned)n), dim3(256), 0, st, p);
      else hxa_launch(quant_rows_kernel<T, 4, 8>, dim3((unsigned)n), dim3(256), 0, st, p);
    }
  };
  if (dtype == HXA_DT_F16) run(hxa_h{});
  else run(hxa_b{});
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HXA_OK : hxa_set_error(HXA_E_HIP, "quantize_rows: %s", hipGetErrorString(e));
}
