// The matrix product of rows in 8-bit integers with weights in 8-bit integers, for sm_100a:
//   y[m, n] = (sum_k a[m, k] * b[n, k]) * sa[m] * sb[n] + bias[n]
// The sum of products of whole numbers is exact (32-bit integers); the three operations behind it round in float32.
#include "runtime.h"

using namespace cgtb;

namespace {

// one thread per result
__global__ void __launch_bounds__(256) int8_product_kernel(const int8_t* __restrict__ a, const float* __restrict__ sa, const int8_t* __restrict__ b,
                                                           const float* __restrict__ sb, const float* __restrict__ bias, long M, long N, long K,
                                                           float* __restrict__ y) {
  for (long o = blockIdx.x * 256L + threadIdx.x; o < M * N; o += gridDim.x * 256L) {
    const long m = o / N, n = o - m * N;
    const int* pa = (const int*)(a + m * K);
    const int* pb = (const int*)(b + n * K);
    int s = 0;
    for (long k = 0; k < K / 4; ++k) s = __dp4a(pa[k], pb[k], s);
    float v = (float)s * sa[m] * sb[n];
    if (bias) v += bias[n];
    y[o] = v;
  }
}

}  // namespace

CGTB_API int cgtb_int8_product(const int8_t* a, const float* sa, const int8_t* b, const float* sb, const float* bias, long M, long N, long K, float* y) {
  if (!require_runtime("cgtb_int8_product")) return 1;
  if (M < 0 || N < 0 || K < 0) return fail("cgtb_int8_product: negative extent");
  if (K % 16) return fail("cgtb_int8_product: rows of %ld codes; they have to be padded with zeros to a multiple of 16", K);
  if (K >= CGTB_INT8_MAX_K) return fail("cgtb_int8_product: rows of %ld codes; the 32-bit sums hold fewer than %d", K, CGTB_INT8_MAX_K);
  if (((uintptr_t)a | (uintptr_t)b) & 15) return fail("cgtb_int8_product: the codes have to start on a 16-byte boundary");
  if (M == 0 || N == 0) return 0;
  const long blocks = cgtb_ceil_div(M * N, 256);
  CGTB_LAUNCH(int8_product_kernel, (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), 256, 0, a, sa, b, sb, bias, M, N, K, y);
  CGTB_CHECK_LAUNCH("int8_product");
  return 0;
}
