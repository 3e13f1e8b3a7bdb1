// Layer norm with its gradients, dropout from a counter-based generator, and rows in 8-bit integers with a scale each, for
// sm_100a.
#include "runtime.h"
#include <cmath>

using namespace cgtb;

namespace {

constexpr int kRowThreads = 256;

// Sum over a block of kRowThreads threads, in a fixed order; every thread gets it. `part`: one value per warp.
template <typename T>
__device__ __forceinline__ T block_sum(T v, T* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();   // the previous sum has been read
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  T s = T(0);
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) s += part[w];
  return s;
}

__device__ __forceinline__ float inverse_root(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double inverse_root(double v) { return 1.0 / sqrt(v); }

// ================================================================================================
// Layer norm: y = (x - m) / sqrt(v + eps) * gain + bias with the row's mean m and variance v (of the centred values, so
// that a large common offset costs no digits).
// ================================================================================================
template <typename T>
__device__ __forceinline__ void row_statistics(const T* x, long C, T eps, T* part, T& mean, T& rstd) {
  T s = T(0);
  for (long c = threadIdx.x; c < C; c += kRowThreads) s += x[c];
  mean = block_sum(s, part) / (T)C;
  T q = T(0);
  for (long c = threadIdx.x; c < C; c += kRowThreads) { const T d = x[c] - mean; q += d * d; }
  rstd = inverse_root(block_sum(q, part) / (T)C + eps);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) norm_forward_kernel(const T* __restrict__ x, const T* __restrict__ gain, const T* __restrict__ bias,
                                                                   long R, long C, T eps, T* __restrict__ y) {
  __shared__ T part[kRowThreads / 32];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    T mean, rstd;
    row_statistics(x + r * C, C, eps, part, mean, rstd);
    for (long c = threadIdx.x; c < C; c += kRowThreads) y[r * C + c] = (x[r * C + c] - mean) * rstd * gain[c] + bias[c];
  }
}

// dx = rstd * (d - mean(d) - xh * mean(d * xh)) with xh = (x - m) * rstd and d = gy * gain; the row's statistics are formed
// again from x, which is read anyway, and kept for the sums over the rows.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) norm_backward_kernel(const T* __restrict__ x, const T* __restrict__ gain, const T* __restrict__ gy,
                                                                    long R, long C, T eps, T* __restrict__ dx, T* __restrict__ stats) {
  __shared__ T part[kRowThreads / 32];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    T mean, rstd;
    row_statistics(x + r * C, C, eps, part, mean, rstd);
    T s1 = T(0), s2 = T(0);
    for (long c = threadIdx.x; c < C; c += kRowThreads) {
      const T d = gy[r * C + c] * gain[c];
      s1 += d;
      s2 += d * ((x[r * C + c] - mean) * rstd);
    }
    s1 = block_sum(s1, part) / (T)C;
    s2 = block_sum(s2, part) / (T)C;
    for (long c = threadIdx.x; c < C; c += kRowThreads) {
      const T d = gy[r * C + c] * gain[c], xh = (x[r * C + c] - mean) * rstd;
      dx[r * C + c] = rstd * (d - s1 - xh * s2);
    }
    if (threadIdx.x == 0) { stats[2 * r] = mean; stats[2 * r + 1] = rstd; }
  }
}

// sums over the rows of slice blockIdx.y: part[slice][0][c] of gy * xh, part[slice][1][c] of gy
template <typename T>
__global__ void __launch_bounds__(kRowThreads) norm_columns_kernel(const T* __restrict__ x, const T* __restrict__ gy, const T* __restrict__ stats,
                                                                   long R, long C, long rows_per_slice, T* __restrict__ part) {
  const long c = (long)blockIdx.x * kRowThreads + threadIdx.x;
  if (c >= C) return;
  const long first = blockIdx.y * rows_per_slice;
  const long last = first + rows_per_slice < R ? first + rows_per_slice : R;
  T s1 = T(0), s2 = T(0);
  for (long r = first; r < last; ++r) {
    const T g = gy[r * C + c];
    s1 += g * ((x[r * C + c] - stats[2 * r]) * stats[2 * r + 1]);
    s2 += g;
  }
  part[(2 * (long)blockIdx.y) * C + c] = s1;
  part[(2 * (long)blockIdx.y + 1) * C + c] = s2;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) norm_fold_kernel(const T* __restrict__ part, long C, int slices, T* __restrict__ dgain, T* __restrict__ dbias) {
  const long c = (long)blockIdx.x * kRowThreads + threadIdx.x;
  if (c >= C) return;
  T s1 = T(0), s2 = T(0);
  for (int s = 0; s < slices; ++s) {
    s1 += part[(2L * s) * C + c];
    s2 += part[(2L * s + 1) * C + c];
  }
  dgain[c] = s1;
  dbias[c] = s2;
}

template <typename T>
int norm_forward(const T* x, long R, long C, const T* gain, const T* bias, double eps, T* y) {
  const long grid = R < 65536 ? R : 65536;
  CGTB_LAUNCH(norm_forward_kernel<T>, (unsigned)grid, kRowThreads, 0, x, gain, bias, R, C, (T)eps, y);
  CGTB_CHECK_LAUNCH("layer_norm_forward");
  return 0;
}

template <typename T>
int norm_backward(const T* x, const T* gain, const T* gy, long R, long C, double eps, T* dx, T* dgain, T* dbias) {
  const long cblocks = cgtb_ceil_div(C, kRowThreads);
  long slices = cgtb_ceil_div(R, 64);
  if (slices > 64) slices = 64;
  T* stats = (T*)scratch((size_t)(2 * R + 2 * slices * C) * sizeof(T));
  if (!stats) return 1;
  T* part = stats + 2 * R;
  const long grid = R < 65536 ? R : 65536;
  CGTB_LAUNCH(norm_backward_kernel<T>, (unsigned)grid, kRowThreads, 0, x, gain, gy, R, C, (T)eps, dx, stats);
  CGTB_LAUNCH(norm_columns_kernel<T>, dim3((unsigned)cblocks, (unsigned)slices), kRowThreads, 0, x, gy, stats, R, C, cgtb_ceil_div(R, slices), part);
  CGTB_LAUNCH(norm_fold_kernel<T>, (unsigned)cblocks, kRowThreads, 0, part, C, (int)slices, dgain, dbias);
  CGTB_CHECK_LAUNCH("layer_norm_backward");
  return 0;
}

int norm_extents(const char* who, long R, long C, double eps) {
  if (R < 0 || C < 0) return fail("%s: negative extent", who);
  if (C > 0x7fffffffL) return fail("%s: rows of %ld elements are too long (at most 2^31 - 1)", who, C);
  if (!(eps >= 0) || std::isinf(eps)) return fail("%s: epsilon has to be a finite number that is not negative", who);
  return 0;
}

// ================================================================================================
// Dropout. Element i takes word i % 4 of the Philox4x32-10 block (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as
// easy as 1, 2, 3; 2011) with key = seed and counter = (i / 4, step, site): the mask is a function of the element's place,
// so the backward pass forms it again and nothing is stored.
// ================================================================================================
__device__ __forceinline__ uint4 philox(uint4 c, uint2 k) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p0 = (unsigned long long)0xD2511F53u * c.x, p1 = (unsigned long long)0xCD9E8D57u * c.z;
    c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k.x, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k.y, (uint32_t)p0);
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, long n, uint32_t threshold, T scale, const long* __restrict__ state,
                                                      uint32_t site, T* y) {
  const unsigned long long seed = (unsigned long long)state[0], step = (unsigned long long)state[1];
  const long blocks = (n + 3) / 4;
  for (long b = blockIdx.x * 256L + threadIdx.x; b < blocks; b += gridDim.x * 256L) {
    const uint4 w = philox(make_uint4((uint32_t)b, (uint32_t)((unsigned long long)b >> 32), (uint32_t)step, site), make_uint2((uint32_t)seed, (uint32_t)(seed >> 32)));
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * b + j < n) y[4 * b + j] = ws[j] >= threshold ? x[4 * b + j] * scale : T(0);
  }
}

// ================================================================================================
// Rows in 8-bit integers: a = max |x|, scale = a / 127, code = 127 x / a rounded to nearest, ties to even.
// ================================================================================================

// The exact code of x: the quotient of two numbers of 31 and 24 bits is never rounded across a tie in 64 bits.
__device__ __noinline__ float code_exact(float x, float largest) { return (float)rint(127.0 * (double)x / (double)largest); }

// `inverse` = 127 / largest in 32 bits. x * inverse is off by less than 127 * 2^-22 = 3e-5: wherever it is not that near to a
// tie, its nearest whole number is the exact quotient's.
__device__ __forceinline__ float code_of(float x, float largest, float inverse) {
  const float t = x * inverse, k = rintf(t);
  return fabsf(t - k) < 0.4999f ? k : code_exact(x, largest);   // also for an inverse that overflows: then t is not finite
}

__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(const float* __restrict__ x, long R, long C, long Cp, int8_t* __restrict__ codes,
                                                                    float* __restrict__ scales) {
  __shared__ uint32_t part[kRowThreads / 32];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    uint32_t m = 0;   // as whole numbers the bits of |x| order like the values, infinities and NaN above all
    for (long c = threadIdx.x; c < C; c += kRowThreads) m = max(m, __float_as_uint(x[r * C + c]) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < kRowThreads / 32; ++w) m = max(m, part[w]);
    const bool finite = m < 0x7f800000u;
    const float largest = __uint_as_float(m), inverse = 127.0f / largest;
    for (long c = threadIdx.x; c < Cp; c += kRowThreads)
      codes[r * Cp + c] = (int8_t)(c < C && finite && m != 0 ? code_of(x[r * C + c], largest, inverse) : 0.0f);
    if (threadIdx.x == 0) scales[r] = finite ? largest / 127.0f : __uint_as_float(0x7fc00000u);
  }
}

}  // namespace

CGTB_API int cgtb_layer_norm_forward(int dtype, const void* x, long R, long C, const void* gain, const void* bias, double epsilon, void* y) {
  if (!require_runtime("cgtb_layer_norm_forward")) return 1;
  if (norm_extents("cgtb_layer_norm_forward", R, C, epsilon)) return 1;
  if (R == 0 || C == 0) return 0;
  if (dtype == cgtb_f4) return norm_forward((const float*)x, R, C, (const float*)gain, (const float*)bias, epsilon, (float*)y);
  if (dtype == cgtb_f8) return norm_forward((const double*)x, R, C, (const double*)gain, (const double*)bias, epsilon, (double*)y);
  return fail("cgtb_layer_norm_forward: unsupported dtype %d", dtype);
}

CGTB_API int cgtb_layer_norm_backward(int dtype, const void* x, const void* gain, const void* gy, long R, long C, double epsilon, void* dx, void* dgain,
                                      void* dbias) {
  if (!require_runtime("cgtb_layer_norm_backward")) return 1;
  if (norm_extents("cgtb_layer_norm_backward", R, C, epsilon)) return 1;
  if (dtype != cgtb_f4 && dtype != cgtb_f8) return fail("cgtb_layer_norm_backward: unsupported dtype %d", dtype);
  if (C == 0) return 0;
  if (R == 0) {   // sums of no rows
    if (cgtb_memset(dgain, 0, C * (dtype == cgtb_f4 ? 4 : 8))) return 1;
    return cgtb_memset(dbias, 0, C * (dtype == cgtb_f4 ? 4 : 8));
  }
  if (dtype == cgtb_f4)
    return norm_backward((const float*)x, (const float*)gain, (const float*)gy, R, C, epsilon, (float*)dx, (float*)dgain, (float*)dbias);
  return norm_backward((const double*)x, (const double*)gain, (const double*)gy, R, C, epsilon, (double*)dx, (double*)dgain, (double*)dbias);
}

CGTB_API int cgtb_dropout(int dtype, const void* x, long n, double p, const int64_t* state, unsigned site, void* y) {
  if (!require_runtime("cgtb_dropout")) return 1;
  if (!(p >= 0 && p < 1)) return fail("cgtb_dropout: the probability has to be in [0, 1)");
  if (n < 0) return fail("cgtb_dropout: negative extent");
  if (dtype != cgtb_f4 && dtype != cgtb_f8) return fail("cgtb_dropout: unsupported dtype %d", dtype);
  if (n == 0) return 0;
  // a word below the threshold drops its element; the largest p below 1 rounds to 2^32, which no word reaches
  const double t = std::nearbyint(p * 4294967296.0);
  const uint32_t threshold = t >= 4294967295.0 ? 4294967295u : (uint32_t)t;
  const double scale = 1.0 / (1.0 - p);
  const long blocks = cgtb_ceil_div(cgtb_ceil_div(n, 4), 256);
  const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
  if (dtype == cgtb_f4)
    CGTB_LAUNCH(dropout_kernel<float>, grid, 256, 0, (const float*)x, n, threshold, (float)scale, (const long*)state, site, (float*)y);
  else
    CGTB_LAUNCH(dropout_kernel<double>, grid, 256, 0, (const double*)x, n, threshold, scale, (const long*)state, site, (double*)y);
  CGTB_CHECK_LAUNCH("dropout");
  return 0;
}

CGTB_API int cgtb_quantize_rows(const float* x, long R, long C, int8_t* codes, float* scales) {
  if (!require_runtime("cgtb_quantize_rows")) return 1;
  if (R < 0 || C < 0) return fail("cgtb_quantize_rows: negative extent");
  if (R == 0) return 0;
  const unsigned grid = (unsigned)(R < 65536 ? R : 65536);
  CGTB_LAUNCH(quantize_rows_kernel, grid, kRowThreads, 0, x, R, C, cgtb_ceil_div(C, 16) * 16, codes, scales);
  CGTB_CHECK_LAUNCH("quantize_rows");
  return 0;
}
