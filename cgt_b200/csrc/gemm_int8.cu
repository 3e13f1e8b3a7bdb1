// The matrix product of rows in 8-bit integers with weights in 8-bit integers, for sm_100a:
//   y[m, n] = (sum_k a[m, k] * b[n, k]) * sa[m] * sb[n] + bias[n]
// The sum of products of whole numbers is exact (32-bit integers); the three operations behind it round in float32.
#include <cuda.h>  // CUtensorMap and its enums; the encoder is looked up at run time, libcuda is not linked

#include <algorithm>

#include "runtime.h"
#include "tc_util.h"

using namespace cgtb;
using namespace cgtb::tc;

namespace {

constexpr int kRows = 128;          // rows of a per tile: the tensor core's M
constexpr int kDepth = 128;         // codes of K per stage: one 128-byte swizzle row
constexpr int kMaxStages = 8;
constexpr int kEpilogueWarps = 4;   // one for each quarter of the accumulator's lanes
constexpr int kThreads = kEpilogueWarps * 32 + 64;
constexpr int kPitch = 36;          // floats per row of an epilogue warp's 32 x 32 block: 16-byte accesses without bank conflicts
constexpr int kGroup = 16;          // row tiles that are walked together: their codes and the weights stay in L2

struct Params {
  const float *sa, *sb, *bias;
  float* y;
  long M, N, K;
  int BN, stages, tmem_cols, a_bytes;
  int mtiles, ntiles;
  long total;
  int vec;
  int* err;
};

struct Tile { long m0, n0; };
__device__ __forceinline__ Tile tile_of(const Params& p, long t) {
  const long per = (long)kGroup * p.ntiles, g = t / per, first = g * kGroup;
  const long rows = p.mtiles - first < kGroup ? p.mtiles - first : kGroup, r = t - g * per;
  return Tile{(first + r % rows) * kRows, (r / rows) * p.BN};
}

// D 32-bit integers, A and B signed 8-bit integers, both K-major
__device__ __forceinline__ uint32_t idesc_int8(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ void mma_int8(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// One CTA per SM walks tiles of 128 x BN results. One thread issues the TMA loads of a ring of stages (128 codes of K: 128 bytes
// of every row of a and of b), one thread the MMAs (four of K = 32 per stage) into one of two accumulators in TMEM, four warps
// turn the other accumulator into results meanwhile. Rows and codes beyond the operands arrive as zeros; what a box that is
// shorter than 128 rows leaves in its stage feeds rows that are not stored.
__global__ void __launch_bounds__(kThreads, 1)
int8_product_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t a_stage = kRows * kDepth, stage_bytes = a_stage + (uint32_t)p.BN * kDepth;
  volatile int* abortp = &abort_flag;
  const int nkb = (int)((p.K + kDepth - 1) / kDepth);

  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), kEpilogueWarps);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kEpilogueWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((uint32_t)p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;

  if (warp < kEpilogueWarps) {
    float* block = reinterpret_cast<float*>(smem + (size_t)p.stages * stage_bytes) + warp * 32 * kPitch;
    uint32_t it = 0;
    for (long t = blockIdx.x; t < p.total; t += gridDim.x, ++it) {
      const Tile c = tile_of(p, t);
      const uint32_t buf = it & 1u;
      bool ok = mbar_wait_or_abort(smem_u32(&acc_full[buf]), (it >> 1) & 1u, abortp);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        *abortp = 1;
        if (lane == 0) { *(volatile int*)p.err = 3; __threadfence_system(); }
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const long mrow = c.m0 + warp * 32 + lane;      // the row of this lane's accumulators
      const float scale = mrow < p.M ? p.sa[mrow] : 0.f;
      const long mfirst = c.m0 + warp * 32;
      const int nrows = (int)(p.M - mfirst < 32 ? p.M - mfirst : 32);
      for (int ch = 0; ch < p.BN / 32; ++ch) {
        uint32_t r[32];
        tmem_ld32(tmem + ((uint32_t)(warp * 32) << 16) + buf * (uint32_t)p.BN + (uint32_t)ch * 32u, r);
        const long n0 = c.n0 + ch * 32;
        __syncwarp();   // the block's previous content has been read
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<float4*>(block + lane * kPitch + 4 * q) =
              make_float4((float)(int)r[4 * q] * scale, (float)(int)r[4 * q + 1] * scale, (float)(int)r[4 * q + 2] * scale, (float)(int)r[4 * q + 3] * scale);
        __syncwarp();
        if (p.vec) {      // N a multiple of four: a warp stores four rows of 128 bytes at a time
          const int q = lane & 7;
          const long n = n0 + 4 * q;
          if (n < p.N) {
            const float4 s = make_float4(p.sb[n], p.sb[n + 1], p.sb[n + 2], p.sb[n + 3]);
            const float4 b = p.bias ? make_float4(p.bias[n], p.bias[n + 1], p.bias[n + 2], p.bias[n + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
            for (int row = lane >> 3; row < nrows; row += 4) {
              const float4 v = *reinterpret_cast<const float4*>(block + row * kPitch + 4 * q);
              *reinterpret_cast<float4*>(p.y + (mfirst + row) * p.N + n) =
                  p.bias ? make_float4(v.x * s.x + b.x, v.y * s.y + b.y, v.z * s.z + b.z, v.w * s.w + b.w)
                         : make_float4(v.x * s.x, v.y * s.y, v.z * s.z, v.w * s.w);
            }
          }
        } else {
          const long n = n0 + lane;
          if (n < p.N) {
            const float s = p.sb[n], b = p.bias ? p.bias[n] : 0.f;
            for (int row = 0; row < nrows; ++row) {
              const float v = block[row * kPitch + lane];
              p.y[(mfirst + row) * p.N + n] = p.bias ? v * s + b : v * s;
            }
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&acc_empty[buf]));
    }
  } else if (warp == kEpilogueWarps) {
    // MMA issuer
    const uint32_t idesc = idesc_int8(p.BN);
    bool ok = true;
    if (elect_one()) {
      int s = 0;
      uint32_t phase = 0, it = 0;
      for (long t = blockIdx.x; t < p.total && ok; t += gridDim.x, ++it) {
        const uint32_t buf = it & 1u;
        ok = mbar_wait_or_abort(smem_u32(&acc_empty[buf]), ((it >> 1) & 1u) ^ 1u, abortp);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + buf * (uint32_t)p.BN;
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait_or_abort(smem_u32(&full[s]), phase, abortp);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t base = smem_u32(smem + (size_t)s * stage_bytes);
          const uint64_t da = make_desc(base), db = make_desc(base + a_stage);
#pragma unroll
          for (int kk = 0; kk < kDepth / 32; ++kk)     // 32 codes: 32 bytes further inside the swizzle row
            mma_int8(d, da + (uint64_t)(kk * 2), db + (uint64_t)(kk * 2), idesc, (kb | kk) ? 1u : 0u);
          mma_commit(smem_u32(&empty[s]));
          if (++s == p.stages) { s = 0; phase ^= 1u; }
        }
        if (ok) mma_commit(smem_u32(&acc_full[buf]));
      }
      if (!ok) { *abortp = 1; *(volatile int*)p.err = 4; __threadfence_system(); }
    }
    __syncwarp();
  } else if (lane == 0) {
    // TMA producer
    long issued = 0;
    bool ok = true;
    int s = 0;
    uint32_t phase = 0;
    const uint32_t tx = (uint32_t)p.a_bytes + (uint32_t)p.BN * kDepth;
    for (long t = blockIdx.x; t < p.total && ok; t += gridDim.x) {
      const Tile c = tile_of(p, t);
      for (int kb = 0; kb < nkb; ++kb) {
        ok = mbar_wait_or_abort(smem_u32(&empty[s]), phase ^ 1u, abortp);
        if (!ok) break;
        const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(smem + (size_t)s * stage_bytes);
        mbar_arrive_expect_tx(bar, tx);
        load_2d(dst, &map_a, kb * kDepth, (int)c.m0, bar);
        load_2d(dst + a_stage, &map_b, kb * kDepth, (int)c.n0, bar);
        ++issued;
        if (++s == p.stages) { s = 0; phase ^= 1u; }
      }
    }
    if (!ok || *abortp) {
      *abortp = 1;
      *(volatile int*)p.err = 5;
      __threadfence_system();
      // copies already issued still write this CTA's shared memory: wait (bounded) until they have landed
      for (long j = (issued > p.stages ? issued - p.stages : 0); j < issued; ++j)
        mbar_wait(smem_u32(&full[j % p.stages]), (uint32_t)(j / p.stages) & 1u);
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == kEpilogueWarps) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)p.tmem_cols) : "memory");
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encoder() {
  static const EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      return (EncodeTiledFn)ptr;
    cudaGetLastError();
    return (EncodeTiledFn) nullptr;
  }();
  return fn;
}
// rows of K codes, in boxes of 128 codes x `box_rows` rows
bool encode(CUtensorMap* map, const int8_t* base, long rows, long K, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)K};
  const cuuint32_t box[2] = {(cuuint32_t)kDepth, (cuuint32_t)box_rows}, steps[2] = {1, 1};
  return encoder() && encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)base, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int product_tc(const int8_t* a, const float* sa, const int8_t* b, const float* sb, const float* bias, long M, long N, long K, float* y) {
  Params p;
  p.err = tc_error_flag();
  if (!p.err) return 1;
  p.sa = sa; p.sb = sb; p.bias = bias; p.y = y;
  p.M = M; p.N = N; p.K = K;
  p.mtiles = (int)cgtb_ceil_div(M, kRows);
  // the widest tile that still gives every SM one
  p.BN = 256;
  while (p.BN > 32 && p.mtiles * cgtb_ceil_div(N, p.BN) < rt().sm_count) p.BN /= 2;
  p.ntiles = (int)cgtb_ceil_div(N, p.BN);
  p.total = (long)p.mtiles * p.ntiles;
  p.tmem_cols = 2 * p.BN;
  const int a_rows = (int)std::min<long>(kRows, cgtb_ceil_div(M, 8) * 8);
  p.a_bytes = a_rows * kDepth;
  p.vec = N % 4 == 0 && ((uintptr_t)y & 15) == 0;
  const int stage_bytes = (kRows + p.BN) * kDepth, epilogue = kEpilogueWarps * 32 * kPitch * 4;
  p.stages = std::min(kMaxStages, (225 * 1024 - 1024 - epilogue) / stage_bytes);
  const int smem = 1024 + p.stages * stage_bytes + epilogue;
  CUtensorMap map_a, map_b;
  if (!encode(&map_a, a, M, K, a_rows) || !encode(&map_b, b, N, K, p.BN)) return fail("cgtb_int8_product: no tensor map for %ld x %ld x %ld", M, N, K);
  static const cudaError_t attribute = cudaFuncSetAttribute(int8_product_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
  if (attribute != cudaSuccess) return fail("cgtb_int8_product: %s", cudaGetErrorString(attribute));
  CGTB_LAUNCH(int8_product_tc_kernel, (unsigned)std::min<long>(p.total, rt().sm_count), kThreads, smem, map_a, map_b, p);
  CGTB_CHECK_LAUNCH("int8_product");
  return 0;
}

// Few rows: one thread per result
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
  if (M > 0x7fffffffL || N > 0x7fffffffL) return fail("cgtb_int8_product: more than 2^31 - 1 rows or channels");
  if (M == 0 || N == 0) return 0;
  if (M > 8 && K > 0) return product_tc(a, sa, b, sb, bias, M, N, K, y);
  const long blocks = cgtb_ceil_div(M * N, 256);
  CGTB_LAUNCH(int8_product_kernel, (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), 256, 0, a, sa, b, sb, bias, M, N, K, y);
  CGTB_CHECK_LAUNCH("int8_product");
  return 0;
}
