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
constexpr int kMaxStages = 32;
constexpr int kEpilogueWarps = 8;   // two for each quarter of the accumulator's lanes
constexpr int kThreads = (kEpilogueWarps + 3) * 32;   // and a warp for the MMAs, one for the loads of a, one for those of b
constexpr int kGroup = 16;          // row tiles that are walked together: their codes and the weights stay in L2
constexpr int kSlotBytes = kRows * 32 * 4;   // 32 columns of a tile's partial sums, column by column

struct Params {
  const float *sa, *sb, *bias;
  float* y;
  long M, N, K;
  int BN, stages, tmem_cols, a_bytes;
  int mtiles, ntiles, tile_rows;
  long total;
  int vec;
  int split, split_log;             // CTAs of a cluster that share a tile, a power of two
  int block_offset;                 // of the epilogue's blocks in shared memory
  int* err;
};

struct Tile { long m0, n0; };
__device__ __forceinline__ Tile tile_of(const Params& p, long t) {
  // fewer than 2^31 tiles: divisions of 64 bits would take 0.1 us before the first load
  const uint32_t per = (uint32_t)kGroup * (uint32_t)p.ntiles, g = (uint32_t)t / per, first = g * kGroup, left = (uint32_t)p.mtiles - first;
  const uint32_t r = (uint32_t)t - g * per, rows = left < kGroup ? left : kGroup, column = left < kGroup ? r / rows : r / kGroup;
  return Tile{(long)(first + r - column * rows) * p.tile_rows, (long)column * p.BN};
}

// D 32-bit integers, A and B signed 8-bit integers, both K-major
__device__ __forceinline__ uint32_t idesc_int8(int n, int m = kRows) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
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
// The epilogue's wait, bounded and abortable: one lane polls, and sleeps in between.
__device__ __forceinline__ bool wait_sleeping(uint32_t bar, uint32_t parity, const volatile int* abort_flag, int lane) {
  int ok = 1;
  if (lane == 0 && !mbar_try(bar, parity)) {
    const long long t0 = clock64();
    ok = 0;
    for (uint32_t spin = 0; spin < kSpinLimit; ++spin) {
      __nanosleep(64);
      if (mbar_try(bar, parity)) { ok = 1; break; }
      if ((spin & 15u) == 15u && (*abort_flag || clock64() - t0 > kWaitCycles)) break;
    }
  }
  ok = __shfl_sync(0xffffffffu, ok, 0);
  if (ok) (void)mbar_try(bar, parity);   // every lane observes the phase itself
  return ok != 0;
}

// 16 columns of this warp's 32 lanes of TMEM; the registers hold them after tmem_arrived()
__device__ __forceinline__ void tmem_request16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :: "memory");
}

// The epilogue warps go on together or not at all: they meet at a barrier in every tile, where none may be missing.
__device__ __forceinline__ bool epilogue_agrees(bool ok) {
  uint32_t failed;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.eq.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(failed) : "r"((uint32_t)ok), "n"(kEpilogueWarps * 32) : "memory");
  return failed == 0;
}

// Word offset of quad q of row `row` in a warp's 32 x 16 block: 16-byte accesses by rows and by quads without bank conflicts
__device__ __forceinline__ int block_at(int row, int q) { return row * 16 + 4 * (q ^ ((row >> 1) & 3)); }

__device__ __forceinline__ float4 finished(float4 v, float4 s, float4 b, bool bias) {
  if (bias) return make_float4(v.x * s.x + b.x, v.y * s.y + b.y, v.z * s.z + b.z, v.w * s.w + b.w);
  return make_float4(v.x * s.x, v.y * s.y, v.z * s.z, v.w * s.w);
}

// 16 columns of a warp's 32 rows: lane l holds row l's sums. They are scaled by the row, turned through shared memory, scaled by
// the column and stored, eight rows of 64 bytes at a time. `columns`: the scales of the 16 columns, 256 floats on their biases.
__device__ __forceinline__ void store_chunk(const Params& p, const uint32_t (&r)[16], float row_scale, long m0, long n0, float* block, const float* columns,
                                            int lane) {
  const int nrows = (int)(p.M - m0 < 32 ? p.M - m0 : 32);
  __syncwarp();   // the block's previous content has been read
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<float4*>(block + block_at(lane, q)) =
        make_float4((float)(int)r[4 * q] * row_scale, (float)(int)r[4 * q + 1] * row_scale, (float)(int)r[4 * q + 2] * row_scale,
                    (float)(int)r[4 * q + 3] * row_scale);
  const bool bias = p.bias != nullptr;
  __syncwarp();
  if (p.vec) {      // N a multiple of four
    const int q = lane & 3, row0 = lane >> 2;
    if (n0 + 4 * q < p.N) {
      const float4 s = *reinterpret_cast<const float4*>(columns + 4 * q), b = *reinterpret_cast<const float4*>(columns + 256 + 4 * q);
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const float4*>(block + block_at(row0 + 8 * i, q));
      float* dst = p.y + (m0 + row0) * p.N + n0 + 4 * q;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row0 + 8 * i < nrows) *reinterpret_cast<float4*>(dst + 8 * i * p.N) = finished(v[i], s, b, bias);
    }
  } else {
    const int c = lane & 15, row0 = lane >> 4;
    if (n0 + c < p.N) {
      const float s = columns[c], b = columns[256 + c];
      float* dst = p.y + (m0 + row0) * p.N + n0 + c;
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = block[block_at(row0 + 2 * i, c >> 2) + (c & 3)];
#pragma unroll
      for (int i = 0; i < 16; ++i, dst += 2 * p.N)
        if (row0 + 2 * i < nrows) *dst = bias ? v[i] * s + b : v[i] * s;
    }
  }
}

// A warp's share of a tile: its 32 rows, every other chunk of 16 columns. The next chunk is on its way from TMEM meanwhile;
// release() is called when nothing more is read there.
template <typename F>
__device__ __forceinline__ void store_tile_rows(const Params& p, uint32_t taddr, int chunks, int half, float row_scale, long m0, long n0, float* block,
                                                const float* scales, int lane, F release) {
  uint32_t r[16], next[16];
  if (half < chunks) tmem_request16(taddr + (uint32_t)half * 16u, next);
  for (int ch = half; ch < chunks; ch += 2) {
    tmem_arrived(next);
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j] = next[j];
    if (ch + 2 < chunks) tmem_request16(taddr + (uint32_t)(ch + 2) * 16u, next);
    else {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      release();
    }
    store_chunk(p, r, row_scale, m0, n0 + ch * 16, block, scales + ch * 16, lane);
  }
}
// What an epilogue thread brings to a tile: its row's scale, and the scale and bias of one column, which go to shared memory. They
// are asked for a tile ahead.
struct Scales { float row, column, bias; };
__device__ __forceinline__ Scales ask_scales(const Params& p, long row, long n0, int tid) {
  const long n = n0 + tid;
  const bool inside = tid < p.BN && n < p.N;
  return Scales{row < p.M ? p.sa[row] : 0.f, inside ? p.sb[n] : 0.f, inside && p.bias ? p.bias[n] : 0.f};
}
__device__ __forceinline__ const float* stage_columns(const Scales& s, float* columns, uint32_t it, int tid) {   // `it`: two places
  float* to = columns + (it & 1u) * 512;
  to[tid] = s.column;
  to[256 + tid] = s.bias;
  asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueWarps * 32) : "memory");
  return to;
}

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote_address(uint32_t local, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
  return at;
}
__device__ __forceinline__ void store_remote(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }

// One CTA per SM walks tiles of 128 x BN results. One thread issues the TMA loads of a, one those of b, into a ring of stages (128
// codes of K: 128 bytes of every row), one thread the MMAs (four of K = 32 per stage) into one of two accumulators in TMEM, eight
// warps turn the other accumulator into results meanwhile. Rows and codes beyond the operands arrive as zeros. With fewer than
// 128 rows the box of a is as short as they are, and the MMAs read on into what lies behind it (at the ring's end the epilogue's
// blocks, 16 KB like a full box): whole numbers that only reach rows which are not stored.
//
// SPLIT: fewer tiles than SMs. The CTAs of a cluster share a tile, each sums over a slice of K; then every CTA sends its partial
// sums to the CTA that finishes their columns (chunk c of 16 columns: CTA c % split), through distributed shared memory, and adds
// what it receives (whole numbers: in any order). An MMA takes a hundred cycles however narrow the tile, so a tile stays wide
// and K is split.
template <bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
int8_product_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  __shared__ __align__(16) float columns[2 * 512];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t a_stage = (uint32_t)p.a_bytes, stage_bytes = a_stage + (uint32_t)p.BN * kDepth;
  volatile int* abortp = &abort_flag;
  const uint32_t rank = SPLIT ? cluster_rank() : 0u;
  const long t_first = SPLIT ? blockIdx.x >> p.split_log : blockIdx.x, t_step = SPLIT ? p.total : gridDim.x;   // SPLIT: one tile
  const int nkb_all = (int)((p.K + kDepth - 1) / kDepth), kb_first = SPLIT ? ((int)rank * nkb_all) >> p.split_log : 0;
  const int nkb = (SPLIT ? (((int)rank + 1) * nkb_all) >> p.split_log : nkb_all) - kb_first;

  if (tid < p.stages) {
    mbar_init(smem_u32(&full[tid]), 2);
    mbar_init(smem_u32(&empty[tid]), 1);
  }
  if (tid == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), kEpilogueWarps);
    }
    abort_flag = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_a)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_b)) : "memory");
  }
  if (warp == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");   // all barriers are this warp's
  if (warp == kEpilogueWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((uint32_t)p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  const int quarter = warp & 3, half = warp >> 2;
  float* block = reinterpret_cast<float*>(smem + p.block_offset) + warp * 512;
  const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
  bool ok = true;
  float row_scale = 0.f;            // SPLIT: kept for the end

  if (warp < kEpilogueWarps) {
    uint32_t it = 0;
    Tile c = tile_of(p, t_first);
    Scales ahead = ask_scales(p, c.m0 + quarter * 32 + lane, c.n0, tid);
    for (long t = t_first; t < p.total; t += t_step, ++it) {
      const uint32_t buf = it & 1u;
      const long m0 = c.m0 + quarter * 32, n0 = c.n0;
      row_scale = ahead.row;
      const float* scales = stage_columns(ahead, columns, it, tid);
      if (!SPLIT && t + t_step < p.total) {
        c = tile_of(p, t + t_step);
        ahead = ask_scales(p, c.m0 + quarter * 32 + lane, c.n0, tid);
      }
      ok = wait_sleeping(smem_u32(&acc_full[buf]), (it >> 1) & 1u, abortp, lane);
      if (!ok) {
        *abortp = 1;
        if (lane == 0) { *(volatile int*)p.err = 3; __threadfence_system(); }
      }
      if (SPLIT) break;
      ok = epilogue_agrees(ok);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      auto release = [&] { if (lane == 0) mbar_arrive(smem_u32(&acc_empty[buf])); };
      if (m0 < p.M) store_tile_rows(p, lanes + buf * (uint32_t)p.BN, p.BN / 16, half, row_scale, m0, n0, block, scales, lane, release);
      else release();
    }
  } else if (warp == kEpilogueWarps) {
    // MMA issuer
    const uint32_t idesc = idesc_int8(p.BN), base = smem_u32(smem), full0 = smem_u32(full), empty0 = smem_u32(empty);
    const uint64_t da0 = make_desc(base), db0 = make_desc(base + a_stage);
    const uint32_t step = stage_bytes >> 4;
    if (elect_one()) {
      uint32_t s = 0, phase = 0, it = 0;
      for (long t = t_first; t < p.total && ok; t += t_step, ++it) {
        const uint32_t buf = it & 1u;
        ok = mbar_wait_or_abort(smem_u32(&acc_empty[buf]), ((it >> 1) & 1u) ^ 1u, abortp);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + buf * (uint32_t)p.BN;
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait_or_abort(full0 + 8u * s, phase, abortp);   // what TMA wrote needs no further fence
          if (!ok) break;
          const uint64_t da = da0 + s * step, db = db0 + s * step;
          mma_int8(d, da, db, idesc, kb > 0);                  // 32 codes: 32 bytes further inside the swizzle row
          mma_int8(d, da + 2, db + 2, idesc, 1u);
          mma_int8(d, da + 4, db + 4, idesc, 1u);
          mma_int8(d, da + 6, db + 6, idesc, 1u);
          mma_commit(empty0 + 8u * s);
          if (++s == (uint32_t)p.stages) { s = 0; phase ^= 1u; }
        }
        if (ok) mma_commit(smem_u32(&acc_full[buf]));
      }
      if (!ok) { *abortp = 1; *(volatile int*)p.err = 4; __threadfence_system(); }
    }
    __syncwarp();
  } else {
    if (elect_one()) {
      // TMA producers: one thread for the boxes of a, one for those of b
      const bool is_b = warp == kEpilogueWarps + 2;
      const CUtensorMap* map = is_b ? &map_b : &map_a;
      const uint32_t tx = is_b ? (uint32_t)p.BN * kDepth : a_stage, dst0 = smem_u32(smem) + (is_b ? a_stage : 0u);
      const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty);
      uint32_t issued = 0, s = 0, phase = 1;
      for (long t = t_first; t < p.total && ok; t += t_step) {
        const Tile c = tile_of(p, t);
        const int row = (int)(is_b ? c.n0 : c.m0);
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait_or_abort(empty0 + 8u * s, phase, abortp);
          if (!ok) break;
          mbar_arrive_expect_tx(full0 + 8u * s, tx);
          load_2d(dst0 + s * stage_bytes, map, (kb_first + kb) * kDepth, row, full0 + 8u * s);
          ++issued;
          if (++s == (uint32_t)p.stages) { s = 0; phase ^= 1u; }
        }
      }
      if (!ok || *abortp) {
        *abortp = 1;
        *(volatile int*)p.err = 5;
        __threadfence_system();
        // copies already issued still write this CTA's shared memory: wait (bounded) until they have landed
        const uint32_t stages = (uint32_t)p.stages;
        for (uint32_t j = (issued > stages ? issued - stages : 0u); j != issued; ++j) mbar_wait(full0 + 8u * (j % stages), (j / stages) & 1u);
      }
    }
    __syncwarp();
  }

  if (SPLIT) {
    // Every CTA passes both barriers, whatever happened to its waits. Behind the first one all MMAs of the cluster have run and
    // the rings are free: they take the partial sums, one slot of 128 rows for each (sender, chunk of 32 columns).
    cluster_sync();
    const Tile c = tile_of(p, t_first);
    const long m0 = c.m0 + quarter * 32;
    const bool takes_part = warp < kEpilogueWarps && ok && m0 < p.M;
    const int chunks = p.BN / 32, mine = (chunks + p.split - 1) >> p.split_log, row = quarter * 32 + lane;
    const uint32_t half_columns = (uint32_t)half * 16u;       // a warp takes 16 of a chunk's 32 columns
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (takes_part) {
      const uint32_t slots = smem_u32(smem) + half_columns * (kRows * 4) + (uint32_t)row * 4u;
      for (int ch = 0; ch < chunks; ++ch) {
        const uint32_t owner = (uint32_t)(ch & (p.split - 1));
        if (owner == rank) continue;
        uint32_t r[16];
        tmem_ld16(lanes + (uint32_t)ch * 32u + half_columns, r);
        const uint32_t sender = rank < owner ? rank : rank - 1u;
        const uint32_t at = remote_address(slots + (sender * (uint32_t)mine + (uint32_t)(ch >> p.split_log)) * kSlotBytes, owner);
#pragma unroll
        for (int j = 0; j < 16; ++j) store_remote(at + (uint32_t)(j * kRows * 4), r[j]);   // a warp stores 128 bytes of a column
      }
    }
    cluster_sync();
    if (takes_part) {
      for (int i = 0; i < mine; ++i) {
        const int ch = (i << p.split_log) + (int)rank;
        if (ch >= chunks) break;
        uint32_t r[16];
        tmem_ld16(lanes + (uint32_t)ch * 32u + half_columns, r);
        for (int sender = 0; sender + 1 < p.split; ++sender) {
          const uint32_t* from = reinterpret_cast<const uint32_t*>(smem + (size_t)(sender * mine + i) * kSlotBytes) + half_columns * kRows + row;
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] += from[j * kRows];
        }
        const int col = ch * 32 + (int)half_columns;
        store_chunk(p, r, row_scale, m0, c.n0 + col, block, columns + col, lane);
      }
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == kEpilogueWarps) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)p.tmem_cols) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------
// Large products: two CTAs of a cluster, on two SMs, share tiles of 256 x 256 results (tcgen05 cta_group::2). Each loads its 128
// rows of a and 128 of the 256 rows of b, and holds its 128 rows of sums in its TMEM; the even CTA's MMA thread issues for both,
// and every tensor core reads both halves of b. A stage is 32 KB in either SM instead of 48 KB: the L2 cache, whose bandwidth
// bounds the kernel above (a stage took 630 cycles, its MMAs 512), delivers a third less, and six stages fit instead of four.
// 8192 x 4096 x 4096: 96 us in a row of calls (2.85 PFLOP/s; alone 89 us, the tensor pipe 85 % active at the 1.6 GHz that the
// power cap leaves), 110 us by the kernel above.
//
// Barriers: `full` is the even CTA's, told by the loads of both; `empty` and `acc_full` are each CTA's own, told by the MMAs'
// commits, which go to both; `acc_empty` is the even CTA's, told by the epilogue warps of both.
// ------------------------------------------------------------------------------------------------
constexpr int kPairRows = 256;

__device__ __forceinline__ void mma_int8_pair(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrives at the barriers at this place in both CTAs when the MMAs issued so far have run
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// into this CTA's memory; the bytes are counted at the barrier of the pair's even CTA (`bar`: an address of the cluster window)
__device__ __forceinline__ void load_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool try_cluster(uint32_t bar, uint32_t parity) {   // sees what the other CTA released
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}

__global__ void __launch_bounds__(kThreads, 1)
int8_product_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  __shared__ __align__(16) float columns[2 * 512];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  constexpr uint32_t kHalf = 128 * kDepth, kStage = 2 * kHalf;
  volatile int* abortp = &abort_flag;
  const uint32_t rank = cluster_rank();
  const long t_first = blockIdx.x >> 1, t_step = gridDim.x >> 1;
  const int nkb = (int)((p.K + kDepth - 1) / kDepth);

  if (tid < p.stages) {
    mbar_init(smem_u32(&full[tid]), 2);            // the even CTA's two loading threads, which announce the other's bytes too
    mbar_init(smem_u32(&empty[tid]), 1);
  }
  if (tid == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), 2 * kEpilogueWarps);
    }
    abort_flag = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_a)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_b)) : "memory");
  }
  if (warp == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  if (warp == kEpilogueWarps) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  bool ok = true;

  if (warp < kEpilogueWarps) {
    const int quarter = warp & 3, half = warp >> 2;
    float* block = reinterpret_cast<float*>(smem + p.block_offset) + warp * 512;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    uint32_t it = 0;
    const long own = (long)rank * 128 + quarter * 32;     // of a tile's rows
    Tile c = tile_of(p, t_first);
    Scales ahead = ask_scales(p, c.m0 + own + lane, c.n0, tid);
    for (long t = t_first; t < p.total; t += t_step, ++it) {
      const uint32_t buf = it & 1u;
      const long m0 = c.m0 + own, n0 = c.n0;
      const float row_scale = ahead.row;
      const float* scales = stage_columns(ahead, columns, it, tid);
      if (t + t_step < p.total) {
        c = tile_of(p, t + t_step);
        ahead = ask_scales(p, c.m0 + own + lane, c.n0, tid);
      }
      ok = wait_sleeping(smem_u32(&acc_full[buf]), (it >> 1) & 1u, abortp, lane);
      if (!ok) {
        *abortp = 1;
        if (lane == 0) { *(volatile int*)p.err = 3; __threadfence_system(); }
      }
      ok = epilogue_agrees(ok);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // relaxed: nothing in memory is handed over, and a release at cluster scope would wait for every store of results
      auto release = [&] {
        if (lane == 0)
          asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_address(smem_u32(&acc_empty[buf]), 0u)) : "memory");
      };
      if (m0 < p.M) store_tile_rows(p, lanes + buf * 256u, 16, half, row_scale, m0, n0, block, scales, lane, release);
      else release();
    }
  } else if (warp == kEpilogueWarps) {
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = idesc_int8(256, kPairRows), base = smem_u32(smem), full0 = smem_u32(full), empty0 = smem_u32(empty);
      const uint64_t da0 = make_desc(base), db0 = make_desc(base + kHalf);
      uint32_t s = 0, phase = 0, it = 0;
      for (long t = t_first; t < p.total && ok; t += t_step, ++it) {
        const uint32_t buf = it & 1u, bar = smem_u32(&acc_empty[buf]), parity = ((it >> 1) & 1u) ^ 1u;
        ok = mbar_wait_or_abort(bar, parity, abortp) && try_cluster(bar, parity);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + buf * 256u;
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait_or_abort(full0 + 8u * s, phase, abortp);
          if (!ok) break;
          const uint64_t da = da0 + s * (kStage >> 4), db = db0 + s * (kStage >> 4);
          mma_int8_pair(d, da, db, idesc, kb > 0);
          mma_int8_pair(d, da + 2, db + 2, idesc, 1u);
          mma_int8_pair(d, da + 4, db + 4, idesc, 1u);
          mma_int8_pair(d, da + 6, db + 6, idesc, 1u);
          mma_commit_pair(empty0 + 8u * s);
          if (++s == (uint32_t)p.stages) { s = 0; phase ^= 1u; }
        }
        if (ok) mma_commit_pair(smem_u32(&acc_full[buf]));
      }
      if (!ok) { *abortp = 1; *(volatile int*)p.err = 4; __threadfence_system(); }
    }
    __syncwarp();
  } else {
    if (elect_one()) {
      const bool is_b = warp == kEpilogueWarps + 2;
      const CUtensorMap* map = is_b ? &map_b : &map_a;
      const uint32_t dst0 = smem_u32(smem) + (is_b ? kHalf : 0u), empty0 = smem_u32(empty), full0 = remote_address(smem_u32(full), 0u);
      uint32_t issued = 0, s = 0, phase = 1;
      for (long t = t_first; t < p.total && ok; t += t_step) {
        const Tile c = tile_of(p, t);
        const int row = (int)((is_b ? c.n0 : c.m0) + (long)rank * 128);
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait_or_abort(empty0 + 8u * s, phase, abortp);
          if (!ok) break;
          if (rank == 0) mbar_arrive_expect_tx(smem_u32(full) + 8u * s, 2 * kHalf);
          load_2d_pair(dst0 + s * kStage, map, kb * kDepth, row, full0 + 8u * s);
          ++issued;
          if (++s == (uint32_t)p.stages) { s = 0; phase ^= 1u; }
        }
      }
      // Copies still write this CTA's memory until the MMAs have read them; before the CTA leaves, every stage issued has to be
      // empty again (bounded; when a wait has expired somewhere, this one does too).
      const uint32_t stages = (uint32_t)p.stages;
      for (uint32_t j = (issued > stages ? issued - stages : 0u); j != issued && ok; ++j) ok = mbar_wait_or_abort(empty0 + 8u * (j % stages), (j / stages) & 1u, abortp);
      if (!ok || *abortp) {
        *abortp = 1;
        *(volatile int*)p.err = 5;
        __threadfence_system();
        const long long t0 = clock64();      // whatever is in flight lands meanwhile
        while (clock64() - t0 < 2000000) __nanosleep(1000);
      }
    }
    __syncwarp();
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();        // neither CTA leaves while the other reads its memory or tells its barriers
  if (warp == kEpilogueWarps) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
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
  // Widths and splits, by what they cost in cycles (measured): a stage takes 400 or, wide, two for each column; tiles follow each
  // other on an SM; a cluster's two barriers and its last step take 3000, what a CTA sends goes at 12 bytes a cycle. At
  // 128 x 4096 x 4096 a width of 32 takes 14.5 us, 128 in clusters of four 11 us.
  const int nkb = (int)cgtb_ceil_div(K, kDepth), sms = rt().sm_count;
  long best = -1;
  for (int bn = 256; bn >= 32; bn /= 2) {
    if (bn > 32 && bn / 2 >= N) continue;
    const long tiles = p.mtiles * cgtb_ceil_div(N, bn), rows = std::min<long>(M, kRows);
    for (int log = 0; log <= 2 && (1 << log) <= nkb; ++log) {      // clusters of eight leave a fifth of the SMs without work
      const int split = 1 << log;
      if (split > 1 && tiles * split > sms) break;
      const long waves = cgtb_ceil_div(tiles * split, sms), blocks = cgtb_ceil_div(nkb, split);
      const long cost = waves * (blocks * std::max(400, 2 * bn) + 500) + (split > 1 ? 3000 + rows * bn * 4 * (split - 1) / split / 12 : 0);
      if (best < 0 || cost < best) { best = cost; p.BN = bn; p.split = split; p.split_log = log; }
    }
  }
  // Pairs of CTAs, where their larger tiles leave none without work
  const bool pairs = p.split == 1 && p.BN == 256 && M > kRows && cgtb_ceil_div(M, kPairRows) * cgtb_ceil_div(N, 256) >= sms / 2;
  p.tile_rows = pairs ? kPairRows : kRows;
  p.mtiles = (int)cgtb_ceil_div(M, p.tile_rows);
  p.ntiles = (int)cgtb_ceil_div(N, p.BN);
  p.total = (long)p.mtiles * p.ntiles;
  if (p.total > 0x7fffffffL) return fail("cgtb_int8_product: %ld x %ld results are too many", M, N);
  p.tmem_cols = (p.split > 1 ? 1 : 2) * p.BN;
  const int a_rows = (int)std::min<long>(kRows, cgtb_ceil_div(M, 8) * 8);
  p.a_bytes = a_rows * kDepth;
  p.vec = N % 4 == 0 && ((uintptr_t)y & 15) == 0;
  const int box_b = pairs ? 128 : p.BN, stage_bytes = p.a_bytes + box_b * kDepth, epilogue = kEpilogueWarps * 512 * 4;
  p.stages = std::min(kMaxStages, (220 * 1024 - 1024 - epilogue) / stage_bytes);
  if (p.split > 1) p.stages = std::min(p.stages, (int)cgtb_ceil_div(nkb, p.split));
  const int slots = (p.split - 1) * (int)cgtb_ceil_div(p.BN / 32, p.split) * kSlotBytes;
  p.block_offset = std::max(p.stages * stage_bytes, slots);
  const int smem = 1024 + p.block_offset + epilogue;
  CUtensorMap map_a, map_b;
  if (!encode(&map_a, a, M, K, a_rows) || !encode(&map_b, b, N, K, box_b)) return fail("cgtb_int8_product: no tensor map for %ld x %ld x %ld", M, N, K);
  static const cudaError_t attribute = [] {
    const cudaError_t e = cudaFuncSetAttribute(int8_product_tc_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
    if (e != cudaSuccess) return e;
    const cudaError_t f = cudaFuncSetAttribute(int8_product_tc_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
    return f != cudaSuccess ? f : cudaFuncSetAttribute(int8_product_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
  }();
  if (attribute != cudaSuccess) return fail("cgtb_int8_product: %s", cudaGetErrorString(attribute));
  if (p.split > 1 || pairs) {
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = pairs ? 2u : (unsigned)p.split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(pairs ? 2 * std::min<long>(p.total, sms / 2) : p.total * p.split));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = (size_t)smem;
    config.stream = rt().stream;
    config.attrs = &attr;
    config.numAttrs = 1;
    CGTB_CUDA_TRY(cudaLaunchKernelEx(&config, pairs ? int8_product_pair_kernel : int8_product_tc_kernel<true>, map_a, map_b, p));
    g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  } else {
    CGTB_LAUNCH(int8_product_tc_kernel<false>, (unsigned)std::min<long>(p.total, sms), kThreads, smem, map_a, map_b, p);
  }
  CGTB_CHECK_LAUNCH("int8_product");
  return 0;
}

// ------------------------------------------------------------------------------------------------
// Small products and few rows, where the kernels above spend most of their time on beginning (5 to 8 us whatever they do). A
// block makes 16 CT output channels x 8 NT TW rows; its eight warps, TW of them beside each other, take turns with 64 codes of K,
// UNROLL such steps in flight, and join their sums in shared memory at the end. The weights are the matrix instructions' A operand (16 channels), the rows their
// B operand (8 rows): with few rows nothing is multiplied in vain. No shared memory in the loop: which codes of K an instruction
// sees in which of its places is free as long as both operands agree, so a thread loads 16 consecutive codes of a row and gives
// them to two instructions as they are, and rows that start on any 16 bytes cost little (the TMA loads above take a quarter longer
// where K is an odd multiple of 16). Bound by latency, then by what the blocks read again from L2: 128 x 256 x 784 2.4 us,
// 500 x 1001 x 1008 6.5 us (tcgen05 8.7), 8 x 4096 x 4096 8 us (2.1 TB/s).
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int CT, int NT, int TW>
struct Small {
  static constexpr int kChannels = 16 * CT, kTokens = 8 * NT * TW, kSlices = 8 / TW;
  static constexpr int kPitch = kChannels + 4;   // the stores of a warp, 8 channels of 4 tokens two apart, reach all banks
  static constexpr int kBytes = kSlices * kTokens * kPitch * 4;
};
template <int CT, int NT, int TW, int UNROLL>
__global__ void __launch_bounds__(256) int8_product_small_kernel(const int8_t* __restrict__ a, const float* __restrict__ sa, const int8_t* __restrict__ b,
                                                                 const float* __restrict__ sb, const float* __restrict__ bias, long M, long N, long K,
                                                                 float* __restrict__ y) {
  using S = Small<CT, NT, TW>;
  extern __shared__ int joined[];         // [slice][token][channel]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, slice = warp / TW, token0 = warp % TW * (8 * NT);
  const long n0 = (long)blockIdx.x * S::kChannels, m0 = (long)blockIdx.y * S::kTokens;
  // rows beyond the operands are read as the last one: their results are not stored
  const int8_t *w[2 * CT], *x[NT];
#pragma unroll
  for (int i = 0; i < 2 * CT; ++i) w[i] = b + (n0 + g + 8 * i < N ? n0 + g + 8 * i : N - 1) * K + t * 16;
#pragma unroll
  for (int j = 0; j < NT; ++j) x[j] = a + (m0 + token0 + g + 8 * j < M ? m0 + token0 + g + 8 * j : M - 1) * K + t * 16;
  int c[CT][NT][4];
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) c[i][j][k] = 0;
  const long last = K - t * 16;      // this thread's codes of a step are there for k < last
  constexpr int kStep = S::kSlices * 64;
  for (long k = slice * 64; k < K; k += kStep * UNROLL) {
    uint4 wv[UNROLL][2 * CT], xv[UNROLL][NT];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const bool there = k + u * kStep < last;
#pragma unroll
      for (int i = 0; i < 2 * CT; ++i) wv[u][i] = there ? __ldg(reinterpret_cast<const uint4*>(w[i] + k + u * kStep)) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int j = 0; j < NT; ++j) xv[u][j] = there ? __ldg(reinterpret_cast<const uint4*>(x[j] + k + u * kStep)) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_16832(c[i][j], wv[u][2 * i].x, wv[u][2 * i + 1].x, wv[u][2 * i].y, wv[u][2 * i + 1].y, xv[u][j].x, xv[u][j].y);
          mma_16832(c[i][j], wv[u][2 * i].z, wv[u][2 * i + 1].z, wv[u][2 * i].w, wv[u][2 * i + 1].w, xv[u][j].z, xv[u][j].w);
        }
  }
  int* own = joined + (slice * S::kTokens + token0) * S::kPitch;
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) own[(8 * j + 2 * t + (k & 1)) * S::kPitch + 16 * i + 8 * (k >> 1) + g] = c[i][j][k];
  __syncthreads();
  const int channel = threadIdx.x % S::kChannels;
  const long n = n0 + channel;
  if (n < N) {
    const float s = sb[n], shift = bias ? bias[n] : 0.f;
    constexpr int kRowsAtOnce = 256 / S::kChannels;
#pragma unroll
    for (int i = 0; i < (S::kTokens + kRowsAtOnce - 1) / kRowsAtOnce; ++i) {
      const int token = threadIdx.x / S::kChannels + i * kRowsAtOnce;
      if (token >= S::kTokens || m0 + token >= M) break;
      int sum = 0;
#pragma unroll
      for (int v = 0; v < S::kSlices; ++v) sum += joined[(v * S::kTokens + token) * S::kPitch + channel];
      const float r = (float)sum * sa[m0 + token] * s;
      y[(m0 + token) * N + n] = bias ? r + shift : r;
    }
  }
}

template <int CT, int NT, int TW, int UNROLL>
int product_small(const int8_t* a, const float* sa, const int8_t* b, const float* sb, const float* bias, long M, long N, long K, float* y) {
  using S = Small<CT, NT, TW>;
  constexpr auto kernel = int8_product_small_kernel<CT, NT, TW, UNROLL>;
  static_assert(S::kBytes <= 48 * 1024);
  const dim3 grid((unsigned)cgtb_ceil_div(N, S::kChannels), (unsigned)cgtb_ceil_div(M, S::kTokens));
  CGTB_LAUNCH(kernel, grid, 256, S::kBytes, a, sa, b, sb, bias, M, N, K, y);
  CGTB_CHECK_LAUNCH("int8_product");
  return 0;
}

// One row, a token at a time, or two: bound by the bytes of the weights. WARPS warps share an output channel, each lane takes 16
// codes of the channel's row at a time, four such loads in flight, and multiplies them with the codes of ROWS rows, which come
// from the L1 cache; whole numbers are added by redux, in any order. 1 x 8192 x 8192: 14.2 us, 4.7 TB/s. Eight blocks on an SM leave
// a thread 32 registers; 12 to 68 bytes are spilled.
template <int ROWS, int WARPS>
__global__ void __launch_bounds__(256, 8) int8_product_rows_kernel(const int8_t* __restrict__ a, const float* __restrict__ sa, const int8_t* __restrict__ b,
                                                                const float* __restrict__ sb, const float* __restrict__ bias, long N, long K,
                                                                float* __restrict__ y) {
  __shared__ int part[8][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slice = warp % WARPS;
  const long n = (long)blockIdx.x * (8 / WARPS) + warp / WARPS;
  int sums[ROWS];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) sums[m] = 0;
  if (n < N) {
    const int8_t* w = b + n * K;
    long k = (slice * 32 + lane) * 16;
    constexpr long kStep = WARPS * 32 * 16;
    for (; k + 3 * kStep < K; k += 4 * kStep) {
      int4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = __ldg(reinterpret_cast<const int4*>(w + k + u * kStep));
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int m = 0; m < ROWS; ++m) {
          const int4 x = __ldg(reinterpret_cast<const int4*>(a + m * K + k + u * kStep));
          sums[m] = __dp4a(v[u].x, x.x, __dp4a(v[u].y, x.y, __dp4a(v[u].z, x.z, __dp4a(v[u].w, x.w, sums[m]))));
        }
    }
    for (; k < K; k += kStep) {
      const int4 v = __ldg(reinterpret_cast<const int4*>(w + k));
#pragma unroll
      for (int m = 0; m < ROWS; ++m) {
        const int4 x = __ldg(reinterpret_cast<const int4*>(a + m * K + k));
        sums[m] = __dp4a(v.x, x.x, __dp4a(v.y, x.y, __dp4a(v.z, x.z, __dp4a(v.w, x.w, sums[m]))));
      }
    }
  }
#pragma unroll
  for (int m = 0; m < ROWS; ++m) sums[m] = __reduce_add_sync(0xffffffffu, sums[m]);
  if (WARPS > 1) {
    if (lane == 0)
#pragma unroll
      for (int m = 0; m < ROWS; ++m) part[warp][m] = sums[m];
    __syncthreads();
    if (slice != 0) return;
#pragma unroll
    for (int m = 0; m < ROWS; ++m)
#pragma unroll
      for (int i = 1; i < WARPS; ++i) sums[m] += part[warp + i][m];
  }
  if (n >= N) return;
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
    if (lane == m) {
      const float v = (float)sums[m] * sa[m] * sb[n];
      y[m * N + n] = bias ? v + bias[n] : v;
    }
}

template <int ROWS>
int product_rows(const int8_t* a, const float* sa, const int8_t* b, const float* sb, const float* bias, long N, long K, float* y) {
  // as many warps for a channel as there are slices of 512 codes in its row, while the SMs are not full of warps
  const long full = (long)rt().sm_count * 32;
  const int warps = K > 2048 && N * 4 <= full ? 8 : K > 512 && N <= full ? 2 : 1;
  const unsigned grid = (unsigned)cgtb_ceil_div(N, 8 / warps);
  if (warps == 8) CGTB_LAUNCH((int8_product_rows_kernel<ROWS, 8>), grid, 256, 0, a, sa, b, sb, bias, N, K, y);
  else if (warps == 2) CGTB_LAUNCH((int8_product_rows_kernel<ROWS, 2>), grid, 256, 0, a, sa, b, sb, bias, N, K, y);
  else CGTB_LAUNCH((int8_product_rows_kernel<ROWS, 1>), grid, 256, 0, a, sa, b, sb, bias, N, K, y);
  CGTB_CHECK_LAUNCH("int8_product");
  return 0;
}

// No terms: y = bias
__global__ void __launch_bounds__(256) int8_product_empty_kernel(const float* __restrict__ sa, const float* __restrict__ sb, const float* __restrict__ bias,
                                                                 long M, long N, float* __restrict__ y) {
  for (long o = blockIdx.x * 256L + threadIdx.x; o < M * N; o += gridDim.x * 256L) {
    const float v = 0.f * sa[o / N] * sb[o % N];
    y[o] = bias ? v + bias[o % N] : v;
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
  if (K == 0) {
    const long blocks = cgtb_ceil_div(M * N, 256);
    CGTB_LAUNCH(int8_product_empty_kernel, (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), 256, 0, sa, sb, bias, M, N, y);
    CGTB_CHECK_LAUNCH("int8_product");
    return 0;
  }
  if (M == 1) return product_rows<1>(a, sa, b, sb, bias, N, K, y);
  if (M == 2) return product_rows<2>(a, sa, b, sb, bias, N, K, y);
  // Measured, in us, for blocks of 16 channels x 8 rows, 16 x 16, 32 x 32, 32 x 64, and tcgen05:
  //   8 x 4096 x 4096     7.9   8.3   9.5  14.8   8.8        128 x 4096 x 1008    -     -   7.8   6.5   8.4
  //   32 x 4096 x 64      3.1   2.5   2.9   2.9   5.0        500 x 1001 x 1008  12.0   9.5  7.6   6.5   8.7
  //   128 x 1024 x 1008   4.8   3.8   3.6   4.8   8.3        500 x 1001 x 2048    -     -   9.2   8.4   8.4
  //   128 x 512 x 1008    3.2   2.8   3.6   4.8   8.3        512 x 2048 x 784     -     -  12.5  10.8   8.0
  //   256 x 1024 x 1008   7.3   5.6   4.6   4.9   8.4        1000 x 1001 x 272    -     -   9.8   7.9   6.9
  //   8192 x 8 x 1008     4.4   3.5   4.4   4.9    -         32 x 4096 x 4096   13.0   9.2  10.5  15.9   9.1
  // The smaller a block, the fewer turns of its threads follow each other, and the more often the operands are read.
  if (M <= 16 || ((double)M * N * K <= 6e8 && M <= 1L << 18 && M * N <= 1L << 19 && N * K <= 1L << 23)) {
    const long sms = rt().sm_count, small = cgtb_ceil_div(M, 16) * cgtb_ceil_div(N, 16), middle = cgtb_ceil_div(M, 32) * cgtb_ceil_div(N, 32);
    if (M <= 8) return product_small<1, 1, 1, 2>(a, sa, b, sb, bias, M, N, K, y);
    if (M <= 16 || 2 * small <= 7 * sms) return product_small<1, 2, 1, 2>(a, sa, b, sb, bias, M, N, K, y);
    if (middle <= 2 * sms) return product_small<2, 4, 1, 2>(a, sa, b, sb, bias, M, N, K, y);
    return product_small<2, 4, 2, 2>(a, sa, b, sb, bias, M, N, K, y);
  }
  return product_tc(a, sa, b, sb, bias, M, N, K, y);
}
