// Layer norm with its gradients, dropout from a counter-based generator, and rows in 8-bit integers with a scale each, for
// sm_100a.
#include "runtime.h"
#include "tc_util.h"
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <type_traits>

using namespace cgtb;

namespace {

// ================================================================================================
// Teams. A team of TEAM threads holds one row in its registers, E = N * VEC elements in each thread: element
// (i * TEAM + thread) * VEC + v, so that a team reads and writes consecutive addresses, 16 bytes a thread where rows start on
// 16-byte boundaries (VEC * sizeof(T) = 16) and element by element otherwise. TEAM is the smallest power of two that covers the
// row: part of a warp (sums by shuffles; several rows per warp), or several warps (shuffles, then shared memory).
// ================================================================================================
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

template <typename T, int VEC, int N, int TEAM>
struct Row {
  static constexpr int E = VEC * N;
  T v[E];
  // elements beyond C are `fill`
  __device__ __forceinline__ void load(const T* row, int C, int t, T fill) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TEAM + t) * VEC;
      if (c < C) {
        const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC>*>(row + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i * VEC + j] = p.v[j];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i * VEC + j] = fill;
      }
    }
  }
  __device__ __forceinline__ void store(T* row, int C, int t) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TEAM + t) * VEC;
      if (c < C) {
        Pack<T, VEC> p;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.v[j] = v[i * VEC + j];
        *reinterpret_cast<Pack<T, VEC>*>(row + c) = p;
      }
    }
  }
};

constexpr int kTeamThreads = 256;   // of a block, unless a team is larger
template <int TEAM> constexpr int team_block() { return TEAM > kTeamThreads ? TEAM : kTeamThreads; }

// Waits for other blocks or for copies are bounded: after `cycles` a thread raises the error flag, the block's `note` of it and kGaveUp
// among its own flags. A thread that has given up, or waits and finds the note, waits no more; thread 0 then asks for no copies, and
// the threads that tell the other blocks something tell them nothing. The block runs through its rows, whose results are
// invalid: it waits in vain once, however many rows there are.
struct Waits {
  int* err;
  uint32_t cycles;
  uint32_t flags;      // of every thread at first; kSilent: nothing is asked for or told, so that every wait is in vain (a self-test)
};
constexpr uint32_t kGaveUp = 1u << 31, kSilent = 1u << 30;
__device__ __forceinline__ bool wait_until(uint32_t bar, uint32_t parity, const Waits& waits, volatile int* note, uint32_t& flags) {
  if (flags & kGaveUp) return false;
  if (tc::mbar_try(bar, parity)) return true;
  const uint32_t t0 = (uint32_t)clock();
  while (!*note && (uint32_t)clock() - t0 < waits.cycles)
    if (tc::mbar_try(bar, parity)) return true;
  flags |= kGaveUp;
  *note = 1;
  *(volatile int*)waits.err = 9;
  __threadfence_system();
  return false;
}

// Sums of one or two values over a team, in a fixed order; every thread gets them. `part`: the block's space for teams of several
// warps, 2 * K * (warps of the block) values; consecutive calls alternate `turn`, so that one barrier separates a call's reads
// from the next but one's writes. Two values cost little more than one: after the first step half of the lanes go on with
// either of them.
template <int TEAM, int K, typename T>
__device__ __forceinline__ void team_sums(T (&s)[K], T* part, int turn) {
  constexpr int kLanes = TEAM < 32 ? TEAM : 32, kWarps = TEAM / 32, kAll = team_block<TEAM>() / 32;
  const int lane = threadIdx.x & 31;
  T v = s[0];
  if constexpr (K == 2 && kLanes > 1) {
    const bool upper = lane & (kLanes / 2);
    v = (upper ? s[1] : s[0]) + __shfl_xor_sync(0xffffffffu, upper ? s[0] : s[1], kLanes / 2);
  }
#pragma unroll
  for (int o = kLanes / (2 * K); o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TEAM <= 32) {
    if constexpr (K == 1) s[0] = v;
    else if constexpr (kLanes > 1) {
      const T other = __shfl_xor_sync(0xffffffffu, v, kLanes / 2);
      const bool upper = lane & (kLanes / 2);
      s[0] = upper ? other : v;
      s[1] = upper ? v : other;
    }
  } else {
    const int warp = threadIdx.x >> 5, first = warp / kWarps * kWarps;
    T* at = part + turn * kAll * K;           // [K][warp]
    if ((lane & 15) == 0 && (K == 2 || lane == 0)) at[(lane >> 4) * kAll + warp] = v;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      T t;
      if constexpr (kWarps <= 8) {            // every thread adds them
        t = at[k * kAll + first];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) t += at[k * kAll + first + w];
      } else {                                // lane w takes warp w's
        t = at[k * kAll + first + (lane & (kWarps - 1))];
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      }
      s[k] = t;
    }
  }
}

// v / C. A division of float64 is a long chain of dependent steps, so there it is a product with 1 / C, one rounding more (gradients of
// 100000 x 65: 43.6 -> 36.6 us); in float32 it is not the slower one (8192 x 4096: 69 us, with a product 72 us). The mean, which
// everything else is centred around, is divided in both.
__device__ __forceinline__ float share(float v, int C, float) { return v / (float)C; }
__device__ __forceinline__ double share(double v, int, double inverse) { return v * inverse; }
__device__ __forceinline__ float inverse_root(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double inverse_root(double v) { return rsqrt(v); }

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a value of another block of the cluster, whose shared memory is laid out like this one's
template <typename T>
__device__ __forceinline__ T load_remote(uint32_t local, int rank) {
  T v;
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
  if constexpr (sizeof(T) == 4) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  else asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
  return v;
}

// Rows that no block holds are shared by the blocks of a cluster, each with the same columns of every row.
struct Part { int rank, blocks, first, count; };      // a block's columns
template <bool SHARED>
__device__ __forceinline__ Part part_of_row(int C) {
  if constexpr (!SHARED) return Part{0, 1, 0, C};
  uint32_t rank, blocks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
  const int share = ((C + (int)blocks - 1) / (int)blocks + 3) / 4 * 4, first = (int)rank * share;
  return Part{(int)rank, (int)blocks, first, min(C - first, share)};
}

// The sums of all blocks of a cluster from theirs, in the blocks' order; every thread gets them. Every block is told the others' by
// stores that count their bytes at its barrier: nothing is released, so no store of results is waited for (with barriers of
// the whole cluster 1677 x 19999 took 182 us, with these stores 110). Consecutive calls alternate `turn`, and the threads of a block meet
// between two calls: a block that is told the sums of a row's turn again has read those before, since it told its own since then.
constexpr int kMaxCluster = 8;
template <typename T, bool SHARED, int K>
struct ClusterSpace {
  T slots[2][SHARED ? kMaxCluster : 1][K];
  uint64_t told[2];
  int note;
};
template <typename T, bool SHARED, int K>
__device__ __forceinline__ void cluster_begin(ClusterSpace<T, SHARED, K>& space) {
  if constexpr (SHARED) {
    if (threadIdx.x == 0) {
      space.note = 0;
      tc::mbar_init(tc::smem_u32(&space.told[0]), 1);
      tc::mbar_init(tc::smem_u32(&space.told[1]), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    cluster_sync();
  }
}
template <typename T, bool SHARED, int K>
__device__ __forceinline__ void cluster_sums(T (&s)[K], ClusterSpace<T, SHARED, K>& space, const Part& mine, int turn, uint32_t parity, const Waits& waits,
                                             uint32_t& flags) {
  if constexpr (SHARED) {
    const uint32_t bar = tc::smem_u32(&space.told[turn]);
    // A thread that has not waited in vain knows that the last use of the barrier is over, and that the others have read the sums
    // that they were told before
    const bool tell = flags < kSilent;
    if (threadIdx.x == 0 && tell) tc::mbar_arrive_expect_tx(bar, mine.blocks * K * (uint32_t)sizeof(T));
    if (threadIdx.x < mine.blocks && tell) {
      uint32_t at, there;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(tc::smem_u32(&space.slots[turn][mine.rank][0])), "r"((uint32_t)threadIdx.x));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(bar), "r"((uint32_t)threadIdx.x));
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if constexpr (sizeof(T) == 4)
          asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(at + k * 4), "f"(s[k]), "r"(there) : "memory");
        else asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.f64 [%0], %1, [%2];" ::"r"(at + k * 8), "d"(s[k]), "r"(there) : "memory");
      }
    }
    if (wait_until(bar, parity, waits, &space.note, flags)) {     // this makes what the other blocks stored visible
      uint32_t seen;
      asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                   : "=r"(seen) : "r"(bar), "r"(parity) : "memory");
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      T t = space.slots[turn][0][k];
#pragma unroll
      for (int q = 1; q < kMaxCluster; ++q)      // all loads at once: a loop over the blocks costs 15 us at 1677 x 19999
        if (q < mine.blocks) t += space.slots[turn][q][k];
      s[k] = t;
    }
  }
}

// The end of a cluster's kernel: no block leaves while it may be told something. What it has not waited for is on its way at most
// when all blocks are here.
template <typename T, bool SHARED, int K>
__device__ __forceinline__ void cluster_end(ClusterSpace<T, SHARED, K>& space) {
  if constexpr (SHARED) {
    __syncwarp();
    cluster_sync();
    const uint32_t t0 = (uint32_t)clock();
    while (*(volatile int*)&space.note && (uint32_t)clock() - t0 < 2000000u) __nanosleep(1000);
  }
}

// ================================================================================================
// Layer norm: y = (x - m) / sqrt(v + eps) * gain + bias with the row's mean m and variance v (of the centred values, so
// that a large common offset costs no digits). Bound by the bytes of x and y: every row is read once, and the next row's loads
// are under way while this row's sums are formed.
// ================================================================================================
template <typename T, int VEC, int N, int TEAM, bool SHARED>
__global__ void __launch_bounds__(team_block<TEAM>()) norm_forward_kernel(const T* __restrict__ x, const T* __restrict__ gain, const T* __restrict__ bias,
                                                                          long R, int C, T eps, T* __restrict__ y, const Waits waits) {
  constexpr int kBlock = team_block<TEAM>(), kTeams = kBlock / TEAM, E = VEC * N;
  __shared__ T part[2 * (kBlock / 32) * 1];
  __shared__ ClusterSpace<T, SHARED, 1> space;
  const Part mine = part_of_row<SHARED>(C);
  uint32_t flags = waits.flags;      // and the parity of the sums' exchanges
  const int team = threadIdx.x / TEAM, t = threadIdx.x % TEAM;
  Row<T, VEC, N, TEAM> g, b, row, next;
  bool inside[N];
#pragma unroll
  for (int i = 0; i < N; ++i) inside[i] = (i * TEAM + t) * VEC < mine.count;
  g.load(gain + mine.first, mine.count, t, T(0));
  b.load(bias + mine.first, mine.count, t, T(0));
  cluster_begin(space);
  // all teams of a block make the same number of steps: they share barriers
  const long group = blockIdx.x / mine.blocks, step = (long)(gridDim.x / mine.blocks) * kTeams;
  const T inverse = T(1) / (T)C;      // float64
  long r = group * kTeams + team;
  if (r < R) next.load(x + r * C + mine.first, mine.count, t, T(0));
  for (long first = group * kTeams; first < R; first += step, r += step) {
    row = next;
    if (r + step < R) next.load(x + (r + step) * C + mine.first, mine.count, t, T(0));
    T s[1] = {T(0)};
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += row.v[e];
    team_sums<TEAM>(s, part, 0);
    cluster_sums(s, space, mine, 0, flags & 1u, waits, flags);
    const T mean = s[0] / (T)C;
    T q[1] = {T(0)};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      row.v[e] -= mean;
      q[0] += inside[e / VEC] ? row.v[e] * row.v[e] : T(0);
    }
    team_sums<TEAM>(q, part, 1);
    cluster_sums(q, space, mine, 1, flags & 1u, waits, flags);
    flags ^= 1u;
    const T rstd = inverse_root(share(q[0], C, inverse) + eps);
    if (r < R) {
#pragma unroll
      for (int e = 0; e < E; ++e) row.v[e] = row.v[e] * rstd * g.v[e] + b.v[e];
      row.store(y + r * C + mine.first, mine.count, t);
    }
  }
  cluster_end(space);
}

// One element group of a thread from global to shared memory, asynchronously
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}

// Gradients, from one pass over x and gy: with d = gy * gain and xh = (x - m) * rstd
//   dx = rstd * (d - mean(d) - xh * mean(d * xh)), dgain[c] = sum_r gy * xh, dbias[c] = sum_r gy.
// The row's statistics are formed again from x, which is read anyway: two rounds of sums per row (x and d; the squares and the
// products of the centred x). A thread sees the same columns in every row, so dgain and dbias are added up in registers; the
// teams of a block join theirs through shared memory, the blocks through part[block][2][C], which norm_fold_kernel adds in order.
// Bound by the bytes of x, gy and dx. What a thread will need of the next kAhead rows is on its way into its own places of shared
// memory (no other thread touches them: no barrier): registers could hold one row more at most.
constexpr int kAhead = 2;
template <typename T, int VEC, int N, int TEAM>
constexpr size_t norm_backward_array() { return (size_t)N * team_block<TEAM>() * VEC * sizeof(T) + (VEC == 1 ? 32 : 0); }   // of one stage
template <typename T, int VEC, int N, int TEAM>
constexpr size_t norm_backward_bytes() { return (kAhead + 1) * 2 * norm_backward_array<T, VEC, N, TEAM>(); }

// VEC 1, for rows that start anywhere among others. Element by element, the copies above are four bytes each and bound the kernel
// (16384 x 2047: 111 us, now 68 us). But the rows that a block's teams take in one step lie one behind the other, so one thread
// brings all of them by a bulk copy, from the 16-byte boundary before the first to the one behind the last. Where that would
// leave the array, at its two ends, the rows are loaded directly.
template <typename T>
struct Span {
  const unsigned char* from;     // on a 16-byte boundary
  uint32_t bytes, shift;         // `shift`: of the first element
  bool inside;
  __device__ __forceinline__ Span(const T* array, long size, long first, long count) {
    const uintptr_t begin = (uintptr_t)array, lo = begin + first * sizeof(T), hi = lo + count * sizeof(T);
    const uintptr_t lo16 = lo & ~(uintptr_t)15, hi16 = (hi + 15) & ~(uintptr_t)15;
    from = (const unsigned char*)lo16;
    bytes = (uint32_t)(hi16 - lo16);
    shift = (uint32_t)(lo - lo16);
    inside = lo16 >= begin && hi16 <= begin + size * sizeof(T);
  }
};
__device__ __forceinline__ void copy_bulk(void* to, const void* from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

template <typename T, int VEC, int N, int TEAM, bool ONE, bool SHARED>
__global__ void __launch_bounds__(team_block<TEAM>(), (TEAM == 1024 || VEC * N * sizeof(T) == 32 && sizeof(T) == 4 ? 1024 : 512) / team_block<TEAM>())
norm_backward_kernel(const T* __restrict__ x, const T* __restrict__ gain, const T* __restrict__ gy, long R, int C, T eps, T* __restrict__ dx,
                     T* __restrict__ part, T* __restrict__ dgain, T* __restrict__ dbias, const Waits waits) {
  constexpr int kBlock = team_block<TEAM>(), kTeams = kBlock / TEAM, E = VEC * N;
  typedef Pack<T, VEC> P;
  extern __shared__ __align__(16) unsigned char ahead_raw[];
  __shared__ __align__(16) T sums[2 * (kBlock / 32) * 2];
  __shared__ ClusterSpace<T, SHARED, 2> space;
  __shared__ __align__(8) uint64_t full[kAhead + 1];
  uint32_t flags = waits.flags;      // bits 0 to kAhead: phases of the stages' barriers; bit 8: parity of the sums' exchanges
  constexpr size_t kArray = norm_backward_array<T, VEC, N, TEAM>();
  P* ahead = reinterpret_cast<P*>(ahead_raw) + threadIdx.x;     // [kAhead + 1][x, gy][N][thread]
  const int team = threadIdx.x / TEAM, t = threadIdx.x % TEAM;
  const Part mine = part_of_row<SHARED>(C);
  const long group = blockIdx.x / mine.blocks, step = (long)(gridDim.x / mine.blocks) * kTeams;
  bool inside[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    inside[i] = (i * TEAM + t) * VEC < mine.count;
    if (VEC > 1 && !inside[i])      // never written again: columns beyond C are zeros in every row
      for (int k = 0; k < 2 * (kAhead + 1); ++k)
        for (int j = 0; j < VEC; ++j) ahead[(k * N + i) * kBlock].v[j] = T(0);
  }
  if (VEC == 1 && threadIdx.x == 0) {
    space.note = 0;
    for (int i = 0; i <= kAhead; ++i) tc::mbar_init(tc::smem_u32(&full[i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (VEC == 1) __syncthreads();
  // r: this team's row; VEC 1: the first team's, by one thread for all
  auto fetch = [&](int stage, long r) {
    if constexpr (VEC == 1) {
      if (threadIdx.x == 0 && r < R) {
        const long rows = R - r < kTeams ? R - r : kTeams;
        const long count = !SHARED ? rows * C : mine.count;
        const Span<T> sx(x, R * C, r * C + mine.first, count), sg(gy, R * C, r * C + mine.first, count);
        if (sx.inside && sg.inside && flags < kSilent) {      // the copy before it into this place has landed
          const uint32_t bar = tc::smem_u32(&full[stage]);
          tc::mbar_arrive_expect_tx(bar, sx.bytes + sg.bytes);
          copy_bulk(ahead_raw + (stage * 2) * kArray, sx.from, sx.bytes, bar);
          copy_bulk(ahead_raw + (stage * 2 + 1) * kArray, sg.from, sg.bytes, bar);
        }
      }
    } else {
      if (r < R) {
        const T *from_x = x + r * C + t * VEC, *from_g = gy + r * C + t * VEC;
        P* to = ahead + stage * (2 * N * kBlock);
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (inside[i]) {
            copy_async<sizeof(P)>(to + i * kBlock, from_x + i * TEAM * VEC);
            copy_async<sizeof(P)>(to + (N + i) * kBlock, from_g + i * TEAM * VEC);
          }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  const T inverse = T(1) / (T)C;      // float64
  long r = group * kTeams + team;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) fetch(i, (VEC == 1 ? group * kTeams : r) + i * step);
  Row<T, VEC, N, TEAM> w, dg, db;
  w.load(gain + mine.first, mine.count, t, T(0));
  cluster_begin(space);
#pragma unroll
  for (int e = 0; e < E; ++e) dg.v[e] = db.v[e] = T(0);
  int stage = 0;
  for (long first = group * kTeams; first < R; first += step, r += step) {
    // VEC 1: the stage that is filled now was read in the step before; teams of several warps met at a barrier since
    if (VEC == 1 && TEAM <= 32) __syncthreads();
    fetch(stage >= 1 ? stage - 1 : kAhead, (VEC == 1 ? first : r) + kAhead * step);
    Row<T, VEC, N, TEAM> a, g;
    if constexpr (VEC == 1) {
      const long rows = R - first < kTeams ? R - first : kTeams;
      const long count = !SHARED ? rows * C : mine.count;
      const Span<T> sx(x, R * C, first * C + mine.first, count), sg(gy, R * C, first * C + mine.first, count);
      if (sx.inside && sg.inside) {
        if (wait_until(tc::smem_u32(&full[stage]), (flags >> stage) & 1u, waits, &space.note, flags)) flags ^= 1u << stage;
        const T* from_x = reinterpret_cast<const T*>(ahead_raw + (stage * 2) * kArray + sx.shift) + team * C + t;
        const T* from_g = reinterpret_cast<const T*>(ahead_raw + (stage * 2 + 1) * kArray + sg.shift) + team * C + t;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          a.v[i] = inside[i] ? from_x[i * TEAM] : T(0);
          g.v[i] = inside[i] ? from_g[i * TEAM] : T(0);
        }
      } else {
        const int valid = r < R ? mine.count : 0;
        a.load(x + r * C + mine.first, valid, t, T(0));
        g.load(gy + r * C + mine.first, valid, t, T(0));
      }
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
      const P* from = ahead + stage * (2 * N * kBlock);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const P px = from[i * kBlock], pg = from[(N + i) * kBlock];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          a.v[i * VEC + j] = px.v[j];
          g.v[i * VEC + j] = pg.v[j];
        }
      }
    }
    if (++stage > kAhead) stage = 0;
    T s[2] = {T(0), T(0)};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s[0] += a.v[e];
      s[1] += g.v[e] * w.v[e];
    }
    team_sums<TEAM>(s, sums, 0);
    cluster_sums(s, space, mine, 0, flags >> 8 & 1u, waits, flags);
    const T mean = s[0] / (T)C, s1 = share(s[1], C, inverse);
    T q[2] = {T(0), T(0)};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      a.v[e] -= mean;
      q[0] += inside[e / VEC] ? a.v[e] * a.v[e] : T(0);
      q[1] += g.v[e] * w.v[e] * a.v[e];      // g is 0 beyond C
    }
    team_sums<TEAM>(q, sums, 1);
    cluster_sums(q, space, mine, 1, flags >> 8 & 1u, waits, flags);
    flags ^= 1u << 8;
    const T rstd = inverse_root(share(q[0], C, inverse) + eps), s2 = share(q[1], C, inverse) * rstd;
    if (r < R) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const T xh = a.v[e] * rstd;
        dg.v[e] += g.v[e] * xh;
        db.v[e] += g.v[e];
        a.v[e] = rstd * (g.v[e] * w.v[e] - s1 - xh * s2);
      }
      a.store(dx + r * C + mine.first, mine.count, t);
    }
  }
  // ONE, for few rows: the whole grid is one cluster, whose blocks leave their sums in their shared memory and then add all
  // blocks' sums of a share of the columns, in order; no second kernel.
  T* joined = reinterpret_cast<T*>(ahead_raw);      // 2 E of the block's threads, or 2 C: less than the rows took
  if (VEC == 1 && threadIdx.x == 0 && flags >= kSilent)      // copies that were not waited for land before their place is written or left
    for (int i = 0; i <= kAhead; ++i) {
      const uint32_t t0 = (uint32_t)clock();
      while (!tc::mbar_try(tc::smem_u32(&full[i]), (flags >> i) & 1u) && (uint32_t)clock() - t0 < 20000000u) {}
    }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (kTeams > 1 || ONE) __syncthreads();
  T* out = ONE ? joined + (kTeams > 1 ? 2 * E * kBlock : 0) : part + group * 2 * C;
  if (kTeams == 1) {
    dg.store(out + mine.first, mine.count, t);
    db.store(out + C + mine.first, mine.count, t);
  } else {
    // [e][thread]; then the columns are added over the teams, in order
#pragma unroll
    for (int e = 0; e < E; ++e) {
      joined[(2 * e) * kBlock + threadIdx.x] = dg.v[e];
      joined[(2 * e + 1) * kBlock + threadIdx.x] = db.v[e];
    }
    __syncthreads();
    for (int k = threadIdx.x; k < 2 * E * TEAM; k += kBlock) {
      const int j = k % TEAM, e = k / TEAM / 2, which = k / TEAM & 1;
      T v = T(0);
      for (int q = 0; q < kTeams; ++q) v += joined[(2 * e + which) * kBlock + q * TEAM + j];
      const int c = (e / VEC * TEAM + j) * VEC + e % VEC;
      if (c < C) out[(long)which * C + c] = v;
    }
  }
  cluster_end(space);
  if constexpr (ONE) {
    cluster_sync();
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(out);
    for (int c = blockIdx.x * kBlock + threadIdx.x; c < 2 * C; c += gridDim.x * kBlock) {
      T v = T(0);
      for (int q = 0; q < (int)gridDim.x; ++q) v += load_remote<T>(at + c * (uint32_t)sizeof(T), q);
      if (c < C) dgain[c] = v;
      else dbias[c - C] = v;
    }
    cluster_sync();      // the others have read this block's sums
  }
}

// dgain and dbias from the blocks' sums part[P][2][C]: 32 groups of VEC of the 2 C columns per block, 32 warps that each add
// every 32nd block's, then the warps' sums in order
constexpr int kFoldGroups = 32;
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kFoldGroups) norm_fold_kernel(const T* __restrict__ part, long C, int P, T* __restrict__ dgain, T* __restrict__ dbias) {
  typedef Pack<T, VEC> V;
  __shared__ V joined[kFoldGroups][32];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  const long c = ((long)blockIdx.x * 32 + lane) * VEC;
  V s;
#pragma unroll
  for (int j = 0; j < VEC; ++j) s.v[j] = T(0);
  if (c < 2 * C) {
#pragma unroll 4
    for (int q = group; q < P; q += kFoldGroups) {
      const V v = *reinterpret_cast<const V*>(part + (long)q * 2 * C + c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s.v[j] += v.v[j];
    }
  }
  joined[group][lane] = s;
  __syncthreads();
  if (group < VEC && c - lane * VEC < 2 * C) {       // warp j adds column j of every group of columns
    const long mine = c + group;
    T v = joined[0][lane].v[group];
#pragma unroll
    for (int q = 1; q < kFoldGroups; ++q) v += joined[q][lane].v[group];
    if (mine < C) dgain[mine] = v;
    else if (mine < 2 * C) dbias[mine - C] = v;
  }
}
template <typename T>
void norm_fold(const T* part, long C, long P, T* dgain, T* dbias) {
  constexpr int VEC = 16 / sizeof(T);      // float64: 2, of which 2 C is a multiple
  if constexpr (VEC > 2)
    if (2 * C % VEC) {
      CGTB_LAUNCH((norm_fold_kernel<T, 1>), (unsigned)cgtb_ceil_div(2 * C, 32), 32 * kFoldGroups, 0, part, C, (int)P, dgain, dbias);
      return;
    }
  CGTB_LAUNCH((norm_fold_kernel<T, VEC>), (unsigned)cgtb_ceil_div(2 * C, 32 * VEC), 32 * kFoldGroups, 0, part, C, (int)P, dgain, dbias);
}

constexpr int kLongThreads = 1024;

// ---- rows that no cluster holds: a block per row that reads it several times (the L2 cache has it) ----
template <typename T>
__device__ __forceinline__ void long_row_statistics(const T* x, long C, T eps, T* part, T& mean, T& rstd) {
  T s[1] = {T(0)};
  for (long c = threadIdx.x; c < C; c += kLongThreads) s[0] += x[c];
  team_sums<kLongThreads>(s, part, 0);
  mean = s[0] / (T)C;
  T q[1] = {T(0)};
  for (long c = threadIdx.x; c < C; c += kLongThreads) { const T d = x[c] - mean; q[0] += d * d; }
  team_sums<kLongThreads>(q, part, 1);
  rstd = inverse_root(q[0] / (T)C + eps);
}
template <typename T>
__global__ void __launch_bounds__(kLongThreads) norm_forward_long_kernel(const T* __restrict__ x, const T* __restrict__ gain, const T* __restrict__ bias,
                                                                         long R, long C, T eps, T* __restrict__ y) {
  __shared__ T part[2 * 32];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    T mean, rstd;
    long_row_statistics(x + r * C, C, eps, part, mean, rstd);
    for (long c = threadIdx.x; c < C; c += kLongThreads) y[r * C + c] = (x[r * C + c] - mean) * rstd * gain[c] + bias[c];
  }
}
template <typename T>
__global__ void __launch_bounds__(kLongThreads) norm_backward_long_kernel(const T* __restrict__ x, const T* __restrict__ gain, const T* __restrict__ gy,
                                                                          long R, long C, T eps, T* __restrict__ dx, T* __restrict__ stats) {
  __shared__ T part[2 * 32 + 32 * 2];
  for (long r = blockIdx.x; r < R; r += gridDim.x) {
    T mean, rstd;
    long_row_statistics(x + r * C, C, eps, part, mean, rstd);
    T s[2] = {T(0), T(0)};
    for (long c = threadIdx.x; c < C; c += kLongThreads) {
      const T d = gy[r * C + c] * gain[c];
      s[0] += d;
      s[1] += d * ((x[r * C + c] - mean) * rstd);
    }
    team_sums<kLongThreads>(s, part + 2 * 32, 0);
    const T s1 = s[0] / (T)C, s2 = s[1] / (T)C;
    for (long c = threadIdx.x; c < C; c += kLongThreads) {
      const T d = gy[r * C + c] * gain[c], xh = (x[r * C + c] - mean) * rstd;
      dx[r * C + c] = rstd * (d - s1 - xh * s2);
    }
    if (threadIdx.x == 0) { stats[2 * r] = mean; stats[2 * r + 1] = rstd; }
  }
}
// sums over the rows of slice blockIdx.y: part[slice][0][c] of gy * xh, part[slice][1][c] of gy
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_kernel(const T* __restrict__ x, const T* __restrict__ gy, const T* __restrict__ stats,
                                                           long R, long C, long rows_per_slice, T* __restrict__ part) {
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  const long first = blockIdx.y * rows_per_slice;
  const long last = first + rows_per_slice < R ? first + rows_per_slice : R;
  T s1 = T(0), s2 = T(0);
#pragma unroll 4
  for (long r = first; r < last; ++r) {
    const T g = gy[r * C + c];
    s1 += g * ((x[r * C + c] - stats[2 * r]) * stats[2 * r + 1]);
    s2 += g;
  }
  part[(2 * (long)blockIdx.y) * C + c] = s1;
  part[(2 * (long)blockIdx.y + 1) * C + c] = s2;
}

template <typename T> bool starts_on_16(long C, std::initializer_list<const void*> arrays) {
  if (C * sizeof(T) % 16) return false;
  for (const void* a : arrays)
    if ((uintptr_t)a & 15) return false;
  return true;
}

// calls f(team) with the smallest team for rows of C elements, E of them a thread; false when none is large enough. Only teams from
// kMinTeam to kMaxTeam are made; where kMinTeam is above 1, the caller has rows that no smaller team holds.
template <int E, int kMinTeam, int kMaxTeam, typename F>
bool with_team(long C, F f) {
  if (C <= (long)kMinTeam * E) {
    f(std::integral_constant<int, kMinTeam>());
    return true;
  }
  if constexpr (kMinTeam < kMaxTeam) return with_team<E, 2 * kMinTeam, kMaxTeam>(C, f);
  else return false;
}

// as many blocks as the SMs hold at a time: the grid of a kernel whose blocks walk the rows
template <auto KERNEL, int THREADS, size_t BYTES>
long resident_blocks() {
  static const long n = [] {
    int per_sm = 0;
    if (BYTES > 32 * 1024) cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BYTES);   // with static memory: over 48 KB
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, KERNEL, THREADS, BYTES) != cudaSuccess || per_sm < 1) per_sm = 1;
    return (long)rt().sm_count * per_sm;
  }();
  return n;
}

// Launches KERNEL, whose clusters of `blocks` blocks walk the rows, with as many of them as the GPU holds at a time; returns their
// number, 0 when it failed.
template <auto KERNEL, int THREADS, size_t BYTES, typename F>
long launch_clusters(const char* who, int blocks, long R, F arguments) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = BYTES;
  config.stream = rt().stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  static std::atomic<int> resident[kMaxCluster + 1];      // by blocks; 0: not asked yet
  int n = resident[blocks].load(std::memory_order_relaxed);
  if (!n) {
    if (BYTES > 32 * 1024) cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BYTES);
    config.gridDim = dim3((unsigned)blocks);
    if (cudaOccupancyMaxActiveClusters(&n, KERNEL, &config) != cudaSuccess || n < 1) n = 1;
    resident[blocks].store(n, std::memory_order_relaxed);
  }
  const long P = std::min<long>(R, n);
  config.gridDim = dim3((unsigned)(P * blocks));
  const cudaError_t e = arguments(config, P);
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  if (e != cudaSuccess) { fail("%s launch failed: %s", who, cudaGetErrorString(e)); return 0; }
  return P;
}

std::atomic<uint32_t> g_selftest_cycles{0};
Waits bounded_waits() {
  const uint32_t cycles = g_selftest_cycles.load();
  return Waits{tc_error_flag(), cycles ? cycles : (uint32_t)tc::kWaitCycles, cycles ? kSilent : 0u};
}

template <typename T>
int norm_forward(const T* x, long R, long C, const T* gain, const T* bias, double eps, T* y) {
  constexpr int E = 32 / sizeof(T);     // 8 float32 or 4 float64 a thread
  const bool wide = starts_on_16<T>(C, {x, gain, bias, y});
  const bool held = with_team<E, 1, 1024>(C, [&](auto team) {
    constexpr int TEAM = decltype(team)::value, kBlock = team_block<TEAM>();
    auto launch = [&](auto width, auto elements) {
      constexpr auto kernel = norm_forward_kernel<T, decltype(width)::value, decltype(elements)::value / decltype(width)::value, TEAM, false>;
      const long blocks = std::min<long>(cgtb_ceil_div(R, kBlock / TEAM), resident_blocks<kernel, kBlock, 0>());
      CGTB_LAUNCH(kernel, (unsigned)blocks, kBlock, 0, x, gain, bias, R, (int)C, (T)eps, y, Waits());
    };
    if (wide) return launch(std::integral_constant<int, 16 / sizeof(T)>(), std::integral_constant<int, E>());
    if constexpr (TEAM > 1)      // fewer places without an element
      if (C <= TEAM * (E * 3 / 4)) return launch(std::integral_constant<int, 1>(), std::integral_constant<int, E * 3 / 4>());
    launch(std::integral_constant<int, 1>(), std::integral_constant<int, E>());
  });
  // Rows that no team holds, by clusters whose blocks hold 16 KB of a row: 1677 x 19999 66 us, 3000 x 9001 63 us (a block of 1024
  // threads for a row: 76 and 78 us; blocks of 512 threads and 16 KB 81 and 79 us). Where one block holds the row it is faster
  // (4096 x 8192 49 us, by clusters 52; gradients 69 and 84 us).
  constexpr int kTeam = 256, kElements = 64 / sizeof(T);
  if (!held && C <= 1L * kTeam * kElements * kMaxCluster) {
    const Waits waits = bounded_waits();
    if (!waits.err) return 1;
    auto launch = [&](auto width) {
      constexpr int VEC = decltype(width)::value;
      constexpr auto kernel = norm_forward_kernel<T, VEC, kElements / VEC, kTeam, true>;
      return launch_clusters<kernel, kTeam, 0>("layer_norm_forward", (int)cgtb_ceil_div(C, kTeam * kElements), R, [&](const cudaLaunchConfig_t& config, long) {
        return cudaLaunchKernelEx(&config, kernel, x, gain, bias, R, (int)C, (T)eps, y, waits);
      });
    };
    if (!(wide ? launch(std::integral_constant<int, 16 / sizeof(T)>()) : launch(std::integral_constant<int, 1>()))) return 1;
  } else if (!held) {
    const unsigned grid = (unsigned)std::min<long>(R, rt().sm_count * 2L);
    CGTB_LAUNCH(norm_forward_long_kernel<T>, grid, kLongThreads, 0, x, gain, bias, R, C, (T)eps, y);
  }
  CGTB_CHECK_LAUNCH("layer_norm_forward");
  return 0;
}

// The gradients by teams of E elements a thread, VEC at a time; dgain and dbias are complete, or in `part` for P blocks. 1: failed,
// -1: no team is that large
template <typename T, int VEC, int E, int kMinTeam, int kMaxTeam>
int norm_backward_teams(const T* x, const T* gain, const T* gy, long R, long C, double eps, T* dx, T* dgain, T* dbias, T*& part, long& P) {
  int failed = 0;
  const Waits waits = bounded_waits();
  if (!waits.err) return 1;
  const bool held = with_team<E, kMinTeam, kMaxTeam>(C, [&](auto team) {
    constexpr int TEAM = decltype(team)::value, kBlock = team_block<TEAM>(), kTeams = kBlock / TEAM;
    constexpr size_t bytes = norm_backward_bytes<T, VEC, E / VEC, TEAM>();
    constexpr auto kernel = norm_backward_kernel<T, VEC, E / VEC, TEAM, false, false>, one = norm_backward_kernel<T, VEC, E / VEC, TEAM, true, false>;
    const long steps = cgtb_ceil_div(R, kTeams), sms = rt().sm_count;
    if (steps <= 8) {       // (512 x 256, 32 steps: 7.0 us by eight blocks, 5.1 us by more and another kernel)
      (void)resident_blocks<one, kBlock, bytes>();      // allows the shared memory
      cudaLaunchAttribute attr = {};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = steps > 4 ? 8 : steps > 2 ? 4 : steps > 1 ? 2 : 1;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cudaLaunchConfig_t config = {};
      config.gridDim = dim3(attr.val.clusterDim.x);
      config.blockDim = dim3(kBlock);
      config.dynamicSmemBytes = bytes;
      config.stream = rt().stream;
      config.attrs = &attr;
      config.numAttrs = 1;
      const cudaError_t e = cudaLaunchKernelEx(&config, one, x, gain, gy, R, (int)C, (T)eps, dx, (T*)nullptr, dgain, dbias, waits);
      if (e != cudaSuccess) failed = fail("layer_norm_backward launch failed: %s", cudaGetErrorString(e));
      g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
      return;
    }
    // at least four rows for a team, so that what the blocks leave for the last kernel stays small against the rows; but no SM
    // without a block where there are rows for it
    P = std::min(std::min(steps, resident_blocks<kernel, kBlock, bytes>()), std::max(cgtb_ceil_div(steps, 4), sms));
    part = (T*)scratch((size_t)P * 2 * C * sizeof(T));     // starts on a 256-byte boundary
    if (!part) failed = 1;
    else CGTB_LAUNCH(kernel, (unsigned)P, kBlock, bytes, x, gain, gy, R, (int)C, (T)eps, dx, part, (T*)nullptr, (T*)nullptr, waits);
  });
  return held ? failed : -1;
}

template <typename T>
int norm_backward(const T* x, const T* gain, const T* gy, long R, long C, double eps, T* dx, T* dgain, T* dbias) {
  T* part = nullptr;
  long P = 0;
  // 64 bytes of a row a thread save steps of the sums (float32, 30000 x 784: 72 us with 32, 48 us with 64; float64, 4000 x 2047: 51
  // and 38 us), 32 bytes where a row has not enough for that, or is short and float64 (100000 x 64: 29 against 33 us). Arrays
  // that start on 16-byte boundaries are read 16 bytes at a time (100000 x 64: 20 against 31 us, 4000 x 5000: 53 against 66 us),
  // but in between, where two or four rows are under way on an SM, by the bulk copies all the same (8192 x 4096: 69 against 86 us).
  const bool starts = starts_on_16<T>(C, {x, gain, gy, dx});
  auto teams = [&](auto width, auto elements, auto least, auto most) {
    return norm_backward_teams<T, decltype(width)::value, decltype(elements)::value, decltype(least)::value, decltype(most)::value>(
        x, gain, gy, R, C, eps, dx, dgain, dbias, part, P);
  };
  constexpr std::integral_constant<int, 16 / sizeof(T)> k16Bytes;
  constexpr std::integral_constant<int, 1> kOne;
  constexpr std::integral_constant<int, 32 / sizeof(T)> kFew;
  constexpr std::integral_constant<int, 64 / sizeof(T)> kMany;
  constexpr std::integral_constant<int, 512> kLargest;
  constexpr std::integral_constant<int, 16 / kFew> kUpTo16;         // the team that holds 16 columns, and the least one for more of them
  constexpr std::integral_constant<int, 32 / kMany> kFrom17;
  int failed;
  if constexpr (sizeof(T) == 8) {
    if (starts && C <= 1024) failed = teams(k16Bytes, kFew, kOne, std::integral_constant<int, 1024 / kFew>());
    else if (C <= 16) failed = teams(kOne, kFew, kOne, kUpTo16);
    else failed = teams(kOne, kMany, kFrom17, kLargest);
  } else {
    if (C <= 16) failed = starts ? teams(k16Bytes, kFew, kOne, kUpTo16) : teams(kOne, kFew, kOne, kUpTo16);
    else if (starts && C <= 1024) failed = teams(k16Bytes, kMany, kFrom17, std::integral_constant<int, 1024 / kMany>());
    else if (starts && C > 4096) failed = teams(k16Bytes, kMany, kLargest, kLargest);
    else failed = teams(kOne, kMany, kFrom17, kLargest);
  }
  if (failed > 0) return 1;
  // Rows that no team holds, by clusters: their blocks hold 32 or 16 KB of a row, of which two fit an SM. The larger ones are faster
  // where the row fills them as well (2000 x 16384: 84 and 101 us), the smaller ones where it does not (1677 x 20000, before the
  // sums of a cluster were loaded at once: 143 and 103 us).
  constexpr long kLarge = 512 * (64 / sizeof(T)), kSmall = kLarge / 2;
  auto clusters = [&](auto threads, int blocks) {
    constexpr int TEAM = decltype(threads)::value, E = 64 / sizeof(T);
    constexpr size_t bytes = norm_backward_bytes<T, 1, E, TEAM>();
    constexpr auto kernel = norm_backward_kernel<T, 1, E, TEAM, false, true>;
    const Waits waits = bounded_waits();
    if (!waits.err) return 0L;
    return launch_clusters<kernel, TEAM, bytes>("layer_norm_backward", blocks, R, [&](const cudaLaunchConfig_t& config, long n) {
      part = (T*)scratch((size_t)n * 2 * C * sizeof(T));
      return part ? cudaLaunchKernelEx(&config, kernel, x, gain, gy, R, (int)C, (T)eps, dx, part, (T*)nullptr, (T*)nullptr, waits) : cudaErrorMemoryAllocation;
    });
  };
  if (failed < 0 && C <= kSmall * kMaxCluster) {
    const int large = (int)cgtb_ceil_div(C, kLarge), small = (int)cgtb_ceil_div(C, kSmall);
    P = small == 2 * large ? clusters(std::integral_constant<int, 512>(), large) : clusters(std::integral_constant<int, 256>(), small);
    if (!P) return 1;
  } else if (failed < 0) {
    const long cblocks = cgtb_ceil_div(C, 256);
    P = cgtb_ceil_div(R, 64);
    if (P > 64) P = 64;
    part = (T*)scratch((size_t)(2 * R + 2 * P * C) * sizeof(T));    // first: the last kernel reads it 16 bytes at a time
    if (!part) return 1;
    T* stats = part + 2 * P * C;
    const long grid = R < rt().sm_count * 2L ? R : rt().sm_count * 2L;
    CGTB_LAUNCH(norm_backward_long_kernel<T>, (unsigned)grid, kLongThreads, 0, x, gain, gy, R, C, (T)eps, dx, stats);
    CGTB_LAUNCH(norm_columns_kernel<T>, dim3((unsigned)cblocks, (unsigned)P), 256, 0, x, gy, stats, R, C, cgtb_ceil_div(R, P), part);
  }
  if (part) norm_fold(part, C, P, dgain, dbias);
  CGTB_CHECK_LAUNCH("layer_norm_backward");
  return 0;
}

int norm_extents(const char* who, int dtype, long R, long C, double eps) {
  if (R < 0 || C < 0) return fail("%s: negative extent", who);
  if (C > 0x7fffffffL) return fail("%s: rows of %ld elements are too long (at most 2^31 - 1)", who, C);
  if (!(eps >= 0) || std::isinf(eps)) return fail("%s: epsilon has to be a finite number that is not negative", who);
  // rounded to 0 or infinity it would turn rows of equal values into NaN or all rows into the bias
  if (dtype == cgtb_f4 && eps != 0 && !(eps >= FLT_MIN && eps <= FLT_MAX)) return fail("%s: epsilon %g is not a normal float32 number", who, eps);
  if (eps != 0 && eps < DBL_MIN) return fail("%s: epsilon %g is not a normal number", who, eps);
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

// A thread makes UNROLL blocks of four words, their elements loaded beforehand, 16 bytes at a time where the arrays start on
// 16-byte boundaries. Bound by the bytes of x and y; the ten rounds of a block are forty multiplications for four elements.
template <typename T, bool WIDE, int UNROLL>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, long n, uint32_t threshold, T scale, const long* __restrict__ state,
                                                      uint32_t site, T* y) {
  constexpr int kPack = WIDE ? 16 / sizeof(T) : 1, kPacks = 4 / kPack;
  typedef Pack<T, kPack> P;
  const unsigned long long seed = (unsigned long long)state[0];
  const uint32_t step = (uint32_t)(unsigned long long)state[1];
  const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
  const long whole = n / 4, stride = (long)gridDim.x * 256;
  long b = (long)blockIdx.x * 256 + threadIdx.x;
  for (; b < whole; b += UNROLL * stride) {
    P v[UNROLL][kPacks];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (b + u * stride < whole)
#pragma unroll
        for (int i = 0; i < kPacks; ++i) v[u][i] = reinterpret_cast<const P*>(x + 4 * (b + u * stride))[i];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const unsigned long long at = (unsigned long long)(b + u * stride);
      if (b + u * stride < whole) {
        const uint4 w = philox(make_uint4((uint32_t)at, (uint32_t)(at >> 32), step, site), key);
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
#pragma unroll
          for (int j = 0; j < kPack; ++j) v[u][i].v[j] = words[i * kPack + j] >= threshold ? v[u][i].v[j] * scale : T(0);
          reinterpret_cast<P*>(y + 4 * at)[i] = v[u][i];
        }
      }
    }
  }
  // the last block's one to three elements
  if (blockIdx.x == 0 && threadIdx.x < n % 4) {
    const uint4 w = philox(make_uint4((uint32_t)whole, (uint32_t)((unsigned long long)whole >> 32), step, site), key);
    const uint32_t mine = threadIdx.x == 0 ? w.x : threadIdx.x == 1 ? w.y : w.z;
    const long i = 4 * whole + threadIdx.x;
    y[i] = mine >= threshold ? x[i] * scale : T(0);
  }
}

template <typename T>
void dropout(const T* x, long n, uint32_t threshold, double scale, const int64_t* state, unsigned site, T* y) {
  const bool wide = (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
  const long blocks = cgtb_ceil_div(cgtb_ceil_div(n, 4), 256);
  auto launch = [&](auto wide16) {
    constexpr int kUnroll = 16 / sizeof(T);
    constexpr auto kernel = dropout_kernel<T, decltype(wide16)::value, kUnroll>;
    const long grid = std::max(cgtb_ceil_div(blocks, kUnroll), std::min(blocks, rt().sm_count * 2L));
    CGTB_LAUNCH(kernel, (unsigned)std::min(grid, 1L << 30), 256, 0, x, n, threshold, (T)scale, (const long*)state, site, y);
  };
  if (wide) launch(std::true_type());
  else launch(std::false_type());
}

// ================================================================================================
// Rows in 8-bit integers: a = max |x|, scale = a / 127, code = 127 x / a rounded to nearest, ties to even.
// ================================================================================================

// The exact code of x: the quotient of two numbers of 31 and 24 bits is never rounded across a tie in 64 bits.
__device__ __noinline__ int code_exact(float x, float largest) { return (int)rint(127.0 * (double)x / (double)largest); }

// The codes of VEC elements in the low bytes of a word. `inverse` = 127 / largest in 32 bits: x * inverse is off by less than
// 127 * 2^-22 = 3e-5, so wherever it is not that near to a tie, its nearest whole number is the exact quotient's. Adding
// 1.5 * 2^23 rounds to that number, ties to even, and leaves it in the low bits: no conversion, whose pipe would bound the kernel.
template <int VEC>
__device__ __forceinline__ uint32_t codes_of(const float* x, float largest, float inverse, bool exact) {
  constexpr float kRound = 12582912.0f;
  uint32_t w[VEC];
  float off = 0.f;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const float t = __fmul_rn(x[j], inverse), k = __fadd_rn(t, kRound);
    off = fmaxf(off, fabsf(__fadd_rn(t, -__fadd_rn(k, -kRound))));
    w[j] = __float_as_uint(k);
  }
  if (off >= 0.4999f || exact)
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[j] = (uint32_t)code_exact(x[j], largest);
  if constexpr (VEC == 1) return w[0];
  else return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}

__device__ __forceinline__ float scale_of(uint32_t bits) {      // of a row whose largest magnitude has these bits
  return bits < 0x7f800000u ? __uint_as_float(bits) / 127.0f : __uint_as_float(0x7fc00000u);
}

// The largest of the team's values; every thread gets it. `part`, `turn`: as team_sums has them.
template <int TEAM>
__device__ __forceinline__ uint32_t team_max(uint32_t m, uint32_t* part, int turn) {
  if constexpr (TEAM >= 32) m = __reduce_max_sync(0xffffffffu, m);
  else
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if constexpr (TEAM > 32) {
    constexpr int kWarps = TEAM / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t* at = part + turn * (team_block<TEAM>() / 32);
    if (lane == 0) at[warp] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, at[warp / kWarps * kWarps + (lane & (kWarps - 1))]);
  }
  return m;
}

// A team holds a row, four consecutive elements of it in a thread at a time, whose codes are one word; rows that do not start on
// 16-byte boundaries are loaded element by element (the four loads of a warp touch the same lines: 500000 x 17 15.5 us, with
// consecutive elements in consecutive threads and stores of single bytes 38 us). The next row's loads are under way meanwhile.
// Bound by the bytes of x.
template <bool WIDE, int N, int TEAM>
__global__ void __launch_bounds__(team_block<TEAM>()) quantize_rows_kernel(const float* __restrict__ x, long R, int C, int Cp, int8_t* __restrict__ codes,
                                                                           float* __restrict__ scales) {
  constexpr int kBlock = team_block<TEAM>(), kTeams = kBlock / TEAM, E = 4 * N;
  __shared__ uint32_t part[2 * (kBlock / 32)];
  const int team = threadIdx.x / TEAM, t = threadIdx.x % TEAM;
  const long step = (long)gridDim.x * kTeams;
  long r = (long)blockIdx.x * kTeams + team;
  Row<float, 4, N, TEAM> row, next;
  auto load = [&](long at) {
    if constexpr (WIDE) next.load(x + at * C, C, t, 0.f);
    else {
      const float* from = x + at * C + 4 * t;
#pragma unroll
      for (int e = 0; e < E; ++e) next.v[e] = (e / 4 * TEAM + t) * 4 + e % 4 < C ? from[e / 4 * TEAM * 4 + e % 4] : 0.f;
    }
  };
  if (r < R) load(r);
  int turn = 0;
  for (long first = (long)blockIdx.x * kTeams; first < R; first += step, r += step, turn ^= 1) {
    row = next;
    if (r + step < R) load(r + step);
    uint32_t m = 0;   // as whole numbers the bits of |x| order like the values, infinities and NaN above all
#pragma unroll
    for (int e = 0; e < E; ++e) m = max(m, __float_as_uint(row.v[e]) & 0x7fffffffu);
    m = team_max<TEAM>(m, part, turn);
    if (r < R) {
      const bool some = m != 0 && m < 0x7f800000u;
      const float largest = __uint_as_float(m), inverse = 127.0f / largest;
      const bool exact = !(inverse <= 3.0e38f);      // rows of the smallest numbers
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (i * TEAM + t) * 4;
        if (c < Cp) *reinterpret_cast<uint32_t*>(codes + r * Cp + c) = some ? codes_of<4>(row.v + i * 4, largest, inverse, exact) : 0u;
      }
      if (t == 0) scales[r] = scale_of(m);
    }
  }
}

// rows that no team holds: read twice
__global__ void __launch_bounds__(kLongThreads) quantize_rows_long_kernel(const float* __restrict__ x, long R, long C, long Cp, int8_t* __restrict__ codes,
                                                                          float* __restrict__ scales) {
  __shared__ uint32_t part[2 * 32];
  int turn = 0;
  for (long r = blockIdx.x; r < R; r += gridDim.x, turn ^= 1) {
    uint32_t m = 0;
    for (long c = threadIdx.x; c < C; c += kLongThreads) m = max(m, __float_as_uint(x[r * C + c]) & 0x7fffffffu);
    m = team_max<kLongThreads>(m, part, turn);
    const bool some = m != 0 && m < 0x7f800000u;
    const float largest = __uint_as_float(m), inverse = 127.0f / largest;
    for (long c = threadIdx.x; c < Cp; c += kLongThreads)
      codes[r * Cp + c] = (int8_t)(c < C && some ? codes_of<1>(x + r * C + c, largest, inverse, !(inverse <= 3.0e38f)) : 0u);
    if (threadIdx.x == 0) scales[r] = scale_of(m);
  }
}

}  // namespace

CGTB_API int cgtb_layer_norm_forward(int dtype, const void* x, long R, long C, const void* gain, const void* bias, double epsilon, void* y) {
  if (!require_runtime("cgtb_layer_norm_forward")) return 1;
  if (norm_extents("cgtb_layer_norm_forward", dtype, R, C, epsilon)) return 1;
  if (R == 0 || C == 0) return 0;
  if (dtype == cgtb_f4) return norm_forward((const float*)x, R, C, (const float*)gain, (const float*)bias, epsilon, (float*)y);
  if (dtype == cgtb_f8) return norm_forward((const double*)x, R, C, (const double*)gain, (const double*)bias, epsilon, (double*)y);
  return fail("cgtb_layer_norm_forward: unsupported dtype %d", dtype);
}

CGTB_API int cgtb_layer_norm_backward(int dtype, const void* x, const void* gain, const void* gy, long R, long C, double epsilon, void* dx, void* dgain,
                                      void* dbias) {
  if (!require_runtime("cgtb_layer_norm_backward")) return 1;
  if (norm_extents("cgtb_layer_norm_backward", dtype, R, C, epsilon)) return 1;
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

CGTB_API int cgtb_layer_norm_selftest_waits(long cycles) {
  if (cycles < 0 || cycles > (long)tc::kWaitCycles) return fail("cgtb_layer_norm_selftest_waits: 0 to %ld cycles", (long)tc::kWaitCycles);
  g_selftest_cycles.store((uint32_t)cycles);
  return 0;
}

CGTB_API int cgtb_dropout(int dtype, const void* x, long n, double p, const int64_t* state, unsigned site, void* y) {
  if (!require_runtime("cgtb_dropout")) return 1;
  if (!(p >= 0 && p < 1)) return fail("cgtb_dropout: the probability has to be in [0, 1)");
  if (n < 0) return fail("cgtb_dropout: negative extent");
  if (dtype != cgtb_f4 && dtype != cgtb_f8) return fail("cgtb_dropout: unsupported dtype %d", dtype);
  if (n == 0) return 0;
  // A word below the threshold drops its element. p above 1 - 2^-33 would round to 2^32, which is no 32-bit number: there the
  // threshold stays at 2^32 - 1, and the element of the largest word is kept
  const double t = std::nearbyint(p * 4294967296.0);
  const uint32_t threshold = t >= 4294967295.0 ? 4294967295u : (uint32_t)t;
  const double scale = 1.0 / (1.0 - p);
  if (dtype == cgtb_f4) dropout((const float*)x, n, threshold, scale, state, site, (float*)y);
  else dropout((const double*)x, n, threshold, scale, state, site, (double*)y);
  CGTB_CHECK_LAUNCH("dropout");
  return 0;
}

CGTB_API int cgtb_quantize_rows(const float* x, long R, long C, int8_t* codes, float* scales) {
  if (!require_runtime("cgtb_quantize_rows")) return 1;
  if (R < 0 || C < 0) return fail("cgtb_quantize_rows: negative extent");
  if ((uintptr_t)codes & 15) return fail("cgtb_quantize_rows: the codes have to start on a 16-byte boundary");
  if (R == 0) return 0;
  const long Cp = cgtb_ceil_div(C, 16) * 16;
  const bool wide = starts_on_16<float>(C, {x});
  auto launch = [&](auto wide16, auto elements, auto team) {
    constexpr int TEAM = decltype(team)::value, kBlock = team_block<TEAM>();
    constexpr auto kernel = quantize_rows_kernel<decltype(wide16)::value, decltype(elements)::value / 4, TEAM>;
    const long blocks = std::min<long>(cgtb_ceil_div(R, kBlock / TEAM), resident_blocks<kernel, kBlock, 0>());
    CGTB_LAUNCH(kernel, (unsigned)blocks, kBlock, 0, x, R, (int)C, (int)Cp, codes, scales);
  };
  auto either = [&](auto elements, auto team) {
    if (wide) launch(std::true_type(), elements, team);
    else launch(std::false_type(), elements, team);
  };
  // Up to 16384 codes 16 elements a thread, up to 20480 20, which fill the 64 registers that 1024 threads leave each (32 bytes are
  // spilled); longer rows are read twice: 2000 x 16384 29 us, x 20480 35 us, x 20496 84 us.
  bool held = with_team<16, 1, 1024>(Cp, [&](auto team) { either(std::integral_constant<int, 16>(), team); });
  if (!held && Cp <= 1024 * 20) {
    either(std::integral_constant<int, 20>(), std::integral_constant<int, 1024>());
    held = true;
  }
  if (!held) CGTB_LAUNCH(quantize_rows_long_kernel, (unsigned)std::min<long>(R, rt().sm_count * 2L), kLongThreads, 0, x, R, C, Cp, codes, scales);
  CGTB_CHECK_LAUNCH("quantize_rows");
  return 0;
}
