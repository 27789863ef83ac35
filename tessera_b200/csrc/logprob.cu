// Log probabilities of given tokens, the entropy of every row and its likeliest tokens, in one pass over the logits (id
// "logprob_rows"): what a server answers beside a token, and what a verified tree's drafts or a scored prompt are measured by.
//   lse = m + log S, m = max x, S = sum e^(x - m);   logprob = x_t - lse;   entropy = log S - T / S, T = sum e^(x - m) (x - m)
// The reference has top_k_rows for the likeliest tokens alone (src/backends/rocm/rocm_kernels.hpp:558-566), whose kernel walks
// a row once for every one of them.
//
// Bound: the logits' bytes (256 rows of 151936: 156 MB, 24 us at the measured copy rate).  A cluster of CTAs takes a row.  A
// CTA walks over its share in tiles of 6144 logits held in registers, the next tile's loads under way, with a running maximum
// and two running sums a thread.  The likeliest tokens come out of the same registers: a logit below the threshold -- the
// top_k-th largest so far -- costs one comparison; the few above it go to a list in shared memory, which is cut back to its
// top_k largest by counting, for each entry, the entries above it.  An entry is its logit's bits in an order-preserving form
// over its inverted index, so that no two are equal and the lowest index wins among equal logits.  The first threshold is a
// bound from the threads' maxima (enough threads are above it), and a tile that floods the list all the same (ascending or
// equal logits) finds its own threshold by bisection over the entries.  The CTAs meet through distributed shared memory.
//
// Measured: 1 row of 151936, 20 tokens 10.3 us (16 CTAs: a launch, two cuts of a list and the meeting of the CTAs); 16 rows, 8
// tokens 14.1 us; 256 rows, 20 tokens 44 us.  Twelve logits a thread are the most that the registers of two CTAs of 512
// threads hold: 16 spilled (11.4, 15.2, 53 us), 8 take 11.0, 14.2 and 50 us.  With 16, 256 threads a CTA, twice as many of them,
// took 57 us where 512 took 55; a look at the list every fourth tile instead of every one 54 us, but 18 for the 16 rows; a
// tile's second reading from memory instead of registers 117 us.  With twelve, tiles by bulk copies through shared memory, four
// under way, took 48 us (16 a thread and three under way 45), two values an instruction 43.4 us: what a tile waits for is its
// barrier and the list, since without a top list the 256 rows take 27 us (one token 38).  108 of 148 SMs have two of the 256 CTAs, the
// others one: 296 rows take no longer.
#include <cuda_runtime.h>

#include <atomic>

#include "codec.cuh"
#include "launch.h"
#include "logprob_plan.h"
#include "tessera_b200.h"

namespace tsr {
namespace {

constexpr int kLpList = 1024;   // entries of the list
constexpr int kLpTop = 32;      // top_k at most, as top_k_rows
constexpr int kLpCut = 96;      // entries from which the list is cut back before the next tile
static_assert(kLpCluster * kLpTop <= kLpMost && kLpCut > kLpTop, "a thread an entry where the CTAs meet");

using Entry64 = unsigned long long;

// An order-preserving form of a logit (NaN lowest, -0 as 0), and its inverse.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return k == 0 ? __uint_as_float(0x7FC00000u) : __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ Entry64 entry_of(float x, uint32_t index) { return static_cast<Entry64>(order_of(x)) << 32 | (0xFFFFFFFFu - index); }

// 2^x without the slow path below the normal numbers (0 there; its neighbours of a sum are 1 or more)
__device__ __forceinline__ float power2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLpLog2e = 1.4426950408889634f, kLpLn2 = 0.6931471805599453f;
struct Sums {  // y = (x - top) log2 e: sums of 2^y and of 2^y y; top is -inf before the first finite logit
  float top, s, t;
};
__device__ __forceinline__ float shift_of(float top) { return top == -INFINITY ? 0.0f : top; }
__device__ __forceinline__ Sums moved(const Sums& a, float top) {  // top >= a.top
  const float by = (shift_of(a.top) - shift_of(top)) * kLpLog2e;
  if (a.s == 0.0f) return Sums{top, a.s, a.t};  // (nothing so far; its top may be -inf)
  const float f = power2(by);
  return Sums{top, a.s * f, f == 0.0f ? 0.0f : f * fmaf(a.s, by, a.t)};  // (by may be -inf: logits of the type's lowest value)
}
// Of a warp's lanes, in every lane.
__device__ __forceinline__ Sums warp_joined(Sums a) {
  float top = a.top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  a = moved(a, top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xFFFFFFFFu, a.s, o);
    a.t += __shfl_xor_sync(0xFFFFFFFFu, a.t, o);
  }
  return a;
}

__device__ __forceinline__ uint32_t shared_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t peer_at(uint32_t local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

struct LogprobShared {
  alignas(16) Entry64 list[kLpList + 256];
  Entry64 cut[kLpTop];
  Sums sums[kLpMost / 32], all;
  uint32_t bound[kLpMost / 32];
  int count;
};

// (Named by both functions below: an address handed to one that is not inlined would be a generic one.)
extern __shared__ __align__(16) unsigned char logprob_smem[];
__device__ __forceinline__ LogprobShared& logprob_shared() { return *reinterpret_cast<LogprobShared*>(logprob_smem); }

// The list's top_k largest to its front, in order; returns the entry that a new one has to exceed (0: none).  Several threads
// count for an entry where there are few.
template <int THREADS>
__device__ __noinline__ Entry64 cut_back(int n, int top_k) {
  LogprobShared& sh = logprob_shared();
  const int tid = threadIdx.x;
  int log = 0;  // 2^log threads an entry
  while (log < 5 && (n << (log + 1)) <= THREADS) ++log;
  const int part = tid & ((1 << log) - 1);
  if (tid < 8 << log) sh.list[n + tid] = 0;  // (they are read eight a thread at a time)
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += THREADS >> log) {
    const int i = i0 + (tid >> log);
    const Entry64 mine = sh.list[min(i, n - 1)];
    int above = 0;
#pragma unroll 1
    for (int j = 2 * part; j < n; j += 8 << log) {
      ulonglong2 e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) e[u] = *reinterpret_cast<const ulonglong2*>(&sh.list[j + u * (2 << log)]);
#pragma unroll
      for (int u = 0; u < 4; ++u) above += (e[u].x > mine ? 1 : 0) + (e[u].y > mine ? 1 : 0);
    }
    for (int o = 1; o < 1 << log; o <<= 1) above += __shfl_xor_sync(0xFFFFFFFFu, above, o);
    if (part == 0 && i < n && above < top_k) sh.cut[above] = mine;
  }
  __syncthreads();
  const int left = min(n, top_k);
  if (tid < left) sh.list[tid] = sh.cut[tid];
  if (tid == 0) sh.count = left;
  const Entry64 least = n >= top_k ? sh.cut[top_k - 1] : 0;
  __syncthreads();
  return least;
}

// grid: (cluster size, rows) in clusters along x
template <int VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
logprob_rows_kernel(const float* __restrict__ logits, const uint32_t* __restrict__ targets, float* __restrict__ logprob,
                    float* __restrict__ entropy, uint32_t* __restrict__ top_ids, float* __restrict__ top_logprobs, uint32_t vocab,
                    int top_k, size_t row_base) {
  constexpr int kWarps = THREADS / 32, kTile = THREADS * kLpPer;
  LogprobShared& sh = logprob_shared();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = blockIdx.x, ranks = gridDim.x;
  const size_t row = blockIdx.y;
  const float* x = logits + (row_base + row) * vocab;
  const uint32_t share = ((vocab + ranks - 1) / ranks + 3) / 4 * 4;
  const uint32_t begin = min(vocab, rank * share), end = min(vocab, begin + share);
  constexpr int kRuns = kLpPer / VEC;
  float next[kLpPer];
  auto index_of = [&](uint32_t tile, int i) { return tile + (i / VEC) * (THREADS * VEC) + tid * VEC + i % VEC; };
  auto load = [&](uint32_t tile) {
    if (VEC == 4 && tile + kTile <= end) {  // a whole tile: no checks, no defaults
      const float4* const from = reinterpret_cast<const float4*>(x + tile) + tid;
#pragma unroll
      for (int r = 0; r < kRuns; ++r) {
        const float4 y = __ldcs(from + r * THREADS);
        next[r * VEC] = y.x, next[r * VEC + 1 % VEC] = y.y, next[r * VEC + 2 % VEC] = y.z, next[r * VEC + 3 % VEC] = y.w;
      }
      return;
    }
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      const uint32_t at = index_of(tile, r * VEC);
      if constexpr (VEC == 4) {
        float4 y = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (at < end) y = __ldcs(reinterpret_cast<const float4*>(x + at));
        next[r * 4] = y.x, next[r * 4 + 1] = y.y, next[r * 4 + 2] = y.z, next[r * 4 + 3] = y.w;
      } else {
        next[r] = at < end ? __ldcs(x + at) : -INFINITY;
      }
    }
  };
  if (tid == 0) sh.count = 0;
  pdl_wait();  // (this kernel's start overlaps the end of the one before it)
  pdl_trigger();
  load(begin);
  float given = -INFINITY;  // the target's logit
  if (rank == 0 && tid == 0) {
    const uint32_t target = targets[row];
    if (target < vocab) given = x[target];
  }
  Sums mine{-INFINITY, 0.0f, 0.0f};
  Entry64 least = 0;             // a new entry has to exceed it
  float threshold = -INFINITY;  // its logit
  __syncthreads();
  for (uint32_t tile = begin; tile < end; tile += kTile) {
    float v[kLpPer];
#pragma unroll
    for (int i = 0; i < kLpPer; ++i) v[i] = next[i];
    if (tile + kTile < end) load(tile + kTile);
    const uint32_t held = min(end - tile, static_cast<uint32_t>(kTile));
    float most = v[0];
#pragma unroll
    for (int i = 1; i < kLpPer; ++i) most = fmaxf(most, v[i]);
    if (most > mine.top) mine = moved(mine, most);
    const float shift = shift_of(mine.top);
    float s[2] = {0.0f, 0.0f}, u[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kLpPer; ++i) {
      const float y = (v[i] - shift) * kLpLog2e, e = power2(y);
      s[i & 1] += e;
      u[i & 1] = fmaf(e, fmaxf(y, -1e30f), u[i & 1]);  // a masked logit is 0 * -1e30
    }
    mine.s += s[0] + s[1], mine.t += u[0] + u[1];
    if (top_k == 0) continue;
    if (tile == begin) {
      // The full[] warps whose every lane holds logits each give the per_warp-th largest of their lanes' maxima: at least
      // top_k logits are not below the least of these.
      const uint32_t full = held / (32 * VEC) < kWarps ? held / (32 * VEC) : kWarps;
      uint32_t bound = 0;
      if (full != 0) {
        const int per_warp = (top_k + static_cast<int>(full) - 1) / static_cast<int>(full);
        uint32_t key = order_of(most);
        for (int r = 0; r < per_warp; ++r) {
          bound = __reduce_max_sync(0xFFFFFFFFu, key);
          const uint32_t who = __ballot_sync(0xFFFFFFFFu, key == bound);
          if (lane == __ffs(who) - 1) key = 0;
        }
        if (lane == 0) sh.bound[warp] = bound;
        __syncthreads();
        bound = __reduce_min_sync(0xFFFFFFFFu, lane < static_cast<int>(full) ? sh.bound[lane] : 0xFFFFFFFFu);
      }
      least = bound == 0 ? 0 : static_cast<Entry64>(bound) << 32;
      threshold = bound == 0 ? -INFINITY : value_of(bound);
    }
    // The few logits that reach the threshold.  (A NaN is above nothing: it comes up only while there is no threshold.)
    int last_slot = -1;
    if (!(most < threshold)) {
      uint32_t above = 0;
#pragma unroll
      for (int i = 0; i < kLpPer; ++i)
        if (!(v[i] < threshold)) above |= 1u << i;
#pragma unroll 1
      for (; above != 0; above &= above - 1) {
        const int which = __ffs(above) - 1;
        float value = v[0];
#pragma unroll
        for (int i = 1; i < kLpPer; ++i) value = which == i ? v[i] : value;
        const uint32_t at = index_of(tile, which);
        const Entry64 e = entry_of(value, at);
        if (at >= end || e <= least) continue;
        last_slot = atomicAdd(&sh.count, 1);
        if (last_slot < kLpList) sh.list[last_slot] = e;
      }
    }
    const bool last = tile + kTile >= end;
    // (the bound will do for one more tile)
    const bool cut_now = last || (tile == begin && end - tile > 2 * kTile);
    if (!__syncthreads_or(last_slot >= kLpCut - 1) && !cut_now) continue;
    int n = sh.count;
    if (n > kLpList) {
      // The list overflowed.  Its first entries, fewer than kLpCut, are those of the tiles before; this tile's are found again:
      // bisection for the top_k-th largest entry of both.
      __syncthreads();
      const Entry64 kept = tid < kLpCut ? sh.list[tid] : 0;
      const uint32_t where = 0xFFFFFFFFu - static_cast<uint32_t>(kept);
      const bool before = tid < kLpCut && (where < tile || where >= tile + kTile);
      Entry64 lo = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const Entry64 trial = lo | (1ull << bit);
        if (tid == 0) sh.count = 0;
        __syncthreads();
        int mine_above = before && kept >= trial ? 1 : 0;
#pragma unroll
        for (int i = 0; i < kLpPer; ++i) {
          const uint32_t at = index_of(tile, i);
          const Entry64 e = entry_of(v[i], at);
          if (at < end && e > least && e >= trial) ++mine_above;
        }
        mine_above = __reduce_add_sync(0xFFFFFFFFu, mine_above);
        if (lane == 0 && mine_above != 0) atomicAdd(&sh.count, mine_above);
        __syncthreads();
        if (sh.count >= top_k) lo = trial;
        __syncthreads();
      }
      if (tid == 0) sh.count = 0;
      __syncthreads();
      if (before && kept >= lo) sh.list[atomicAdd(&sh.count, 1)] = kept;
#pragma unroll 1
      for (int i = 0; i < kLpPer; ++i) {
        const uint32_t at = index_of(tile, i);
        if (at >= end) continue;
        const Entry64 e = entry_of(x[at], at);
        if (e > least && e >= lo) sh.list[atomicAdd(&sh.count, 1)] = e;
      }
      __syncthreads();
      n = sh.count;
    }
    const Entry64 cut = cut_back<THREADS>(n, top_k);
    if (cut != 0) least = cut, threshold = value_of(static_cast<uint32_t>(cut >> 32));
  }

  // the threads' sums, then the CTAs'
  const Sums none{-INFINITY, 0.0f, 0.0f};
  mine = warp_joined(mine);
  if (lane == 0) sh.sums[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    mine = warp_joined(lane < kWarps ? sh.sums[lane] : none);
    if (lane == 0) sh.all = mine;
  }
  if (ranks > 1) {
    cluster_meet();
    if (rank != 0) {
      cluster_meet();  // this CTA's shared memory is read until here
      return;
    }
    if (warp == 0) {
      Sums other = none;
      if (lane < static_cast<int>(ranks)) {
        const uint32_t at = peer_at(shared_at(&sh.all), lane);
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.top) : "r"(at) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.s) : "r"(at + 4) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.t) : "r"(at + 8) : "memory");
      }
      other = warp_joined(other);
      if (lane == 0) sh.sums[0] = other;
    }
    // A thread an entry.  What is below the last of some CTA's full list is not among the row's top_k.
    Entry64 least_of = 0;
    if (lane < static_cast<int>(ranks) && top_k != 0) {
      uint32_t n;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n) : "r"(peer_at(shared_at(&sh.count), lane)) : "memory");
      asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(least_of) : "r"(peer_at(shared_at(&sh.list[top_k - 1]), lane)) : "memory");
      if (n < static_cast<uint32_t>(top_k)) least_of = 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Entry64 other = __shfl_xor_sync(0xFFFFFFFFu, least_of, o);
      least_of = other > least_of ? other : least_of;
    }
    static_assert(THREADS >= kLpCluster * kLpTop, "one entry a thread");
    Entry64 e = 0;
    if (tid < static_cast<int>(ranks) * top_k) {
      const uint32_t r = tid / top_k, i = tid % top_k;
      uint32_t n;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n) : "r"(peer_at(shared_at(&sh.count), r)) : "memory");
      asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(e) : "r"(peer_at(shared_at(&sh.list[i]), r)) : "memory");
      if (i >= n || e < least_of) e = 0;
    }
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // (and not waited for: nobody reads this CTA's memory)
    if (tid == 0) sh.all = sh.sums[0], sh.count = 0;
    __syncthreads();
    if (e != 0) sh.list[atomicAdd(&sh.count, 1)] = e;
    __syncthreads();
    if (top_k != 0) cut_back<THREADS>(sh.count, top_k);
    if (tid < top_k && tid >= sh.count) sh.list[tid] = tid;  // below every entry, and no two alike: the row has fewer logits
    __syncthreads();
  } else {
    if (tid < top_k && tid >= sh.count) sh.list[tid] = tid;
    __syncthreads();
  }
  const Sums all = sh.all;
  const bool nothing = all.s == 0.0f;  // every logit is -inf
  const float log_s = logf(all.s), top = shift_of(all.top);
  if (tid == 0) {
    logprob[row] = all.s != all.s ? all.s : nothing ? -INFINITY : (given - top) - log_s;
    entropy[row] = nothing ? 0.0f : log_s - all.t / all.s * kLpLn2;
  }
  if (tid < top_k) {
    const Entry64 e = sh.list[tid];
    const bool some = e >= kLpMost;  // (a place without an entry holds its number: the row has fewer logits than top_k)
    top_ids[row * top_k + tid] = some ? 0xFFFFFFFFu - static_cast<uint32_t>(e) : 0u;
    top_logprobs[row * top_k + tid] = all.s != all.s ? all.s : !some || nothing ? -INFINITY : (value_of(static_cast<uint32_t>(e >> 32)) - top) - log_s;
  }
}

// How many clusters of `ctas` CTAs (a power of two) the device runs at a time.
template <int VEC, int THREADS>
int logprob_resident(unsigned ctas) {
  static std::atomic<int> known[64][5];  // the number plus one; 0: not asked
  int dev = 0, log = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  while ((1u << log) < ctas) ++log;
  if (const int v = known[dev][log].load(std::memory_order_relaxed)) return v - 1;
  const auto kernel = logprob_rows_kernel<VEC, THREADS>;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = ctas;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = sizeof(LogprobShared);
  config.attrs = &cluster;
  config.numAttrs = 1;
  int clusters = 0;
  if ((ctas > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
      cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess) {
    cudaGetLastError();
    clusters = 0;
  }
  known[dev][log].store(clusters + 1, std::memory_order_relaxed);
  return clusters;
}

template <int VEC, int THREADS>
int launch_logprob(uint64_t rows, const float* logits, const uint32_t* targets, float* logprob, float* entropy, uint32_t* top_ids,
                   float* top_logprobs, uint64_t vocab, uint64_t top_k, uint64_t row_base, cudaStream_t st) {
  const auto kernel = logprob_rows_kernel<VEC, THREADS>;
  const unsigned ctas = logprob_ctas(rows, vocab, logprob_resident<VEC, THREADS>);
  const void* const out[4] = {logprob, entropy, top_ids, top_logprobs};
  const size_t out_bytes[4] = {rows * 4, rows * 4, rows * top_k * 4, rows * top_k * 4};
  const bool pdl = pdl_allowed_ranges(st, nullptr, nullptr, 0, out, out_bytes, 4);
  const cudaError_t e = launch_kernel_cluster(kernel, dim3(ctas, static_cast<unsigned>(rows)), dim3(THREADS), sizeof(LogprobShared), st, pdl, ctas, logits, targets, logprob,
                                              entropy, top_ids, top_logprobs, static_cast<uint32_t>(vocab), static_cast<int>(top_k), row_base);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return kDeviceError;
  }
  return check_launch();
}

}  // namespace

int logprob_rows(const float* logits, const uint32_t* targets, float* logprob, float* entropy, uint32_t* top_ids,
                                float* top_logprobs, uint64_t rows, uint64_t vocab, uint64_t top_k, uint64_t row_base, bool dry, cudaStream_t st) {
  if (!logits || !targets || !logprob || !entropy || rows == 0 || rows > 65535 || vocab == 0 || vocab > 0x7FFFFFFFull - kLpMost * kLpPer || top_k > kLpTop ||
      row_base > 0x7FFFFFFFull || (top_k != 0 && (!top_ids || !top_logprobs)))
    return kInvalidArgument;
  struct {
    const void* at;
    uint64_t bytes;
  } const in[2] = {{logits + row_base * vocab, rows * vocab * 4}, {targets, rows * 4}},
          out[4] = {{logprob, rows * 4}, {entropy, rows * 4}, {top_ids, rows * top_k * 4}, {top_logprobs, rows * top_k * 4}};
  auto meet = [](const auto& a, const auto& b) {
    const auto *x = static_cast<const unsigned char*>(a.at), *y = static_cast<const unsigned char*>(b.at);
    return a.bytes != 0 && x < y + b.bytes && y < x + a.bytes;
  };
  for (int i = 0; i < 4; ++i) {  // a row's results are written while others are read
    for (const auto& r : in)
      if (meet(out[i], r)) return kInvalidArgument;
    for (int j = 0; j < i; ++j)
      if (out[j].bytes != 0 && meet(out[i], out[j])) return kInvalidArgument;
  }
  if (dry) return kOk;
  const bool wide = vocab % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15u) == 0;
  return wide ? launch_logprob<4, kLpMost>(rows, logits, targets, logprob, entropy, top_ids, top_logprobs, vocab, top_k, row_base, st)
              : launch_logprob<1, kLpMost>(rows, logits, targets, logprob, entropy, top_ids, top_logprobs, vocab, top_k, row_base, st);
}

}  // namespace tsr

extern "C" int tsr_logprob_rows(const float* logits, const uint32_t* targets, float* logprob, float* entropy, uint32_t* top_ids,
                                float* top_logprobs, uint64_t rows, uint64_t vocab, uint64_t top_k, uint64_t row_base, void* stream) {
  return tsr::logprob_rows(logits, targets, logprob, entropy, top_ids, top_logprobs, rows, vocab, top_k, row_base, false,
                           static_cast<cudaStream_t>(stream));
}
