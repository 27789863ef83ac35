// Attention of the rows of a drafted tree over the key / value cache (ids "attention_tree", "attention_tree_q8" / "_q4" /
// "_fp8"): the causal attention of attention.cu (AttentionRef and its cache formats, src/core/numerics/attention.cpp:45-214 of the
// reference) for a speculative step that verifies several continuations at once.  The cache holds n past rows and behind them
// the tree's m rows; row i of the tree sees the past, its ancestors and itself, in that order; a window keeps the last of these.
// parents[i] is a row before i, or -1 for a child of the last past row; a row with any other value, or below one, is not used: it
// sees nothing, nobody sees it and its result is zero, so that a step of fixed size serves smaller trees.
#include <cuda_fp16.h>

#include "attention.cuh"
#include "codec.cuh"
#include "launch.h"
#include "pipeline.cuh"
#include "tessera_b200.h"

namespace tsr {

__device__ unsigned int g_tree_timeouts = 0;

namespace {

constexpr int kTreeRows = 256;  // of a tree at most
constexpr int kTreeWords = kTreeRows / 32;
constexpr int kTreeWarps = 8;

struct TreeParams {
  const float* q;
  const unsigned char *k, *v;
  const float *ks, *vs;
  const int* parents;
  float* out;
  int m, n, heads, kv_heads, window;
};

// What row i sees: bit j of `path` for row j of the tree, the past rows from `first` on (n: none).
struct TreeRow {
  uint32_t path[kTreeWords];
  int first;
};

// Walks up from row i; `parents` in shared memory.
__device__ __forceinline__ void tree_row(const int* parents, int i, int n, int window, TreeRow& row) {
#pragma unroll
  for (int w = 0; w < kTreeWords; ++w) row.path[w] = 0;
  int at = i, length = 0;
  while (at >= 0) {
    const int up = parents[at];
    if (up < -1 || up >= at) break;
    if (window == 0 || length < window) {
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) row.path[w] |= w == at >> 5 ? 1u << (at & 31) : 0u;
      ++length;
    }
    at = up;
  }
  row.first = window != 0 ? max(0, n - (window - length)) : 0;
  if (at != -1) {  // stopped at a row that is not used
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) row.path[w] = 0;
    row.first = n;
  }
}

// Cache element e of a row, as fp32.
template <int KV>
__device__ __forceinline__ float tree_element(const unsigned char* row, int e) {
  if (KV == kKvF32) return reinterpret_cast<const float*>(row)[e];
  if (KV == kKvF16) return __half2float(reinterpret_cast<const __half*>(row)[e]);
  if (KV == kKvFp8) return e4m3_to_float(row[e]);
  if (KV == kKvInt8) return static_cast<float>(static_cast<signed char>(row[e]));
  return static_cast<float>(static_cast<int>(static_cast<uint32_t>(row[e >> 1]) << (28 - 4 * (e & 1))) >> 28);
}

// grid: (heads, rows): a CTA a (row, head), a warp every kTreeWarps-th key, key by key in fp32.
template <int KV, int D>
__global__ void __launch_bounds__(kTreeWarps * 32) attention_tree_rows_kernel(const TreeParams p) {
  constexpr bool kScaled = KV >= kKvFp8;
  constexpr size_t kRowBytes = static_cast<size_t>(D) * kv_bits<KV>() / 8;
  __shared__ int parents_s[kTreeRows];
  __shared__ TreeRow row_s;
  __shared__ float acc_s[kTreeWarps][D], top_s[kTreeWarps], total_s[kTreeWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = blockIdx.x, i = blockIdx.y;
  for (int r = tid; r <= i; r += kTreeWarps * 32) parents_s[r] = p.parents[r];
  __syncthreads();
  if (tid == 0) {
    TreeRow row;
    tree_row(parents_s, i, p.n, p.window, row);
    row_s = row;
  }
  const size_t kv_at = static_cast<size_t>(h / (p.heads / p.kv_heads)) * kRowBytes, row_bytes = p.kv_heads * kRowBytes;
  const size_t at = (static_cast<size_t>(i) * p.heads + h) * D;
  float x[D / 32], acc[D / 32], top = kNoKey, total = 0.0f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) x[e] = p.q[at + e * 32 + lane] * (kLog2e / sqrtf(static_cast<float>(D))), acc[e] = 0.0f;
  __syncthreads();
  for (int j = row_s.first + warp; j < p.n + p.m; j += kTreeWarps) {
    if (j >= p.n && !(row_s.path[(j - p.n) >> 5] >> ((j - p.n) & 31) & 1u)) continue;
    const unsigned char *kr = p.k + j * row_bytes + kv_at, *vr = p.v + j * row_bytes + kv_at;
    float dot = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) dot = fmaf(x[e], tree_element<KV>(kr, e * 32 + lane), dot);
    const float sc = warp_sum(dot) * (kScaled ? p.ks[j] : 1.0f), now = fmaxf(top, sc);
    const float corr = exp2f(top - now), w = exp2f(sc - now), wv = w * (kScaled ? p.vs[j] : 1.0f);
    total = fmaf(total, corr, w);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(wv, tree_element<KV>(vr, e * 32 + lane), acc[e] * corr);
    top = now;
  }
#pragma unroll
  for (int e = 0; e < D / 32; ++e) acc_s[warp][e * 32 + lane] = acc[e];
  if (lane == 0) top_s[warp] = top, total_s[warp] = total;
  __syncthreads();
  top = top_s[0];
  for (int w = 1; w < kTreeWarps; ++w) top = fmaxf(top, top_s[w]);
  for (int e = tid; e < D; e += kTreeWarps * 32) {
    float num = 0.0f, den = 0.0f;
    for (int w = 0; w < kTreeWarps; ++w) {
      const float f = exp2f(top_s[w] - top);
      den = fmaf(f, total_s[w], den), num = fmaf(f, acc_s[w][e], num);
    }
    p.out[at + e] = den == 0.0f ? 0.0f : num / den;
  }
}

// ---- the tensor kernel ----
// A CTA takes 128 (tree row, head) pairs of one kv head and walks over its share of the keys in tiles of 64, on tcgen05 binary16
// MMAs with fp32 accumulators.  Cache elements are exact in binary16 (fp32 ones are two terms of a row scaled by a power of
// two), a query element or a softmax weight is two terms, as in attention_tile.cu.  Everything the MMAs take from the left
// lies in tensor memory: the queries' two terms for the whole call, a tile's weights over its scores.  Columns of tensor memory:
// queries 256, two tiles' scores or weights 64 each, and 128 for the outputs of a tile, which are read after every tile -- half
// of head_dim at a time -- and added to fp32 registers, so that what an accumulator cuts off does not add up over the keys.
//   warps 0-7   a thread a row (tensor memory lane), warps 0-3 keys 0-31 of a tile and outputs 0-63 of a half, 4-7 the rest
//   warps 8-10  keys and values: global memory -> binary16 in the operands' layout
//   warp 11     one thread issues the MMAs: a tile's outputs, then the scores of the tile after next over its weights
// Measured, 24 heads over 4 of 256 unless said: FP8, 16 rows behind 512 18.1 us; fp16, 61 rows behind 4000, 16 heads over 2 of 128
// 25 us; fp32, 8 rows behind 4096 36 us; FP8, 64 rows behind 32768 151 us (the MMAs' operations alone 31 us).
// A kernel key by key (as attention_tree_rows_kernel) took 61, 391, 981 and 10389 us.  What bounds: one tile costs 12 us
// (tensor memory, paths, two terms of the queries, the first scores) and the second launch, which joins the chunks, 3 to 4.  In a
// long row of tiles one takes 5900 clocks, of which the issuing thread spends 3300 on its 48 MMAs (2900 by their rates: 55 clocks
// with 64 columns, 70 with 128) and waits 730 for a half of the outputs to be read, both halves having one accumulator, and 1250
// for keys, weights, values and the last outputs (tensor pipe 42 % busy).  The fp32 cache: its loaders, which scale and split
// every row (9 us a tile; 12 with stores of a row at a time, 16 of them to the same banks).  Tiles of 64 keys, since two tiles'
// weights lie over their scores and columns of tensor memory are short.  Bytes by bulk copies of a key each 295 us for the long case, by tiled copies 152.
constexpr int kSoftThreads = 256, kLoadThreads = 96, kTcThreads = kSoftThreads + kLoadThreads + 32;
constexpr int kTcRows = 128, kTcKeys = 64;
constexpr uint32_t kColQ = 0, kColS = 256, kColO = 384;  // of tensor memory; tile t's scores and weights: kColS + 64 (t % 2)
constexpr int kScaleBufs = 4;
constexpr int kNoExponent = -1000;
constexpr int kUnused = 0x7FFFFFFF;
constexpr int kWideScales = 16;  // exponents apart
// Of the values' scales where weights are formed: a weight is at most 2^(14 - e), and a thread's 32 have a finite sum (a tile of zero
// values alone, as of a cache that has just been cleared, would give 2^124 each).
constexpr int kLowestExponent = -108;

struct TcParams {
  TreeParams t;
  float *pacc, *pmax, *psum;  // partials of chunks as in AttnParams; null: one chunk, the result itself
  int group, row_tiles, splits, tiles_per_split, first_key;
};

template <int KV, int D>
struct TcShape {
  static constexpr int kTerms = KV == kKvF32 ? 2 : 1;
  static constexpr int kBufs = KV == kKvF32 ? 1 : 2;  // of a tile's keys and of its values
  static constexpr int kTermBytes = kTcKeys * D * 2, kTileBytes = kTerms * kTermBytes;
  static constexpr int kRowBytes = D * kv_bits<KV>() / 8;
  static constexpr bool kRaw = KV != kKvF32 && KV != kKvF16;          // raw bytes pass through shared memory
  static constexpr int kBox = kRowBytes < 128 ? kRowBytes : 128;      // bytes of a key in a box of raw bytes; 128: swizzled
  static constexpr int kRawBytes = kRaw ? kTcKeys * kRowBytes : 0;
  static constexpr int kRuns = 768 / D, kPitch = kRowBytes + 16;      // fp32: runs of eight rows of a warp under way
  static constexpr int kRing = KV == kKvF32 ? kLoadThreads / 32 * kRuns * 8 * kPitch : 0;
  static constexpr int kHalves = D / 128;
  static constexpr uint32_t kGroupBytes = D / 8 * 128;                // eight keys
  static constexpr int kSmem = 1024 + 2 * kBufs * kTileBytes + 4 * kRawBytes + kRing;
};

// A parity wait tells a phase from the one before it, so no barrier may come two phases ahead of one who waits on it: scores and
// weights have a barrier for either buffer, since the softmax warps give away a tile's weights before the MMAs have taken the
// tile's before it; a phase of each other one is followed by the next only when everybody who waits for it has been heard of.
struct TcShared {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full, o_read, drained, raw_full[2][2];
  uint32_t tmem;
  uint32_t used[kTreeWords];               // rows of the tree that are used
  uint32_t path[kTreeRows][kTreeWords + 1];  // what each row sees of the tree
  int parents[kTreeRows];
  alignas(16) float scale[kScaleBufs][2][kTcKeys];  // keys', values'; read four at a time
  int range[kScaleBufs][kLoadThreads / 32][2];      // largest and smallest exponent of the values' scales
  float top[2][2][kTcRows];                         // [tile & 1][half of the keys][row]: largest score
  float weighed[2][kTcRows];                        // the same of score + log2 of the value's scale
  uint32_t q_most[2][kTcRows];
  float sum[2][kTcRows];
  int to[kTcRows], bad[kTcRows], any_bad;           // (bad: something that is not finite)
};

__device__ __forceinline__ void tc_alloc(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_free(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}
// D (tensor memory) [+]= A (tensor memory) B (shared memory)
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{.reg .pred p; setp.ne.b32 p, %4, 0; "
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_load32(uint32_t at, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"  // (one statement: the registers are not the results before the wait)
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tc_store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tc_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void to_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Operand B without swizzle: core matrices of eight rows of 16 bytes; `lead` and `stride`: bytes between core matrices.  Keys
// (elements along head_dim contract): lead along head_dim, stride along the keys.  Values (keys contract, head_dim runs within a
// core matrix' rows): lead along the keys, stride along head_dim.
__device__ __forceinline__ uint64_t tc_operand(uint32_t addr, uint32_t lead, uint32_t stride) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | static_cast<uint64_t>((lead >> 4) & 0x3FFF) << 16 |
         static_cast<uint64_t>((stride >> 4) & 0x3FFF) << 32 | 1ull << 46;
}
// fp32 results of binary16 operands, 128 rows, n columns; turned: B's rows are the contracted index
__device__ __forceinline__ uint32_t tc_shape(uint32_t n, bool turned) {
  return (1u << 4) | (turned ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((kTcRows >> 4) << 24);
}

__device__ __forceinline__ uint32_t tree_pack(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ void tree_split(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = tree_pack(h);
  lo = tree_pack(__floats2half2_rn(x - f.x, y - f.y));
}
// The same of the products x u and y v, with one rounding.
__device__ __forceinline__ void tree_split_product(float x, float y, float u, float v, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x * u, y * v);
  const float2 f = __half22float2(h);
  hi = tree_pack(h);
  lo = tree_pack(__floats2half2_rn(fmaf(x, u, -f.x), fmaf(y, v, -f.y)));
}
// Bits [a, b) of a word, a and b anything.
__device__ __forceinline__ uint32_t bits_between(int a, int b) {
  a = max(a, 0), b = min(b, 32);
  return a >= b ? 0u : (0xFFFFFFFFu >> (32 - (b - a))) << a;
}

// Four cache elements of a 32-bit word (eight of 4 bits) as binary16.
template <int KV>
__device__ __forceinline__ void tree_expand(uint32_t w, uint32_t (&h)[KV == kKvInt4 ? 4 : 2]) {
  auto minus = [](uint32_t a, uint32_t b) { return tree_pack(__hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b))); };
  if constexpr (KV == kKvFp8) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      h[i] = tree_pack(__half2(__half2_raw(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((w >> (16 * i)) & 0xFFFFu), __NV_E4M3))));
  } else if constexpr (KV == kKvInt8) {  // 1024 + (b + 128) - 1152, exact
    const uint32_t u = w ^ 0x80808080u;
    h[0] = minus(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u);
    h[1] = minus(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u);
  } else {  // two's-complement nibbles, element 2i low: 1024 + (v + 8) - 1032
    const uint32_t t = w ^ 0x88888888u, even = t & 0x0F0F0F0Fu, odd = (t >> 4) & 0x0F0F0F0Fu;
    const uint32_t x = __byte_perm(even, odd, 0x5140), y = __byte_perm(even, odd, 0x7362);
    h[0] = minus(__byte_perm(x, 0x64646464u, 0x4140), 0x64086408u);
    h[1] = minus(__byte_perm(x, 0x64646464u, 0x4342), 0x64086408u);
    h[2] = minus(__byte_perm(y, 0x64646464u, 0x4140), 0x64086408u);
    h[3] = minus(__byte_perm(y, 0x64646464u, 0x4342), 0x64086408u);
  }
}
// exp2 without the slow path for results below the normal numbers, which are 0
__device__ __forceinline__ float tree_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^e, e in [-126, 127]
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// Every row's path: pointer doubling, a thread a row of the tree; then the window.  All threads of the CTA.
__device__ __forceinline__ void tree_paths(TcShared& sh, int m, int window) {
  const int i = threadIdx.x;
  int up = -2;
  uint32_t mine[kTreeWords];
  if (i < m) {
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) sh.path[i][w] = mine[w] = w == i >> 5 ? 1u << (i & 31) : 0u;
    sh.path[i][kTreeWords] = 0;
    const int p = sh.parents[i];
    up = p < -1 || p >= i ? -2 : p;
  }
  __syncthreads();
  if (i < m) sh.parents[i] = up;
  while (__syncthreads_or(up >= 0)) {
    int next = up;
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) mine[w] |= sh.path[up][w];
      next = sh.parents[up];
    }
    __syncthreads();
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) sh.path[i][w] = mine[w];
      sh.parents[i] = next;
    }
    up = next;
  }
  if (i < m) {
    int length = 0;
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) {
      if (up != -1) mine[w] = 0;
      length += __popc(mine[w]);
    }
    if (length != 0) atomicOr(&sh.used[i >> 5], 1u << (i & 31));
    if (window != 0) {  // the nearest ancestors have the highest bits
      int over = length - window;
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) {
        const int here = __popc(mine[w]);
        if (over >= here) mine[w] = 0;
        else
          for (int x = 0; x < over; ++x) mine[w] &= mine[w] - 1;
        over -= here;
        if (over < 0) over = 0;
      }
    }
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) sh.path[i][w] = mine[w];
  }
  __syncthreads();
}

// Pair r of (tree row, head) over keys [c0, c1), by a warp and key by key in fp32: where something is not finite.
template <int KV, int D>
__device__ __noinline__ void tree_scalar_row(const TcParams& p, const TcShared& sh, int kv, int r, int c0, int c1, int split) {
  constexpr bool kScaled = KV >= kKvFp8;
  constexpr size_t kRowBytes = static_cast<size_t>(D) * kv_bits<KV>() / 8;
  const int lane = threadIdx.x & 31, n = p.t.n;
  const size_t row_bytes = p.t.kv_heads * kRowBytes;
  const int i = r / p.group, h = kv * p.group + r - i * p.group;
  int length = 0;
  for (int w = 0; w < kTreeWords; ++w) length += __popc(sh.path[i][w]);
  const int first = length == 0 ? n : p.t.window != 0 ? max(0, n - (p.t.window - length)) : 0;
  const size_t at = (static_cast<size_t>(i) * p.t.heads + h) * D;
  float x[D / 32], acc[D / 32], top = kNoKey, total = 0.0f;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) x[e] = p.t.q[at + e * 32 + lane] * (kLog2e / sqrtf(static_cast<float>(D))), acc[e] = 0.0f;
  for (int j = max(first, c0); j < c1; ++j) {
    if (j >= n && !(sh.path[i][(j - n) >> 5] >> ((j - n) & 31) & 1u)) continue;
    const unsigned char *kr = p.t.k + j * row_bytes + kv * kRowBytes, *vr = p.t.v + j * row_bytes + kv * kRowBytes;
    float dot = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) dot = fmaf(x[e], tree_element<KV>(kr, e * 32 + lane), dot);
    const float sc = warp_sum(dot) * (kScaled ? p.t.ks[j] : 1.0f), now = fmaxf(top, sc);
    const float corr = exp2f(top - now), w = exp2f(sc - now), wv = w * (kScaled ? p.t.vs[j] : 1.0f);
    total = fmaf(total, corr, w);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(wv, tree_element<KV>(vr, e * 32 + lane), acc[e] * corr);
    top = now;
  }
  const size_t part = (static_cast<size_t>(i) * p.t.heads + h) * p.splits + split;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) {
    if (p.pacc != nullptr) p.pacc[part * D + e * 32 + lane] = acc[e];
    else p.t.out[at + e * 32 + lane] = total == 0.0f ? 0.0f : acc[e] / total;
  }
  if (p.pacc != nullptr && lane == 0) p.pmax[part] = top, p.psum[part] = total;
}

// The loading warps' part: tile t of the keys (VALUES: of the values) into its operand buffer, raw bytes from `raw`.
template <int KV, int D>
struct TcLoader {
  using S = TcShape<KV, D>;
  const TcParams& p;
  TcShared& sh;
  const CUtensorMap *k_map, *v_map;
  int kv, c0, c1, tiles;

  __device__ __forceinline__ const unsigned char* base(bool values) const {
    return (values ? p.t.v : p.t.k) + static_cast<size_t>(kv) * S::kRowBytes;
  }
  __device__ __forceinline__ size_t pitch() const { return static_cast<size_t>(p.t.kv_heads) * S::kRowBytes; }
  // whether key j is a row of the tree that nobody sees: read as zeros
  __device__ __forceinline__ bool unseen(int j) const {
    const int i = j - p.t.n;
    return i >= 0 && !(sh.used[i >> 5] >> (i & 31) & 1u);
  }
  // A warp takes 16-byte pieces of a tile four neighbours of eight keys at a time, so that its stores to the operand's layout are
  // conflict-free and it reads 64 bytes of a key side by side.  Piece `it` of a thread:
  static constexpr int kTimes = kTcKeys * S::kRowBytes / 512;
  static __device__ __forceinline__ int key_of(int it, int lane) { return (it & 7) * 8 + (lane & 7); }
  static __device__ __forceinline__ int piece_of(int it, int lane) { return (it >> 3) * 4 + (lane >> 3); }
  static __device__ __forceinline__ uint32_t operand_at(int it, int lane, int c) { return (it & 7) * S::kGroupBytes + (lane & 7) * 16 + c * 128; }
  // Raw bytes, by one thread (rows beyond the cache's last come as zeros).
  __device__ __forceinline__ void fetch_raw(bool values, int t, unsigned char* raw) const {
    if (t >= tiles) return;
    uint64_t* bar = &sh.raw_full[t & 1][values ? 1 : 0];
    mbar_expect_tx(bar, S::kRawBytes);
#pragma unroll
    for (int b = 0; b < S::kRowBytes / S::kBox; ++b)
      tma_load_2d(raw + b * kTcKeys * S::kBox, values ? v_map : k_map, kv * S::kRowBytes + b * S::kBox, c0 + t * kTcKeys, bar);
  }
  // fp16: straight into the operand's layout
  __device__ __forceinline__ void fetch(bool values, int t, unsigned char* dst, int tid) const {
    if (t < tiles) {
      const int warp = tid >> 5, lane = tid & 31, j0 = c0 + t * kTcKeys;
      const unsigned char* src = base(values) + static_cast<size_t>(j0) * pitch();
      const int last = c1 - 1 - j0;
#pragma unroll 4
      for (int it = warp; it < kTimes; it += kLoadThreads / 32) {
        const int c = piece_of(it, lane);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst) + operand_at(it, lane, c)),
                     "l"(src + static_cast<size_t>(min(key_of(it, lane), last)) * pitch() + c * 16)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Rows of the tree that nobody sees are zeros: what they hold may be anything.
  __device__ __forceinline__ void convert(int t, const unsigned char* raw, unsigned char* dst, int tid) const {
    const int warp = tid >> 5, lane = tid & 31, j0 = c0 + t * kTcKeys;
    const bool past = j0 + kTcKeys <= p.t.n;
    if constexpr (KV == kKvF16) {
      if (past) return;
      for (int it = warp; it < kTimes; it += kLoadThreads / 32)
        if (unseen(min(j0 + key_of(it, lane), c1 - 1)))
          *reinterpret_cast<uint4*>(dst + operand_at(it, lane, piece_of(it, lane))) = make_uint4(0u, 0u, 0u, 0u);
    } else {
      constexpr int kWords = KV == kKvInt4 ? 4 : 2;  // of 16 bytes of operand a piece becomes
      constexpr int kRun = KV == kKvInt4 ? 2 : 4;    // pieces in flight
      auto raw_at = [&](int it) {  // piece c of a key lies at c ^ (key & 7) of its 128 bytes
        const int c = piece_of(it, lane), key = key_of(it, lane);
        return S::kBox == 128 ? raw + (c >> 3) * (kTcKeys * 128) + key * 128 + (((c ^ key) & 7) << 4) : raw + key * S::kBox + c * 16;
      };
#pragma unroll 1
      for (int i0 = warp; i0 < kTimes; i0 += kRun * (kLoadThreads / 32)) {
        uint4 y[kRun];
#pragma unroll
        for (int u = 0; u < kRun; ++u) {
          const int it = min(i0 + u * (kLoadThreads / 32), kTimes - 1);
          y[u] = *reinterpret_cast<const uint4*>(raw_at(it));
          if (!past && unseen(min(j0 + key_of(it, lane), c1 - 1))) y[u] = make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < kRun; ++u) {
          const int it = i0 + u * (kLoadThreads / 32);
          const uint32_t w[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
          uint32_t h[4][KV == kKvInt4 ? 4 : 2];
#pragma unroll
          for (int i = 0; i < 4; ++i) tree_expand<KV>(w[i], h[i]);
          unsigned char* at = dst + operand_at(it, lane, piece_of(it, lane) * kWords);
          if (it < kTimes) {
#pragma unroll
            for (int o = 0; o < kWords; ++o)
              *reinterpret_cast<uint4*>(at + o * 128) = KV == kKvInt4 ? make_uint4(h[o][0], h[o][1], h[o][2 % kWords], h[o][3 % kWords])
                                                                     : make_uint4(h[2 * (o & 1)][0], h[2 * (o & 1)][1], h[2 * (o & 1) + 1][0], h[2 * (o & 1) + 1][1]);
          }
        }
      }
    }
  }
  // fp32 rows pass through a warp's own ring, eight keys (a group of the operand's layout) a run.  Of a tile's eight runs of keys
  // warp w takes w, w + 3, ..., of its eight runs of values (w + 2) % 3 and so on: five, six and five.
  __device__ __forceinline__ int runs_of_keys(int warp) const { return warp == 2 ? 2 : 3; }
  __device__ __forceinline__ int runs_of_tile(int warp) const { return warp == 1 ? 6 : 5; }
  __device__ __forceinline__ unsigned char* run_at(int s, unsigned char* ring, int warp) const {
    return ring + (warp * S::kRuns + s % S::kRuns) * 8 * S::kPitch;
  }
  __device__ __forceinline__ void ask_rows(int s, unsigned char* ring, int tid) const {
    static_assert(kLoadThreads == 96, "three warps");
    const int lane = tid & 31, warp = tid >> 5, of_tile = runs_of_tile(warp), of_keys = runs_of_keys(warp);
    const int t = s / of_tile, x = s - t * of_tile;
    if (t < tiles) {
      const bool values = x >= of_keys;
      const int group = values ? (warp + 2) % 3 + 3 * (x - of_keys) : warp + 3 * x;
      unsigned char* dst = run_at(s, ring, warp) + lane * 16;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = min(c0 + t * kTcKeys + group * 8 + u, c1 - 1);
        const unsigned char* src = base(values) + j * pitch() + lane * 16;
#pragma unroll
        for (int i = 0; i < D / 128; ++i)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst) + u * S::kPitch + i * 512), "l"(src + i * 512) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Each row scaled by a power of two to [2^13, 2^14), two terms.  Row by row for its largest element; then a lane has a row,
  // eight elements at a time, so that the ring's rows (16 bytes apart in their banks) and the operand's are free of conflicts.
  __device__ __forceinline__ void split_rows(bool values, int t, unsigned char* ring, unsigned char* dst, int tid) const {
    const int lane = tid & 31, warp = tid >> 5, of_keys = runs_of_keys(warp), key = lane & 7;
    const int runs = values ? runs_of_tile(warp) - of_keys : of_keys;
    int high = kNoExponent, low = -kNoExponent;
#pragma unroll 1
    for (int b = 0; b < runs; ++b) {
      const int s = t * runs_of_tile(warp) + (values ? of_keys : 0) + b, group = (values ? (warp + 2) % 3 : warp) + 3 * b;
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kRuns - 1) : "memory");
      __syncwarp();
      const unsigned char* const rows = run_at(s, ring, warp);
      uint32_t most[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        most[u] = 0;
#pragma unroll
        for (int i = 0; i < D / 128; ++i) {
          const uint4 y = *reinterpret_cast<const uint4*>(rows + u * S::kPitch + i * 512 + lane * 16);
          most[u] = max(max(most[u], max(y.x & 0x7FFFFFFFu, y.y & 0x7FFFFFFFu)), max(y.z & 0x7FFFFFFFu, y.w & 0x7FFFFFFFu));
        }
      }
      uint32_t mine = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint32_t all = __reduce_max_sync(0xFFFFFFFFu, most[u]);
        mine = key == u ? all : mine;
      }
      const int j = min(c0 + t * kTcKeys + group * 8 + key, c1 - 1);
      const bool zero = j >= p.t.n && unseen(j);
      if (zero) mine = 0;
      // (a row of zeros has the smallest scale: its weight, which is relative to the other rows' scales, may be large)
      const int e = mine == 0 ? -126 : max(-110, min(114, static_cast<int>(mine >> 23) - 127 - 13));
      const float up = power_of_two(-e);
      if (mine != 0) high = max(high, e), low = min(low, e);
      if (lane < 8) sh.scale[t % kScaleBufs][values ? 1 : 0][group * 8 + key] = power_of_two(e);
#pragma unroll 4
      for (int it = 0; it < D / 32; ++it) {
        const int c = it * 4 + (lane >> 3);
        float4 x = *reinterpret_cast<const float4*>(rows + key * S::kPitch + c * 32), y = *reinterpret_cast<const float4*>(rows + key * S::kPitch + c * 32 + 16);
        if (zero) x = y = make_float4(0.f, 0.f, 0.f, 0.f);
        uint4 hi, lo;
        tree_split(x.x * up, x.y * up, hi.x, lo.x);
        tree_split(x.z * up, x.w * up, hi.y, lo.y);
        tree_split(y.x * up, y.y * up, hi.z, lo.z);
        tree_split(y.z * up, y.w * up, hi.w, lo.w);
        unsigned char* const at = dst + group * S::kGroupBytes + key * 16 + c * 128;
        *reinterpret_cast<uint4*>(at) = hi;
        *reinterpret_cast<uint4*>(at + S::kTermBytes) = lo;
      }
      __syncwarp();  // the run's place is free
      ask_rows(s + S::kRuns, ring, tid);
    }
    if (!values) return;
    high = __reduce_max_sync(0xFFFFFFFFu, high), low = __reduce_min_sync(0xFFFFFFFFu, low);
    if (lane == 0) sh.range[t % kScaleBufs][warp][0] = high, sh.range[t % kScaleBufs][warp][1] = low;
  }
  // a quantised tile's scales: asked for a tile ahead, put where the weights are formed
  __device__ __forceinline__ void next_scales(int t, int tid, float& k, float& v) const {
    k = v = 0.0f;
    if (tid >= kTcKeys || t >= tiles) return;
    const int j = min(c0 + t * kTcKeys + tid, c1 - 1);
    if (!unseen(j)) k = __ldg(p.t.ks + j), v = __ldg(p.t.vs + j);
  }
  __device__ __forceinline__ void put_scales(int t, int tid, float k, float v) const {
    const uint32_t bits = __float_as_uint(v) & 0x7FFFFFFFu;
    const int e = static_cast<int>(bits >> 23) - 126;  // |v| < 2^e
    const int high = __reduce_max_sync(0xFFFFFFFFu, bits != 0 ? e : kNoExponent), low = __reduce_min_sync(0xFFFFFFFFu, bits != 0 ? e : -kNoExponent);
    if ((tid & 31) == 0) sh.range[t % kScaleBufs][tid >> 5][0] = high, sh.range[t % kScaleBufs][tid >> 5][1] = low;
    if (tid < kTcKeys) sh.scale[t % kScaleBufs][0][tid] = k, sh.scale[t % kScaleBufs][1][tid] = v;
  }
};

template <int KV, int D>
__global__ void __launch_bounds__(kTcThreads, 1) attention_tree_tc_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                                                                         const TcParams p) {
  using S = TcShape<KV, D>;
  constexpr bool kScaled = KV != kKvF16;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(16) TcShared sh;
  unsigned char* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* const k_s = smem;                               // [kBufs][terms][64 keys][D]
  unsigned char* const v_s = k_s + S::kBufs * S::kTileBytes;
  unsigned char* const raw_s = v_s + S::kBufs * S::kTileBytes;  // [2][keys, values]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kv = blockIdx.x % p.t.kv_heads, row0 = static_cast<int>(blockIdx.x) / p.t.kv_heads * kTcRows, split = blockIdx.y;
  const int rows = min(kTcRows, p.t.m * p.group - row0), n = p.t.n;
  const int c0 = p.first_key + split * p.tiles_per_split * kTcKeys;
  const int c1 = static_cast<int>(min(static_cast<long long>(n) + p.t.m, static_cast<long long>(c0) + static_cast<long long>(p.tiles_per_split) * kTcKeys));
  const int tiles = (c1 - c0 + kTcKeys - 1) / kTcKeys;
  const bool loading = warp >= kSoftThreads / 32 && warp < (kSoftThreads + kLoadThreads) / 32;
  const int load_tid = tid - kSoftThreads;
  TcLoader<KV, D> loader{p, sh, &k_map, &v_map, kv, c0, c1, tiles};

  if (tid < kTreeWords) sh.used[tid] = 0;
  if (tid < kTcRows) sh.bad[tid] = 0;
  if (tid == 0) {
    sh.any_bad = 0;
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh.k_full[b], kLoadThreads / 32), mbar_init(&sh.v_full[b], kLoadThreads / 32);
      mbar_init(&sh.k_empty[b], 1), mbar_init(&sh.v_empty[b], 1);
    }
    mbar_init(&sh.s_full[0], 1), mbar_init(&sh.s_full[1], 1), mbar_init(&sh.o_full, 1), mbar_init(&sh.drained, 1);
    for (int b = 0; b < 4; ++b) mbar_init(&sh.raw_full[b >> 1][b & 1], 1);
    mbar_init(&sh.p_full[0], kSoftThreads / 32), mbar_init(&sh.p_full[1], kSoftThreads / 32), mbar_init(&sh.o_read, kSoftThreads / 32);
    mbar_fence_init();
  }
  if (warp == kTcThreads / 32 - 1) tc_alloc(&sh.tmem);
  // So far this kernel's start overlaps the end of the one before it.  (It lets no other start under its own end: the registers are
  // taken, and CTAs that wait elsewhere cost the long case 5 of 151 us.)
  pdl_wait();
  if (tid < p.t.m) sh.parents[tid] = p.t.parents[tid];
  // Queries, to begin with as they are, in the operands' buffers: 16-byte piece c of a row at c ^ (row & 7).
  if (warp < kSoftThreads / 32) {
    constexpr int kRowsOf = kTcRows / (kSoftThreads / 32);
    const int r0 = warp * kRowsOf;
    int i = (row0 + r0) / p.group, g = (row0 + r0) - i * p.group;
#pragma unroll 4
    for (int u = 0; u < kRowsOf; ++u) {
      const int r = r0 + u;
      const float* src = p.t.q + (static_cast<size_t>(i) * p.t.heads + kv * p.group + g) * D + lane * 4;
      if (r < rows) {
#pragma unroll
        for (int k = 0; k < D / 128; ++k)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem) + r * (D * 4) + (((k * 32 + lane) ^ (r & 7)) << 4)), "l"(src + k * 128) : "memory");
      }
      if (++g == p.group) g = 0, ++i;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (S::kRaw && load_tid == 0)  // raw bytes of the first tiles
    for (int t = 0; t < 4; ++t) loader.fetch_raw((t & 1) != 0, t >> 1, raw_s + t * S::kRawBytes);
  if (KV == kKvF32 && loading)
    for (int s = 0; s < S::kRuns; ++s) loader.ask_rows(s, raw_s, load_tid);
  tree_paths(sh, p.t.m, p.t.window);
  const uint32_t tmem = sh.tmem;
  // a thread's row
  const int half = warp >> 2, row = (warp & 3) * 32 + lane;  // (of warps 0-7)
  const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
  const int tree_i = row < rows ? (row0 + row) / p.group : 0;
  float row_f = 0.0f;
  int first = kUnused;
  if (warp < kSoftThreads / 32) {
    // a thread half a row: scaled by a power of two to [2^13, 2^14), two terms to tensor memory
    if (row < rows) {
      int length = 0;
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) length += __popc(sh.path[tree_i][w]);
      if (length != 0) first = p.t.window != 0 ? max(0, n - (p.t.window - length)) : 0;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const unsigned char* src = smem + row * (D * 4);
    const int c0q = half * (D / 8);
    uint32_t most = 0;
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {
      const uint4 y = *reinterpret_cast<const uint4*>(src + (((c0q + c) ^ (row & 7)) << 4));
      most = max(max(most, max(y.x & 0x7FFFFFFFu, y.y & 0x7FFFFFFFu)), max(y.z & 0x7FFFFFFFu, y.w & 0x7FFFFFFFu));
    }
    sh.q_most[half][row] = most;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    most = first == kUnused ? 0u : max(most, sh.q_most[half ^ 1][row]);
    const int e = most == 0 ? 0 : max(-110, min(114, static_cast<int>(most >> 23) - 127 - 13));
    const float up = power_of_two(-e);
    row_f = power_of_two(e) * (kLog2e / sqrtf(static_cast<float>(D)));
#pragma unroll 1
    for (int i = 0; i < D / 64; ++i) {
      uint32_t hi[16], lo[16];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float4 y = *reinterpret_cast<const float4*>(src + (((c0q + i * 8 + u) ^ (row & 7)) << 4));
        tree_split(y.x * up, y.y * up, hi[2 * u], lo[2 * u]);
        tree_split(y.z * up, y.w * up, hi[2 * u + 1], lo[2 * u + 1]);
        if (first == kUnused) hi[2 * u] = hi[2 * u + 1] = lo[2 * u] = lo[2 * u + 1] = 0;  // (what the buffer holds may be anything)
      }
      tc_store16(tmem + lanes + kColQ + half * (D / 4) + i * 16, hi);
      tc_store16(tmem + lanes + kColQ + D / 2 + half * (D / 4) + i * 16, lo);
    }
    tc_store_wait();
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (KV == kKvF16 && loading) {
    loader.fetch(false, 0, k_s, load_tid), loader.fetch(true, 0, v_s, load_tid);
    loader.fetch(false, 1, k_s + S::kTileBytes, load_tid), loader.fetch(true, 1, v_s + S::kTileBytes, load_tid);
  }

  // the softmax warps hold 128 sums a thread where head_dim is 256: 256 * 208 + 128 * 88 registers, the launch's 384 * 168
  if (D == 256) {
    if (warp < kSoftThreads / 32) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  }
  // Once a wait has given up (counted, and told to the host) a thread waits no more and goes on to the end of its loop, so that
  // everybody comes to the barriers.
  bool ok = true;
  auto wait = [&](uint64_t* bar, int phase) {
    if (ok) ok = mbar_wait(bar, phase & 1, &g_tree_timeouts);
  };
  if (warp < kSoftThreads / 32) {
    float o[S::kHalves][64];
#pragma unroll
    for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
      for (int c = 0; c < 64; ++c) o[h][c] = 0.0f;
    float mx = kNoKey, sum = 0.0f, unit = 0.0f;  // mx: a whole number, so that everything is rescaled by powers of two
    // half of a tile's outputs, relative to the maximum when its weights were formed
    auto take = [&](float (&acc)[64]) {
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        uint32_t y[32];
        tc_load32(tmem + lanes + kColO + half * 64 + part * 32, y);
#pragma unroll
        for (int c = 0; c < 32; ++c) acc[part * 32 + c] = fmaf(__uint_as_float(y[c]), unit, acc[part * 32 + c]);
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.o_read);
    };
    auto take_tile = [&](int t) {
#pragma unroll
      for (int h = 0; h < S::kHalves; ++h) {
        wait(&sh.o_full, S::kHalves * t + h);
        tc_after();
        take(o[h]);
      }
    };
    for (int t = 0; t < tiles; ++t) {
      const uint32_t s_at = tmem + lanes + kColS + (t & 1) * 64;
      wait(&sh.s_full[t & 1], t >> 1);
      tc_after();
      uint32_t s[32];
      tc_load32(s_at + half * 32, s);
      if (S::kBufs == 1) {  // a tile's values, whose scales come with them, wait for the products of the tile before
        if (t > 0) take_tile(t - 1);
        wait(&sh.v_full[0], t);
      }
      // which of the 32 keys the row sees
      const int j0 = c0 + t * kTcKeys + half * 32;
      uint32_t see = 0xFFFFFFFFu;
      if (j0 < first || j0 + 32 > n) {
        see = first == kUnused ? 0u : bits_between(first - j0, n - j0);
        const int off = j0 - n;
        if (off > -32 && row < rows) {
          const uint32_t* path = sh.path[tree_i];
          if (off < 0) see |= path[0] << -off;
          else if (off < kTreeRows) see |= __funnelshift_r(path[off >> 5], path[(off >> 5) + 1], off & 31);
        }
      }
      const float* ks = sh.scale[t % kScaleBufs][0] + half * 32;
      const float* vs = sh.scale[t % kScaleBufs][1] + half * 32;
      // scores over row_f, -infinity for a key that the row does not see
      if constexpr (kScaled) {
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 f = *reinterpret_cast<const float4*>(ks + c);
          const float y[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) s[c + u] = __float_as_uint(__uint_as_float(s[c + u]) * y[u]);
        }
      }
      if (__any_sync(0xFFFFFFFFu, see != 0xFFFFFFFFu)) {
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if (!(see >> c & 1u)) s[c] = 0xFF800000u;
      }
      float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 32; ++c) tops[c & 3] = fmaxf(tops[c & 3], __uint_as_float(s[c]));
      float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      sh.top[t & 1][half][row] = top;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      top = fmaxf(top, sh.top[t & 1][half ^ 1][row]);
      const float now = fmaxf(mx, ceilf(top * row_f));
      const float corr = tree_exp2(mx - now);  // 1 while the row has had no key (kNoKey - kNoKey)
      mx = now;
      // The power of two that takes weights (at most 1) times their values' scales to at most 2^14.  What binary16 cuts off is 2^-39
      // of that, so one for all keys will do while their scales lie within 2^16; else each row's is made for its largest.
      int e = 0;
      if (kScaled) {
        const int(*range)[2] = sh.range[t % kScaleBufs];
        int high = range[0][0], low = range[0][1];
#pragma unroll
        for (int w = 1; w < kLoadThreads / 32; ++w) high = max(high, range[w][0]), low = min(low, range[w][1]);
        e = high;
        if (high - low > kWideScales) {
          float most = kNoKey;
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const uint32_t bits = __float_as_uint(vs[c]) & 0x7FFFFFFFu;
            if (bits != 0) most = fmaxf(most, fmaf(__uint_as_float(s[c]), row_f, -now) + static_cast<float>(static_cast<int>(bits >> 23) - 126));
          }
          asm volatile("bar.sync 1, 256;" ::: "memory");  // (the tile before may still be reading)
          sh.weighed[half][row] = most;
          asm volatile("bar.sync 1, 256;" ::: "memory");
          most = fmaxf(most, sh.weighed[half ^ 1][row]);
          e = static_cast<int>(fminf(fmaxf(ceilf(most), -110.0f), 110.0f));
        }
        e = max(kLowestExponent, min(110, e));
      }
      const float shift = now == kNoKey ? 0.0f : static_cast<float>(14 - e) - now;
      uint32_t hi[16], lo[16];
      float part[2] = {0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 f = kScaled ? *reinterpret_cast<const float4*>(vs + c) : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        const float y[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int u = 0; u < 4; u += 2) {
          float w[2];
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            w[v] = tree_exp2(fmaf(__uint_as_float(s[c + u + v]), row_f, shift));
            part[v] += w[v];
          }
          if (kScaled) tree_split_product(w[0], w[1], y[u], y[u + 1], hi[(c + u) / 2], lo[(c + u) / 2]);
          else tree_split(w[0], w[1], hi[(c + u) / 2], lo[(c + u) / 2]);
        }
      }
      const float next_unit = power_of_two(e - 14);
      sum = fmaf(part[0] + part[1], next_unit, sum * corr);
      // the weights over the scores (the other half's threads have read theirs: they were at the barrier above)
      tc_store16(s_at + half * 16, hi);
      tc_store16(s_at + 32 + half * 16, lo);
      tc_store_wait();
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[t & 1]);
      if (S::kBufs == 2 && t > 0) take_tile(t - 1);
      if (__any_sync(0xFFFFFFFFu, corr != 1.0f)) {
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
          for (int c = 0; c < 64; ++c) o[h][c] *= corr;
      }
      unit = next_unit;
    }
    take_tile(tiles - 1);
    // Through shared memory (the operands' buffers are free), so that a warp writes whole rows.  A NaN or an infinity among a
    // row's operands has made its sums so (that of a key which it does not see as well: its weight of 0 does not mask it).
    float all = sum;
#pragma unroll
    for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        all = fmaf((o[h][c] + o[h][c + 1]) + (o[h][c + 2] + o[h][c + 3]), 0.0f, all);
        *reinterpret_cast<float4*>(smem + row * (D * 4) + (((h * 32 + half * 16 + c / 4) ^ (row & 7)) << 4)) =
            make_float4(o[h][c], o[h][c + 1], o[h][c + 2], o[h][c + 3]);
      }
    sh.sum[half][row] = sum;
    if (half == 0) {
      sh.top[0][0][row] = mx;
      sh.to[row] = tree_i * p.t.heads + kv * p.group + (row0 + row) - tree_i * p.group;  // its (row, head)
    }
    if (row < rows && !(fabsf(all) <= 3.402823466e38f)) sh.bad[row] = sh.any_bad = 1;
    asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 4
    for (int r = warp; r < rows; r += kSoftThreads / 32) {
      const size_t at = static_cast<size_t>(sh.to[r]);
      const float total = sh.sum[0][r] + sh.sum[1][r], f = p.pacc != nullptr ? 1.0f : total == 0.0f ? 0.0f : 1.0f / total;
      float4* dst = reinterpret_cast<float4*>(p.pacc != nullptr ? p.pacc + (at * p.splits + split) * D : p.t.out + at * D);
      const bool bad = sh.bad[r] != 0;
#pragma unroll
      for (int k = 0; k < D / 128; ++k) {
        const float4 y = *reinterpret_cast<const float4*>(smem + r * (D * 4) + (((k * 32 + lane) ^ (r & 7)) << 4));
        if (!bad) dst[k * 32 + lane] = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
      }
      if (p.pacc != nullptr && lane == 0 && !bad) p.pmax[at * p.splits + split] = sh.top[0][0][r], p.psum[at * p.splits + split] = total;
    }
    if (sh.any_bad != 0)
      for (int r = warp; r < rows; r += kSoftThreads / 32)
        if (sh.bad[r] != 0) tree_scalar_row<KV, D>(p, sh, kv, row0 + r, c0, c1, split);
  } else if (loading) {
    float k_next = 0.0f, v_next = 0.0f;  // the next tile's scales
    if (S::kRaw) loader.next_scales(0, load_tid, k_next, v_next);
    for (int t = 0; t < tiles; ++t) {
      const int kb = t % S::kBufs, k_use = t / S::kBufs, vb = t % S::kBufs, v_use = t / S::kBufs;
      unsigned char *const k_dst = k_s + kb * S::kTileBytes, *const v_dst = v_s + vb * S::kTileBytes;
      unsigned char* const raw = raw_s + (t & 1) * 2 * S::kRawBytes;
      // keys: the buffer is free once the scores that read it are there
      if (KV != kKvF16 && k_use > 0) wait(&sh.k_empty[kb], k_use - 1);
      if constexpr (KV == kKvF32) {
        loader.split_rows(false, t, raw_s, k_dst, load_tid);
      } else {
        if constexpr (S::kRaw) {
          loader.put_scales(t, load_tid, k_next, v_next);
          loader.next_scales(t + 1, load_tid, k_next, v_next);
          wait(&sh.raw_full[t & 1][0], t >> 1);
        } else {
          asm volatile("cp.async.wait_group 2;" ::: "memory");
        }
        loader.convert(t, raw, k_dst, load_tid);
      }
      to_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.k_full[kb]);
      if constexpr (S::kRaw) {  // everybody has read the raw bytes
        asm volatile("bar.sync 2, 96;" ::: "memory");
        if (load_tid == 0) loader.fetch_raw(false, t + 2, raw);
      }
      // values: the buffer is free once the outputs that read it are there
      if (KV != kKvF16 && v_use > 0) wait(&sh.v_empty[vb], v_use - 1);
      if constexpr (KV == kKvF32) {
        loader.split_rows(true, t, raw_s, v_dst, load_tid);
      } else {
        if constexpr (S::kRaw) wait(&sh.raw_full[t & 1][1], t >> 1);
        else asm volatile("cp.async.wait_group 1;" ::: "memory");
        loader.convert(t, raw + S::kRawBytes, v_dst, load_tid);
      }
      to_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.v_full[vb]);
      if constexpr (S::kRaw) {
        asm volatile("bar.sync 2, 96;" ::: "memory");
        if (load_tid == 0) loader.fetch_raw(true, t + 2, raw + S::kRawBytes);
      }
      if constexpr (KV == kKvF16) {
        // The next tile's values and the keys of the one after it, straight into their buffers.  (The values of this tile's
        // buffer are in use until the scores of the next tile have been issued, for which its keys have to be published first.)
        if (t > 0) {
          if (t + 1 < tiles) wait(&sh.v_empty[vb ^ 1], (t - 1) / 2);
          loader.fetch(true, t + 1, v_s + (vb ^ 1) * S::kTileBytes, load_tid);
        } else {
          asm volatile("cp.async.commit_group;" ::: "memory");  // (its values are under way already)
        }
        if (t + 2 < tiles) wait(&sh.k_empty[kb], k_use);
        loader.fetch(false, t + 2, k_dst, load_tid);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (!ok) {  // bulk copies may be under way still: a millisecond for them
      const long long begin = clock64();
      while (clock64() - begin < 2000000) {
      }
    }
  } else if (lane == 0) {
    const uint32_t s_shape = tc_shape(kTcKeys, false), o_shape = tc_shape(128, true);
    auto scores = [&](int t) {
      const uint32_t d = tmem + kColS + (t & 1) * 64;
      const uint32_t at = smem_u32(k_s + (t % S::kBufs) * S::kTileBytes);
#pragma unroll 4
      for (int kk = 0; kk < D / 16; ++kk) {  // the small products first
        const uint64_t b = tc_operand(at + kk * 256, 128, S::kGroupBytes);
        tc_mma(d, tmem + kColQ + D / 2 + kk * 8, b, s_shape, kk != 0);
        if (S::kTerms == 2) tc_mma(d, tmem + kColQ + kk * 8, tc_operand(at + S::kTermBytes + kk * 256, 128, S::kGroupBytes), s_shape, 1);
      }
#pragma unroll 4
      for (int kk = 0; kk < D / 16; ++kk)
        tc_mma(d, tmem + kColQ + kk * 8, tc_operand(at + kk * 256, 128, S::kGroupBytes), s_shape, 1);
      tc_commit(&sh.s_full[t & 1]);
      tc_commit(&sh.k_empty[t % S::kBufs]);
    };
    auto outputs = [&](int t, int h) {
      const uint32_t w = tmem + kColS + (t & 1) * 64;
      const uint32_t at = smem_u32(v_s + (t % S::kBufs) * S::kTileBytes) + h * 2048;
#pragma unroll
      for (int kk = 0; kk < kTcKeys / 16; ++kk) {
        const uint64_t b = tc_operand(at + kk * 2 * S::kGroupBytes, S::kGroupBytes, 128);
        tc_mma(tmem + kColO, w + 32 + kk * 8, b, o_shape, kk != 0);
        if (S::kTerms == 2) tc_mma(tmem + kColO, w + kk * 8, tc_operand(at + S::kTermBytes + kk * 2 * S::kGroupBytes, S::kGroupBytes, 128), o_shape, 1);
      }
#pragma unroll
      for (int kk = 0; kk < kTcKeys / 16; ++kk)
        tc_mma(tmem + kColO, w + kk * 8, tc_operand(at + kk * 2 * S::kGroupBytes, S::kGroupBytes, 128), o_shape, 1);
      tc_commit(&sh.o_full);
      if (h == S::kHalves - 1) tc_commit(&sh.v_empty[t % S::kBufs]);
    };
    auto next_scores = [&](int t) {
      if (t >= tiles) return;
      wait(&sh.k_full[t % S::kBufs], t / S::kBufs);
      tc_after();
      if (ok) scores(t);
    };
    next_scores(0);
    next_scores(1);
    for (int t = 0; t < tiles && ok; ++t) {
      // outputs of a half: the weights and values are there, and the half before has been read
      wait(&sh.p_full[t & 1], t >> 1);
      wait(&sh.v_full[t % S::kBufs], t / S::kBufs);
#pragma unroll
      for (int h = 0; h < S::kHalves; ++h) {
        if (t + h > 0) wait(&sh.o_read, S::kHalves * t + h - 1);
        tc_after();
        if (ok) outputs(t, h);
      }
      if (t + 2 < tiles) wait(&sh.o_full, S::kHalves * (t + 1) - 1);  // the next scores go over this tile's weights
      next_scores(t + 2);
    }
    if (!ok) {  // products may be under way still: not while tensor memory is given back
      tc_commit(&sh.drained);
      mbar_wait(&sh.drained, 0, &g_tree_timeouts);
    }
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == kTcThreads / 32 - 1) tc_free(tmem);
}

// The chunks of a (row, head), at most 64, by a warp; zero where no chunk had a key.
constexpr int kMergeWarps = 4, kMostSplits = 64;
template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32)
attention_tree_merge_kernel(const float* __restrict__ pacc, const float* __restrict__ pmax, const float* __restrict__ psum,
                            float* __restrict__ out, int splits, int total) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const size_t row = static_cast<size_t>(blockIdx.x) * kMergeWarps + (threadIdx.x >> 5);
  if (row >= static_cast<size_t>(total)) return;
  const size_t base = row * splits;
  float top[2], sum[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int s = lane + 32 * u;
    top[u] = s < splits ? pmax[base + s] : kNoKey, sum[u] = s < splits ? psum[base + s] : 0.0f;
  }
  float most = fmaxf(top[0], top[1]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
  const float w[2] = {exp2f(top[0] - most), exp2f(top[1] - most)};
  const float den = warp_sum(fmaf(w[0], sum[0], w[1] * sum[1]));
  float4 num[D / 128];
#pragma unroll
  for (int k = 0; k < D / 128; ++k) num[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* src = reinterpret_cast<const float4*>(pacc) + base * (D / 4) + lane;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    const float ws = __shfl_sync(0xFFFFFFFFu, s < 32 ? w[0] : w[1], s & 31);
#pragma unroll
    for (int k = 0; k < D / 128; ++k) {
      const float4 x = __ldcs(src + s * (D / 4) + k * 32);
      num[k].x = fmaf(ws, x.x, num[k].x), num[k].y = fmaf(ws, x.y, num[k].y), num[k].z = fmaf(ws, x.z, num[k].z), num[k].w = fmaf(ws, x.w, num[k].w);
    }
  }
  const float f = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll
  for (int k = 0; k < D / 128; ++k)
    reinterpret_cast<float4*>(out)[row * (D / 4) + k * 32 + lane] = make_float4(num[k].x * f, num[k].y * f, num[k].z * f, num[k].w * f);
}

template <int KV, int D>
int launch_tree_tc(TcParams p, cudaStream_t st) {
  using S = TcShape<KV, D>;
  static_assert(S::kSmem + sizeof(TcShared) <= 227 * 1024, "shared memory of a CTA");
  const auto kernel = attention_tree_tc_kernel<KV, D>;
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), S::kSmem)) return rc;
  CUtensorMap maps[2] = {};
  if (S::kRaw) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.t.kv_heads) * S::kRowBytes, static_cast<uint64_t>(p.t.n) + p.t.m}, stride = dims[0];
    const uint32_t box[2] = {S::kBox, kTcKeys};
    for (int i = 0; i < 2; ++i)
      if (int rc = encode_tensor_map(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, i ? p.t.v : p.t.k, dims, &stride, box, S::kBox == 128)) return rc;
  }
  const dim3 grid(static_cast<unsigned>(p.t.kv_heads * p.row_tiles), static_cast<unsigned>(p.splits));
  const bool pdl = pdl_allowed(st, nullptr, 0, p.t.out, static_cast<size_t>(p.t.m) * p.t.heads * D * 4);
  if (launch_kernel(kernel, grid, dim3(kTcThreads), S::kSmem, st, pdl, maps[0], maps[1], p) != cudaSuccess) {
    cudaGetLastError();
    return kDeviceError;
  }
  if (int rc = check_launch(); rc != kOk || p.pacc == nullptr) return rc;
  const int total = p.t.m * p.t.heads;
  // (its launch overlaps the end of the chunks' kernel, which it waits for before it reads or writes anything)
  if (launch_kernel(attention_tree_merge_kernel<D>, dim3(static_cast<unsigned>((total + kMergeWarps - 1) / kMergeWarps)), dim3(kMergeWarps * 32), 0, st, true,
                    p.pacc, p.pmax, p.psum, p.t.out, p.splits, total) != cudaSuccess) {
    cudaGetLastError();
    return kDeviceError;
  }
  return check_launch();
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int KV>
int launch_tree(const TreeParams& t, uint64_t head_dim, cudaStream_t st) {
  if (!on16(t.q) || !on16(t.k) || !on16(t.v) || !on16(t.out)) {
    const dim3 grid(static_cast<unsigned>(t.heads), static_cast<unsigned>(t.m));
    if (head_dim == 256) attention_tree_rows_kernel<KV, 256><<<grid, kTreeWarps * 32, 0, st>>>(t);
    else attention_tree_rows_kernel<KV, 128><<<grid, kTreeWarps * 32, 0, st>>>(t);
    return check_launch();
  }
  TcParams p{};
  p.t = t;
  p.group = t.heads / t.kv_heads;
  p.row_tiles = (t.m * p.group + kTcRows - 1) / kTcRows;
  p.first_key = t.window != 0 && t.window < t.n ? t.n - t.window : 0;
  const long keys = static_cast<long>(t.n) + t.m - p.first_key, tiles = (keys + kTcKeys - 1) / kTcKeys;
  const long units = static_cast<long>(t.kv_heads) * p.row_tiles;
  // Chunks of the key range: whole waves of one CTA a SM, a CTA's start counted as four tiles; a tile of the fp32 cache costs its
  // loaders three of the others' (65 tiles of 8 rows, 4 kv heads: 33 chunks of two tiles 39 us, 22 of three 49, 17 of four 58).
  const double tile_cost = KV == kKvF32 ? (head_dim == 256 ? 3.0 : 1.5) : 1.0;
  static const int sms = [] {
    int dev = 0, v = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    return v > 0 ? v : 148;
  }();
  long best_splits = 1;
  double best = 0.0;
  for (long s = 1; s <= kMostSplits && s <= tiles; ++s) {
    const long per = (tiles + s - 1) / s;
    if ((tiles + per - 1) / per != s) continue;
    const double waves = static_cast<double>((units * s + sms - 1) / sms);
    const double cost = waves * (per * tile_cost + 4.0) + (s > 1 ? 2.0 + 0.1 * s : 0.0);
    if (s == 1 || cost < best) best = cost, best_splits = s;
  }
  p.splits = static_cast<int>(best_splits);
  p.tiles_per_split = static_cast<int>((tiles + best_splits - 1) / best_splits);
  if (p.splits > 1) {
    const size_t parts = static_cast<size_t>(t.m) * t.heads * p.splits;
    const size_t acc_bytes = parts * head_dim * 4, stat_bytes = (parts * 4 + 255) / 256 * 256;
    unsigned char* scratch = stream_scratch(st, acc_bytes + 2 * stat_bytes, 5);
    if (scratch != nullptr) {
      p.pacc = reinterpret_cast<float*>(scratch);
      p.pmax = reinterpret_cast<float*>(scratch + acc_bytes);
      p.psum = reinterpret_cast<float*>(scratch + acc_bytes + stat_bytes);
    } else {  // a capture before the first plain launch: no chunks
      p.splits = 1;
      p.tiles_per_split = static_cast<int>(tiles);
    }
  }
  return head_dim == 256 ? launch_tree_tc<KV, 256>(p, st) : launch_tree_tc<KV, 128>(p, st);
}

}  // namespace

int tree_wait_timeouts(unsigned int* count) {
  return cudaMemcpyFromSymbol(count, g_tree_timeouts, sizeof(*count)) == cudaSuccess ? kOk : kDeviceError;
}
int tree_set_error_word(unsigned int* word) { return set_host_error_word(word); }

int attention_tree(int kv_format, const float* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                                  const int32_t* parents, float* out, uint64_t m, uint64_t n, uint64_t heads, uint64_t kv_heads,
                                  uint64_t head_dim, uint64_t row_base, uint64_t window, bool dry, cudaStream_t st) {
  if (!q || !k || !v || !parents || !out || m == 0 || n > 0x7FFFFFFFull - kTreeRows || heads == 0 || heads > 65535 || kv_heads == 0 ||
      head_dim == 0 || heads % kv_heads != 0 || row_base > 0x7FFFFFFFull || window > 0x7FFFFFFFull || kv_format < TSR_KV_F32 || kv_format > TSR_KV_FP8)
    return kInvalidArgument;
  if (kv_format >= TSR_KV_INT8 && (!k_scale || !v_scale)) return kInvalidArgument;
  const uintptr_t item = kv_format == TSR_KV_F32 ? 4 : kv_format == TSR_KV_F16 ? 2 : 1;  // what the cache is read by at least
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % item != 0) return kInvalidArgument;
  if (m > kTreeRows || (head_dim != 128 && head_dim != 256) || heads / kv_heads > kAttnMaxGroup) return kUnsupportedFeature;
  const size_t skip = row_base * heads * head_dim;
  {  // a row's result is written while other rows are read; over its own queries it may go
    const uint64_t cols = kv_heads * head_dim, rows = n + m, bytes = m * heads * head_dim * 4;
    const uint64_t cache = kv_format == TSR_KV_F32 ? rows * cols * 4 : kv_format == TSR_KV_F16 ? rows * cols * 2 : kv_format == TSR_KV_INT4 ? rows * cols / 2 : rows * cols;
    const bool scaled = kv_format >= TSR_KV_INT8;
    struct {
      const void* at;
      uint64_t bytes;
    } const in[6] = {{q + skip, q == out ? 0 : bytes}, {k, cache}, {v, cache}, {k_scale, scaled ? rows * 4 : 0}, {v_scale, scaled ? rows * 4 : 0}, {parents, m * 4}};
    const auto* y = reinterpret_cast<const unsigned char*>(out + skip);
    for (const auto& r : in) {
      const auto* x = static_cast<const unsigned char*>(r.at);
      if (r.bytes != 0 && x < y + bytes && y < x + r.bytes) return kInvalidArgument;
    }
  }
  if (dry) return kOk;
  const TreeParams p{q + skip, static_cast<const unsigned char*>(k), static_cast<const unsigned char*>(v), k_scale, v_scale, parents, out + skip,
                     static_cast<int>(m), static_cast<int>(n), static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(window)};
  switch (kv_format) {
    case TSR_KV_F32: return launch_tree<kKvF32>(p, head_dim, st);
    case TSR_KV_F16: return launch_tree<kKvF16>(p, head_dim, st);
    case TSR_KV_INT8: return launch_tree<kKvInt8>(p, head_dim, st);
    case TSR_KV_INT4: return launch_tree<kKvInt4>(p, head_dim, st);
    default: return launch_tree<kKvFp8>(p, head_dim, st);
  }
}

}  // namespace tsr

extern "C" int tsr_attention_tree(int kv_format, const float* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                                  const int32_t* parents, float* out, uint64_t m, uint64_t n, uint64_t heads, uint64_t kv_heads,
                                  uint64_t head_dim, uint64_t row_base, uint64_t window, void* stream) {
  return tsr::attention_tree(kv_format, q, k, v, k_scale, v_scale, parents, out, m, n, heads, kv_heads, head_dim, row_base, window, false,
                             static_cast<cudaStream_t>(stream));
}
