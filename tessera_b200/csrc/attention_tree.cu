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
#include "tessera_b200.h"

namespace tsr {
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

template <int KV>
int launch_tree(const TreeParams& p, uint64_t head_dim, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.heads), static_cast<unsigned>(p.m));
  if (head_dim == 256) attention_tree_rows_kernel<KV, 256><<<grid, kTreeWarps * 32, 0, st>>>(p);
  else attention_tree_rows_kernel<KV, 128><<<grid, kTreeWarps * 32, 0, st>>>(p);
  return check_launch();
}

}  // namespace

int attention_tree(int kv_format, const float* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                                  const int32_t* parents, float* out, uint64_t m, uint64_t n, uint64_t heads, uint64_t kv_heads,
                                  uint64_t head_dim, uint64_t row_base, uint64_t window, bool dry, cudaStream_t st) {
  if (!q || !k || !v || !parents || !out || m == 0 || n > 0x7FFFFFFFull - kTreeRows || heads == 0 || heads > 65535 || kv_heads == 0 ||
      head_dim == 0 || heads % kv_heads != 0 || row_base > 0x7FFFFFFFull || window > 0x7FFFFFFFull || kv_format < TSR_KV_F32 || kv_format > TSR_KV_FP8)
    return kInvalidArgument;
  if (kv_format >= TSR_KV_INT8 && (!k_scale || !v_scale)) return kInvalidArgument;
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
