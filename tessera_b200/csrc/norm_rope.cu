// What a full-attention layer does to its queries and keys before attention, for any number of rows in one launch:
// per-head rmsnorm of q and k, their rotation to each row's position (t, h, w), and the append of the k and v rows to the
// key / value cache in its format (ids "qk_norm_rope", "qk_norm_rope_append", "_q8" / "_q4" / "_fp8").  The reference
// issues these as two rmsnorms, two mropes and a cache writer for each of k and v (src/models/qwen3_5/trunk.cpp:374-391,
// trunk_batch.cpp:212-300); the arithmetic of each step is that of those ids:
//   y = x / sqrt(mean(x^2) + eps) * w;   (y_j, y_j+p) turned by pos[section of j] * theta^(-2j / rope_dim), p = rope_dim / 2,
//   angle, sine and cosine in double precision;   codes and scales as quantize_q8, quantize_q4, quantize_fp8_pack.
// The squares of a head are added in another order than rmsnorm's, so results agree to fp32 rounding.
//
// A warp takes a head: its elements stay in registers from the one read to the one write, and meet their partners of the
// rotation through the warp's row of shared memory.  CTA (row, 0) has the row's k and v heads (a quantised row's scale is the
// maximum over all kv heads), the other CTAs the query heads.
//
// Bound: for few rows the launch and one head's chain (16 rows of 24 + 4 heads of 256, FP8 cache: 5.7 us in the kernel, 6.4 us a
// call), for many the barrier behind the angles, which one warp of a CTA forms in double precision while the others wait (512
// rows, fp16 cache: 8.8 us, of which 1.5 under the launch before; half of the issue slots taken; the bytes alone 4.8 us).  There four elements
// at a time in the rotation, a head's norm ahead of the barrier that the angles need and the next head's elements under way
// brought 12.3 to 10.3 us; registers cut for more CTAs an SM cost (48: 12.4, 40: 14.5 us, spilled), and so did a table of
// frequencies from the host (1.2 us a call).
#include <cuda_fp16.h>

#include <cmath>

#include "codec.cuh"
#include "launch.h"
#include "tessera_b200.h"

namespace tsr {
namespace {

constexpr int kNormThreads = 256, kNormWarps = kNormThreads / 32;
constexpr int kNormMaxDim = 256;    // head_dim: eight elements a lane
constexpr int kNormMaxCols = 8192;  // kv_heads * head_dim of the quantised formats: a row of k waits in shared memory

struct NormRopeParams {
  const float *q, *k, *v, *q_w, *k_w;
  const unsigned long long* pos;
  float *q_out, *k_out;  // k_out: the form without a cache
  unsigned char *k_cache, *v_cache;  // at the first appended row
  float *k_scale, *v_scale;
  double log2_theta;
  float eps;
  int heads, kv_heads, head_dim, rope_dim, sec_t, sec_h, heads_per_cta;
};

enum : int { kToFloat = -1 };  // beside the cache formats: k rows as fp32 to k_out, v untouched

template <int N>
__device__ __forceinline__ void store_halves(__half* dst, const float (&x)[N]) {
  if constexpr (N == 4) {
    const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    *dst = __float2half_rn(x[0]);
  }
}
template <int N>
__device__ __forceinline__ void load_floats(float (&x)[N], const float* src) {
  if constexpr (N == 4) {
    const float4 y = *reinterpret_cast<const float4*>(src);
    x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
  } else {
    x[0] = *src;
  }
}
template <int N>
__device__ __forceinline__ void store_floats(float* dst, const float (&x)[N]) {
  if constexpr (N == 4) *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
  else *dst = x[0];
}

// The code of one value, its row's scale s given.
template <int FMT>
__device__ __forceinline__ uint32_t cache_code(float x, float s) {
  const float y = __fdiv_rn(x, s);
  if constexpr (FMT == TSR_KV_FP8) return e4m3_code(y < -448.0f ? -448.0f : (448.0f < y ? 448.0f : y));
  constexpr float kLimit = FMT == TSR_KV_INT8 ? 127.0f : 7.0f;
  return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(roundf(y), -kLimit), kLimit)));
}
template <int FMT>
__device__ __forceinline__ float cache_scale(float amax) {
  if constexpr (FMT == TSR_KV_FP8) return fmaxf(__fdiv_rn(amax, 448.0f), 1.0f / (448.0f * 512.0f));
  return amax > 0.0f ? __fdiv_rn(amax, FMT == TSR_KV_INT8 ? 127.0f : 7.0f) : 1.0f;
}
template <int FMT>
__device__ __forceinline__ void store_codes(unsigned char* row, const float* x, int cols, float s) {
  constexpr int kPer = FMT == TSR_KV_INT4 ? 8 : 4;  // codes of a 32-bit word
  constexpr int kBits = 32 / kPer;
  for (int c = threadIdx.x; c < cols / kPer; c += kNormThreads) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) w |= (cache_code<FMT>(x[c * kPer + e], s) & ((1u << kBits) - 1u)) << (kBits * e);
    reinterpret_cast<uint32_t*>(row)[c] = w;
  }
}

// grid: (rows, 1 + CTAs of query heads).  VEC: elements of a lane that lie side by side.
template <int OUT, int VEC>
__global__ void __launch_bounds__(kNormThreads) qk_norm_rope_kernel(const NormRopeParams p) {
  constexpr bool kQuant = OUT == TSR_KV_INT8 || OUT == TSR_KV_INT4 || OUT == TSR_KV_FP8;
  constexpr int kRuns = kNormMaxDim / (32 * VEC);
  extern __shared__ float k_row[];  // quantised formats: the row's k heads
  __shared__ __align__(16) float cos_s[kNormMaxDim / 2], sin_s[kNormMaxDim / 2];
  __shared__ __align__(16) float head_s[kNormWarps][kNormMaxDim];
  __shared__ float most_s[2][kNormWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dim = p.head_dim, pairs = p.rope_dim / 2;
  const size_t row = blockIdx.x;
  const bool keys = blockIdx.y == 0;
  const int h0 = keys ? 0 : (static_cast<int>(blockIdx.y) - 1) * p.heads_per_cta;
  const int h1 = keys ? p.kv_heads : min(p.heads, h0 + p.heads_per_cta);
  const float* src = (keys ? p.k : p.q) + row * (keys ? p.kv_heads : p.heads) * dim;
  const float* weight = keys ? p.k_w : p.q_w;
  float next[kRuns][VEC];  // a head ahead
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int e = (i * 32 + lane) * VEC;
#pragma unroll
      for (int c = 0; c < VEC; ++c) next[i][c] = 0.0f;
      if (h < h1 && e < dim) load_floats(next[i], src + static_cast<size_t>(h) * dim + e);
    }
  };
  // (this kernel's start overlaps the end of the one before it, which may write anything that is read from here on)
  const double freq = tid < pairs ? exp2(p.log2_theta * (-2.0 * tid / p.rope_dim)) : 0.0;
  pdl_wait();
  pdl_trigger();
  load(h0 + warp);
  if (tid < pairs) {
    const unsigned long long at = p.pos[row * 3 + (tid < p.sec_t ? 0 : tid < p.sec_t + p.sec_h ? 1 : 2)];
    const double angle = static_cast<double>(at) * freq;
    double s, c;
    sincos(angle, &s, &c);
    cos_s[tid] = static_cast<float>(c), sin_s[tid] = static_cast<float>(s);
  }
  float w[kRuns][VEC];
#pragma unroll
  for (int i = 0; i < kRuns; ++i) {
    const int e = (i * 32 + lane) * VEC;
    if (e < dim) load_floats(w[i], weight + e);
  }
  float most = 0.0f, x[kRuns][VEC];
  auto normalise = [&](int h) {  // x of head h; what is rotated to shared memory too
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kRuns; ++i)
#pragma unroll
      for (int c = 0; c < VEC; ++c) x[i][c] = next[i][c], sum = fmaf(x[i][c], x[i][c], sum);
    load(h + kNormWarps);  // (in place: another head)
    const float gain = 1.0f / sqrtf(warp_sum(sum) / static_cast<float>(dim) + p.eps);
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int e = (i * 32 + lane) * VEC;
      if (e >= dim) continue;
#pragma unroll
      for (int c = 0; c < VEC; ++c) x[i][c] = x[i][c] * gain * w[i][c];
      if (e < p.rope_dim) store_floats(&head_s[warp][e], x[i]);
    }
    __syncwarp();
  };
  normalise(h0 + warp);
  __syncthreads();  // the angles, formed meanwhile
  for (int h = h0 + warp; h < h1; h += kNormWarps) {
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int e = (i * 32 + lane) * VEC;
      if (e >= dim) continue;
      if (e < p.rope_dim) {  // (VEC divides the pairs)
        const bool first = e < pairs;
        const int d = first ? e : e - pairs;
        float other[VEC], cosine[VEC], sine[VEC];
        load_floats(other, &head_s[warp][first ? e + pairs : d]);
        load_floats(cosine, &cos_s[d]), load_floats(sine, &sin_s[d]);
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          const float turned = __fmul_rn(other[c], sine[c]);
          x[i][c] = __fadd_rn(__fmul_rn(x[i][c], cosine[c]), first ? -turned : turned);
        }
      }
      if constexpr (kQuant)
#pragma unroll
        for (int c = 0; c < VEC; ++c) most = fmaxf(most, fabsf(x[i][c]));
      if (!keys) {
        store_floats(p.q_out + (row * p.heads + h) * dim + e, x[i]);
      } else {
        const size_t at = static_cast<size_t>(h) * dim + e, cache_at = row * p.kv_heads * dim + at;
        if constexpr (kQuant) store_floats(k_row + at, x[i]);
        else if constexpr (OUT == TSR_KV_F16) store_halves(reinterpret_cast<__half*>(p.k_cache) + cache_at, x[i]);
        else store_floats(OUT == kToFloat ? p.k_out + cache_at : reinterpret_cast<float*>(p.k_cache) + cache_at, x[i]);
      }
    }
    __syncwarp();
    if (h + kNormWarps < h1) normalise(h + kNormWarps);
  }
  if (!keys || OUT == kToFloat) return;
  // the row of v
  const int cols = p.kv_heads * dim;
  const float* v = p.v + row * cols;
  if constexpr (!kQuant) {
    for (int e = tid * VEC; e < cols; e += kNormThreads * VEC) {
      float y[VEC];
      load_floats(y, v + e);
      if constexpr (OUT == TSR_KV_F16) store_halves(reinterpret_cast<__half*>(p.v_cache) + row * cols + e, y);
      else store_floats(reinterpret_cast<float*>(p.v_cache) + row * cols + e, y);
    }
  } else {
    float v_most = 0.0f;
    for (int e = tid * VEC; e < cols; e += kNormThreads * VEC) {
      float y[VEC];
      load_floats(y, v + e);
#pragma unroll
      for (int c = 0; c < VEC; ++c) v_most = fmaxf(v_most, fabsf(y[c]));  // fmaxf drops NaN, as the cache writers do
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
      v_most = fmaxf(v_most, __shfl_xor_sync(0xFFFFFFFFu, v_most, o));
    }
    if (lane == 0) most_s[0][warp] = most, most_s[1][warp] = v_most;
    __syncthreads();
    most = most_s[0][0], v_most = most_s[1][0];
#pragma unroll
    for (int i = 1; i < kNormWarps; ++i) most = fmaxf(most, most_s[0][i]), v_most = fmaxf(v_most, most_s[1][i]);
    const float ks = cache_scale<OUT>(most), vs = cache_scale<OUT>(v_most);
    if (tid == 0) p.k_scale[row] = ks, p.v_scale[row] = vs;
    const size_t row_bytes = OUT == TSR_KV_INT4 ? cols / 2 : cols;
    store_codes<OUT>(p.k_cache + row * row_bytes, k_row, cols, ks);
    store_codes<OUT>(p.v_cache + row * row_bytes, v, cols, vs);
  }
}

bool wide(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15u) == 0; }

struct Range {
  const void* at;
  uint64_t bytes;
  bool meets(const Range& o) const {
    const auto *x = static_cast<const unsigned char*>(at), *y = static_cast<const unsigned char*>(o.at);
    return x != nullptr && y != nullptr && x < y + o.bytes && y < x + bytes;
  }
};

// out: everything the launch writes, which a projection behind it may read as its weights (an FP8 cache and its scales are gemm_fp8's)
template <int OUT, int N>
int launch_norm_rope(NormRopeParams& p, uint64_t rows, bool vec, const Range (&out)[N], cudaStream_t st) {
  constexpr bool kQuant = OUT == TSR_KV_INT8 || OUT == TSR_KV_INT4 || OUT == TSR_KV_FP8;
  // A warp a head while that does not fill the machine, then all of a row's query heads in one CTA: the row's angles are formed
  // once a CTA (512 rows, before the last step: 12.4 us, with a warp a head 14.5).
  const int parts = rows <= 148 ? (p.heads + kNormWarps - 1) / kNormWarps : 1;
  p.heads_per_cta = (p.heads + parts - 1) / parts;
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(1 + parts));
  const size_t smem = kQuant ? static_cast<size_t>(p.kv_heads) * p.head_dim * 4 : 0;
  const void* written[N];
  size_t written_bytes[N];
  for (int i = 0; i < N; ++i) written[i] = out[i].at, written_bytes[i] = out[i].bytes;
  const bool pdl = pdl_allowed_ranges(st, nullptr, nullptr, 0, written, written_bytes, N);
  if (launch_kernel(vec ? qk_norm_rope_kernel<OUT, 4> : qk_norm_rope_kernel<OUT, 1>, grid, dim3(kNormThreads), smem, st, pdl, p) != cudaSuccess) {
    cudaGetLastError();
    return kDeviceError;
  }
  return check_launch();
}

// Checks shared by the two forms; fills the parameters they share.
int check_norm_rope(const float* q, const float* k, const float* q_w, const float* k_w, const uint64_t* pos, const float* q_out,
                    uint64_t rows, uint64_t heads, uint64_t kv_heads, uint64_t head_dim, uint64_t rope_dim, float theta, uint64_t sec_t,
                    uint64_t sec_h, uint64_t sec_w, float eps, NormRopeParams* p) {
  if (!q || !k || !q_w || !k_w || !pos || !q_out || rows == 0 || rows > 0x7FFFFFFFull || heads == 0 || heads > 65535 || kv_heads == 0 ||
      kv_heads > 65535 || head_dim == 0 || head_dim > 65535 || head_dim % 2 != 0 || rope_dim == 0 || rope_dim > head_dim || rope_dim % 2 != 0 ||
      sec_t > rope_dim || sec_h > rope_dim || sec_w > rope_dim || sec_t + sec_h + sec_w > rope_dim / 2 || !(theta > 0.0f) ||
      !std::isfinite(theta) || !(eps >= 0.0f))
    return kInvalidArgument;
  if (head_dim > kNormMaxDim) return kUnsupportedFeature;
  *p = NormRopeParams{};
  p->q = q, p->k = k, p->q_w = q_w, p->k_w = k_w, p->pos = reinterpret_cast<const unsigned long long*>(pos);
  p->q_out = const_cast<float*>(q_out);
  p->log2_theta = std::log2(static_cast<double>(theta));
  p->eps = eps;
  p->heads = static_cast<int>(heads), p->kv_heads = static_cast<int>(kv_heads), p->head_dim = static_cast<int>(head_dim);
  p->rope_dim = static_cast<int>(rope_dim), p->sec_t = static_cast<int>(sec_t), p->sec_h = static_cast<int>(sec_h);
  return kOk;
}

}  // namespace

int qk_norm_rope(const float* q, const float* k, const float* q_w, const float* k_w, const uint64_t* pos, float* q_out, float* k_out,
                     uint64_t rows, uint64_t heads, uint64_t kv_heads, uint64_t head_dim, uint64_t rope_dim, float theta, uint64_t sec_t,
                     uint64_t sec_h, uint64_t sec_w, float eps, bool dry, cudaStream_t st) {
  NormRopeParams p;
  if (int rc = check_norm_rope(q, k, q_w, k_w, pos, q_out, rows, heads, kv_heads, head_dim, rope_dim, theta, sec_t, sec_h, sec_w, eps, &p)) return rc;
  if (!k_out) return kInvalidArgument;
  // in place head by head, else apart: a head is read whole before it is written, another CTA's may not be there yet
  const uint64_t q_bytes = rows * heads * head_dim * 4, k_bytes = rows * kv_heads * head_dim * 4;
  const Range in[5] = {{q, q_bytes}, {k, k_bytes}, {q_w, head_dim * 4}, {k_w, head_dim * 4}, {pos, rows * 24}};
  const Range out[2] = {{q_out, q_bytes}, {k_out, k_bytes}}, &qo = out[0], &ko = out[1];
  if (qo.meets(ko)) return kInvalidArgument;
  for (int i = 0; i < 5; ++i)  // (by its place: keys or weights may lie where the queries do)
    if ((qo.meets(in[i]) && !(i == 0 && q_out == q)) || (ko.meets(in[i]) && !(i == 1 && k_out == k))) return kInvalidArgument;
  if (dry) return kOk;
  p.k_out = k_out;
  const bool vec = head_dim % 4 == 0 && rope_dim % 8 == 0 && wide(q) && wide(k) && wide(q_w) && wide(k_w) && wide(q_out) && wide(k_out);
  return launch_norm_rope<kToFloat>(p, rows, vec, out, st);
}

int qk_norm_rope_append(int kv_format, const float* q, const float* k, const float* v, const float* q_w, const float* k_w, const uint64_t* pos,
                            float* q_out, void* k_cache, void* v_cache, float* k_scale, float* v_scale, uint64_t rows, uint64_t cache_row,
                            uint64_t heads, uint64_t kv_heads, uint64_t head_dim, uint64_t rope_dim, float theta, uint64_t sec_t,
                            uint64_t sec_h, uint64_t sec_w, float eps, bool dry, cudaStream_t st) {
  NormRopeParams p;
  if (int rc = check_norm_rope(q, k, q_w, k_w, pos, q_out, rows, heads, kv_heads, head_dim, rope_dim, theta, sec_t, sec_h, sec_w, eps, &p)) return rc;
  if (!v || !k_cache || !v_cache || cache_row > 0x7FFFFFFFull) return kInvalidArgument;
  const uint64_t cols = kv_heads * head_dim;
  uint64_t row_bytes = cols, item = 4;  // item: what the cache's rows are written by
  bool quant = true;
  switch (kv_format) {
    case TSR_KV_F32: row_bytes = cols * 4, quant = false; break;
    case TSR_KV_F16: row_bytes = cols * 2, item = 2, quant = false; break;
    case TSR_KV_INT4: row_bytes = cols / 2; break;
    case TSR_KV_INT8: case TSR_KV_FP8: break;
    default: return kInvalidArgument;
  }
  if (reinterpret_cast<uintptr_t>(k_cache) % item != 0 || reinterpret_cast<uintptr_t>(v_cache) % item != 0) return kInvalidArgument;
  if (quant) {
    if (!k_scale || !v_scale || cols % (kv_format == TSR_KV_INT4 ? 8 : 4) != 0) return kInvalidArgument;
    if (cols > kNormMaxCols) return kUnsupportedFeature;
  }
  p.v = v;
  p.k_cache = static_cast<unsigned char*>(k_cache) + cache_row * row_bytes;
  p.v_cache = static_cast<unsigned char*>(v_cache) + cache_row * row_bytes;
  p.k_scale = quant ? k_scale + cache_row : nullptr, p.v_scale = quant ? v_scale + cache_row : nullptr;
  const uint64_t q_bytes = rows * heads * head_dim * 4, k_bytes = rows * cols * 4;
  const Range in[6] = {{q, q_bytes}, {k, k_bytes}, {v, k_bytes}, {q_w, head_dim * 4}, {k_w, head_dim * 4}, {pos, rows * 24}};
  const uint64_t scale_bytes = quant ? rows * 4 : 0;
  const Range out[5] = {{q_out, q_bytes}, {p.k_cache, rows * row_bytes}, {p.v_cache, rows * row_bytes}, {p.k_scale, scale_bytes}, {p.v_scale, scale_bytes}};
  for (int i = 0; i < 5; ++i) {
    for (int j = 0; j < 6; ++j)
      if (out[i].meets(in[j]) && !(i == 0 && j == 0 && q_out == q)) return kInvalidArgument;
    for (int j = 0; j < i; ++j)
      if (out[i].meets(out[j])) return kInvalidArgument;
  }
  const bool vec = head_dim % 4 == 0 && rope_dim % 8 == 0 && wide(q) && wide(k) && wide(v) && wide(q_w) && wide(k_w) && wide(q_out) &&
                   (quant || (wide(p.k_cache) && wide(p.v_cache)));
  if (dry) return kOk;
  switch (kv_format) {
    case TSR_KV_F32: return launch_norm_rope<TSR_KV_F32>(p, rows, vec, out, st);
    case TSR_KV_F16: return launch_norm_rope<TSR_KV_F16>(p, rows, vec, out, st);
    case TSR_KV_INT8: return launch_norm_rope<TSR_KV_INT8>(p, rows, vec, out, st);
    case TSR_KV_INT4: return launch_norm_rope<TSR_KV_INT4>(p, rows, vec, out, st);
    default: return launch_norm_rope<TSR_KV_FP8>(p, rows, vec, out, st);
  }
}

}  // namespace tsr

extern "C" {

int tsr_qk_norm_rope(const float* q, const float* k, const float* q_w, const float* k_w, const uint64_t* pos, float* q_out, float* k_out,
                     uint64_t rows, uint64_t heads, uint64_t kv_heads, uint64_t head_dim, uint64_t rope_dim, float theta, uint64_t sec_t,
                     uint64_t sec_h, uint64_t sec_w, float eps, void* stream) {
  return tsr::qk_norm_rope(q, k, q_w, k_w, pos, q_out, k_out, rows, heads, kv_heads, head_dim, rope_dim, theta, sec_t, sec_h, sec_w, eps, false,
                           static_cast<cudaStream_t>(stream));
}

int tsr_qk_norm_rope_append(int kv_format, const float* q, const float* k, const float* v, const float* q_w, const float* k_w, const uint64_t* pos,
                            float* q_out, void* k_cache, void* v_cache, float* k_scale, float* v_scale, uint64_t rows, uint64_t cache_row,
                            uint64_t heads, uint64_t kv_heads, uint64_t head_dim, uint64_t rope_dim, float theta, uint64_t sec_t,
                            uint64_t sec_h, uint64_t sec_w, float eps, void* stream) {
  return tsr::qk_norm_rope_append(kv_format, q, k, v, q_w, k_w, pos, q_out, k_cache, v_cache, k_scale, v_scale, rows, cache_row, heads, kv_heads,
                                  head_dim, rope_dim, theta, sec_t, sec_h, sec_w, eps, false, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
