// The gated delta rule over many rows in its chunked form (id "delta_chunk_heads"): what delta_step_heads computes row by row
// (DeltaStepHeadsRef, src/core/numerics/attention.cpp:290-334 of the reference), for a prompt's chunk or a chain of drafted
// tokens.  Per head, with state S (dk x dv), c_t = beta_t (v_t - alpha_t S_{t-1}^T k_t):
//   S_t = alpha_t S_{t-1} + k_t c_t^T,   o_t = S_t^T q_t.
// Over a chunk of 32 rows that starts from S, with G(t, s) = prod_{s < r <= t} alpha_r and g_t = G(t, start):
//   c_t + beta_t sum_{s < t} G(t, s) (k_s . k_t) c_s = beta_t (v_t - g_t S^T k_t)      a unit lower triangular system
//   o_t = g_t S^T q_t + sum_{s <= t} G(t, s) (k_s . q_t) c_s,    S' = g_C S + sum_s G(C, s) k_s c_s^T.
// The decays are products, not exponentials of differences of logarithms, so alpha = 0 and products that underflow are exact.
//
// Two launches.  delta_chunk_prepare: all chunks at once, what does not depend on the state.  With T the inverse of the system
// times beta (forward substitution, a lane a column), c = u - W S with u = T v and W = T diag(g) K; the weights
// P = G (k . q); keys and queries.  A key head's Gram matrices serve all value heads that share it.  delta_chunk_scan: the chunks
// in turn.  Two warps carry 16 state columns (S^T, 16 x dk, half of dk each, in registers as fp32) through S^T W^T and the update;
// two more form the outputs a chunk behind them.  All products are m16n8k16 binary16 MMAs; the left operand is made of registers,
// the accumulators' layout being that operand's.  Each operand enters as two binary16 terms of a row scaled by a power of two, 22
// bits below the row's largest element, and three products of terms; in the scan small products have accumulators of their own
// (the MMA cuts off what falls below its accumulator).
//
// Bound: the chain of the chunks.  48 heads over 16 key heads of 128 x 128, 33 rows: 16 us; 512 rows: 63 us, of which 22 the first kernel (44 % of
// its issue slots, a chain of short phases) and 48 the scan, 2.9 us a chunk; 32 heads, 2048 rows: 179 us, 61 and 128, 2.0 us a chunk
// (tensor pipe 30 % busy, a third of the issue slots: what a warp waits for is its own last instruction).  Row by row the same
// takes 155 us for 512 rows; 33 rows 25 us with the two repeat_heads that it needs, one row 11 us against 13 here, two rows 14.  Steps: one warp for 16 whole columns, outputs by the same warp 78 and 261; outputs by warps of
// their own, copies of 16 bytes by all threads 75 and 270 (the copies' issue held up everybody); T folded into W, half of dk a
// warp 82 and 260; bulk copies by one thread 75 and 235; u as a bulk copy too, operands of the MMAs a step ahead 68 and 186.
#include <cuda_fp16.h>

#include "codec.cuh"
#include "launch.h"
#include "pipeline.cuh"
#include "tessera_b200.h"

namespace tsr {
namespace {

constexpr int kChunk = 32;       // rows
constexpr int kMostChunks = 64;  // of a pair of launches
constexpr int kSms = 148;
__device__ unsigned int g_delta_timeouts = 0;

// One chunk's operands as they lie in the workspace and in shared memory: K and Q (per key head), W and P (per value head).  Every
// row: the leading terms, then the rest; its 16-byte piece c at c ^ (row & 7), so that ldmatrix is conflict-free.
template <int DK>
struct ChunkShape {
  static constexpr int kRowBytes = 4 * DK;
  static constexpr int kKeyBytes = kChunk * kRowBytes;       // of K, Q or W
  static constexpr int kMatBytes = kChunk * 4 * kChunk;      // of P
};
// What a chunk's columns of results are multiplied by: the decay with the power of two that takes an operand's row back.
struct Factors {
  float solve[2][kChunk];  // 2^e(W_t), of either half of its elements
  float query[kChunk];     // g_t 2^e(q_t): of S^T q_t
  float out[kChunk];       // 2^e(P_t)
  float put[kChunk];       // G(C, s) 2^e(k_s): of c_s in the update
  float state;             // g_C
  float unused[3];
};
static_assert(sizeof(Factors) % 16 == 0, "copied in pieces of 16 bytes");

struct DeltaChunkParams {
  const float *s, *k, *v, *q, *alpha, *beta;  // s, alpha, beta at their bases
  float *o, *s_out;
  unsigned char *keys, *mats;                 // [key head][chunk][K, Q], [head][chunk][W, P]
  float4* u;                                  // [head][16 columns][chunk][eight rows][lane]: as the scan holds them
  Factors* factors;                           // [head][chunk]
  int heads, k_heads, dv, rows, chunks;
};

// The power of two that takes a row's largest element (its bits as an integer) to [2^13, 2^14), and its inverse.
__device__ __forceinline__ void row_unit(uint32_t most, float& up, float& unit) {
  int e = static_cast<int>(most >> 23) - 127 - 13;
  e = most == 0 ? 0 : max(-110, min(114, e));
  up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  unit = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
// (x, y) as binary16 and what binary16 lost of them
__device__ __forceinline__ void two_terms(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = half2_bits(h);
  lo = half2_bits(__floats2half2_rn(x - f.x, y - f.y));
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void load_matrices_turned(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x (rows of the accumulators' layout, N tiles of eight columns) as the left operand of a product: two terms of each row
// scaled by a power of two; unit: what takes rows lane / 4 and lane / 4 + 8 back.
template <int N>
__device__ __forceinline__ void as_operand(const float (&x)[N][4], uint32_t (&hi)[N / 2][4], uint32_t (&lo)[N / 2][4], float (&unit)[2]) {
  uint32_t most[2] = {0, 0};
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) most[c >> 1] = max(most[c >> 1], abs_bits(x[n][c]));
  float up[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    most[u] = max(most[u], __shfl_xor_sync(0xFFFFFFFFu, most[u], 1));
    most[u] = max(most[u], __shfl_xor_sync(0xFFFFFFFFu, most[u], 2));
    row_unit(most[u], up[u], unit[u]);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    two_terms(x[n][0] * up[0], x[n][1] * up[0], hi[n / 2][2 * (n & 1)], lo[n / 2][2 * (n & 1)]);
    two_terms(x[n][2] * up[1], x[n][3] * up[1], hi[n / 2][2 * (n & 1) + 1], lo[n / 2][2 * (n & 1) + 1]);
  }
}

template <int N>
struct Const {
  static constexpr int n = N;
};

// y += A M of two terms each, for a right operand of two tiles of eight columns: matrices (tile 0 rows 0-7, rows 8-15, tile 1 ...)
__device__ __forceinline__ void mma3(float (&hi0)[4], float (&hi1)[4], float (&lo0)[4], float (&lo1)[4], const uint32_t (&ah)[4],
                                     const uint32_t (&al)[4], const uint32_t (&bh)[4], const uint32_t (&bl)[4]) {
  mma(lo0, al, bh[0], bh[1]);
  mma(lo1, al, bh[2], bh[3]);
  mma(hi0, ah, bh[0], bh[1]);
  mma(hi1, ah, bh[2], bh[3]);
  mma(lo0, ah, bl[0], bl[1]);
  mma(lo1, ah, bl[2], bl[3]);
}
// what this thread wrote to shared memory, for a bulk copy that a thread issues after the next barrier
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, __shfl_xor_sync(0xFFFFFFFFu, x, 1));
  return max(x, __shfl_xor_sync(0xFFFFFFFFu, x, 2));
}

// grid: (chunks, key heads, parts of a key head's value heads), 8 warps.  Up to four value heads at a time: the substitution is a warp's, everything else is spread
// over all warps.
constexpr int kPrepThreads = 256, kPrepWarps = kPrepThreads / 32, kPrepHeads = 4, kPitch = kChunk + 4;
struct PrepHead {
  float solve[kChunk][kPitch];  // the system, then T
  float out[kChunk][kPitch];    // the decays G, then P
};
struct PrepShared {
  float gram[2][kChunk][kPitch];            // k_t . k_s and q_t . k_s
  float fold[kPrepHeads][kChunk];           // g_s 2^e(k_s)
  float beta[kPrepHeads][kChunk];
  float unit[2][kChunk];
};
template <int DK, int PER_SM>
__global__ void __launch_bounds__(kPrepThreads, PER_SM) delta_chunk_prepare_kernel(const DeltaChunkParams p) {
  using S = ChunkShape<DK>;
  extern __shared__ __align__(128) unsigned char prep_smem[];
  // K and Q as two terms, as in the workspace: bulk copies take them there; W takes Q's place
  unsigned char *const op_s = prep_smem, *const w_s = prep_smem + S::kKeyBytes;
  PrepShared& sh = *reinterpret_cast<PrepShared*>(prep_smem + 2 * S::kKeyBytes);
  PrepHead* const hd = reinterpret_cast<PrepHead*>(prep_smem + 2 * S::kKeyBytes + sizeof(PrepShared));  // as many as there are, at most kPrepHeads
  pdl_wait();     // (this kernel's start overlaps the end of the one before it)
  pdl_trigger();  // once every CTA is here, the scan's may start: not earlier, since they read the state ahead of their wait
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int chunk = blockIdx.x, kh = blockIdx.y, t0 = chunk * kChunk, rows = min(kChunk, p.rows - t0);
  const int factor = p.heads / p.k_heads, per = (factor + gridDim.z - 1) / gridDim.z, f_begin = blockIdx.z * per, f_end = min(factor, f_begin + per);
  float alpha = 1.0f, beta = 0.0f;  // of row `lane` and the value head that the warp solves
  auto load_gates = [&](int f) {
    if (warp >= kPrepHeads || f >= f_end || lane >= rows) return alpha = 1.0f, beta = 0.0f, void();
    const size_t at = static_cast<size_t>(t0 + lane) * p.heads + kh + f * p.k_heads;
    alpha = p.alpha[at], beta = p.beta[at];
  };
  load_gates(f_begin + warp);
  // eight lanes a row
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int t = tid >> 3, part = tid & 7;
    const float* src = (which ? p.q : p.k) + (static_cast<size_t>(t0 + t) * p.k_heads + kh) * DK + part * 8;
    float x[DK / 64][8];
    uint32_t most = 0;
    const bool wide = (reinterpret_cast<uintptr_t>(src) & 15) == 0;  // (the same for every row)
#pragma unroll
    for (int j = 0; j < DK / 64; ++j) {
      if (t >= rows) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
      } else if (wide) {
        *reinterpret_cast<float4*>(&x[j][0]) = *reinterpret_cast<const float4*>(src + 64 * j);
        *reinterpret_cast<float4*>(&x[j][4]) = *reinterpret_cast<const float4*>(src + 64 * j + 4);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = src[64 * j + i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) most = max(most, abs_bits(x[j][i]));
    }
    most = quad_max(most);
    most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 4));
    float up, unit;
    row_unit(most, up, unit);
    if (part == 0) sh.unit[which][t] = unit;
#pragma unroll
    for (int j = 0; j < DK / 64; ++j) {
      uint4 hi, lo;
      two_terms(x[j][0] * up, x[j][1] * up, hi.x, lo.x);
      two_terms(x[j][2] * up, x[j][3] * up, hi.y, lo.y);
      two_terms(x[j][4] * up, x[j][5] * up, hi.z, lo.z);
      two_terms(x[j][6] * up, x[j][7] * up, hi.w, lo.w);
      const int c = part + 8 * j;
      unsigned char* const at = op_s + which * S::kKeyBytes + t * S::kRowBytes;
      *reinterpret_cast<uint4*>(at + ((c ^ (t & 7)) << 4)) = hi;
      *reinterpret_cast<uint4*>(at + (((c + DK / 8) ^ (t & 7)) << 4)) = lo;
    }
  }
  const uint32_t k_at = smem_u32(op_s);
  const size_t step_v = static_cast<size_t>(p.heads) * p.dv;
  fence_async();
  __syncthreads();
  if (tid == 0 && blockIdx.z == 0) bulk_store(p.keys + (static_cast<size_t>(kh) * p.chunks + chunk) * 2 * S::kKeyBytes, op_s, 2 * S::kKeyBytes);
  {  // the Gram matrices: 16 rows by 16 columns a warp; what lies above the diagonal is not used
    const int which = warp >> 2, m = warp >> 1 & 1, n = warp & 1;
    if (n <= m) {
      const int ar = m * 16 + (lane & 15), ac = lane >> 4, br = n * 16 + (lane & 7) + ((lane >> 4) << 3), bc = lane >> 3 & 1;
      const uint32_t a_at = k_at + which * S::kKeyBytes + ar * S::kRowBytes, b_at = k_at + br * S::kRowBytes;
      float hi[2][4] = {}, lo[2][4] = {};
#pragma unroll
      for (int step = 0; step < DK / 16; ++step) {
        uint32_t ah[4], al[4], bh[4], bl[4];
        load_matrices(ah, a_at + (((2 * step + ac) ^ (ar & 7)) << 4));
        load_matrices(al, a_at + (((2 * step + ac + DK / 8) ^ (ar & 7)) << 4));
        load_matrices(bh, b_at + (((2 * step + bc) ^ (br & 7)) << 4));
        load_matrices(bl, b_at + (((2 * step + bc + DK / 8) ^ (br & 7)) << 4));
        mma3(hi[0], hi[1], lo[0], lo[1], ah, al, bh, bl);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = m * 16 + g + 8 * (c >> 1), s = n * 16 + e * 8 + 2 * t4 + (c & 1);
          sh.gram[which][r][s] = (hi[e][c] + lo[e][c]) * sh.unit[which][r] * sh.unit[0][s];
        }
    }
  }
  for (int f0 = f_begin; f0 < f_end; f0 += kPrepHeads) {
    const int heads = min(kPrepHeads, f_end - f0);
    Factors* const fac = p.factors + static_cast<size_t>(kh + f0 * p.k_heads) * p.chunks + chunk;
    const size_t fac_step = static_cast<size_t>(p.k_heads) * p.chunks;
    unsigned char* const mats = p.mats + (static_cast<size_t>(kh + f0 * p.k_heads) * p.chunks + chunk) * (S::kKeyBytes + S::kMatBytes);
    const size_t mats_step = fac_step * (S::kKeyBytes + S::kMatBytes);
    if (warp < heads) {
      float decay = 0.0f, start = 1.0f, mine = 1.0f;  // G(t, lane), g_t, g_lane
#pragma unroll
      for (int t = 0; t < kChunk; ++t) {
        const float a = __shfl_sync(0xFFFFFFFFu, alpha, t);
        decay = lane == t ? 1.0f : lane < t ? decay * a : 0.0f;
        start *= a;
        if (lane == t) mine = start;
        hd[warp].out[t][lane] = decay;
      }
      Factors* const f = fac + warp * fac_step;
      f->query[lane] = mine * sh.unit[1][lane], f->put[lane] = decay * sh.unit[0][lane];
      if (lane == 0) f->state = start;
      sh.fold[warp][lane] = mine * sh.unit[0][lane], sh.beta[warp][lane] = beta;
    }
    __syncthreads();
    for (int i = tid; i < heads * kChunk * kChunk / 4; i += kPrepThreads) {
      const int w = i / (kChunk * kChunk / 4), t = i / (kChunk / 4) % kChunk, s = i % (kChunk / 4) * 4;
      const float4 d = *reinterpret_cast<const float4*>(&hd[w].out[t][s]), kk = *reinterpret_cast<const float4*>(&sh.gram[0][t][s]),
                   qk = *reinterpret_cast<const float4*>(&sh.gram[1][t][s]);
      const float b = sh.beta[w][t];
      *reinterpret_cast<float4*>(&hd[w].solve[t][s]) = make_float4(s < t ? b * d.x * kk.x : 0.0f, s + 1 < t ? b * d.y * kk.y : 0.0f,
                                                                   s + 2 < t ? b * d.z * kk.z : 0.0f, s + 3 < t ? b * d.w * kk.w : 0.0f);
      *reinterpret_cast<float4*>(&hd[w].out[t][s]) =
          make_float4(s <= t ? d.x * qk.x : 0.0f, s + 1 <= t ? d.y * qk.y : 0.0f, s + 2 <= t ? d.z * qk.z : 0.0f, s + 3 <= t ? d.w * qk.w : 0.0f);
    }
    __syncthreads();
    // values of u's warps: 16 columns, [tile][row 2 t, 2 t + 1, + 8, ...], loaded ahead
    float v[2][8];
    auto load_values = [&](int w, int c0) {
      const float* const src = p.v + (static_cast<size_t>(t0) * p.heads + kh + (f0 + w) * p.k_heads) * p.dv + c0 + g;
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int s = (i >> 1) * 8 + 2 * t4 + (i & 1);
          v[e][i] = s < rows && c0 < p.dv ? src[s * step_v + 8 * e] : 0.0f;
        }
    };
    const int first = (warp - 4) * 16;
    if (warp >= 4) load_values(0, first);
    if (warp < heads) {
      float x[kChunk];  // a column of the inverse
#pragma unroll
      for (int t = 0; t < kChunk; ++t) {
        float sum[4] = {lane == t ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < (t + 3) / 4; ++s) {
          const float4 row = *reinterpret_cast<const float4*>(&hd[warp].solve[t][4 * s]);
          sum[0] = fmaf(-row.x, x[4 * s], sum[0]);
          if (4 * s + 1 < t) sum[1] = fmaf(-row.y, x[4 * s + 1], sum[1]);
          if (4 * s + 2 < t) sum[2] = fmaf(-row.z, x[4 * s + 2], sum[2]);
          if (4 * s + 3 < t) sum[3] = fmaf(-row.w, x[4 * s + 3], sum[3]);
        }
        x[t] = lane <= t ? (sum[0] + sum[1]) + (sum[2] + sum[3]) : 0.0f;
      }
      __syncwarp();
      const float b = sh.beta[warp][lane];
#pragma unroll
      for (int t = 0; t < kChunk; ++t) hd[warp].solve[t][lane] = x[t] * b;
      load_gates(f0 + kPrepHeads + warp);
    } else {  // P, eight lanes a row
      for (int i = (warp - heads) * 4 + (lane >> 3); i < heads * kChunk; i += (kPrepWarps - heads) * 4) {
        const int w = i / kChunk, t = i % kChunk, part = lane & 7;
        const float4 x = *reinterpret_cast<const float4*>(&hd[w].out[t][4 * part]);
        uint32_t most = quad_max(max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w))));
        most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 4));
        float up, unit;
        row_unit(most, up, unit);
        uint2 hi, lo;
        two_terms(x.x * up, x.y * up, hi.x, lo.x);
        two_terms(x.z * up, x.w * up, hi.y, lo.y);
        unsigned char* const row = mats + w * mats_step + S::kKeyBytes + t * 4 * kChunk;
        *reinterpret_cast<uint2*>(row + (((part >> 1) ^ (t & 7)) << 4) + 8 * (part & 1)) = hi;
        *reinterpret_cast<uint2*>(row + (((part >> 1) + kChunk / 8 ^ (t & 7)) << 4) + 8 * (part & 1)) = lo;
        if (part == 0) fac[w * fac_step].out[t] = unit;
      }
    }
    __syncthreads();
    // rows 16 m + g and 16 m + g + 8 of T diag(fold) as a left operand; unit: what takes them back
    auto left = [&](int w, int m, uint32_t(&ah)[2][4], uint32_t(&al)[2][4], float(&unit)[2]) {
      float x[2][2][4];  // [step][row][column 2 t, 2 t + 1, + 8, + 9]
      uint32_t most[2] = {0, 0};
      float up[2];
#pragma unroll
      for (int step = 0; step < 2; ++step)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float2 y = make_float2(0.0f, 0.0f);
            const int s = step * 16 + 8 * c + 2 * t4;
            if (step <= m) {
              y = *reinterpret_cast<const float2*>(&hd[w].solve[m * 16 + g + 8 * r][s]);
              y.x *= sh.fold[w][s], y.y *= sh.fold[w][s + 1];
            }
            x[step][r][2 * c] = y.x, x[step][r][2 * c + 1] = y.y;
            most[r] = max(most[r], max(abs_bits(y.x), abs_bits(y.y)));
          }
#pragma unroll
      for (int r = 0; r < 2; ++r) row_unit(quad_max(most[r]), up[r], unit[r]);
#pragma unroll
      for (int step = 0; step < 2; ++step)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c) two_terms(x[step][r][2 * c] * up[r], x[step][r][2 * c + 1] * up[r], ah[step][2 * c + r], al[step][2 * c + r]);
    };
    for (int w = 0; w < heads; ++w) {
      // W: 16 rows by half of the elements a warp.  Large and small products share an accumulator: there are two steps of them, and
      // accumulators of their own left the results' errors as they were (2.3e-7, 2.9e-7) and spilled (512 rows: 64.8 us against 63.1).
      if (warp < 4) {
        const int half = warp & 1, m = warp >> 1;
        constexpr int kTiles = DK / 16;
        uint32_t ah[2][4], al[2][4];
        float unit[2], hi[kTiles][4] = {}, up[2], unit_w[2];
        left(w, m, ah, al, unit);
        const int ur = lane & 15, uc = lane >> 4;
#pragma unroll
        for (int step = 0; step < 2; ++step) {
          if (step > m) continue;
          const int r = step * 16 + ur;
#pragma unroll
          for (int pair = 0; pair < kTiles / 2; ++pair) {
            uint32_t bh[4], bl[4];
            const int c = half * kTiles + pair * 2 + uc;
            load_matrices_turned(bh, k_at + r * S::kRowBytes + ((c ^ (r & 7)) << 4));
            load_matrices_turned(bl, k_at + r * S::kRowBytes + (((c + DK / 8) ^ (r & 7)) << 4));
            mma3(hi[2 * pair], hi[2 * pair + 1], hi[2 * pair], hi[2 * pair + 1], ah[step], al[step], bh, bl);
          }
        }
        if (tid == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the W before this one has left
        asm volatile("bar.sync 1, 128;" ::: "memory");
        uint32_t most[2] = {0, 0};
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) hi[n][c] *= unit[c >> 1], most[c >> 1] = max(most[c >> 1], abs_bits(hi[n][c]));
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          row_unit(quad_max(most[r]), up[r], unit_w[r]);
          const int t = m * 16 + g + 8 * r;
          if (t4 == 0) fac[w * fac_step].solve[half][t] = unit_w[r];
          uint32_t* const row = reinterpret_cast<uint32_t*>(w_s + t * S::kRowBytes) + t4;
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            uint32_t h, l;
            two_terms(hi[n][2 * r] * up[r], hi[n][2 * r + 1] * up[r], h, l);
            const int c = half * kTiles + n;
            row[(c ^ (t & 7)) << 2] = h, row[((c + DK / 8) ^ (t & 7)) << 2] = l;
          }
        }
        fence_async();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (tid == 0) bulk_store(mats + w * mats_step, w_s, S::kKeyBytes);
      } else {  // u: 16 columns a warp and turn, all rows
        // T as a right operand, rows 8 n + g; unit: what takes rows 8 n + 2 t, 2 t + 1 back
        uint32_t th[4][2][2], tl[4][2][2];
        float unit[4][2];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          float2 y[2][2];
          uint32_t most = 0;
#pragma unroll
          for (int step = 0; step <= n / 2; ++step)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              y[step][c] = *reinterpret_cast<const float2*>(&hd[w].solve[8 * n + g][step * 16 + 8 * c + 2 * t4]);
              most = max(most, max(abs_bits(y[step][c].x), abs_bits(y[step][c].y)));
            }
          float up, mine;
          row_unit(quad_max(most), up, mine);
          unit[n][0] = __shfl_sync(0xFFFFFFFFu, mine, 8 * t4), unit[n][1] = __shfl_sync(0xFFFFFFFFu, mine, 8 * t4 + 4);
#pragma unroll
          for (int step = 0; step <= n / 2; ++step)
#pragma unroll
            for (int c = 0; c < 2; ++c) two_terms(y[step][c].x * up, y[step][c].y * up, th[n][step][c], tl[n][step][c]);
        }
        float4* const u = p.u + static_cast<size_t>(kh + (f0 + w) * p.k_heads) * (p.dv / 16) * p.chunks * 128;
#pragma unroll 1
        for (int c0 = first; c0 < p.dv; c0 += 64) {
          uint32_t ah[2][4], al[2][4];
          float unit_c[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t most = 0;
            float up;
#pragma unroll
            for (int i = 0; i < 8; ++i) most = max(most, abs_bits(v[e][i]));
            row_unit(quad_max(most), up, unit_c[e]);
#pragma unroll
            for (int i = 0; i < 4; ++i) two_terms(v[e][2 * i] * up, v[e][2 * i + 1] * up, ah[i >> 1][2 * (i & 1) + e], al[i >> 1][2 * (i & 1) + e]);
          }
          if (c0 + 64 < p.dv)
            load_values(w, c0 + 64);
          else if (w + 1 < heads)
            load_values(w + 1, first);
#pragma unroll
          for (int n = 0; n < 4; n += 2) {
            float hi[2][4] = {}, lo[2][4] = {};
#pragma unroll
            for (int step = 0; step <= n / 2; ++step) {
              const uint32_t bh[4] = {th[n][step][0], th[n][step][1], th[n + 1][step][0], th[n + 1][step][1]};
              const uint32_t bl[4] = {tl[n][step][0], tl[n][step][1], tl[n + 1][step][0], tl[n + 1][step][1]};
              mma3(hi[0], hi[1], lo[0], lo[1], ah[step], al[step], bh, bl);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float y[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) y[c] = (hi[e][c] + lo[e][c]) * (unit[n + e][c & 1] * unit_c[c >> 1]);
              u[(static_cast<size_t>(c0 / 16) * p.chunks + chunk) * 128 + (n + e) * 32 + lane] = make_float4(y[0], y[1], y[2], y[3]);
            }
          }
        }
      }
    }
    __syncthreads();
  }
  if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// grid: (value heads, columns / 16 / groups).  Four warps a group of 16 state columns: two carry half of dk each, two form the
// outputs of 16 rows each, a chunk behind: they find the state (as the operand of S^T W^T) and the corrections in shared memory.
constexpr int kMostGroups = 4;
template <int DK>
struct ScanShape {
  using S = ChunkShape<DK>;
  static constexpr int kSteps = DK / 32;  // of half of dk
  static constexpr int kStateBytes = 2 * S::kKeyBytes, kOutBytes = S::kKeyBytes + S::kMatBytes;
  // of a group, what a chunk hands over: two halves' operands, [half][step][term][lane], their columns' units, c
  static constexpr int kUnitAt = 2 * kSteps * 2 * 512, kCAt = kUnitAt + 512, kHand = kCAt + 4 * 512;
  static constexpr int kSumBytes = 2 * 4 * 512;  // two halves' sums
  static constexpr int kUBytes = 4 * 512;
  static constexpr int smem(int groups) { return 2 * (kStateBytes + kOutBytes) + 3 * static_cast<int>(sizeof(Factors)) + groups * (2 * kHand + kSumBytes + 2 * kUBytes); }
};
template <int DK, int GROUPS>
__global__ void __launch_bounds__(GROUPS * 128, 1) delta_chunk_scan_kernel(const DeltaChunkParams p) {
  using S = ChunkShape<DK>;
  using Z = ScanShape<DK>;
  constexpr int kTiles = DK / 16, kRowTiles = kChunk / 8;  // of half of dk; of the rows
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t full_s[2];
  unsigned char* const state_s = smem;                       // [2][K, W]
  unsigned char* const out_s = state_s + 2 * Z::kStateBytes;  // [2][Q, P]
  Factors* const fac_s = reinterpret_cast<Factors*>(out_s + 2 * Z::kOutBytes);  // [3]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int group = warp >> 2, role = (warp + 2 * group) & 3, half = role & 1;  // (a scheduler gets carriers and others)
  const int groups = blockDim.x >> 7;
  const bool carries = role < 2;
  unsigned char* const u_s = reinterpret_cast<unsigned char*>(fac_s + 3);  // [2][groups]
  unsigned char* const hand_s = u_s + groups * 2 * Z::kUBytes + group * (2 * Z::kHand + Z::kSumBytes);
  float4* const sums_s = reinterpret_cast<float4*>(hand_s + 2 * Z::kHand);
  const int h = blockIdx.x, kh = h % p.k_heads, col = (blockIdx.y * groups + group) * 16;
  const bool active = col < p.dv;
  const unsigned char* const keys = p.keys + static_cast<size_t>(kh) * p.chunks * 2 * S::kKeyBytes;
  const unsigned char* const mats = p.mats + static_cast<size_t>(h) * p.chunks * Z::kOutBytes;
  const Factors* const factors = p.factors + static_cast<size_t>(h) * p.chunks;
  const float4* const u = p.u + (static_cast<size_t>(h) * (p.dv / 16) + blockIdx.y * groups) * p.chunks * 128;
  const int own_groups = min(groups, p.dv / 16 - static_cast<int>(blockIdx.y) * groups);
  // bulk copies by one thread, the state's operands of a chunk with the outputs' of the one before it
  auto stage = [&](int chunk) {
    uint64_t* const bar = &full_s[chunk & 1];
    const unsigned char* const key = keys + static_cast<size_t>(chunk) * 2 * S::kKeyBytes;
    const unsigned char* const mat = mats + static_cast<size_t>(chunk) * Z::kOutBytes;
    mbar_expect_tx(bar, (chunk < p.chunks ? Z::kStateBytes + sizeof(Factors) + own_groups * Z::kUBytes : 0) + (chunk > 0 ? Z::kOutBytes : 0));
    if (chunk < p.chunks) {
      unsigned char* const dst = state_s + (chunk & 1) * Z::kStateBytes;
      bulk_load(dst + S::kKeyBytes, mat, S::kKeyBytes, bar);
      bulk_load(dst, key, S::kKeyBytes, bar);
      bulk_load(fac_s + chunk % 3, factors + chunk, sizeof(Factors), bar);
      for (int i = 0; i < own_groups; ++i)
        bulk_load(u_s + ((chunk & 1) * groups + i) * Z::kUBytes, u + (static_cast<size_t>(i) * p.chunks + chunk) * 128, Z::kUBytes, bar);
    }
    if (chunk > 0) {
      unsigned char* const dst = out_s + (chunk & 1 ^ 1) * Z::kOutBytes;
      bulk_load(dst, key - S::kKeyBytes, S::kKeyBytes, bar);
      bulk_load(dst + S::kKeyBytes, mat - S::kMatBytes, S::kMatBytes, bar);
    }
  };
  // o: (row 8 n + 2 t + {0, 1}, columns g and g + 8)
  const size_t o_step = static_cast<size_t>(p.heads) * p.dv, o_at = static_cast<size_t>(h) * p.dv + col + g;
  float s[kTiles][4];  // S^T: columns g, g + 8 of the state, rows 8 n + 2 t + {0, 1} of this half
  const size_t state = (static_cast<size_t>(h) * DK + half * (DK / 2)) * p.dv + col + g;
  if (carries && active) {  // (the kernel before this one does not write it, and has waited for those that may have)
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[n][c] = __ldcg(p.s + state + static_cast<size_t>(8 * n + 2 * t + (c & 1)) * p.dv + 8 * (c >> 1));
  }
  const bool stages = warp == 2 && lane == 0;  // (of a warp that does not carry)
  if (stages) {
    mbar_init(&full_s[0], 1), mbar_init(&full_s[1], 1);
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  if (stages) stage(0);
  bool ok = true;
  // matrices of an ldmatrix: rows 0-7 / 8-15 (lane / 16), first / second eight elements of a step (lane / 8 % 2)
  const int br = (lane & 7) + ((lane >> 4) << 3), bc = (lane >> 3) & 1;
  // ... key rows 0-7 / 8-15 of the step (lane / 8 % 2), elements 0-7 / 8-15 (lane / 16)
  const int ur = lane & 15, uc = lane >> 4;

  for (int chunk = 0; chunk <= p.chunks; ++chunk) {
    if (ok) ok = mbar_wait(&full_s[chunk & 1], chunk >> 1 & 1, &g_delta_timeouts);
    // The chunk is there for everybody, and everybody is done with the ones before.
    if (!__syncthreads_and(ok)) {  // a copy did not come: a millisecond for those under way
      const long long begin = clock64();
      while (clock64() - begin < 2000000) {
      }
      return;
    }
    if (stages && chunk < p.chunks) stage(chunk + 1);
    if (!active) continue;
    if (carries) {
      if (chunk == p.chunks) break;  // (the last iteration)
      const uint32_t k_at = smem_u32(state_s) + (chunk & 1) * Z::kStateBytes, w_at = k_at + S::kKeyBytes;
      const Factors* const f = fac_s + chunk % 3;
      unsigned char* const hand = hand_s + (chunk & 1) * Z::kHand;
      float x[kRowTiles][4];  // c
      {
        float hi[kRowTiles][4] = {}, lo[kRowTiles][4] = {};
        uint32_t bh[2][kRowTiles / 2][4], bl[2][kRowTiles / 2][4];  // a step ahead
        auto load = [&](int step) {
#pragma unroll
          for (int pair = 0; pair < kRowTiles / 2; ++pair) {
            const int r = pair * 16 + br, c = half * (DK / 16) + step * 2 + bc;
            load_matrices(bh[step & 1][pair], w_at + r * S::kRowBytes + ((c ^ (r & 7)) << 4));
            load_matrices(bl[step & 1][pair], w_at + r * S::kRowBytes + (((c + DK / 8) ^ (r & 7)) << 4));
          }
        };
        load(0);
        uint32_t most[2] = {0, 0};
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) most[c >> 1] = max(most[c >> 1], abs_bits(s[n][c]));
        float up[2], unit[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) row_unit(quad_max(most[v]), up[v], unit[v]);
        uint4* const op = reinterpret_cast<uint4*>(hand) + half * Z::kSteps * 64 + lane;
#pragma unroll
        for (int step = 0; step < Z::kSteps; ++step) {
          uint32_t ah[4], al[4];
          if (step + 1 < Z::kSteps) load(step + 1);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float(&y)[4] = s[2 * step + e];
            two_terms(y[0] * up[0], y[1] * up[0], ah[2 * e], al[2 * e]);
            two_terms(y[2] * up[1], y[3] * up[1], ah[2 * e + 1], al[2 * e + 1]);
          }
          op[step * 64] = make_uint4(ah[0], ah[1], ah[2], ah[3]);
          op[step * 64 + 32] = make_uint4(al[0], al[1], al[2], al[3]);
#pragma unroll
          for (int pair = 0; pair < kRowTiles / 2; ++pair)
            mma3(hi[2 * pair], hi[2 * pair + 1], lo[2 * pair], lo[2 * pair + 1], ah, al, bh[step & 1][pair], bl[step & 1][pair]);
        }
        reinterpret_cast<float2*>(hand + Z::kUnitAt)[half * 32 + lane] = make_float2(unit[0], unit[1]);
        float own[kRowTiles][4];  // u of half 0, less the halves' products
        const float4* const u_at = reinterpret_cast<const float4*>(u_s + ((chunk & 1) * groups + group) * Z::kUBytes) + lane;
#pragma unroll
        for (int n = 0; n < kRowTiles; ++n) {
          const float2 fs = *reinterpret_cast<const float2*>(&f->solve[half][8 * n + 2 * t]);
          const float4 un = half == 0 ? u_at[n * 32] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          own[n][0] = fmaf(hi[n][0] + lo[n][0], -unit[0] * fs.x, un.x), own[n][1] = fmaf(hi[n][1] + lo[n][1], -unit[0] * fs.y, un.y);
          own[n][2] = fmaf(hi[n][2] + lo[n][2], -unit[1] * fs.x, un.z), own[n][3] = fmaf(hi[n][3] + lo[n][3], -unit[1] * fs.y, un.w);
          sums_s[(half * kRowTiles + n) * 32 + lane] = make_float4(own[n][0], own[n][1], own[n][2], own[n][3]);
        }
        asm volatile("bar.sync %0, 64;" ::"r"(1 + group) : "memory");
#pragma unroll
        for (int n = 0; n < kRowTiles; ++n) {
          const float4 other = sums_s[((half ^ 1) * kRowTiles + n) * 32 + lane];
          x[n][0] = own[n][0] + other.x, x[n][1] = own[n][1] + other.y, x[n][2] = own[n][2] + other.z, x[n][3] = own[n][3] + other.w;
          if (n >> 1 == half) reinterpret_cast<float4*>(hand + Z::kCAt)[n * 32 + lane] = make_float4(x[n][0], x[n][1], x[n][2], x[n][3]);
        }
      }
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
        const float2 fp = *reinterpret_cast<const float2*>(&f->put[8 * n + 2 * t]);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[n][c] *= (c & 1) ? fp.y : fp.x;
      }
      uint32_t key_hi[2][kChunk / 16][4], key_lo[2][kChunk / 16][4];  // 16 elements of the keys, ahead
      auto load_keys = [&](int pair) {
#pragma unroll
        for (int step = 0; step < kChunk / 16; ++step) {
          const int r = step * 16 + ur, c = half * (DK / 16) + pair * 2 + uc;
          load_matrices_turned(key_hi[pair & 1][step], k_at + r * S::kRowBytes + ((c ^ (r & 7)) << 4));
          load_matrices_turned(key_lo[pair & 1][step], k_at + r * S::kRowBytes + (((c + DK / 8) ^ (r & 7)) << 4));
        }
      };
      load_keys(0);
      uint32_t ah[kRowTiles / 2][4], al[kRowTiles / 2][4];
      float unit[2];
      as_operand<kRowTiles>(x, ah, al, unit);
      const float keep = f->state;
#pragma unroll
      for (int pair = 0; pair < kTiles / 2; ++pair) {
        float hi[2][4] = {}, lo[2][4] = {};
        if (pair + 1 < kTiles / 2) load_keys(pair + 1);
#pragma unroll
        for (int step = 0; step < kChunk / 16; ++step) mma3(hi[0], hi[1], lo[0], lo[1], ah[step], al[step], key_hi[pair & 1][step], key_lo[pair & 1][step]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[2 * pair + e][c] = fmaf(hi[e][c] + lo[e][c], unit[c >> 1], keep * s[2 * pair + e][c]);
      }
    } else if (chunk > 0) {
      const int done = chunk - 1, t0 = done * kChunk, r = half * 16 + br;  // `half` of the rows
      const uint32_t q_at = smem_u32(out_s) + (done & 1) * Z::kOutBytes + r * S::kRowBytes;
      const uint32_t p_at = smem_u32(out_s) + (done & 1) * Z::kOutBytes + S::kKeyBytes + r * 4 * kChunk;
      const Factors* const f = fac_s + done % 3;
      const unsigned char* const hand = hand_s + (done & 1) * Z::kHand;
      float o[2][4] = {};
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        float hi[2][4] = {}, lo[2][4] = {};
#pragma unroll
        for (int step = 0; step < Z::kSteps; ++step) {
          const uint4* const op = reinterpret_cast<const uint4*>(hand) + (part * Z::kSteps + step) * 64 + lane;
          const uint4 a = op[0], b = op[32];
          const uint32_t ah[4] = {a.x, a.y, a.z, a.w}, al[4] = {b.x, b.y, b.z, b.w};
          const int c = part * (DK / 16) + step * 2 + bc;
          uint32_t bh[4], bl[4];
          load_matrices(bh, q_at + ((c ^ (r & 7)) << 4));
          load_matrices(bl, q_at + (((c + DK / 8) ^ (r & 7)) << 4));
          mma3(hi[0], hi[1], lo[0], lo[1], ah, al, bh, bl);
        }
        const float2 unit = reinterpret_cast<const float2*>(hand + Z::kUnitAt)[part * 32 + lane];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[n][c] = fmaf(hi[n][c] + lo[n][c], c >> 1 ? unit.y : unit.x, o[n][c]);
      }
      float x[kRowTiles][4];
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) *reinterpret_cast<float4*>(x[n]) = reinterpret_cast<const float4*>(hand + Z::kCAt)[n * 32 + lane];
      uint32_t ah[kRowTiles / 2][4], al[kRowTiles / 2][4];
      float unit[2], hi[2][4] = {}, lo[2][4] = {};
      as_operand<kRowTiles>(x, ah, al, unit);
#pragma unroll
      for (int step = 0; step < kChunk / 16; ++step) {
        if (step > half) continue;  // P is a lower triangle
        uint32_t bh[4], bl[4];
        load_matrices(bh, p_at + (((step * 2 + bc) ^ (r & 7)) << 4));
        load_matrices(bl, p_at + (((step * 2 + bc + kChunk / 8) ^ (r & 7)) << 4));
        mma3(hi[0], hi[1], lo[0], lo[1], ah[step], al[step], bh, bl);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int at = half * 16 + 8 * n + 2 * t;
        const float2 fq = *reinterpret_cast<const float2*>(&f->query[at]), fo = *reinterpret_cast<const float2*>(&f->out[at]);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (t0 + at + (c & 1) < p.rows)
            p.o[(t0 + at + (c & 1)) * o_step + o_at + 8 * (c >> 1)] =
                fmaf(hi[n][c] + lo[n][c], unit[c >> 1] * ((c & 1) ? fo.y : fo.x), o[n][c] * ((c & 1) ? fq.y : fq.x));
      }
    }
  }
  if (!active || !carries) return;
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) p.s_out[state + static_cast<size_t>(8 * n + 2 * t + (c & 1)) * p.dv + 8 * (c >> 1)] = s[n][c];
}

template <int DK>
int launch_delta_chunk(DeltaChunkParams p, cudaStream_t st) {
  using S = ChunkShape<DK>;
  using Z = ScanShape<DK>;
  // Long prompts in pieces of kMostChunks, which bound the workspace.  It comes in three sizes, 4, 16 and 64 chunks, since a stream
  // keeps the smaller ones when it grows (48 heads over 16 key heads of 128: 9, 37 and 149 MB).
  const int rows = p.rows;
  int most = 4;
  while (most < kMostChunks && most * kChunk < rows) most *= 4;
  const size_t key_bytes = static_cast<size_t>(p.k_heads) * most * 2 * S::kKeyBytes;
  const size_t mat_bytes = static_cast<size_t>(p.heads) * most * Z::kOutBytes;
  const size_t factor_bytes = static_cast<size_t>(p.heads) * most * sizeof(Factors);
  const size_t u_bytes = static_cast<size_t>(p.heads) * most * kChunk * p.dv * 4;
  unsigned char* scratch = stream_scratch(st, key_bytes + mat_bytes + u_bytes + factor_bytes, kScratchDelta);
  if (scratch == nullptr) return kUnsupportedFeature;  // a capture before the first plain launch of this size
  p.keys = scratch, p.mats = scratch + key_bytes;
  p.u = reinterpret_cast<float4*>(scratch + key_bytes + mat_bytes);
  p.factors = reinterpret_cast<Factors*>(scratch + key_bytes + mat_bytes + u_bytes);
  // The scan's CTAs as narrow as one wave of them allows, so that fewer warps share a scheduler (a chunk of 32 columns a CTA
  // 2.0 us, of 48 2.9 us).
  int groups = 2;
  while (groups < kMostGroups && static_cast<long long>(p.heads) * ((p.dv + 16 * groups - 1) / (16 * groups)) > kSms) ++groups;
  constexpr int kPrepMost = 2 * S::kKeyBytes + static_cast<int>(sizeof(PrepShared)) + kPrepHeads * static_cast<int>(sizeof(PrepHead));
  static_assert(2 * kPrepMost <= 226 * 1024 && Z::smem(kMostGroups) <= 227 * 1024, "shared memory of an SM");
  const auto scan = groups == 2 ? delta_chunk_scan_kernel<DK, 2> : groups == 3 ? delta_chunk_scan_kernel<DK, 3> : delta_chunk_scan_kernel<DK, 4>;
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(scan), Z::smem(groups))) return rc;
  for (int r0 = 0; r0 < rows; r0 += kMostChunks * kChunk) {
    p.rows = min(rows - r0, kMostChunks * kChunk);
    p.chunks = (p.rows + kChunk - 1) / kChunk;
    // Where that leaves SMs without a CTA, the value heads of a key head are spread over several (33 rows: 3 of 19 us).
    const int factor = p.heads / p.k_heads, parts = max(1, min(factor, kSms / (p.chunks * p.k_heads))), per = (factor + parts - 1) / parts;
    const int prep_smem = 2 * S::kKeyBytes + static_cast<int>(sizeof(PrepShared)) + min(kPrepHeads, per) * static_cast<int>(sizeof(PrepHead));
    // one CTA an SM: 255 registers a thread against 128 (64 rows: 20.6 us against 22.6; 2048 rows, seven CTAs an SM: 192 against 181)
    const auto prepare = p.chunks * p.k_heads * ((factor + per - 1) / per) <= kSms ? delta_chunk_prepare_kernel<DK, 1> : delta_chunk_prepare_kernel<DK, 2>;
    if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(prepare), kPrepMost)) return rc;  // (once a kernel: the most it may ask for)
    const void* const out[2] = {p.o, p.s_out};
    const size_t out_bytes[2] = {static_cast<size_t>(p.rows) * p.heads * p.dv * 4, static_cast<size_t>(p.heads) * DK * p.dv * 4};
    const bool pdl = pdl_allowed_ranges(st, nullptr, nullptr, 0, out, out_bytes, 2);
    if (launch_kernel(prepare, dim3(static_cast<unsigned>(p.chunks), static_cast<unsigned>(p.k_heads), static_cast<unsigned>((factor + per - 1) / per)), dim3(kPrepThreads), static_cast<size_t>(prep_smem), st,
                      pdl, p) != cudaSuccess) {
      cudaGetLastError();
      return kDeviceError;
    }
    if (int rc = check_launch()) return rc;
    // (may start once the first kernel's CTAs have: it loads the state, which they do not write, and waits)
    if (launch_kernel(scan, dim3(static_cast<unsigned>(p.heads), static_cast<unsigned>((p.dv + 16 * groups - 1) / (16 * groups))), dim3(128 * groups),
                      Z::smem(groups), st, true, p) != cudaSuccess) {
      cudaGetLastError();
      return kDeviceError;
    }
    if (int rc = check_launch()) return rc;
    const size_t taken = p.rows;
    p.k += taken * p.k_heads * DK, p.q += taken * p.k_heads * DK, p.v += taken * p.heads * p.dv, p.o += taken * p.heads * p.dv;
    p.alpha += taken * p.heads, p.beta += taken * p.heads;
    p.s = p.s_out;
  }
  return kOk;
}

}  // namespace

int delta_wait_timeouts(unsigned int* count) {
  return cudaMemcpyFromSymbol(count, g_delta_timeouts, sizeof(*count)) == cudaSuccess ? kOk : kDeviceError;
}
int delta_set_error_word(unsigned int* word) { return set_host_error_word(word); }

int delta_chunk_heads(const float* s, const float* k, const float* v, const float* q, float* o, const float* alpha,
                                     const float* beta, float* s_out, uint64_t heads, uint64_t k_heads, uint64_t dk, uint64_t dv, uint64_t rows,
                                     uint64_t sbase, uint64_t abase, bool dry, cudaStream_t st) {
  if (!s || !k || !v || !q || !o || !alpha || !beta || !s_out || heads == 0 || heads > 65535 || k_heads == 0 || heads % k_heads != 0 || dk == 0 ||
      dk > 65535 || dv == 0 || dv > 65535 || rows == 0 || rows > 0x7FFFFFFFull - kChunk)
    return kInvalidArgument;
  if ((dk != 64 && dk != 128) || dv % 16 != 0) return kUnsupportedFeature;
  const uint64_t state = heads * dk * dv;
  struct {
    const float* at;
    uint64_t count;
  } const in[6] = {{k, rows * k_heads * dk}, {q, rows * k_heads * dk}, {v, rows * heads * dv}, {alpha + abase, rows * heads}, {beta + abase, rows * heads}, {s + sbase, state}},
          out[2] = {{o, rows * heads * dv}, {s_out + sbase, state}};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 6; ++j) {
      if (i == 1 && j == 5 && s_out == s) continue;  // the state in place
      if (in[j].at < out[i].at + out[i].count && out[i].at < in[j].at + in[j].count) return kInvalidArgument;
    }
  if (out[0].at < out[1].at + out[1].count && out[1].at < out[0].at + out[0].count) return kInvalidArgument;
  if (dry) return kOk;
  DeltaChunkParams p{};
  p.s = s + sbase, p.k = k, p.v = v, p.q = q, p.alpha = alpha + abase, p.beta = beta + abase, p.o = o, p.s_out = s_out + sbase;
  p.heads = static_cast<int>(heads), p.k_heads = static_cast<int>(k_heads), p.dv = static_cast<int>(dv), p.rows = static_cast<int>(rows);
  return dk == 128 ? launch_delta_chunk<128>(p, st) : launch_delta_chunk<64>(p, st);
}

}  // namespace tsr

extern "C" int tsr_delta_chunk_heads(const float* s, const float* k, const float* v, const float* q, float* o, const float* alpha,
                                     const float* beta, float* s_out, uint64_t heads, uint64_t k_heads, uint64_t dk, uint64_t dv, uint64_t rows,
                                     uint64_t sbase, uint64_t abase, void* stream) {
  return tsr::delta_chunk_heads(s, k, v, q, o, alpha, beta, s_out, heads, k_heads, dk, dv, rows, sbase, abase, false,
                                static_cast<cudaStream_t>(stream));
}
