// The gated delta rule over many rows in its chunked form (id "delta_chunk_heads"): what delta_step_heads computes row by row
// (DeltaStepHeadsRef, src/core/numerics/attention.cpp:290-334 of the reference), for a prompt's chunk or a chain of drafted
// tokens.  Per head, with state S (dk x dv), c_t = beta_t (v_t - alpha_t S_{t-1}^T k_t):
//   S_t = alpha_t S_{t-1} + k_t c_t^T,   o_t = S_t^T q_t.
// Over a chunk of 32 rows that starts from S, with G(t, s) = prod_{s < r <= t} alpha_r and g_t = G(t, start):
//   c_t + beta_t sum_{s < t} G(t, s) (k_s . k_t) c_s = beta_t (v_t - g_t S^T k_t)      a unit lower triangular system
//   o_t = g_t S^T q_t + sum_{s <= t} G(t, s) (k_s . q_t) c_s,    S' = g_C S + sum_s G(C, s) k_s c_s^T.
// The decays are products, not exponentials of differences of logarithms, so alpha = 0 and products that underflow are exact.
//
// Two launches.  delta_chunk_prepare: all chunks at once, what does not depend on the state: the inverse of the system
// (forward substitution, a lane a column), the weights G (k . q), and keys and queries as two binary16 terms.  A key head's
// Gram matrices serve all value heads that share it.  delta_chunk_scan: the chunks in turn.  A warp owns 16 state columns
// (S^T, 16 x dk, in registers as fp32) and never waits for another one: S^T K^T, S^T Q^T, the system's solution, the outputs and
// the update are m16n8k16 binary16 MMAs whose left operand is made of registers, the accumulators' layout being that operand's.
// Each operand enters as two binary16 terms of a row scaled by a power of two, 22 bits below the row's largest element, and
// three products of terms; small products have accumulators of their own (the MMA cuts off what falls below its
// accumulator).
#include <cuda_fp16.h>

#include "codec.cuh"
#include "launch.h"
#include "tessera_b200.h"

namespace tsr {
namespace {

constexpr int kChunk = 32;                 // rows
constexpr int kPrepThreads = 256;
constexpr int kMostChunks = 128;           // of a pair of launches
constexpr int kScanWarps = 4, kScanThreads = kScanWarps * 32, kScanCols = 16 * kScanWarps;

// One chunk's operands, in the order the scan copies them: keys and queries (per key head), then the solution's and the
// output's matrices (per value head).  Every row: the leading terms, then the rest.
template <int DK>
struct ChunkShape {
  static constexpr int kRowHalves = 2 * DK;
  static constexpr int kKeyHalves = kChunk * kRowHalves;            // of K or Q
  static constexpr int kMatHalves = kChunk * 2 * kChunk;            // of T or P
  static constexpr int kHeadFloats = 5 * kChunk + 4;                // per value head: see Factors
  static constexpr int kKeyBytes = kKeyHalves * 2, kMatBytes = kMatHalves * 2;
  static constexpr int kFactorBytes = (kHeadFloats * 4 + 15) / 16 * 16;
  static constexpr int kStage = 2 * kKeyBytes + 2 * kMatBytes + kFactorBytes;  // bytes of a chunk in shared memory
};
// What a chunk's columns of results are multiplied by: the decay with the power of two that takes an operand's row back.
struct Factors {
  float key[kChunk];   // g_t 2^e(k_t): of S^T k_t
  float query[kChunk]; // g_t 2^e(q_t): of S^T q_t
  float solve[kChunk]; // 2^e(T_t)
  float out[kChunk];   // 2^e(P_t)
  float put[kChunk];   // G(C, s) 2^e(k_s): of c_s in the update
  float state;         // g_C
  float unused[3];
};
static_assert(sizeof(Factors) == (5 * kChunk + 4) * 4, "as copied");

struct DeltaChunkParams {
  const float *s, *k, *v, *q, *alpha, *beta;  // s, alpha, beta at their bases
  float *o, *s_out;
  __half *keys, *mats;  // [key head][chunk][K, Q], [head][chunk][T, P]
  Factors* factors;     // [head][chunk]
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

// grid: (chunks, key heads)
template <int DK>
__global__ void __launch_bounds__(kPrepThreads) delta_chunk_prepare_kernel(const DeltaChunkParams p) {
  using S = ChunkShape<DK>;
  constexpr int kPitch = DK + 4;
  // K and Q, until their products are formed; then each warp's system
  constexpr int kRowsFloats = 2 * kChunk * kPitch, kLowFloats = kPrepThreads / 32 * kChunk * (kChunk + 4);
  __shared__ __align__(16) float both_s[kRowsFloats > kLowFloats ? kRowsFloats : kLowFloats];
  __shared__ float gram_s[2][kChunk][kChunk + 1];  // k_t . k_s and q_t . k_s
  __shared__ float unit_s[2][kChunk];
  auto* const rows_s = reinterpret_cast<float(*)[kChunk][kPitch]>(both_s);
  auto* const low_s = reinterpret_cast<float(*)[kChunk][kChunk + 4]>(both_s);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunk = blockIdx.x, kh = blockIdx.y, t0 = chunk * kChunk, rows = min(kChunk, p.rows - t0);
  // a warp a row: as it is to shared memory, as two terms to the workspace
  for (int r = warp; r < 2 * kChunk; r += kPrepThreads / 32) {
    const int which = r / kChunk, t = r % kChunk;
    const float* src = (which ? p.q : p.k) + (static_cast<size_t>(t0 + t) * p.k_heads + kh) * DK;
    float x[DK / 32];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) {
      x[2 * i] = x[2 * i + 1] = 0.0f;
      if (t < rows) x[2 * i] = src[i * 64 + lane * 2], x[2 * i + 1] = src[i * 64 + lane * 2 + 1];
      most = max(most, max(abs_bits(x[2 * i]), abs_bits(x[2 * i + 1])));
    }
    float up, unit;
    row_unit(__reduce_max_sync(0xFFFFFFFFu, most), up, unit);
    if (lane == 0) unit_s[which][t] = unit;
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.keys + (static_cast<size_t>(kh) * p.chunks + chunk) * 2 * S::kKeyHalves +
                                                which * S::kKeyHalves + t * S::kRowHalves);
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) {
      rows_s[which][t][i * 64 + lane * 2] = x[2 * i], rows_s[which][t][i * 64 + lane * 2 + 1] = x[2 * i + 1];
      uint32_t hi, lo;
      two_terms(x[2 * i] * up, x[2 * i + 1] * up, hi, lo);
      dst[i * 32 + lane] = hi, dst[DK / 2 + i * 32 + lane] = lo;
    }
  }
  __syncthreads();
  {
    const int t = tid / 8, s0 = tid % 8;
    float kk[4] = {}, qk[4] = {};
#pragma unroll 4
    for (int d = 0; d < DK; d += 4) {
      const float4 a = *reinterpret_cast<const float4*>(&rows_s[0][t][d]), b = *reinterpret_cast<const float4*>(&rows_s[1][t][d]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 c = *reinterpret_cast<const float4*>(&rows_s[0][s0 + 8 * j][d]);
        kk[j] = fmaf(a.x, c.x, fmaf(a.y, c.y, fmaf(a.z, c.z, fmaf(a.w, c.w, kk[j]))));
        qk[j] = fmaf(b.x, c.x, fmaf(b.y, c.y, fmaf(b.z, c.z, fmaf(b.w, c.w, qk[j]))));
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) gram_s[0][t][s0 + 8 * j] = kk[j], gram_s[1][t][s0 + 8 * j] = qk[j];
  }
  __syncthreads();
  // a warp a value head; a lane a column s
  for (int h = kh + warp * p.k_heads; h < p.heads; h += (kPrepThreads / 32) * p.k_heads) {
    const size_t at = static_cast<size_t>(t0 + lane) * p.heads + h;
    const float alpha = lane < rows ? p.alpha[at] : 1.0f, beta = lane < rows ? p.beta[at] : 0.0f;
    uint32_t* mats = reinterpret_cast<uint32_t*>(p.mats + (static_cast<size_t>(h) * p.chunks + chunk) * 2 * S::kMatHalves);
    Factors* f = p.factors + static_cast<size_t>(h) * p.chunks + chunk;
    float decay = 0.0f, start = 1.0f;  // G(t, lane), g_t
    // rows of P on the way: G(t, s) (k_s . q_t); pairs of columns meet in the even lane
    auto store_row = [&](uint32_t* row, float x, float* factor) {
      float up, unit;
      row_unit(__reduce_max_sync(0xFFFFFFFFu, abs_bits(x)), up, unit);
      const float y = __shfl_xor_sync(0xFFFFFFFFu, x, 1);
      uint32_t hi, lo;
      two_terms(x * up, y * up, hi, lo);
      if ((lane & 1) == 0) row[lane / 2] = hi, row[kChunk / 2 + lane / 2] = lo;
      if (lane == 0) *factor = unit;
    };
#pragma unroll 4
    for (int t = 0; t < kChunk; ++t) {
      const float a = __shfl_sync(0xFFFFFFFFu, alpha, t), b = __shfl_sync(0xFFFFFFFFu, beta, t);
      decay = lane == t ? 1.0f : lane < t ? decay * a : 0.0f;
      start *= a;
      low_s[warp][t][lane] = lane < t ? b * decay * gram_s[0][t][lane] : 0.0f;
      store_row(mats + S::kMatHalves / 2 + t * kChunk, lane <= t ? decay * gram_s[1][t][lane] : 0.0f, &f->out[t]);
      if (lane == 0) f->key[t] = start * unit_s[0][t], f->query[t] = start * unit_s[1][t];
    }
    f->put[lane] = decay * unit_s[0][lane];
    if (lane == 0) f->state = start;
    __syncwarp();
    float x[kChunk];
#pragma unroll
    for (int t = 0; t < kChunk; ++t) {
      float sum = lane == t ? 1.0f : 0.0f, more = 0.0f;
#pragma unroll
      for (int s = 0; s < t; s += 2) {
        sum = fmaf(-low_s[warp][t][s], x[s], sum);
        if (s + 1 < t) more = fmaf(-low_s[warp][t][s + 1], x[s + 1], more);
      }
      x[t] = lane <= t ? sum + more : 0.0f;
    }
    for (int t = 0; t < kChunk; ++t) {
      float y = 0.0f;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) y = i == t ? x[i] : y;
      store_row(mats + t * kChunk, y * beta, &f->solve[t]);
    }
    __syncwarp();
  }
}

__device__ __forceinline__ uint32_t shared_of(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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

// grid: (value heads, columns / 64)
template <int DK>
__global__ void __launch_bounds__(kScanThreads, 1) delta_chunk_scan_kernel(const DeltaChunkParams p) {
  using S = ChunkShape<DK>;
  constexpr int kTiles = DK / 8, kRowTiles = kChunk / 8;
  extern __shared__ __align__(128) unsigned char smem[];  // two stages
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int h = blockIdx.x, kh = h % p.k_heads, col = blockIdx.y * kScanCols + warp * 16;
  const bool active = col < p.dv;
  // 16-byte piece c of row r at c ^ (r & 7): ldmatrix is conflict-free
  auto stage = [&](int chunk) {
    const uint32_t dst = shared_of(smem) + (chunk & 1) * S::kStage;
    const unsigned char* keys = reinterpret_cast<const unsigned char*>(p.keys + (static_cast<size_t>(kh) * p.chunks + chunk) * 2 * S::kKeyHalves);
    const unsigned char* mats = reinterpret_cast<const unsigned char*>(p.mats + (static_cast<size_t>(h) * p.chunks + chunk) * 2 * S::kMatHalves);
    const unsigned char* fac = reinterpret_cast<const unsigned char*>(p.factors + static_cast<size_t>(h) * p.chunks + chunk);
    constexpr int kPieces = S::kRowHalves / 8;
#pragma unroll 4
    for (int i = tid; i < 2 * S::kKeyBytes / 16; i += kScanThreads) {
      const int r = i / kPieces, c = i % kPieces;
      copy16(dst + r * S::kRowHalves * 2 + ((c ^ (r & 7)) << 4), keys + i * 16);
    }
#pragma unroll
    for (int i = tid; i < 2 * S::kMatBytes / 16; i += kScanThreads) {
      const int r = i / 8, c = i % 8;
      copy16(dst + 2 * S::kKeyBytes + r * 128 + ((c ^ (r & 7)) << 4), mats + i * 16);
    }
    if (tid < S::kFactorBytes / 16) copy16(dst + 2 * S::kKeyBytes + 2 * S::kMatBytes + tid * 16, fac + tid * 16);
  };
  stage(0);
  asm volatile("cp.async.commit_group;" ::: "memory");
  // values: (row 8 n + 2 t + {0, 1}, columns g and g + 8)
  float v_next[kRowTiles][4];
  const size_t v_step = static_cast<size_t>(p.heads) * p.dv, v_at = static_cast<size_t>(h) * p.dv + col + g;
  auto load_values = [&](int t0) {
#pragma unroll
    for (int n = 0; n < kRowTiles; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int r = t0 + 8 * n + 2 * t + (c & 1);
        v_next[n][c] = active && r < p.rows ? p.v[r * v_step + v_at + 8 * (c >> 1)] : 0.0f;
      }
  };
  load_values(0);
  float s[kTiles][4];  // S^T: columns g, g + 8 of the state, its rows 8 n + 2 t + {0, 1}
  const size_t state = static_cast<size_t>(h) * DK * p.dv + col + g;
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      s[n][c] = active ? p.s[state + static_cast<size_t>(8 * n + 2 * t + (c & 1)) * p.dv + 8 * (c >> 1)] : 0.0f;

  for (int chunk = 0; chunk < p.chunks; ++chunk) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the chunk is there for everybody, and everybody is done with the one before
    if (chunk + 1 < p.chunks) stage(chunk + 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (!active) continue;
    const unsigned char* const base = smem + (chunk & 1) * S::kStage;
    const uint32_t k_at = shared_of(base), q_at = k_at + S::kKeyBytes, t_at = q_at + S::kKeyBytes, p_at = t_at + S::kMatBytes;
    const Factors* f = reinterpret_cast<const Factors*>(base + 2 * S::kKeyBytes + 2 * S::kMatBytes);
    float x[kRowTiles][4], o[kRowTiles][4];  // v - g S^T k, then its solution c; outputs
    {
      float k_hi[kRowTiles][4] = {}, k_lo[kRowTiles][4] = {}, q_hi[kRowTiles][4] = {}, q_lo[kRowTiles][4] = {};
      uint32_t most[2] = {0, 0};
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) most[c >> 1] = max(most[c >> 1], abs_bits(s[n][c]));
      float up[2], unit[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        most[u] = max(most[u], __shfl_xor_sync(0xFFFFFFFFu, most[u], 1));
        most[u] = max(most[u], __shfl_xor_sync(0xFFFFFFFFu, most[u], 2));
        row_unit(most[u], up[u], unit[u]);
      }
      // matrices of an ldmatrix: rows 0-7 / 8-15 (lane / 16), first / second eight elements of the step (lane / 8 % 2)
      const int br = (lane & 7) + ((lane >> 4) << 3), bc = (lane >> 3) & 1;
#pragma unroll
      for (int step = 0; step < DK / 16; ++step) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float(&y)[4] = s[2 * step + half];
          two_terms(y[0] * up[0], y[1] * up[0], ah[2 * half], al[2 * half]);
          two_terms(y[2] * up[1], y[3] * up[1], ah[2 * half + 1], al[2 * half + 1]);
        }
#pragma unroll
        for (int pair = 0; pair < kRowTiles / 2; ++pair) {
          const int r = pair * 16 + br;
          const uint32_t hi_at = r * S::kRowHalves * 2 + (((step * 2 + bc) ^ (r & 7)) << 4);
          const uint32_t lo_at = r * S::kRowHalves * 2 + (((step * 2 + bc + DK / 8) ^ (r & 7)) << 4);
          uint32_t bh[4], bl[4];
          load_matrices(bh, k_at + hi_at);
          load_matrices(bl, k_at + lo_at);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mma(k_lo[2 * pair + e], al, bh[2 * e], bh[2 * e + 1]);
            mma(k_hi[2 * pair + e], ah, bh[2 * e], bh[2 * e + 1]);
            mma(k_lo[2 * pair + e], ah, bl[2 * e], bl[2 * e + 1]);
          }
          load_matrices(bh, q_at + hi_at);
          load_matrices(bl, q_at + lo_at);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mma(q_lo[2 * pair + e], al, bh[2 * e], bh[2 * e + 1]);
            mma(q_hi[2 * pair + e], ah, bh[2 * e], bh[2 * e + 1]);
            mma(q_lo[2 * pair + e], ah, bl[2 * e], bl[2 * e + 1]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
        const float2 fk = *reinterpret_cast<const float2*>(&f->key[8 * n + 2 * t]), fq = *reinterpret_cast<const float2*>(&f->query[8 * n + 2 * t]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x[n][c] = fmaf(-(k_hi[n][c] + k_lo[n][c]), unit[c >> 1] * ((c & 1) ? fk.y : fk.x), v_next[n][c]);
          o[n][c] = (q_hi[n][c] + q_lo[n][c]) * (unit[c >> 1] * ((c & 1) ? fq.y : fq.x));
        }
      }
    }
    const int t0 = chunk * kChunk;
    load_values(t0 + kChunk);  // (rows beyond the last are not read)
    // y = x M^T of a 32 x 32 matrix M whose rows are given as two terms
    auto times = [&](const float (&a)[kRowTiles][4], uint32_t m_at, float (&hi)[kRowTiles][4], float (&lo)[kRowTiles][4], float (&unit)[2]) {
      uint32_t ah[kRowTiles / 2][4], al[kRowTiles / 2][4];
      as_operand<kRowTiles>(a, ah, al, unit);
      const int br = (lane & 7) + ((lane >> 4) << 3), bc = (lane >> 3) & 1;
#pragma unroll
      for (int step = 0; step < kChunk / 16; ++step)
#pragma unroll
        for (int pair = 0; pair < kRowTiles / 2; ++pair) {
          if (step > pair) continue;  // lower triangular: rows 0-15 have no columns from 16 on
          const int r = pair * 16 + br;
          uint32_t bh[4], bl[4];
          load_matrices(bh, m_at + r * 128 + (((step * 2 + bc) ^ (r & 7)) << 4));
          load_matrices(bl, m_at + r * 128 + (((step * 2 + bc + 4) ^ (r & 7)) << 4));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mma(lo[2 * pair + e], al[step], bh[2 * e], bh[2 * e + 1]);
            mma(hi[2 * pair + e], ah[step], bh[2 * e], bh[2 * e + 1]);
            mma(lo[2 * pair + e], ah[step], bl[2 * e], bl[2 * e + 1]);
          }
        }
    };
    {
      float hi[kRowTiles][4] = {}, lo[kRowTiles][4] = {}, unit[2];
      times(x, t_at, hi, lo, unit);
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
        const float2 fs = *reinterpret_cast<const float2*>(&f->solve[8 * n + 2 * t]);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[n][c] = (hi[n][c] + lo[n][c]) * (unit[c >> 1] * ((c & 1) ? fs.y : fs.x));
      }
    }
    {
      float hi[kRowTiles][4] = {}, lo[kRowTiles][4] = {}, unit[2];
      times(x, p_at, hi, lo, unit);
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
        const float2 fo = *reinterpret_cast<const float2*>(&f->out[8 * n + 2 * t]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = t0 + 8 * n + 2 * t + (c & 1);
          if (r < p.rows) p.o[r * v_step + v_at + 8 * (c >> 1)] = fmaf(hi[n][c] + lo[n][c], unit[c >> 1] * ((c & 1) ? fo.y : fo.x), o[n][c]);
        }
      }
    }
    {
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
        const float2 fp = *reinterpret_cast<const float2*>(&f->put[8 * n + 2 * t]);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[n][c] *= (c & 1) ? fp.y : fp.x;
      }
      uint32_t ah[kRowTiles / 2][4], al[kRowTiles / 2][4];
      float unit[2];
      as_operand<kRowTiles>(x, ah, al, unit);
      const float keep = f->state;
      // matrices of an ldmatrix: key rows 0-7 / 8-15 of the step (lane / 8 % 2), elements 0-7 / 8-15 (lane / 16)
      const int br = lane & 15, bc = lane >> 4;
#pragma unroll
      for (int pair = 0; pair < kTiles / 2; ++pair) {
        float hi[2][4] = {}, lo[2][4] = {};
#pragma unroll
        for (int step = 0; step < kChunk / 16; ++step) {
          const int r = step * 16 + br;
          uint32_t bh[4], bl[4];
          load_matrices_turned(bh, k_at + r * S::kRowHalves * 2 + (((pair * 2 + bc) ^ (r & 7)) << 4));
          load_matrices_turned(bl, k_at + r * S::kRowHalves * 2 + (((pair * 2 + bc + DK / 8) ^ (r & 7)) << 4));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mma(lo[e], al[step], bh[2 * e], bh[2 * e + 1]);
            mma(hi[e], ah[step], bh[2 * e], bh[2 * e + 1]);
            mma(lo[e], ah[step], bl[2 * e], bl[2 * e + 1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[2 * pair + e][c] = fmaf(hi[e][c] + lo[e][c], unit[c >> 1], keep * s[2 * pair + e][c]);
      }
    }
  }
  if (!active) return;
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) p.s_out[state + static_cast<size_t>(8 * n + 2 * t + (c & 1)) * p.dv + 8 * (c >> 1)] = s[n][c];
}

template <int DK>
int launch_delta_chunk(DeltaChunkParams p, cudaStream_t st) {
  using S = ChunkShape<DK>;
  // long prompts in pieces of kMostChunks, which bound the workspace (48 heads over 16 key heads of 128: 116 MB)
  const int rows = p.rows, most = min((rows + kChunk - 1) / kChunk, kMostChunks);
  const size_t key_bytes = static_cast<size_t>(p.k_heads) * most * 2 * S::kKeyBytes;
  const size_t mat_bytes = static_cast<size_t>(p.heads) * most * 2 * S::kMatBytes;
  const size_t factor_bytes = static_cast<size_t>(p.heads) * most * sizeof(Factors);
  unsigned char* scratch = stream_scratch(st, key_bytes + mat_bytes + factor_bytes, 4);
  if (scratch == nullptr) return kUnsupportedFeature;  // a capture before the first plain launch of this size
  p.keys = reinterpret_cast<__half*>(scratch);
  p.mats = reinterpret_cast<__half*>(scratch + key_bytes);
  p.factors = reinterpret_cast<Factors*>(scratch + key_bytes + mat_bytes);
  auto scan = delta_chunk_scan_kernel<DK>;
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(scan), 2 * S::kStage)) return rc;
  for (int r0 = 0; r0 < rows; r0 += kMostChunks * kChunk) {
    p.rows = min(rows - r0, kMostChunks * kChunk);
    p.chunks = (p.rows + kChunk - 1) / kChunk;
    delta_chunk_prepare_kernel<DK><<<dim3(static_cast<unsigned>(p.chunks), static_cast<unsigned>(p.k_heads)), kPrepThreads, 0, st>>>(p);
    if (int rc = check_launch()) return rc;
    scan<<<dim3(static_cast<unsigned>(p.heads), static_cast<unsigned>((p.dv + kScanCols - 1) / kScanCols)), kScanThreads, 2 * S::kStage, st>>>(p);
    if (int rc = check_launch()) return rc;
    const size_t taken = p.rows;
    p.k += taken * p.k_heads * DK, p.q += taken * p.k_heads * DK, p.v += taken * p.heads * p.dv, p.o += taken * p.heads * p.dv;
    p.alpha += taken * p.heads, p.beta += taken * p.heads;
    p.s = p.s_out;
  }
  return kOk;
}

}  // namespace

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
