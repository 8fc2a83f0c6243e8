// Gated delta rule: what its kernels share.
//
// A head's state S [Dk, Dv] follows, token by token,
//     S <- e^g S,   u = beta (v - S^T k),   S <- S + k u^T,   o = scale S^T q.
// Over a chunk of 64 tokens, with G the running sum of g, the same is
//     M_ij = e^{G_i - G_j} k_i . k_j (i > j)     P_ij = e^{G_i - G_j} q_i . k_j (i >= j)
//     X = beta (V - e^G (K S0))                  U = T X,  T = (1 + diag(beta) M)^-1
//     O = scale (e^G (Q S0) + P U)               S = e^{G_C} S0 + K^T (e^{G_C - G} U),
// which turns 64 dependent steps into matrix products.  delta_prepare builds
// T and P of every chunk in parallel; delta_sweep walks the chunks of a
// sequence with S in registers.
//
// Products run on the tensor cores in fp16 with fp32 accumulators.  An fp32
// operand is split into planes, hi = fp16(x f), lo = fp16(x f - hi), after
// multiplying by a power of two f that brings its row's largest value near
// 2^12: f is exact, every finite value has a finite plane, and hi + lo
// keep 22 bits of a value (values 2^-26 below the row's largest keep fewer,
// with an error below 2^-38 of the largest).  16-bit inputs fit one plane: a
// bfloat16 has 8 bits, so only values 2^-22 below the row's largest lose any.
// Products of two lo planes are below 2^-22 and left out.  bf16 planes would
// need three of them for the same precision.  Results of 16-bit types are
// computed like fp32 ones and rounded once.  One plane for what only a bf16
// result sees takes less time (4096 tokens of 32 heads of 128, forward and
// backward: 850 us, two planes 1250), but its error, up to 2^-12 of a token's
// norm, comes on top of the rounding.
#pragma once

#include "seq_common.cuh"

namespace pla {
namespace seq {

constexpr int kChunk = 64;
constexpr int kPlanes = 2;  // of every operand but inputs of 16-bit types

// Per-chunk, per-head coefficients over the chunk's tokens (rows of 64 floats).
enum DeltaCoef {
  kBeta = 0,   // beta
  kDown = 1,   // beta e^G f_k: weight of K S0 in X
  kTail = 2,   // e^{G_C - G} f_k: weight of U in the state's update
  kTRow = 3,   // scale of the rows of T's planes
  kOutQ = 4,   // scale e^G f_q: weight of Q S0 in O
  kOutP = 5,   // scale * scale of the rows of P's planes
  kSumHi = 6,  // G as an unevaluated sum of two floats
  kSumLo = 7,
  kKRow = 8,   // f_k, f_q: what a row of the K / Q planes is to be multiplied by
  kQRow = 9,
  kDecay = 10, // e^{G_C} in every place
  kBounds = 11,  // largest sum of |T| over a row; of the same times kTail; of |kDown|
  kCoefs = 12
};

struct DeltaParams {
  const void *q, *k, *v, *g, *beta;
  long long q_batch, q_token, q_head, k_batch, k_token, k_head, v_batch, v_token, v_head;
  long long g_batch, g_token, g_head, beta_batch, beta_token, beta_head;
  const int* cu;
  const float* state_in;
  float* state_out;
  void* o;  // dense
  int batch, tokens, sequences, hk, hv, dk, dv, gates32;
  float scale;
  int row_chunks;    // dense: chunks of a batch row
  int chunk_bound;   // chunks the workspace has room for
  int* plan;         // ragged: lo [N], len [N], first chunk [N + 1], sequences by length [N]
  int4* table;       // ragged: sequence (-1: none), first token, tokens of every chunk
  char* tiles;       // K, Q planes of every (chunk, key head)
  char* heads;       // T, P planes and coefficients of every (chunk, value head)
  // backward
  const void* d_o;
  long long do_batch, do_token, do_head;
  const float* dstate_out;
  float* dstate_in;
  // planes of S and U (kept by the forward sweep), of dS at the chunks' ends and of
  // dX: [chunk, value head][plane][rows][Dk or 64], tiles of delta_common's order
  char *states, *us, *dstates, *dxs;
  float* scales;     // the inverses of their scales: [chunk, value head][S, dS, U, dX][rows]
  int rows;          // dv rounded up to 64
  void *dq, *dk_out, *dv_out, *dg, *dbeta;
  int slabs;         // ceil(dv / 16)
  int vec_qk, vec_v, vec_o, vec_do, pair_qk;  // whole accesses: of 16 bytes (q, k: 4 elements; dq, dk: 2)
};

struct ChunkAt {
  int sequence, batch, token, len;  // first token and number of tokens
};

__device__ __forceinline__ bool chunk_at(const DeltaParams& p, int chunk, ChunkAt* c) {
  if (!p.cu) {
    c->sequence = c->batch = chunk / p.row_chunks;
    c->token = (chunk % p.row_chunks) * kChunk;
    c->len = min(kChunk, p.tokens - c->token);
    return true;
  }
  const int4 t = p.table[chunk];
  if (t.x < 0) return false;
  c->sequence = t.x;
  c->batch = 0;
  c->token = t.y;
  c->len = t.z;
  return true;
}

// Ragged batches: first token, length and first chunk of every sequence.  A
// running maximum over the clamped entries keeps sequences in order and apart
// whatever cu_seqlens holds, so their chunks never exceed tokens / 64 + N.
__global__ void __launch_bounds__(1024) delta_plan(const int* cu, int tokens, int n, int* plan, int4* table, int chunks) {
  __shared__ int scan[1024];
  __shared__ int carry_max, carry_sum;
  const int i = threadIdx.x;
  if (i == 0) {
    carry_max = clamp_token(cu[0], tokens);
    carry_sum = 0;
  }
  __syncthreads();
  for (int base = 0; base < n; base += 1024) {
    const int s = base + i;
    scan[i] = s < n ? clamp_token(cu[s + 1], tokens) : 0;
    __syncthreads();
    for (int o = 1; o < 1024; o <<= 1) {
      const int v = i >= o ? scan[i - o] : 0;
      __syncthreads();
      scan[i] = max(scan[i], v);
      __syncthreads();
    }
    const int hi = max(scan[i], carry_max), lo = i ? max(scan[i - 1], carry_max) : carry_max;
    __syncthreads();
    const int chunks = s < n ? (hi - lo + kChunk - 1) / kChunk : 0;
    scan[i] = chunks;
    __syncthreads();
    for (int o = 1; o < 1024; o <<= 1) {
      const int v = i >= o ? scan[i - o] : 0;
      __syncthreads();
      scan[i] += v;
      __syncthreads();
    }
    if (s < n) {
      plan[s] = lo;
      plan[n + s] = hi - lo;
      plan[2 * n + s] = carry_sum + scan[i] - chunks;
      if (s == n - 1) plan[3 * n] = carry_sum + scan[i];
    }
    __syncthreads();
    if (i == 1023) {
      carry_max = hi;
      carry_sum += scan[i];
    }
    __syncthreads();
  }
  // the longest sequences first, so that the last blocks to start are short; a
  // comparison of all with all, left out for very many
  for (int s = i; s < n; s += 1024) {
    int rank = s;
    if (n <= 2048) {
      const int len = plan[n + s];
      rank = 0;
      for (int j = 0; j < n; ++j) rank += plan[n + j] > len || (plan[n + j] == len && j < s);
    }
    plan[3 * n + 1 + rank] = s;
  }
  for (int chunk = i; chunk < chunks; chunk += 1024) {
    const int at = find_sequence(plan + 2 * n, n, chunk);
    int4 t = make_int4(-1, 0, 0, 0);
    if (at >= 0) {
      const int from = (chunk - plan[2 * n + at]) * kChunk;
      t = make_int4(at, plan[at] + from, min(kChunk, plan[n + at] - from), 0);
    }
    table[chunk] = t;
  }
}

// ---- planes ----------------------------------------------------------------
// Power of two that brings `largest` into [2^12, 2^13), and its inverse; both
// finite for every input (zero, subnormal, infinite or NaN too).
struct Pow2 {
  float f, inverse;
};
__device__ __forceinline__ Pow2 pow2_for(float largest) {
  int e = static_cast<int>((__float_as_uint(largest) >> 23) & 0xff);
  e = min(max(e, 32), 254);  // f in [2^-115, 2^107]
  return {__int_as_float((127 + 12 - e + 127) << 23), __int_as_float((e - 12) << 23)};
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// hi and, with two planes, lo of a pair of values that are already scaled.
template <int PLANES = kPlanes>
__device__ __forceinline__ void split(float a, float b, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(a, b);
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  if (PLANES > 1) {
    const float2 back = __half22float2(h);
    *lo = pack_half2(a - back.x, b - back.y);
  }
}

__device__ __forceinline__ uint32_t shared_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// D += A B, A 16 x 16 row-major, B 16 x 8 column-major, fp16 with fp32 sums.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from zero.
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}

// Tiles of fp16 rows of W features (64 or 128): 16-byte units of a row are
// permuted by the row number so that eight rows at one column, and one row's
// neighbours, fall into different banks.
template <int W>
__device__ __forceinline__ uint32_t tile_at(int row, int unit) {
  return static_cast<uint32_t>(row * W * 2 + ((unit ^ (row & 7)) << 4));
}
// B fragments of two 8-wide column tiles: B[k][n] = tile[n0 + n][k0 + k] ...
template <int W>
__device__ __forceinline__ uint32_t at_nk(int lane, int n0, int k0) {
  const int m = lane >> 3;
  return tile_at<W>(n0 + (m >> 1) * 8 + (lane & 7), (k0 >> 3) + (m & 1));
}
// ... or B[k][n] = tile[k0 + k][n0 + n] (transposing loads).
template <int W>
__device__ __forceinline__ uint32_t at_kn(int lane, int n0, int k0) {
  const int m = lane >> 3;
  return tile_at<W>(k0 + (m & 1) * 8 + (lane & 7), (n0 >> 3) + (m >> 1));
}
// A fragment (16 x 16): A[m][k] = tile[m0 + m][k0 + k].
template <int W>
__device__ __forceinline__ uint32_t at_mk(int lane, int m0, int k0) {
  const int m = lane >> 3;
  return tile_at<W>(m0 + (m & 1) * 8 + (lane & 7), (k0 >> 3) + (m >> 1));
}

// A fragment from a tile that holds the transpose: A[m][k] = tile[k0 + k][m0 + m] (transposing loads).
template <int W>
__device__ __forceinline__ uint32_t at_km(int lane, int m0, int k0) {
  const int m = lane >> 3;
  return tile_at<W>(k0 + (m >> 1) * 8 + (lane & 7), (m0 >> 3) + (m & 1));
}

// A lane's ldmatrix addresses walk a tile along a row by 16 columns a step:
// step k's address is (base ^ 32 (k % 4)) + 128 (k / 4), because the unit
// permutation only touches address bits 4 to 6.  The four permuted bases are
// computed once, the rest are instruction offsets.
struct Walk {
  uint32_t at[4];
  __device__ __forceinline__ explicit Walk(uint32_t base) {
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = base ^ (i << 5);
  }
  __device__ __forceinline__ uint32_t operator[](int k) const { return at[k & 3] + (k >> 2) * 128; }
};

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// e^(hi + lo), lo below half a unit of hi's last place.
__device__ __forceinline__ float exp_sum(float hi, float lo) {
  const float e = expf(hi);
  return fmaf(e, lo, e);
}

// e^x by the hardware's 2^x: off by 2^-22 |x| relative, that is below 2^-23 of
// 1 for x <= 0.
__device__ __forceinline__ float exp_fast(float x) { return exp2f(x * 1.4426950408889634f); }

// Planes of the inputs of a type.
template <typename T>
struct DeltaType {
  static constexpr int kIn = sizeof(T) == 4 ? 2 : 1;
};

// Workspace of a chunk.
template <typename T, int DK>
struct DeltaLayout {
  static constexpr int kIn = DeltaType<T>::kIn;
  static constexpr uint32_t kTile = kChunk * DK * 2;
  static constexpr uint32_t kTiles = 2 * kIn * kTile;  // K planes, Q planes
  static constexpr uint32_t kSquare = kChunk * kChunk * 2;
  static constexpr uint32_t kT = kPlanes * kSquare;
  static constexpr uint32_t kP = kPlanes * kSquare;
  static constexpr uint32_t kCoef = kCoefs * kChunk * 4;
  static constexpr uint32_t kHead = kT + kP + kCoef;
  static constexpr uint32_t kStage = kTiles + kHead;
};

}  // namespace seq
}  // namespace pla
