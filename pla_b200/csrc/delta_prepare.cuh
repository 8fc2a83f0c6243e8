// delta_prepare: everything of a chunk that does not depend on the state, for
// one (chunk, key head) a block and the value heads that share the key head:
// the fp16 planes of K and Q, T = (1 + diag(beta) M)^-1 and P as planes, and
// the per-token coefficients (delta_common.cuh).
#pragma once

#include "delta_common.cuh"

namespace pla {
namespace seq {

constexpr int kPrepThreads = 128;

template <typename T, int DK>
struct PrepShared {
  alignas(16) __half tile[2][DeltaType<T>::kIn][kChunk * DK];  // K, Q planes
  float kk[kChunk][kChunk + 1], qk[kChunk][kChunk + 1];
  alignas(16) float a[kChunk][kChunk + 4];  // diag(beta) M, then T
  float row[2][kChunk];      // what K / Q rows are to be multiplied by
  float hi[kChunk], lo[kChunk], beta[kChunk];
};

// Rows of q or k as planes, in shared memory and in the workspace.
template <typename T, int DK>
__device__ __forceinline__ void prepare_rows(const DeltaParams& p, const T* x, long long step, int vec, int len, int tid,
                                             __half* tile, float* factor, char* out) {
  constexpr int IN = DeltaType<T>::kIn, E = DK / 32;
  const int lane = tid & 31, warp = tid >> 5;
#pragma unroll 4
  for (int i = 0; i < kChunk / 4; ++i) {
    const int row = warp * (kChunk / 4) + i;
    float f[E] = {};
    if (row < len) {
      const T* r = x + row * step;
      if (vec) {
        if (lane * E < p.dk) load<T, E>(r + lane * E, f);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (lane * E + e < p.dk) f[e] = up(r[lane * E + e]);
      }
    }
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, fabsf(f[e]));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const Pow2 s = pow2_for(m);
    if (lane == 0) factor[row] = s.inverse;
    uint32_t hi[E / 2], lo[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) split<IN>(f[2 * e] * s.f, f[2 * e + 1] * s.f, &hi[e], &lo[e]);
    const uint32_t at = tile_at<DK>(row, lane * E / 8) + (lane * E % 8) * 2;
#pragma unroll
    for (int plane = 0; plane < IN; ++plane) {
      const uint32_t* w = plane ? lo : hi;
      char* s_to = reinterpret_cast<char*>(tile) + plane * kChunk * DK * 2 + at;
      char* g_to = out + plane * kChunk * DK * 2 + at;
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        reinterpret_cast<uint32_t*>(s_to)[e] = w[e];
        reinterpret_cast<uint32_t*>(g_to)[e] = w[e];
      }
    }
  }
}

// One row of a 64 x 64 matrix as planes: a lane holds columns 2 lane, 2 lane + 1.
template <int PLANES>
__device__ __forceinline__ float store_square_row(char* out, int row, int lane, float a, float b) {
  float m = fmaxf(fabsf(a), fabsf(b));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const Pow2 s = pow2_for(m);
  uint32_t hi, lo;
  split<PLANES>(a * s.f, b * s.f, &hi, &lo);
  const uint32_t at = tile_at<kChunk>(row, lane / 4) + (lane % 4) * 4;
  *reinterpret_cast<uint32_t*>(out + at) = hi;
  if (PLANES > 1) *reinterpret_cast<uint32_t*>(out + kChunk * kChunk * 2 + at) = lo;
  return s.inverse;
}

template <typename T, int DK, int PS, int PO>
__global__ void __launch_bounds__(kPrepThreads) delta_prepare(DeltaParams p) {
  using L = DeltaLayout<T, DK, PS, PO>;
  extern __shared__ char shared_bytes[];
  PrepShared<T, DK>& s = *reinterpret_cast<PrepShared<T, DK>*>(shared_bytes);
  const int chunk = blockIdx.x / p.hk, kh = blockIdx.x % p.hk;
  ChunkAt c;
  if (!chunk_at(p, chunk, &c)) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  char* tiles = p.tiles + (static_cast<long long>(chunk) * p.hk + kh) * L::kTiles;
  const T* k = static_cast<const T*>(p.k) + c.batch * p.k_batch + c.token * p.k_token + kh * p.k_head;
  const T* q = static_cast<const T*>(p.q) + c.batch * p.q_batch + c.token * p.q_token + kh * p.q_head;
  prepare_rows<T, DK>(p, k, p.k_token, p.vec_qk, c.len, tid, s.tile[0][0], s.row[0], tiles);
  prepare_rows<T, DK>(p, q, p.q_token, p.vec_qk, c.len, tid, s.tile[1][0], s.row[1], tiles + L::kIn * L::kTile);
  __syncthreads();

  // k_i . k_j and q_i . k_j for the 16 rows of this warp, columns up to them
  const uint32_t kt = shared_u32(s.tile[0][0]), qt = shared_u32(s.tile[1][0]);
  {
    float dk[8][4] = {}, dq[8][4] = {};
#pragma unroll
    for (int kk = 0; kk < DK / 16; ++kk)
#pragma unroll
      for (int pa = 0; pa < L::kIn; ++pa) {
        uint32_t ak[4], aq[4];
        ldsm(ak, kt + pa * L::kTile + at_mk<DK>(lane, warp * 16, kk * 16));
        ldsm(aq, qt + pa * L::kTile + at_mk<DK>(lane, warp * 16, kk * 16));
#pragma unroll
        for (int pb = 0; pb + pa < L::kIn; ++pb)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            if (n > warp) break;
            uint32_t b[4];
            ldsm(b, kt + pb * L::kTile + at_nk<DK>(lane, n * 16, kk * 16));
            mma(dk[2 * n], ak, b[0], b[1]);
            mma(dk[2 * n + 1], ak, b[2], b[3]);
            mma(dq[2 * n], aq, b[0], b[1]);
            mma(dq[2 * n + 1], aq, b[2], b[3]);
          }
      }
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = warp * 16 + (lane >> 2) + (e >> 1) * 8, j = n * 8 + (lane & 3) * 2 + (e & 1);
        s.kk[i][j] = dk[n][e] * s.row[0][j] * s.row[0][i];
        s.qk[i][j] = dq[n][e] * s.row[0][j] * s.row[1][i];
      }
  }

  const int group = p.hv / p.hk;
  for (int sub = 0; sub < group; ++sub) {
    const int vh = kh * group + sub;
    char* head = p.heads + (static_cast<long long>(chunk) * p.hv + vh) * L::kHead;
    float* coef = reinterpret_cast<float*>(head + L::kT + L::kP);
    __syncthreads();
    if (warp == 0) {  // running sum of g in 64 bits, kept as two floats
      double sum[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 2 * lane + e;
        float g = 0.f, b = 0.f;
        if (t < c.len) {
          const long long gi = c.batch * p.g_batch + (c.token + t) * p.g_token + vh * p.g_head;
          const long long bi = c.batch * p.beta_batch + (c.token + t) * p.beta_token + vh * p.beta_head;
          g = p.gates32 ? static_cast<const float*>(p.g)[gi] : up(static_cast<const T*>(p.g)[gi]);
          b = p.gates32 ? static_cast<const float*>(p.beta)[bi] : up(static_cast<const T*>(p.beta)[bi]);
        }
        // e^-200 is 0 in fp32 already: a smaller g, -inf among them, is the same reset
        sum[e] = g < -200.f ? -200.f : g;
        s.beta[t] = b;
      }
      sum[1] += sum[0];
      double total = sum[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, total, o);
        if (lane >= o) total += v;
      }
      const double before = total - sum[1];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const double v = before + sum[e];
        s.hi[2 * lane + e] = static_cast<float>(v);
        s.lo[2 * lane + e] = static_cast<float>(v - static_cast<double>(static_cast<float>(v)));
      }
    }
    __syncthreads();
    // diag(beta) M below the diagonal; P as planes
    char* to_p = head + L::kT;
    for (int i = 0; i < kChunk / 4; ++i) {
      const int row = warp * (kChunk / 4) + i;
      float pv[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = 2 * lane + e;
        const float decay = j <= row ? expf((s.hi[row] - s.hi[j]) + (s.lo[row] - s.lo[j])) : 0.f;
        pv[e] = j <= row ? decay * s.qk[row][j] : 0.f;
        s.a[row][j] = j < row ? s.beta[row] * (decay * s.kk[row][j]) : 0.f;
      }
      const float back = store_square_row<PO>(to_p, row, lane, pv[0], pv[1]);
      if (lane == 0) coef[kOutP * kChunk + row] = p.scale * back;
    }
    __syncthreads();
    // column j of T by forward substitution, in registers
    float x[kChunk];
    if (tid < kChunk) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        float sum[4] = {};
#pragma unroll
        for (int l = 0; l + 4 <= i + 3; l += 4) {
          const float4 a = *reinterpret_cast<const float4*>(&s.a[i][l]);
          sum[0] = fmaf(a.x, l < i ? x[l] : 0.f, sum[0]);
          if (l + 1 < i) sum[1] = fmaf(a.y, x[l + 1], sum[1]);
          if (l + 2 < i) sum[2] = fmaf(a.z, x[l + 2], sum[2]);
          if (l + 3 < i) sum[3] = fmaf(a.w, x[l + 3], sum[3]);
        }
        x[i] = (i == tid ? 1.f : 0.f) - ((sum[0] + sum[1]) + (sum[2] + sum[3]));
      }
    }
    __syncthreads();
    if (tid < kChunk)
#pragma unroll
      for (int i = 0; i < kChunk; ++i) s.a[i][tid] = x[i];
    __syncthreads();
    for (int i = 0; i < kChunk / 4; ++i) {
      const int row = warp * (kChunk / 4) + i;
      const float2 v = *reinterpret_cast<const float2*>(&s.a[row][2 * lane]);
      const float back = store_square_row<PS>(head, row, lane, v.x, v.y);
      if (lane == 0) coef[kTRow * kChunk + row] = back;
    }
    if (tid < kChunk) {
      const float gamma = exp_sum(s.hi[tid], s.lo[tid]), b = s.beta[tid];
      const float tail = expf((s.hi[kChunk - 1] - s.hi[tid]) + (s.lo[kChunk - 1] - s.lo[tid]));
      coef[kBeta * kChunk + tid] = b;
      coef[kDown * kChunk + tid] = b * gamma * s.row[0][tid];
      coef[kTail * kChunk + tid] = tail * s.row[0][tid];
      coef[kOutQ * kChunk + tid] = p.scale * gamma * s.row[1][tid];
      coef[kSumHi * kChunk + tid] = s.hi[tid];
      coef[kSumLo * kChunk + tid] = s.lo[tid];
      coef[kKRow * kChunk + tid] = s.row[0][tid];
      coef[kQRow * kChunk + tid] = s.row[1][tid];
      coef[kDecay * kChunk + tid] = exp_sum(s.hi[kChunk - 1], s.lo[kChunk - 1]);
    }
  }
}

}  // namespace seq
}  // namespace pla
