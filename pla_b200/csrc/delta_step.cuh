// One token of the gated delta rule for every sequence, the state [Dk, Dv] of
// a head updated in place:
//     S' = e^g S,  u = beta (v - S'^T k),  S <- S' + k u^T,  o = scale S^T q.
// Bound by HBM: the state is read and written once (8 Dk Dv bytes a head, 6
// flops an entry).  A block owns one head and 32 V columns of it; a warp holds
// every WARPS-th row of them in registers, so one pass gives S'^T k and S'^T q
// together, and o = scale (S'^T q + (q . k) u) needs no second sum over the
// updated state.  Sums are fp32; the warps' partial sums meet once in shared
// memory, in warp order.
#pragma once

#include "seq_common.cuh"

namespace pla {
namespace seq {

struct DeltaStepParams {
  const void *q, *k, *v, *g, *beta;
  long long q_row, q_head, k_row, k_head, v_row, v_head, g_row, g_head, beta_row, beta_head;
  float* state;
  long long state_row;  // elements between sequences; [hv, dk, dv] of one is dense
  void* o;              // dense [n, hv, dv]
  int n, hk, hv, dk, dv, gates32;
  float scale;
};

constexpr int kStepWarps = 8;

// ROWS: rows of S a warp holds, Dk <= ROWS * kStepWarps.  V: columns of a lane.
template <typename T, int ROWS, int V>
__global__ void __launch_bounds__(kStepWarps * 32) delta_step(DeltaStepParams p) {
  __shared__ float sq[ROWS * kStepWarps], sk[ROWS * kStepWarps];
  __shared__ float part[2][kStepWarps][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int parts = (p.dv + 32 * V - 1) / (32 * V);
  int b = blockIdx.x;
  const int col = (b % parts) * 32 * V + lane * V;
  b /= parts;
  const int vh = b % p.hv, kh = vh / (p.hv / p.hk);
  const long long n = b / p.hv;
  float* state = p.state + n * p.state_row + static_cast<long long>(vh) * p.dk * p.dv + col;
  const bool mine = col < p.dv;

  float s[ROWS][V];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = i * kStepWarps + warp;
#pragma unroll
    for (int e = 0; e < V; ++e) s[i][e] = 0.f;
    if (mine && row < p.dk) load<float, V>(state + static_cast<long long>(row) * p.dv, s[i]);
  }
  if (threadIdx.x < ROWS * kStepWarps) {
    const int d = threadIdx.x;
    sq[d] = d < p.dk ? up(static_cast<const T*>(p.q)[n * p.q_row + kh * p.q_head + d]) : 0.f;
    sk[d] = d < p.dk ? up(static_cast<const T*>(p.k)[n * p.k_row + kh * p.k_head + d]) : 0.f;
  }
  float g, beta, v[V];
  {
    const long long gi = n * p.g_row + vh * p.g_head, bi = n * p.beta_row + vh * p.beta_head;
    g = p.gates32 ? static_cast<const float*>(p.g)[gi] : up(static_cast<const T*>(p.g)[gi]);
    beta = p.gates32 ? static_cast<const float*>(p.beta)[bi] : up(static_cast<const T*>(p.beta)[bi]);
#pragma unroll
    for (int e = 0; e < V; ++e)
      v[e] = mine ? up(static_cast<const T*>(p.v)[n * p.v_row + vh * p.v_head + col + e]) : 0.f;
  }
  __syncthreads();
  const float decay = expf(g);
  float with_k[V] = {}, with_q[V] = {}, qk = 0.f;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const float kr = sk[i * kStepWarps + warp], qr = sq[i * kStepWarps + warp];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s[i][e] *= decay;
      with_k[e] = fmaf(s[i][e], kr, with_k[e]);
      with_q[e] = fmaf(s[i][e], qr, with_q[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    part[0][warp][lane * V + e] = with_k[e];
    part[1][warp][lane * V + e] = with_q[e];
  }
  // q . k: every warp the same sum in the same order
#pragma unroll
  for (int d = 0; d < ROWS * kStepWarps / 32; ++d) qk = fmaf(sq[d * 32 + lane], sk[d * 32 + lane], qk);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) qk += __shfl_xor_sync(0xffffffffu, qk, o);
  __syncthreads();
  float u[V], out[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float a = 0.f, c = 0.f;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) {
      a += part[0][w][lane * V + e];
      c += part[1][w][lane * V + e];
    }
    u[e] = beta * (v[e] - a);
    out[e] = p.scale * fmaf(qk, u[e], c);
  }
  if (!mine) return;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = i * kStepWarps + warp;
    const float kr = sk[row];
    float r[V];
#pragma unroll
    for (int e = 0; e < V; ++e) r[e] = fmaf(kr, u[e], s[i][e]);
    if (row < p.dk) store<float, V>(state + static_cast<long long>(row) * p.dv, r);
  }
  if (warp == 0) store<T, V>(static_cast<T*>(p.o) + (n * p.hv + vh) * p.dv + col, out);
}

}  // namespace seq
}  // namespace pla
