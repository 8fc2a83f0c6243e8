// One token of the gated delta rule for every sequence, the state [Dk, Dv] of
// a head updated in place:
//     S' = e^g S,  u = beta (v - S'^T k),  S <- S' + k u^T,  o = scale S^T q.
// Bound by HBM: the state is read and written once (8 Dk Dv bytes a head, 6
// flops an entry).  A pass over the state gives S^T k and S^T q together, and
// o = scale (e^g S^T q + (q . k) u) needs no second sum over the updated
// state.  Sums are fp32 in a fixed order: rows of a warp, then the warps.
//
// delta_step holds the state in shared memory: one bulk copy brings a head's
// whole state, one takes it back, and three blocks an SM keep up to 192 KB in
// flight, with few instructions beside.  delta_step_any takes any sizes and
// alignments, a warp holding every 16th row of 32 columns in registers.
#pragma once

#include "delta_sweep.cuh"

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

template <typename T>
__device__ __forceinline__ float2 step_gates(const DeltaStepParams& p, long long n, int vh) {
  const long long gi = n * p.g_row + vh * p.g_head, bi = n * p.beta_row + vh * p.beta_head;
  const float g = p.gates32 ? static_cast<const float*>(p.g)[gi] : up(static_cast<const T*>(p.g)[gi]);
  const float b = p.gates32 ? static_cast<const float*>(p.beta)[bi] : up(static_cast<const T*>(p.beta)[bi]);
  return make_float2(expf(g), b);
}

constexpr int kStepWarps = 8;

// dv = 4 * 32 / ROWS_A_TIME: a warp takes that many rows at a time, 16 bytes a
// lane.  The state follows the other shared memory.
template <typename T>
__global__ void __launch_bounds__(kStepWarps * 32, 3) delta_step(DeltaStepParams p) {
  __shared__ float sq[128], sk[128];
  __shared__ __align__(16) float su[128];  // read four values at a time
  __shared__ __align__(16) float part[2][kStepWarps][128];
  __shared__ uint64_t full;
  extern __shared__ __align__(128) float held[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int vh = blockIdx.x % p.hv, kh = vh / (p.hv / p.hk);
  const long long n = blockIdx.x / p.hv;
  const int size = p.dk * p.dv;
  float* state = p.state + n * p.state_row + static_cast<long long>(vh) * size;
  if (tid == 0) {
    barrier_init(&full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    barrier_expect(&full, size * 4);
    bulk_copy(held, state, size * 4, &full);
  }
  if (tid < 128) {
    sq[tid] = tid < p.dk ? up(static_cast<const T*>(p.q)[n * p.q_row + kh * p.q_head + tid]) : 0.f;
    sk[tid] = tid < p.dk ? up(static_cast<const T*>(p.k)[n * p.k_row + kh * p.k_head + tid]) : 0.f;
  }
  const float2 gates = step_gates<T>(p, n, vh);  // e^g, beta
  const float v = tid < p.dv ? up(static_cast<const T*>(p.v)[n * p.v_row + vh * p.v_head + tid]) : 0.f;
  __syncthreads();
  float qk = 0.f;  // every warp the same sum in the same order
#pragma unroll
  for (int d = 0; d < 4; ++d) qk = fmaf(sq[d * 32 + lane], sk[d * 32 + lane], qk);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) qk += __shfl_xor_sync(0xffffffffu, qk, o);
  // lanes_row lanes a row, the warp's rows 32 / lanes_row at a time
  const int lanes_row = p.dv / 4, at_once = 32 / lanes_row, sub = lane / lanes_row, col = lane % lanes_row * 4;
  const int step = at_once * kStepWarps;
  const bool there = barrier_wait(&full, 0);
  float with_k[4] = {}, with_q[4] = {};
#pragma unroll 4
  for (int row = warp * at_once + sub; row < p.dk; row += step) {
    const float4 s = *reinterpret_cast<const float4*>(held + row * p.dv + col);
    const float kr = sk[row], qr = sq[row];
    with_k[0] = fmaf(s.x, kr, with_k[0]), with_q[0] = fmaf(s.x, qr, with_q[0]);
    with_k[1] = fmaf(s.y, kr, with_k[1]), with_q[1] = fmaf(s.y, qr, with_q[1]);
    with_k[2] = fmaf(s.z, kr, with_k[2]), with_q[2] = fmaf(s.z, qr, with_q[2]);
    with_k[3] = fmaf(s.w, kr, with_k[3]), with_q[3] = fmaf(s.w, qr, with_q[3]);
  }
  for (int o = lanes_row; o < 32; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      with_k[e] += __shfl_xor_sync(0xffffffffu, with_k[e], o);
      with_q[e] += __shfl_xor_sync(0xffffffffu, with_q[e], o);
    }
  if (sub == 0) {
    store<float, 4>(&part[0][warp][col], with_k);
    store<float, 4>(&part[1][warp][col], with_q);
  }
  if (!__syncthreads_and(there)) {  // the state stays as it was
    if (tid == 0) barrier_wait(&full, 0);  // more time for the copy: the block's shared memory is held meanwhile
    return;
  }
  if (tid < p.dv) {
    float a = 0.f, c = 0.f;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) a += part[0][w][tid], c += part[1][w][tid];
    const float u = gates.y * (v - gates.x * a);
    su[tid] = u;
    static_cast<T*>(p.o)[(n * p.hv + vh) * p.dv + tid] = down<T>(p.scale * fmaf(qk, u, gates.x * c));
  }
  __syncthreads();
  const float4 u = *reinterpret_cast<const float4*>(su + col);
#pragma unroll 4
  for (int row = warp * at_once + sub; row < p.dk; row += step) {
    float4 s = *reinterpret_cast<const float4*>(held + row * p.dv + col);
    const float kr = sk[row];
    s.x = fmaf(kr, u.x, gates.x * s.x), s.y = fmaf(kr, u.y, gates.x * s.y);
    s.z = fmaf(kr, u.z, gates.x * s.z), s.w = fmaf(kr, u.w, gates.x * s.w);
    *reinterpret_cast<float4*>(held + row * p.dv + col) = s;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(state), "r"(shared_u32(held)), "r"(size * 4)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
}

constexpr int kStepAnyWarps = 16;

// ROWS: rows of S a warp holds, Dk <= 16 ROWS.
template <typename T, int ROWS>
__global__ void __launch_bounds__(kStepAnyWarps * 32) delta_step_any(DeltaStepParams p) {
  __shared__ float sq[ROWS * kStepAnyWarps], sk[ROWS * kStepAnyWarps];
  __shared__ float part[2][kStepAnyWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int parts = (p.dv + 31) / 32;
  int b = blockIdx.x;
  const int col = (b % parts) * 32 + lane;
  b /= parts;
  const int vh = b % p.hv, kh = vh / (p.hv / p.hk);
  const long long n = b / p.hv;
  float* state = p.state + n * p.state_row + static_cast<long long>(vh) * p.dk * p.dv + col;
  const bool mine = col < p.dv;
  float s[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = i * kStepAnyWarps + warp;
    s[i] = mine && row < p.dk ? state[static_cast<long long>(row) * p.dv] : 0.f;
  }
  if (threadIdx.x < ROWS * kStepAnyWarps) {
    const int d = threadIdx.x;
    sq[d] = d < p.dk ? up(static_cast<const T*>(p.q)[n * p.q_row + kh * p.q_head + d]) : 0.f;
    sk[d] = d < p.dk ? up(static_cast<const T*>(p.k)[n * p.k_row + kh * p.k_head + d]) : 0.f;
  }
  const float2 gates = step_gates<T>(p, n, vh);
  const float v = mine ? up(static_cast<const T*>(p.v)[n * p.v_row + vh * p.v_head + col]) : 0.f;
  __syncthreads();
  float with_k = 0.f, with_q = 0.f, qk = 0.f;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    with_k = fmaf(s[i], sk[i * kStepAnyWarps + warp], with_k);
    with_q = fmaf(s[i], sq[i * kStepAnyWarps + warp], with_q);
  }
  part[0][warp][lane] = with_k;
  part[1][warp][lane] = with_q;
#pragma unroll
  for (int d = 0; d < ROWS * kStepAnyWarps / 32; ++d) qk = fmaf(sq[d * 32 + lane], sk[d * 32 + lane], qk);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) qk += __shfl_xor_sync(0xffffffffu, qk, o);
  __syncthreads();
  float a = 0.f, c = 0.f;
#pragma unroll
  for (int w = 0; w < kStepAnyWarps; ++w) a += part[0][w][lane], c += part[1][w][lane];
  const float u = gates.y * (v - gates.x * a);
  if (!mine) return;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = i * kStepAnyWarps + warp;
    if (row < p.dk) state[static_cast<long long>(row) * p.dv] = fmaf(sk[row], u, gates.x * s[i]);
  }
  if (warp == 0) static_cast<T*>(p.o)[(n * p.hv + vh) * p.dv + col] = down<T>(p.scale * fmaf(qk, u, gates.x * c));
}

}  // namespace seq
}  // namespace pla
