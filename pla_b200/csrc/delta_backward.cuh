// Backward pass of the gated delta rule.  With do' = scale do and D the
// gradient of the state at a chunk's end (names as in delta_common.cuh):
//     dU = P^T do' + e^{G_C - G} (K D)          dX = T^T dU          dv = beta dX
//     dS0 = e^{G_C} D + Q^T (e^G do') - K^T (beta e^G dX)
// is the reverse of the forward's chain and runs like it (delta_sweep_back:
// D in registers, chunks from the last to the first).  What remains has no dependence between chunks (delta_gradient):
//     dP = tril(do' U^T)       dA = -stril(dX U^T)
//     N = Gamma . dP           B = beta Gamma . dA          Gamma_ij = e^{G_i - G_j}
//     dq = e^G (do' S0^T) + N K
//     dk = -beta e^G (dX S0^T) + e^{G_C - G} (U D^T) + N^T Q + (B + B^T) K
//     dbeta = -e^G k . (dX S0^T) + dX . v + rowsum(Gamma . dA . K K^T)
//     dG = beta part of the same + q . dq_state + rowsum(Z) - colsum(Z) - H,
//          Z = N . (Q K^T) + B . (K K^T),  H = e^{G_C - G} k . (U D^T),
//     dG_C += e^{G_C} <S0, D> + sum H,      dg = sums of dG from each token to the chunk's end.
// S0 and U come from the forward's sweep run again: the forward keeps only its
// inputs.  Every sum has a fixed order.
#pragma once

#include "delta_sweep.cuh"

namespace pla {
namespace seq {

template <typename T, int DK, int PS, int PO, int VB>
__global__ void __launch_bounds__(VB * 8) delta_sweep_back(DeltaParams p, int stages) {
  using L = DeltaLayout<T, DK, PS, PO>;
  using M = SweepShared<T, DK, PS, PO, VB, true>;
  constexpr int IN = L::kIn, QN = DK / 32;
  extern __shared__ __align__(128) char shared_bytes[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = warp % (VB / 16), wn = warp / (VB / 16), m0 = wm * 16;
  const SweepAt a = sweep_at(p, VB);
  Ring<L> ring;
  ring.begin(shared_bytes, stages, VB / 4);
  M& m = *reinterpret_cast<M*>(shared_bytes + kSweepRing + stages * L::kStage);
  const uint32_t dt = shared_u32(m.s), yt = shared_u32(m.a), xt = shared_u32(m.b), wt = shared_u32(m.c), ft = shared_u32(m.d);
  const T* d_o = static_cast<const T*>(p.d_o) + a.batch * p.do_batch + a.lo * p.do_token + a.vh * p.do_head + a.column;
  const long long dv_step = static_cast<long long>(p.hv) * p.dv;
  T* dv = static_cast<T*>(p.dv_out) + (static_cast<long long>(a.batch) * p.tokens + a.lo) * dv_step +
          static_cast<long long>(a.vh) * p.dv + a.column;
  if (threadIdx.x == 0)
    for (int i = 0; i < stages && i < a.chunks; ++i) ring.fill(p, i, a.first + a.chunks - 1 - i, a.kh, a.vh);
  if (a.chunks)
    slab_fetch<T, VB>(m.slab[0], d_o + (a.chunks - 1) * kChunk * p.do_token, p.do_token, a.len - (a.chunks - 1) * kChunk,
                      a.width, p.vec_do);
  const Walk dw(dt + at_mk<DK>(lane, m0, 0)), yw(yt + at_mk<kChunk>(lane, m0, 0));  // planes of D and Y; the others follow Y's
  const Walk kw(at_nk<DK>(lane, wn * 16, 0));                                       // in K
  const uint32_t ts = at_kn<kChunk>(lane, wn * 16, 0);                              // in T and P
  uint32_t ks[QN / 2];                                                              // in K and Q, for the state's update
#pragma unroll
  for (int n = 0; n < QN / 2; ++n) ks[n] = at_kn<DK>(lane, wn * (DK / 4) + n * 16, 0);
  float d[QN][4];
  state_load(p.dstate_out, p, a, m0, wn * (DK / 4), lane, d);
  tile_write<PS, DK>(m.s, M::kWide, m0, wn * (DK / 4), lane, d, &m.scale[0][wn][m0]);

  for (int turn = 0; turn < a.chunks; ++turn) {
    const int c = a.chunks - 1 - turn, len = min(kChunk, a.len - c * kChunk);
    const long long slab_at = (static_cast<long long>(a.first + c) * p.hv + a.vh) * p.slabs + a.column / 16 + wm;
    const bool kept = m0 < a.width;
    if (kept) fragments_store(p.dstates + slab_at * 16 * DK, p.largest + (slab_at * 4 + wn) * 4 + 1, wn * QN, lane, d);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    const char* stage = ring.wait(turn);
    __syncthreads();  // planes of D and this chunk's do are there; the other slab is free
    if (c > 0)
      slab_fetch<T, VB>(m.slab[~turn & 1], d_o + (c - 1) * kChunk * p.do_token, p.do_token, kChunk, a.width, p.vec_do);
    const uint32_t kt = shared_u32(stage), qt = kt + IN * L::kTile, tt = kt + L::kTiles, pt = tt + L::kT;
    const char* coef = stage + L::kTiles + L::kT + L::kP;
    float2 w[2];
    {  // do' with the weights of P's rows and with e^G
      float f[2][4], g[2][4];
      slab_read<T, VB>(m.slab[turn & 1], wn * 16, m0, lane, f);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) g[n][e] = f[n][e];
      coef_read(coef, kOutP, wn * 2, lane, w);
      scale_columns(f, w);
      tile_write<PO, kChunk>(m.c, M::kNarrow, m0, wn * 16, lane, f, &m.scale[3][wn][m0]);
      coef_read(coef, kOutQ, wn * 2, lane, w);
      scale_columns(g, w);
      tile_write<PS, kChunk>(m.d, M::kNarrow, m0, wn * 16, lane, g, &m.scale[4][wn][m0]);
    }
    // (K D)^T
    float du[2][4] = {};
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      float bx[2][4] = {};
#pragma unroll
      for (int k = 0; k < DK / 64; ++k) {
        const int kk = b * (DK / 64) + k;
        uint32_t hi[4], lo[4];
        tile_operand<PS>(dw[kk], M::kWide, hi, lo);
        product<PS, IN, false>(bx[0], bx[1], hi, lo, kt + kw[kk], L::kTile);
      }
      add_scaled(du, bx, &m.scale[0][b][m0], lane);
    }
    coef_read(coef, kTail, wn * 2, lane, w);
    scale_columns(du, w);
    __syncthreads();
    // dU = P^T do' + e^{G_C - G} (K D): tokens j take from i >= j
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (VB == 64 && kk < wn) continue;  // the other blocks are zero
      uint32_t hi[4], lo[4];
      float bx[2][4] = {};
      tile_operand<PO>(yw[kk] + (wt - yt), M::kNarrow, hi, lo);
      product<PO, PO, true>(bx[0], bx[1], hi, lo, pt + ts + kk * 16 * kChunk * 2, L::kSquare);
      add_scaled(du, bx, &m.scale[3][kk][m0], lane);
    }
    coef_read(coef, kTRow, wn * 2, lane, w);
    scale_columns(du, w);
    tile_write<PS, kChunk>(m.a, M::kNarrow, m0, wn * 16, lane, du, &m.scale[1][wn][m0]);
    __syncthreads();
    // dX^T = (T^T dU)^T
    float x[2][4] = {};
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (VB == 64 && kk < wn) continue;  // the other blocks are zero
      uint32_t hi[4], lo[4];
      float bx[2][4] = {};
      tile_operand<PS>(yw[kk], M::kNarrow, hi, lo);
      product<PS, PS, true>(bx[0], bx[1], hi, lo, tt + ts + kk * 16 * kChunk * 2, L::kSquare);
      add_scaled(x, bx, &m.scale[1][kk][m0], lane);
    }
    if (kept) fragments_store(p.dxs + slab_at * 16 * kChunk, p.largest + (slab_at * 4 + wn) * 4 + 3, wn * 2, lane, x);
    {
      float out[2][4], minus[2][4];
      float2 b[2];
      coef_read(coef, kBeta, wn * 2, lane, b);
      coef_read(coef, kDown, wn * 2, lane, w);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          out[n][e] = (e & 1 ? b[n].y : b[n].x) * x[n][e];
          minus[n][e] = (e & 1 ? -w[n].y : -w[n].x) * x[n][e];
        }
      tile_write<PS, kChunk>(m.b, M::kNarrow, m0, wn * 16, lane, minus, &m.scale[2][wn][m0]);
      strip_store<T>(m.strip[warp], lane, out, dv + (c * kChunk + wn * 16) * dv_step + m0, dv_step, len - wn * 16, a.width - m0,
                     p.vec_o);
    }
    __syncthreads();
    // D = e^{G_C} D + (e^G do')^T Q - (beta e^G dX)^T K
    const float decay = reinterpret_cast<const float*>(coef)[kDecay * kChunk];
#pragma unroll
    for (int n = 0; n < QN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) d[n][e] *= decay;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4];
      float bs[QN][4] = {}, bt[QN][4] = {};
      tile_operand<PS>(yw[kk] + (ft - yt), M::kNarrow, hi, lo);
#pragma unroll
      for (int n = 0; n < QN / 2; ++n)
        product<PS, IN, true>(bs[2 * n], bs[2 * n + 1], hi, lo, qt + ks[n] + kk * 16 * DK * 2, L::kTile);
      add_scaled(d, bs, &m.scale[4][kk][m0], lane);
      tile_operand<PS>(yw[kk] + (xt - yt), M::kNarrow, hi, lo);
#pragma unroll
      for (int n = 0; n < QN / 2; ++n)
        product<PS, IN, true>(bt[2 * n], bt[2 * n + 1], hi, lo, kt + ks[n] + kk * 16 * DK * 2, L::kTile);
      add_scaled(d, bt, &m.scale[2][kk][m0], lane);
    }
    tile_write<PS, DK>(m.s, M::kWide, m0, wn * (DK / 4), lane, d, &m.scale[0][wn][m0]);
    ring.done(turn, lane);
    if (threadIdx.x == 0 && turn + stages < a.chunks)
      ring.fill(p, turn + stages, a.first + a.chunks - 1 - turn - stages, a.kh, a.vh);
    __syncwarp();
  }
  if (p.dstate_in) state_store(p.dstate_in, p, a, m0, wn * (DK / 4), lane, d);
}

// ---- what is left, in parallel over chunks ---------------------------------
constexpr int kGradThreads = 256;
constexpr int kGradBlock = 64;  // value features at a time

template <typename T, int DK, int PS>
struct GradShared {
  static constexpr int IN = DeltaType<T>::kIn;
  alignas(128) __half tile[2][IN][kChunk * DK];  // K, Q planes
  union {
    struct {
      alignas(128) __half s[PS][kGradBlock * DK], d[PS][kGradBlock * DK];               // S^T, D^T
      __half u[PS][kGradBlock * kChunk], x[PS][kGradBlock * kChunk];                    // U^T, dX^T
      __half o[PS][kChunk * kGradBlock];                                                // do
    } in;
    alignas(128) __half square[4][PS][kChunk * kChunk];  // N f_k, N f_q (rows), B f_k, B f_k (rows)
  };
  float kk[kChunk][kChunk + 2], qk[kChunk][kChunk + 2];
  float krow[kChunk], qrow[kChunk], orow[kChunk], oscale[kChunk];
  float beta[kChunk], hi[kChunk], lo[kChunk], down[kChunk], tail[kChunk];  // down: e^G, tail: e^{G_C - G}
  float dots[2][3][kChunk];    // column halves: k.r1, q.dq, k.r3
  float rows[2][2][kChunk];    // column halves: row sums of Z, of Gamma dA K K^T
  float cols[4][kChunk];       // row blocks: column sums of Z
  float warp_sum[8];
  unsigned int most[4];
  float xv[kChunk];            // dX . v
};

// Fragments [slab][tile n][lane][4] of a [feature][W] matrix as planes in shared memory.
template <int PS, int W>
__device__ __forceinline__ void tile_from_fragments(const float4& f, float scale, char* tile, uint32_t plane, int slab, int n, int lane) {
  const int row = slab * 16 + (lane >> 2);
  uint32_t hi, lo;
  uint32_t at = tile_at<W>(row, n) + (lane & 3) * 4;
  split<PS>(f.x * scale, f.y * scale, &hi, &lo);
  *reinterpret_cast<uint32_t*>(tile + at) = hi;
  if (PS > 1) *reinterpret_cast<uint32_t*>(tile + plane + at) = lo;
  at = tile_at<W>(row + 8, n) + (lane & 3) * 4;
  split<PS>(f.z * scale, f.w * scale, &hi, &lo);
  *reinterpret_cast<uint32_t*>(tile + at) = hi;
  if (PS > 1) *reinterpret_cast<uint32_t*>(tile + plane + at) = lo;
}

// acc[2 n], acc[2 n + 1] += A B over PA x PB planes, lo x lo left out.
template <int PA, int PB, bool A_T, bool B_T>
__device__ __forceinline__ void tile_product(float (&d0)[4], float (&d1)[4], uint32_t a_at, uint32_t a_plane, uint32_t b_at,
                                             uint32_t b_plane) {
#pragma unroll
  for (int i = 0; i < PA; ++i) {
    uint32_t a[4];
    if (A_T) ldsm_t(a, a_at + i * a_plane); else ldsm(a, a_at + i * a_plane);
#pragma unroll
    for (int j = 0; i + j < (PA > PB ? PA : PB) && j < PB; ++j) {
      uint32_t b[4];
      if (B_T) ldsm_t(b, b_at + j * b_plane); else ldsm(b, b_at + j * b_plane);
      mma(d0, a, b[0], b[1]);
      mma(d1, a, b[2], b[3]);
    }
  }
}

__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

template <typename G>
__device__ __forceinline__ void store_pair(G* to, float a, float b, int n) {
  if (n > 0) to[0] = down<G>(a);
  if (n > 1) to[1] = down<G>(b);
}

template <typename T, int DK, int PS, int PO>
__global__ void __launch_bounds__(kGradThreads) delta_gradient(DeltaParams p) {
  using L = DeltaLayout<T, DK, PS, PO>;
  constexpr int IN = L::kIn;
  constexpr uint32_t kWide = kGradBlock * DK * 2, kNarrow = kGradBlock * kChunk * 2, kSq = kChunk * kChunk * 2;
  constexpr int NT = DK / 16;  // column tiles of a warp's half of the DK columns
  extern __shared__ __align__(128) char shared_bytes[];
  GradShared<T, DK, PS>& s = *reinterpret_cast<GradShared<T, DK, PS>*>(shared_bytes);
  const int chunk = blockIdx.x / p.hk, kh = blockIdx.x % p.hk;
  ChunkAt c;
  if (!chunk_at(p, chunk, &c)) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rb = warp & 3, half = warp >> 2;  // 16 tokens, half of the columns
  const int r0 = rb * 16 + (lane >> 2);
  const uint32_t kt = shared_u32(s.tile[0][0]), qt = shared_u32(s.tile[1][0]);
  {
    const uint4* from = reinterpret_cast<const uint4*>(p.tiles + (static_cast<long long>(chunk) * p.hk + kh) * L::kTiles);
    for (int i = tid; i < static_cast<int>(L::kTiles / 16); i += kGradThreads) reinterpret_cast<uint4*>(s.tile)[i] = from[i];
    const float* coef = reinterpret_cast<const float*>(
        p.heads + (static_cast<long long>(chunk) * p.hv + kh * (p.hv / p.hk)) * L::kHead + L::kT + L::kP);
    if (tid < kChunk) {
      s.krow[tid] = coef[kKRow * kChunk + tid];
      s.qrow[tid] = coef[kQRow * kChunk + tid];
    }
  }
  __syncthreads();
  {  // k_i . k_j and q_i . k_j: 16 rows, 32 columns a warp
    float a[4][4] = {}, b[4][4] = {};
#pragma unroll
    for (int kk = 0; kk < DK / 16; ++kk)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t am = at_mk<DK>(lane, rb * 16, kk * 16), bm = kt + at_nk<DK>(lane, half * 32 + n * 16, kk * 16);
        tile_product<IN, IN, false, false>(a[2 * n], a[2 * n + 1], kt + am, L::kTile, bm, L::kTile);
        tile_product<IN, IN, false, false>(b[2 * n], b[2 * n + 1], qt + am, L::kTile, bm, L::kTile);
      }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = r0 + (e >> 1) * 8, j = half * 32 + n * 8 + (lane & 3) * 2 + (e & 1);
        s.kk[i][j] = a[n][e] * s.krow[i] * s.krow[j];
        s.qk[i][j] = b[n][e] * s.qrow[i] * s.krow[j];
      }
  }
  float dq[NT][4] = {}, dk[NT][4] = {};
  const int group = p.hv / p.hk;
  for (int sub = 0; sub < group; ++sub) {
    const int vh = kh * group + sub;
    const long long head_at = static_cast<long long>(chunk) * p.hv + vh;
    const float* coef = reinterpret_cast<const float*>(p.heads + head_at * L::kHead + L::kT + L::kP);
    __syncthreads();
    if (tid < kChunk) {
      s.beta[tid] = coef[kBeta * kChunk + tid];
      s.hi[tid] = coef[kSumHi * kChunk + tid];
      s.lo[tid] = coef[kSumLo * kChunk + tid];
      s.down[tid] = exp_sum(s.hi[tid], s.lo[tid]);
      s.tail[tid] = expf((coef[kSumHi * kChunk + kChunk - 1] - s.hi[tid]) + (coef[kSumLo * kChunk + kChunk - 1] - s.lo[tid]));
    }
    if (tid < 4) s.most[tid] = 0;
    const float decay = coef[kDecay * kChunk];
    float most[4] = {};
    for (int i = 0; i < p.slabs * 4; ++i) {
      const float4 m = *reinterpret_cast<const float4*>(p.largest + (head_at * p.slabs * 4 + i) * 4);
      most[0] = fmaxf(most[0], m.x);
      most[1] = fmaxf(most[1], m.y);
      most[2] = fmaxf(most[2], m.z);
      most[3] = fmaxf(most[3], m.w);
    }
    const Pow2 fs = pow2_for(most[0]), fd = pow2_for(most[1]), fu = pow2_for(most[2]), fx = pow2_for(most[3]);

    const T* d_o = static_cast<const T*>(p.d_o) + c.batch * p.do_batch + c.token * p.do_token + vh * p.do_head;
    for (int row = warp; row < kChunk; row += 8) {  // one scale for each row of do
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (row < c.len && lane + 32 * e < p.dv) m = fmaxf(m, fabsf(up(d_o[row * p.do_token + lane + 32 * e])));
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const Pow2 fo = pow2_for(m);
      if (lane == 0) {
        s.oscale[row] = fo.f;
        s.orow[row] = fo.inverse;
      }
    }

    float a_q[NT][4] = {}, a_x[NT][4] = {}, a_u[NT][4] = {}, a_p[4][4] = {}, a_a[4][4] = {};
    float sd_sum = 0.f, xv[2] = {};
    for (int block = 0; block * kGradBlock < p.slabs * 16; ++block) {
      __syncthreads();
      // S^T, D^T (64 features), U^T, dX^T as planes; <S, D>
      for (int i = warp; i < 4 * (DK / 8); i += 8) {
        const int slab = i / (DK / 8), n = i % (DK / 8), at = block * 4 + slab;
        float4 f = make_float4(0, 0, 0, 0), g = f;
        if (at < p.slabs) {
          const long long where = (head_at * p.slabs + at) * 16 * DK + (n * 32 + lane) * 4;
          f = *reinterpret_cast<const float4*>(p.states + where);
          g = *reinterpret_cast<const float4*>(p.dstates + where);
        }
        sd_sum += (f.x * g.x + f.y * g.y) + (f.z * g.z + f.w * g.w);
        tile_from_fragments<PS, DK>(f, fs.f, reinterpret_cast<char*>(s.in.s), kWide, slab, n, lane);
        tile_from_fragments<PS, DK>(g, fd.f, reinterpret_cast<char*>(s.in.d), kWide, slab, n, lane);
      }
      for (int i = warp; i < 4 * 8; i += 8) {
        const int slab = i / 8, n = i % 8, at = block * 4 + slab;
        float4 f = make_float4(0, 0, 0, 0), g = f;
        if (at < p.slabs) {
          const long long where = (head_at * p.slabs + at) * 16 * kChunk + (n * 32 + lane) * 4;
          f = *reinterpret_cast<const float4*>(p.us + where);
          g = *reinterpret_cast<const float4*>(p.dxs + where);
        }
        tile_from_fragments<PS, kChunk>(f, fu.f, reinterpret_cast<char*>(s.in.u), kNarrow, slab, n, lane);
        tile_from_fragments<PS, kChunk>(g, fx.f, reinterpret_cast<char*>(s.in.x), kNarrow, slab, n, lane);
        // dX . v of the tokens: this lane's features
        const T* v = static_cast<const T*>(p.v) + c.batch * p.v_batch + vh * p.v_head;
        float two[2] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = n * 8 + (lane & 3) * 2 + (e & 1), col = at * 16 + (lane >> 2) + (e >> 1) * 8;
          const float x = e == 0 ? g.x : e == 1 ? g.y : e == 2 ? g.z : g.w;
          if (t < c.len && col < p.dv) two[e & 1] = fmaf(x, up(v[(c.token + t) * p.v_token + col]), two[e & 1]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) two[e] += __shfl_xor_sync(0xffffffffu, two[e], o);
        }
        // a warp meets token tile n = warp once a slab, in slab order
        xv[0] += two[0];
        xv[1] += two[1];
      }
      // do, this block's features
      for (int row = warp; row < kChunk; row += 8) {
        float f[2] = {};
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (row < c.len && block * kGradBlock + lane * 2 + e < p.dv)
            f[e] = up(d_o[row * p.do_token + block * kGradBlock + lane * 2 + e]) * s.oscale[row];
        uint32_t hi, lo;
        split<PS>(f[0], f[1], &hi, &lo);
        const uint32_t at = tile_at<kGradBlock>(row, lane / 4) + (lane % 4) * 4;
        *reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(s.in.o) + at) = hi;
        if (PS > 1) *reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(s.in.o) + kNarrow + at) = lo;
      }
      __syncthreads();
      const uint32_t st = shared_u32(s.in.s), dt = shared_u32(s.in.d), ut = shared_u32(s.in.u), xt = shared_u32(s.in.x),
                     ot = shared_u32(s.in.o);
#pragma unroll
      for (int kk = 0; kk < kGradBlock / 16; ++kk) {
        const uint32_t o_at = ot + at_mk<kGradBlock>(lane, rb * 16, kk * 16);
        const uint32_t u_at = ut + at_km<kChunk>(lane, rb * 16, kk * 16), x_at = xt + at_km<kChunk>(lane, rb * 16, kk * 16);
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
          const uint32_t b = at_kn<DK>(lane, half * (DK / 2) + n * 16, kk * 16);
          tile_product<PS, PS, false, true>(a_q[2 * n], a_q[2 * n + 1], o_at, kNarrow, st + b, kWide);
          tile_product<PS, PS, true, true>(a_x[2 * n], a_x[2 * n + 1], x_at, kNarrow, st + b, kWide);
          tile_product<PS, PS, true, true>(a_u[2 * n], a_u[2 * n + 1], u_at, kNarrow, dt + b, kWide);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint32_t b = ut + at_kn<kChunk>(lane, half * 32 + n * 16, kk * 16);
          tile_product<PS, PS, false, true>(a_p[2 * n], a_p[2 * n + 1], o_at, kNarrow, b, kNarrow);
          tile_product<PS, PS, true, true>(a_a[2 * n], a_a[2 * n + 1], x_at, kNarrow, b, kNarrow);
        }
      }
    }
    // <S, D> of the block; dX . v of this warp's token tile
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sd_sum += __shfl_xor_sync(0xffffffffu, sd_sum, o);
    if (lane == 0) s.warp_sum[warp] = sd_sum;
    if (lane < 4) {
      s.xv[warp * 8 + lane * 2] = xv[0];
      s.xv[warp * 8 + lane * 2 + 1] = xv[1];
    }

    // parts of dq and dk that see the states, and their products with q and k
    {
      float dot[3][2] = {};
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = r0 + (e >> 1) * 8, col = half * (DK / 2) + n * 8 + (lane & 3) * 2 + (e & 1);
          const uint32_t at = tile_at<DK>(i, col >> 3) + (col & 7) * 2;
          float kv = 0.f, qv = 0.f;
#pragma unroll
          for (int plane = 0; plane < IN; ++plane) {
            kv += __half2float(*reinterpret_cast<const __half*>(reinterpret_cast<const char*>(s.tile[0][plane]) + at));
            qv += __half2float(*reinterpret_cast<const __half*>(reinterpret_cast<const char*>(s.tile[1][plane]) + at));
          }
          kv *= s.krow[i];
          qv *= s.qrow[i];
          const float one = -s.down[i] * (a_x[n][e] * (fx.inverse * fs.inverse));
          const float two = p.scale * s.down[i] * (a_q[n][e] * s.orow[i] * fs.inverse);
          const float three = s.tail[i] * (a_u[n][e] * (fu.inverse * fd.inverse));
          dot[0][e >> 1] = fmaf(kv, one, dot[0][e >> 1]);
          dot[1][e >> 1] = fmaf(qv, two, dot[1][e >> 1]);
          dot[2][e >> 1] = fmaf(kv, three, dot[2][e >> 1]);
          dq[n][e] += two;
          dk[n][e] += fmaf(s.beta[i], one, three);
        }
#pragma unroll
      for (int w = 0; w < 3; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float v = quad_sum(dot[w][h]);
          if ((lane & 3) == 0) s.dots[half][w][r0 + h * 8] = v;
        }
    }
    // N, B, their row and column sums with Q K^T and K K^T
    float n_k[4][4], n_q[4][4], b_k[4][4], b_r[4][4], top[4] = {};
    {
      float row_z[2] = {}, row_a[2] = {}, col_z[4][2];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        col_z[n][0] = col_z[n][1] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = r0 + (e >> 1) * 8, j = half * 32 + n * 8 + (lane & 3) * 2 + (e & 1);
          const float gamma = j <= i ? expf((s.hi[i] - s.hi[j]) + (s.lo[i] - s.lo[j])) : 0.f;
          const float nn = j <= i ? gamma * (p.scale * (a_p[n][e] * s.orow[i] * fu.inverse)) : 0.f;
          const float ga = j < i ? -gamma * (a_a[n][e] * (fx.inverse * fu.inverse)) : 0.f;
          const float with = j < i ? ga * s.kk[i][j] : 0.f;
          const float z = (j <= i ? nn * s.qk[i][j] : 0.f) + s.beta[i] * with;
          row_z[e >> 1] += z;
          row_a[e >> 1] += with;
          col_z[n][e & 1] += z;
          n_k[n][e] = nn * s.krow[j];
          n_q[n][e] = nn * s.qrow[i];
          b_k[n][e] = s.beta[i] * ga * s.krow[j];
          b_r[n][e] = s.beta[i] * ga * s.krow[i];
          top[0] = fmaxf(top[0], fabsf(n_k[n][e]));
          top[1] = fmaxf(top[1], fabsf(n_q[n][e]));
          top[2] = fmaxf(top[2], fabsf(b_k[n][e]));
          top[3] = fmaxf(top[3], fabsf(b_r[n][e]));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float z = quad_sum(row_z[h]), v = quad_sum(row_a[h]);
        if ((lane & 3) == 0) {
          s.rows[half][0][r0 + h * 8] = z;
          s.rows[half][1][r0 + h * 8] = v;
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float z = col_z[n][e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
          if (lane < 4) s.cols[rb][half * 32 + n * 8 + lane * 2 + e] = z;
        }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float m = quad_max(top[w]);
        m = warp_max(m);
        // non-negative floats order as integers: the maximum does not depend on the order
        if (lane == 0) atomicMax(&s.most[w], __float_as_uint(m));
      }
    }
    __syncthreads();
    const Pow2 f[4] = {pow2_for(__uint_as_float(s.most[0])), pow2_for(__uint_as_float(s.most[1])),
                       pow2_for(__uint_as_float(s.most[2])), pow2_for(__uint_as_float(s.most[3]))};
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = tile_at<kChunk>(r0 + h * 8, half * 4 + n) + (lane & 3) * 4;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float(&m)[4] = w == 0 ? n_k[n] : w == 1 ? n_q[n] : w == 2 ? b_k[n] : b_r[n];
          uint32_t hi, lo;
          split<PS>(m[2 * h] * f[w].f, m[2 * h + 1] * f[w].f, &hi, &lo);
          char* to = reinterpret_cast<char*>(s.square[w]);
          *reinterpret_cast<uint32_t*>(to + at) = hi;
          if (PS > 1) *reinterpret_cast<uint32_t*>(to + kSq + at) = lo;
        }
      }
    // the gates' gradients
    if (warp == 0) {
      float h[2], dg[2];
      float sum_h = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 2 * lane + e;
        h[e] = s.dots[0][2][t] + s.dots[1][2][t];
        sum_h += h[e];
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) sum_h += __shfl_xor_sync(0xffffffffu, sum_h, o);
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) total += s.warp_sum[w];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 2 * lane + e;
        const float k1 = s.dots[0][0][t] + s.dots[1][0][t], q1 = s.dots[0][1][t] + s.dots[1][1][t];
        const float z = (s.rows[0][0][t] + s.rows[1][0][t]) - ((s.cols[0][t] + s.cols[1][t]) + (s.cols[2][t] + s.cols[3][t]));
        dg[e] = s.beta[t] * k1 + q1 + z - h[e];
        const float db = k1 + s.xv[t] + (s.rows[0][1][t] + s.rows[1][1][t]);
        if (t < c.len) {
          const long long at = (static_cast<long long>(c.batch) * p.tokens + c.token + t) * p.hv + vh;
          if (p.gates32)
            static_cast<float*>(p.dbeta)[at] = db;
          else
            static_cast<T*>(p.dbeta)[at] = down<T>(db);
        }
      }
      if (lane == 31) dg[1] += decay * total + sum_h;
      dg[0] += dg[1];
      float after = dg[0];  // sums from this pair to the end
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float v = __shfl_down_sync(0xffffffffu, after, o);
        if (lane + o < 32) after += v;
      }
      const float rest = after - dg[0];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 2 * lane + e;
        if (t < c.len) {
          const long long at = (static_cast<long long>(c.batch) * p.tokens + c.token + t) * p.hv + vh;
          if (p.gates32)
            static_cast<float*>(p.dg)[at] = dg[e] + rest;
          else
            static_cast<T*>(p.dg)[at] = down<T>(dg[e] + rest);
        }
      }
    }
    __syncthreads();
    // dq += N K; dk += N^T Q + B K + B^T K, the matrices lower triangular
    {
      float b_q[NT][4] = {}, b_n[NT][4] = {}, b_b[NT][4] = {}, b_t[NT][4] = {};
      const uint32_t sq = shared_u32(s.square);
      constexpr uint32_t one = PS * kSq;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const uint32_t mk = at_mk<kChunk>(lane, rb * 16, kk * 16), km = at_km<kChunk>(lane, rb * 16, kk * 16);
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
          const uint32_t b = at_kn<DK>(lane, half * (DK / 2) + n * 16, kk * 16);
          if (kk <= rb) {
            tile_product<PS, IN, false, true>(b_q[2 * n], b_q[2 * n + 1], sq + mk, kSq, kt + b, L::kTile);
            tile_product<PS, IN, false, true>(b_b[2 * n], b_b[2 * n + 1], sq + 2 * one + mk, kSq, kt + b, L::kTile);
          }
          if (kk >= rb) {
            tile_product<PS, IN, true, true>(b_n[2 * n], b_n[2 * n + 1], sq + one + km, kSq, qt + b, L::kTile);
            tile_product<PS, IN, true, true>(b_t[2 * n], b_t[2 * n + 1], sq + 3 * one + km, kSq, kt + b, L::kTile);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dq[n][e] = fmaf(b_q[n][e], f[0].inverse, dq[n][e]);
          dk[n][e] += fmaf(b_n[n][e], f[1].inverse, fmaf(b_b[n][e], f[2].inverse, b_t[n][e] * f[3].inverse));
        }
    }
  }
  // dq, dk: dense [batch, tokens, key heads, Dk]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = r0 + h * 8, col = half * (DK / 2) + n * 8 + (lane & 3) * 2;
      if (t >= c.len) continue;
      const long long at = ((static_cast<long long>(c.batch) * p.tokens + c.token + t) * p.hk + kh) * p.dk + col;
      store_pair(static_cast<T*>(p.dq) + at, dq[n][2 * h], dq[n][2 * h + 1], p.dk - col);
      store_pair(static_cast<T*>(p.dk_out) + at, dk[n][2 * h], dk[n][2 * h + 1], p.dk - col);
    }
}

// Ragged batches: gradients of rows that belong to no sequence are zero.
template <typename T>
__global__ void __launch_bounds__(256) delta_clear_rows(DeltaParams p) {
  const int first = p.plan[0], last = p.plan[p.sequences - 1] + p.plan[2 * p.sequences - 1];
  const int outside = first + (p.tokens - last);
  for (int i = blockIdx.x; i < outside; i += gridDim.x) {
    const long long t = i < first ? i : last + (i - first);
    for (int j = threadIdx.x; j < p.hk * p.dk; j += 256) {
      static_cast<T*>(p.dq)[t * p.hk * p.dk + j] = down<T>(0.f);
      static_cast<T*>(p.dk_out)[t * p.hk * p.dk + j] = down<T>(0.f);
    }
    for (int j = threadIdx.x; j < p.hv * p.dv; j += 256) static_cast<T*>(p.dv_out)[t * p.hv * p.dv + j] = down<T>(0.f);
    for (int j = threadIdx.x; j < p.hv; j += 256) {
      if (p.gates32) {
        static_cast<float*>(p.dg)[t * p.hv + j] = 0.f;
        static_cast<float*>(p.dbeta)[t * p.hv + j] = 0.f;
      } else {
        static_cast<T*>(p.dg)[t * p.hv + j] = down<T>(0.f);
        static_cast<T*>(p.dbeta)[t * p.hv + j] = down<T>(0.f);
      }
    }
  }
}

}  // namespace seq
}  // namespace pla
