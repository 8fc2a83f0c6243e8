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
//     dbeta = k . (Y - e^G dX S0^T) + dX . v,    Y = (Gamma . dA) K
//     dG = beta k . (Y - e^G dX S0^T) + q . dq - k . (N^T Q + B^T K) - H,    H = e^{G_C - G} k . (U D^T)
//     dG_C += e^{G_C} <S0, D> + sum H,      dg = sums of dG from each token to the chunk's end.
// S0 and U come from the forward's sweep run again: the forward keeps only its
// inputs.  Every sum has a fixed order.
#pragma once

#include "delta_sweep.cuh"

namespace pla {
namespace seq {

template <typename T, int DK, int VB, int STAGES, int PER_SM>
__global__ void __launch_bounds__(VB * 8, PER_SM) delta_sweep_back(DeltaParams p) {
  using L = DeltaLayout<T, DK>;
  using M = SweepShared<T, DK, VB, true>;
  constexpr int IN = L::kIn, QN = DK / 32, kPitch = Slab<T, VB>::kPitch;
  extern __shared__ __align__(128) char shared_bytes[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = warp % (VB / 16), wn = warp / (VB / 16), m0 = wm * 16;
  const SweepAt a = sweep_at(p, VB);
  Ring<L, STAGES> ring;
  ring.begin(shared_bytes, VB / 4);
  M& m = *reinterpret_cast<M*>(shared_bytes + kSweepRing + STAGES * L::kStage);
  const uint32_t dt = shared_u32(m.s), yt = shared_u32(m.a), xt = shared_u32(m.b), wt = shared_u32(m.c), ft = shared_u32(m.d);
  const T* d_o = static_cast<const T*>(p.d_o) + a.batch * p.do_batch + a.lo * p.do_token + a.vh * p.do_head + a.column;
  const long long dv_step = static_cast<long long>(p.hv) * p.dv;
  T* dv = static_cast<T*>(p.dv_out) + (static_cast<long long>(a.batch) * p.tokens + a.lo) * dv_step +
          static_cast<long long>(a.vh) * p.dv + a.column;
  if (threadIdx.x == 0)
    for (int i = 0; i < STAGES && i < a.chunks; ++i) ring.fill(p, i, a.first + a.chunks - 1 - i, a.kh, a.vh);
  if (a.chunks)
    slab_fetch<T, VB>(m.slab[0], d_o + (a.chunks - 1) * kChunk * p.do_token, p.do_token, a.len - (a.chunks - 1) * kChunk,
                      a.width, p.vec_do);
  const Walk dw(dt + at_mk<DK>(lane, m0, 0)), yw(yt + at_mk<kChunk>(lane, m0, 0));  // planes of D and Y; the others follow Y's
  const Walk kw(at_nk<DK>(lane, wn * 16, 0));                                       // in K
  const uint32_t ts = at_kn<kChunk>(lane, wn * 16, 0);                              // in T and P
  uint32_t ks[QN / 2];                                                              // in K and Q, for the state's update
#pragma unroll
  for (int n = 0; n < QN / 2; ++n) ks[n] = at_kn<DK>(lane, wn * (DK / 4) + n * 16, 0);
  float d[QN][4], top[2];
  Pow2 fd[2];
  state_load(p.dstate_out, p, a, m0, wn * (DK / 4), lane, d);
  {
    row_max(d, top);
    share(m.most_s, wn, m0, lane, top[0], top[1]);
    __syncthreads();
    float4 all[2];
    shared_of(m.most_s, m0, lane, all);
    fd[0] = scale_below(most_of(all[0]));
    fd[1] = scale_below(most_of(all[1]));
    tile_write<DK>(m.s, M::kWide, m0, wn * (DK / 4), lane, d, fd);
  }

  for (int turn = 0; turn < a.chunks; ++turn) {
    const int c = a.chunks - 1 - turn, len = min(kChunk, a.len - c * kChunk);
    const long long head_at = static_cast<long long>(a.first + c) * p.hv + a.vh;
    if (wn == 0 && (lane & 3) == 0) {
      m.keep_s[m0 + (lane >> 2)] = fd[0].inverse;
      m.keep_s[m0 + (lane >> 2) + 8] = fd[1].inverse;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // planes of D and this chunk's do are there; the other slab is free
    if (!__syncthreads_and(ring.wait())) return ring.give_up(a.chunks - turn);
    const char* stage = ring.stage();
    if (c > 0)
      slab_fetch<T, VB>(m.slab[~turn & 1], d_o + (c - 1) * kChunk * p.do_token, p.do_token, kChunk, a.width, p.vec_do);
    keep_tile<VB, DK>(m.s, m.keep_s, p.dstates + kept_at<DK>(p, head_at), p.scales + (head_at * 4 + 1) * p.rows, p.rows,
                          a.column);
    const uint32_t kt = shared_u32(stage), qt = kt + IN * L::kTile, tt = kt + L::kTiles, pt = tt + L::kT;
    const char* coef = stage + L::kTiles + L::kT + L::kP;
    const float4 bounds = *reinterpret_cast<const float4*>(coef + kBounds * kChunk * 4);
    const float decay = reinterpret_cast<const float*>(coef)[kDecay * kChunk];
    float2 w[2];
    float g[2][4];  // e^G do'
    {
      float f[2][4];
      slab_read<T, VB>(m.slab[turn & 1], wn * 16, m0, lane, f);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) g[n][e] = f[n][e];
      coef_read(coef, kOutP, wn * 2, lane, w);
      scale_columns(f, w);
      row_max(f, top);
      const Pow2 fw[2] = {pow2_for(top[0]), pow2_for(top[1])};
      share(m.scale_c, wn, m0, lane, fw[0].inverse, fw[1].inverse);
      tile_write<kChunk>(m.c, M::kNarrow, m0, wn * 16, lane, f, fw);
      coef_read(coef, kOutQ, wn * 2, lane, w);
      scale_columns(g, w);
      row_max(g, top);
      share(m.most_d, wn, m0, lane, top[0], top[1]);
    }
    // (K D)^T
    float du[2][4];
#pragma unroll
    for (int kk = 0; kk < DK / 16; ++kk) {
      uint32_t hi[4], lo[4];
      tile_operand(dw[kk], M::kWide, hi, lo);
      product<IN, false>(du[0], du[1], hi, lo, kt + kw[kk], L::kTile, kk == 0);
    }
    float4 most[2];
    shared_of(m.most_s, m0, lane, most);
    coef_read(coef, kTail, wn * 2, lane, w);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) du[n][e] *= (e & 1 ? w[n].y : w[n].x) * fd[e >> 1].inverse;
    __syncthreads();
    // dU = P^T do' + e^{G_C - G} (K D): tokens j take from i >= j
    float4 back[2], most_g[2];
    shared_of(m.scale_c, m0, lane, back);
    shared_of(m.most_d, m0, lane, most_g);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4];
      float bx[2][4];
      tile_operand(yw[kk] + (wt - yt), M::kNarrow, hi, lo);
      product<kPlanes, true>(bx[0], bx[1], hi, lo, pt + ts + kk * 16 * kChunk * 2, L::kSquare, true);
      add_scaled(du, bx, element(back[0], kk), element(back[1], kk));
    }
    coef_read(coef, kTRow, wn * 2, lane, w);
    scale_columns(du, w);
    {
      row_max(du, top);
      const Pow2 fy[2] = {pow2_for(top[0]), pow2_for(top[1])};
      share(m.scale_a, wn, m0, lane, fy[0].inverse, fy[1].inverse);
      tile_write<kChunk>(m.a, M::kNarrow, m0, wn * 16, lane, du, fy);
    }
    __syncthreads();
    // dX^T = (T^T dU)^T
    float x[2][4] = {};
    shared_of(m.scale_a, m0, lane, back);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4];
      float bx[2][4];
      tile_operand(yw[kk], M::kNarrow, hi, lo);
      product<kPlanes, true>(bx[0], bx[1], hi, lo, tt + ts + kk * 16 * kChunk * 2, L::kSquare, true);
      add_scaled(x, bx, element(back[0], kk), element(back[1], kk));
    }
    const float bound_x[2] = {kSumTop * kPlaneTop * most_of(back[0]), kSumTop * kPlaneTop * most_of(back[1])};
    // dX is kept, at a scale from its bound; do' is done with
    const Pow2 fk[2] = {scale_below(bound_x[0]), scale_below(bound_x[1])};
    tile_write<kChunk>(m.c, M::kNarrow, m0, wn * 16, lane, x, fk);
    if (wn == 0 && (lane & 3) == 0) {
      m.keep_c[m0 + (lane >> 2)] = fk[0].inverse;
      m.keep_c[m0 + (lane >> 2) + 8] = fk[1].inverse;
    }
    // e^G do' and -beta e^G dX at one scale
    float bound_f[2];
    Pow2 ff[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bound_f[h] = fmaxf(most_of(most_g[h]), bounds.z * bound_x[h]);
      ff[h] = scale_below(bound_f[h]);
    }
    tile_write<kChunk>(m.d, M::kNarrow, m0, wn * 16, lane, g, ff);
    {
      float out[2][4];
      float2 b[2];
      coef_read(coef, kBeta, wn * 2, lane, b);
      coef_read(coef, kDown, wn * 2, lane, w);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          out[n][e] = (e & 1 ? b[n].y : b[n].x) * x[n][e];
          x[n][e] *= e & 1 ? -w[n].y : -w[n].x;
        }
      tile_write<kChunk>(m.b, M::kNarrow, m0, wn * 16, lane, x, ff);
      strip_store<T, kPitch>(m.slab[turn & 1] + wn * 16 * kPitch + m0 * sizeof(T), lane, out, dv + (c * kChunk + wn * 16) * dv_step + m0, dv_step, len - wn * 16, a.width - m0,
                     p.vec_o);
    }
    __syncthreads();
    keep_tile<VB, kChunk>(m.c, m.keep_c, p.dxs + kept_at<kChunk>(p, head_at), p.scales + (head_at * 4 + 3) * p.rows,
                              p.rows, a.column);
    // D = e^{G_C} D + (e^G do')^T Q - (beta e^G dX)^T K
    float bs[QN][4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4];
      tile_operand(yw[kk] + (ft - yt), M::kNarrow, hi, lo);
#pragma unroll
      for (int n = 0; n < QN / 2; ++n)
        product<IN, true>(bs[2 * n], bs[2 * n + 1], hi, lo, qt + ks[n] + kk * 16 * DK * 2, L::kTile, kk == 0);
      tile_operand(yw[kk] + (xt - yt), M::kNarrow, hi, lo);
#pragma unroll
      for (int n = 0; n < QN / 2; ++n)
        product<IN, true>(bs[2 * n], bs[2 * n + 1], hi, lo, kt + ks[n] + kk * 16 * DK * 2, L::kTile, false);
    }
#pragma unroll
    for (int n = 0; n < QN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) d[n][e] = fmaf(bs[n][e], ff[e >> 1].inverse, decay * d[n][e]);
#pragma unroll
    for (int h = 0; h < 2; ++h) fd[h] = scale_below(fmaf(decay, most_of(most[h]), 2 * kSumTop * bound_f[h]));
    tile_write<DK>(m.s, M::kWide, m0, wn * (DK / 4), lane, d, fd);
    row_max(d, top);
    share(m.most_s, wn, m0, lane, top[0], top[1]);
    ring.next(p, turn + STAGES < a.chunks ? a.first + a.chunks - 1 - turn - STAGES : -1, a.kh, a.vh);
  }
  if (p.dstate_in) state_store(p.dstate_in, p, a, m0, wn * (DK / 4), lane, d);
}

// ---- what is left, in parallel over chunks ---------------------------------
// One (chunk, key head) a block, its value heads one after another, 64 value
// features at a time; 16 warps, each 16 tokens of a quarter of Dk (and of the
// 64 x 64 matrices).  S0, D, U and dX come as the planes that the sweeps had as
// operands; their row scales are brought to one by exact powers of two on the
// way to shared memory, because here the value features are summed over (an
// error of about 2^-27 of the head's largest: features far below it keep fewer
// bits).  The
// row and column sums over N . (Q K^T) and B . (K K^T) are taken as q . (N K),
// k . (N^T Q) and so on, so neither Q K^T nor K K^T is needed.
constexpr int kGradThreads = 512;
constexpr int kGradBlock = 64;  // value features at a time

template <typename T, int DK>
struct GradShared {
  static constexpr int IN = DeltaType<T>::kIn;
  alignas(128) __half tile[2][IN][kChunk * DK];  // K, Q planes
  union {
    struct {
      alignas(128) __half s[kPlanes][kGradBlock * DK], d[kPlanes][kGradBlock * DK];               // S^T, D^T
      __half u[kPlanes][kGradBlock * kChunk], x[kPlanes][kGradBlock * kChunk];                    // U^T, dX^T
      __half o[kPlanes][kChunk * kGradBlock];                                                // do
    } in;
    alignas(128) __half square[4][kPlanes][kChunk * kChunk];  // N f_k, N f_q (rows), Gamma dA f_k, B f_k (rows), all below the diagonal
  };
  alignas(16) float krow[kChunk];
  float qrow[kChunk], orow[kChunk];
  float beta[kChunk], hi[kChunk], lo[kChunk], down[kChunk], tail[kChunk];  // down: e^G, tail: e^{G_C - G}
  float ratio[4][128];         // a row's scale over the common one: S, dS, U, dX
  float dots[4][4][kChunk];    // quarters of Dk: k.r1, q.dq, k.(r3 + ..), k.Y
  float xv[8][kChunk];         // dX . v, groups of value features
  float warp_sum[16];
  float diagonal[kChunk];      // of N
  unsigned int common[4], most[4];
};

__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// d0, d1 += A B over planes, lo x lo left out.  The tensor cores cut a sum's
// last bits at every step, towards zero, so the small products are summed first
// (LOW) over all steps and the large ones after them: a third of the cuts happen
// at full size.
template <int PB, bool LOW>
__device__ __forceinline__ void planes_product(float (&d0)[4], float (&d1)[4], const uint32_t (&a)[kPlanes][4], const uint32_t (&b)[PB][4]) {
#pragma unroll
  for (int i = 0; i < kPlanes; ++i)
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      if (i + j >= kPlanes || LOW != (i + j > 0)) continue;
      mma(d0, a[i], b[j][0], b[j][1]);
      mma(d1, a[i], b[j][2], b[j][3]);
    }
}
// Two neighbours of a tile as the sum of its planes, times their row's factor.
template <int PLANES>
__device__ __forceinline__ void tile_pair(const __half* tile, uint32_t plane, uint32_t at, float row, float (&f)[2]) {
#pragma unroll
  for (int i = 0; i < PLANES; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(reinterpret_cast<const char*>(tile) + i * plane + at));
    f[0] = i ? f[0] + v.x : v.x;
    f[1] = i ? f[1] + v.y : v.y;
  }
  f[0] *= row, f[1] *= row;
}
template <int PLANES, bool TRANS>
__device__ __forceinline__ void planes_load(uint32_t (&f)[PLANES][4], uint32_t at, uint32_t plane) {
#pragma unroll
  for (int i = 0; i < PLANES; ++i)
    if (TRANS) ldsm_t(f[i], at + i * plane); else ldsm(f[i], at + i * plane);
}

// Rows [row0, row0 + 64) of kept planes: into registers, and from there, times
// their rows' ratios, into a tile.
template <int W>
struct Kept {
  static constexpr int kUnits = kGradBlock * W / 8 / kGradThreads;
  uint4 v[kUnits][kPlanes];
  __device__ __forceinline__ void fetch(const char* from, int rows, int row0, int used, int tid) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int at = i * kGradThreads + tid;
#pragma unroll
      for (int n = 0; n < kPlanes; ++n) {
        v[i][n] = make_uint4(0, 0, 0, 0);
        if (row0 + at / (W / 8) < used)
          v[i][n] = __ldg(reinterpret_cast<const uint4*>(from + (static_cast<long long>(n) * rows + row0) * W * 2) + at);
      }
    }
  }
  __device__ __forceinline__ void put(const float* ratio, int row0, int used, char* tile, int tid) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int at = i * kGradThreads + tid, row = row0 + at / (W / 8);
      const __half2 f = __float2half2_rn(row < used ? ratio[row] : 0.f);
#pragma unroll
      for (int n = 0; n < kPlanes; ++n) {
        __half2* h = reinterpret_cast<__half2*>(&v[i][n]);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = __hmul2(h[e], f);
        reinterpret_cast<uint4*>(tile + n * kGradBlock * W * 2)[at] = v[i][n];
      }
    }
  }
};

// Asks L2 for what a block will read of a (chunk, value head).
template <int DK>
__device__ __forceinline__ void prefetch_kept(const DeltaParams& p, long long head, int tid) {
  const int used = p.slabs * 16;
  const auto ask = [&](const char* from, int bytes) {
    for (int at = tid * 128; at < bytes; at += kGradThreads * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(from + at));
  };
#pragma unroll
  for (int n = 0; n < kPlanes; ++n) {
    const long long wide = static_cast<long long>(n) * p.rows * DK * 2, narrow = static_cast<long long>(n) * p.rows * kChunk * 2;
    ask(p.states + kept_at<DK>(p, head) + wide, used * DK * 2);
    ask(p.dstates + kept_at<DK>(p, head) + wide, used * DK * 2);
    ask(p.us + kept_at<kChunk>(p, head) + narrow, used * kChunk * 2);
    ask(p.dxs + kept_at<kChunk>(p, head) + narrow, used * kChunk * 2);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_row(T* to, const float (&f)[N], int count, bool whole) {
  if (whole) {
    store<T, N>(to, f);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < count) to[i] = down<T>(f[i]);
  }
}

template <typename T, int DK>
__global__ void __launch_bounds__(kGradThreads, 1) delta_gradient(DeltaParams p) {
  using L = DeltaLayout<T, DK>;
  constexpr int IN = L::kIn, NT = DK / 32;  // column tiles of a warp
  constexpr uint32_t kWide = kGradBlock * DK * 2, kNarrow = kGradBlock * kChunk * 2, kSq = kChunk * kChunk * 2;
  extern __shared__ __align__(128) char shared_bytes[];
  GradShared<T, DK>& s = *reinterpret_cast<GradShared<T, DK>*>(shared_bytes);
  const int chunk = blockIdx.x / p.hk, kh = blockIdx.x % p.hk;
  ChunkAt c;
  if (!chunk_at(p, chunk, &c)) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rb = warp & 3, cg = warp >> 2;  // 16 tokens; a quarter of the columns
  const int r0 = rb * 16 + (lane >> 2);
  const uint32_t kt = shared_u32(s.tile[0][0]), qt = shared_u32(s.tile[1][0]);
  const int group = p.hv / p.hk, used = p.slabs * 16;
  prefetch_kept<DK>(p, static_cast<long long>(chunk) * p.hv + kh * group, tid);
  {
    const uint4* from = reinterpret_cast<const uint4*>(p.tiles + (static_cast<long long>(chunk) * p.hk + kh) * L::kTiles);
#pragma unroll
    for (int i = 0; i < static_cast<int>(L::kTiles / 16 / kGradThreads); ++i)
      reinterpret_cast<uint4*>(s.tile)[i * kGradThreads + tid] = from[i * kGradThreads + tid];
    const float* coef = reinterpret_cast<const float*>(p.heads + (static_cast<long long>(chunk) * p.hv + kh * group) * L::kHead +
                                                       L::kT + L::kP);
    if (tid < kChunk) {
      s.krow[tid] = coef[kKRow * kChunk + tid];
      s.qrow[tid] = coef[kQRow * kChunk + tid];
    }
  }
  float dq[NT][4] = {}, dk[NT][4] = {};
  for (int sub = 0; sub < group; ++sub) {
    const int vh = kh * group + sub;
    const long long head_at = static_cast<long long>(chunk) * p.hv + vh;
    const float* coef = reinterpret_cast<const float*>(p.heads + head_at * L::kHead + L::kT + L::kP);
    // everything that the head's first steps need is on its way before any of it is waited for
    Kept<DK> ks, kd;
    Kept<kChunk> ku, kx;
    const auto fetch = [&](int v0) {
      ks.fetch(p.states + kept_at<DK>(p, head_at), p.rows, v0, used, tid);
      kd.fetch(p.dstates + kept_at<DK>(p, head_at), p.rows, v0, used, tid);
      ku.fetch(p.us + kept_at<kChunk>(p, head_at), p.rows, v0, used, tid);
      kx.fetch(p.dxs + kept_at<kChunk>(p, head_at), p.rows, v0, used, tid);
    };
    const float decay = __ldg(coef + kDecay * kChunk);
    const int kind = tid >> 7, scale_row = tid & 127;
    const float row_scale = scale_row < used ? __ldg(p.scales + (head_at * 4 + kind) * p.rows + scale_row) : 0.f;
    float c_hi = 0.f, c_lo = 0.f, c_beta = 0.f, c_last = 0.f, c_last_lo = 0.f;
    if (tid < kChunk) {
      c_hi = __ldg(coef + kSumHi * kChunk + tid), c_lo = __ldg(coef + kSumLo * kChunk + tid);
      c_beta = __ldg(coef + kBeta * kChunk + tid);
      c_last = __ldg(coef + kSumHi * kChunk + kChunk - 1), c_last_lo = __ldg(coef + kSumLo * kChunk + kChunk - 1);
    }
    // do: 8 threads a row, 8 features each of both blocks; one scale a row
    const int o_row = tid >> 3, o_col = (tid & 7) * 8;
    float o[2][8] = {};
    if (o_row < c.len) {
      const T* from = static_cast<const T*>(p.d_o) + c.batch * p.do_batch + (c.token + o_row) * p.do_token + vh * p.do_head;
      constexpr int V = 16 / sizeof(T) < 8 ? 16 / sizeof(T) : 8;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int col = b * kGradBlock + o_col;
        if (p.vec_do) {
#pragma unroll
          for (int e = 0; e < 8; e += V)
            if (col + e < p.dv) load<T, V>(from + col + e, *reinterpret_cast<float(*)[V]>(&o[b][e]));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < p.dv) o[b][e] = up(from[col + e]);
        }
      }
    }
    fetch(0);
    if (sub + 1 < group) prefetch_kept<DK>(p, head_at + 1, tid);
    __syncthreads();  // the last head is done with
    if (tid < 4) s.common[tid] = s.most[tid] = 0;
    if (tid < kChunk) {
      s.beta[tid] = c_beta;
      s.hi[tid] = c_hi;
      s.lo[tid] = c_lo;
      s.down[tid] = exp_sum(c_hi, c_lo);
      s.tail[tid] = expf((c_last - c_hi) + (c_last_lo - c_lo));
    }
    {
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fmaxf(fabsf(o[0][e]), fabsf(o[1][e])));
#pragma unroll
      for (int w = 4; w >= 1; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
      const Pow2 f = pow2_for(m);
      if ((tid & 7) == 0) s.orow[o_row] = f.inverse;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[0][e] *= f.f, o[1][e] *= f.f;
    }
    // scales of the kept planes: the largest of each kind is the common one
    {
      const unsigned int m = __reduce_max_sync(0xffffffffu, __float_as_uint(row_scale));
      // non-negative floats order as integers: the maximum does not depend on the order
      __syncthreads();  // common is cleared
      if (lane == 0) atomicMax(&s.common[kind], m);
    }
    __syncthreads();
    float common[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) common[i] = __uint_as_float(s.common[i]);
    s.ratio[kind][scale_row] = row_scale / __uint_as_float(s.common[kind]);

    float a_q[NT][4] = {}, a_x[NT][4] = {}, a_u[NT][4] = {}, a_p[2][4] = {}, a_a[2][4] = {};
    float sd = 0.f, xv = 0.f;
#pragma unroll 1
    for (int block = 0; block * kGradBlock < used; ++block) {
      const int v0 = block * kGradBlock;
      if (block) fetch(v0);
      __syncthreads();
      ks.put(s.ratio[0], v0, used, reinterpret_cast<char*>(s.in.s), tid);
      kd.put(s.ratio[1], v0, used, reinterpret_cast<char*>(s.in.d), tid);
      ku.put(s.ratio[2], v0, used, reinterpret_cast<char*>(s.in.u), tid);
      kx.put(s.ratio[3], v0, used, reinterpret_cast<char*>(s.in.x), tid);
      {
        Vec<uint32_t, 4> plane[kPlanes];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          split(block ? o[1][2 * e] : o[0][2 * e], block ? o[1][2 * e + 1] : o[0][2 * e + 1], &plane[0].e[e], &plane[1].e[e]);
#pragma unroll
        for (int n = 0; n < kPlanes; ++n)
          *reinterpret_cast<Vec<uint32_t, 4>*>(reinterpret_cast<char*>(s.in.o) + n * kNarrow + tile_at<kGradBlock>(o_row, tid & 7)) = plane[n];
      }
      float v[8] = {};  // of token tid & 63, eight features
      {
        const int t = tid & 63, col = v0 + (tid >> 6) * 8;
        const T* from = static_cast<const T*>(p.v) + c.batch * p.v_batch + (c.token + t) * p.v_token + vh * p.v_head;
        constexpr int V = 16 / sizeof(T) < 8 ? 16 / sizeof(T) : 8;
        if (t < c.len) {
          if (p.vec_v) {
#pragma unroll
            for (int e = 0; e < 8; e += V)
              if (col + e < p.dv) load<T, V>(from + col + e, *reinterpret_cast<float(*)[V]>(&v[e]));
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (col + e < p.dv) v[e] = up(from[col + e]);
          }
        }
      }
      __syncthreads();
      const uint32_t st = shared_u32(s.in.s), dt = shared_u32(s.in.d), ut = shared_u32(s.in.u), xt = shared_u32(s.in.x),
                     ot = shared_u32(s.in.o);
      {  // dX . v and <S, D>
        const int t = tid & 63, row = (tid >> 6) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t at = tile_at<kChunk>(row + e, t >> 3) + (t & 7) * 2;
#pragma unroll
          for (int n = 0; n < kPlanes; ++n)
            xv = fmaf(common[3] * __half2float(*reinterpret_cast<const __half*>(reinterpret_cast<const char*>(s.in.x) + n * kNarrow + at)), v[e], xv);
        }
#pragma unroll
        for (int i = 0; i < kGradBlock * DK / 8 / kGradThreads; ++i) {
          float f[8], g[8];
#pragma unroll
          for (int n = 0; n < kPlanes; ++n) {
            const uint4 a = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(s.in.s) + n * kWide)[i * kGradThreads + tid];
            const uint4 b = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(s.in.d) + n * kWide)[i * kGradThreads + tid];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 x = __half22float2(reinterpret_cast<const __half2*>(&a)[e]), y = __half22float2(reinterpret_cast<const __half2*>(&b)[e]);
              if (n == 0)
                f[2 * e] = x.x, f[2 * e + 1] = x.y, g[2 * e] = y.x, g[2 * e + 1] = y.y;
              else
                f[2 * e] += x.x, f[2 * e + 1] += x.y, g[2 * e] += y.x, g[2 * e + 1] += y.y;
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) sd = fmaf(f[e], g[e], sd);
        }
      }
      const auto products = [&](auto low) {
      constexpr bool LOW = decltype(low)::value;
#pragma unroll 1
      for (int kk = 0; kk < kGradBlock / 16; ++kk) {
        uint32_t fo[kPlanes][4], fu[kPlanes][4], fx[kPlanes][4], b[kPlanes][4];
        planes_load<kPlanes, false>(fo, ot + at_mk<kGradBlock>(lane, rb * 16, kk * 16), kNarrow);
        planes_load<kPlanes, true>(fu, ut + at_km<kChunk>(lane, rb * 16, kk * 16), kNarrow);
        planes_load<kPlanes, true>(fx, xt + at_km<kChunk>(lane, rb * 16, kk * 16), kNarrow);
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
          const uint32_t at = at_kn<DK>(lane, cg * (DK / 4) + n * 16, kk * 16);
          planes_load<kPlanes, true>(b, st + at, kWide);
          planes_product<kPlanes, LOW>(a_q[2 * n], a_q[2 * n + 1], fo, b);
          planes_product<kPlanes, LOW>(a_x[2 * n], a_x[2 * n + 1], fx, b);
          planes_load<kPlanes, true>(b, dt + at, kWide);
          planes_product<kPlanes, LOW>(a_u[2 * n], a_u[2 * n + 1], fu, b);
        }
        planes_load<kPlanes, true>(b, ut + at_kn<kChunk>(lane, cg * 16, kk * 16), kNarrow);
        planes_product<kPlanes, LOW>(a_p[0], a_p[1], fo, b);
        planes_product<kPlanes, LOW>(a_a[0], a_a[1], fx, b);
      }
      };
      products(std::true_type{});
      products(std::false_type{});
    }
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) sd += __shfl_xor_sync(0xffffffffu, sd, w);
    if (lane == 0) s.warp_sum[warp] = sd;
    s.xv[tid >> 6][tid & 63] = xv;

    // parts of dq and dk that see the states, and their products with q and k
    float dot[4][2] = {};
    float to_one[2], to_two[2], to_three[2], beta[2], k_row[2], q_row[2];  // of this lane's rows
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = r0 + h * 8;
      to_one[h] = -s.down[i] * (common[3] * common[0]);
      to_two[h] = p.scale * s.down[i] * (s.orow[i] * common[0]);
      to_three[h] = s.tail[i] * (common[2] * common[1]);
      beta[h] = s.beta[i];
      k_row[h] = s.krow[i], q_row[h] = s.qrow[i];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = r0 + h * 8;
        const uint32_t at = tile_at<DK>(i, cg * (DK / 32) + n) + (lane & 3) * 4;
        float kv[2], qv[2];
        tile_pair<IN>(s.tile[0][0], L::kTile, at, k_row[h], kv);
        tile_pair<IN>(s.tile[1][0], L::kTile, at, q_row[h], qv);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at_e = 2 * h + e;
          const float one = to_one[h] * a_x[n][at_e], two = to_two[h] * a_q[n][at_e], three = to_three[h] * a_u[n][at_e];
          dot[0][h] = fmaf(kv[e], one, dot[0][h]);
          dot[1][h] = fmaf(qv[e], two, dot[1][h]);
          dot[2][h] = fmaf(kv[e], three, dot[2][h]);
          dq[n][at_e] += two;
          dk[n][at_e] += fmaf(beta[h], one, three);
        }
      }
    // sum of H = e^{G_C - G} k . (U D^T) over the chunk, before the rest joins that dot
    float h_part = quad_sum(dot[2][0]) + quad_sum(dot[2][1]);

    // N, Gamma dA and B with the row factors of what they meet
    float sq[4][2][4], top[4] = {};
    {
      float row_hi[2], row_lo[2], row_n[2], row_k[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = r0 + h * 8;
        row_hi[h] = s.hi[i], row_lo[h] = s.lo[i], row_k[h] = beta[h] * k_row[h];
        row_n[h] = p.scale * (s.orow[i] * common[2]);
      }
      const float to_a = -(common[3] * common[2]);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int j0 = cg * 16 + n * 8 + (lane & 3) * 2;
        const float2 hi = *reinterpret_cast<const float2*>(&s.hi[j0]), lo = *reinterpret_cast<const float2*>(&s.lo[j0]),
                     kj = *reinterpret_cast<const float2*>(&s.krow[j0]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1, i = r0 + h * 8, j = j0 + (e & 1);
          const float gamma = exp_fast((row_hi[h] - (e & 1 ? hi.y : hi.x)) + (row_lo[h] - (e & 1 ? lo.y : lo.x)));
          if (i == j) s.diagonal[i] = row_n[h] * a_p[n][e];
          const float nn = j < i ? gamma * (row_n[h] * a_p[n][e]) : 0.f, ga = j < i ? gamma * (to_a * a_a[n][e]) : 0.f;
          sq[0][n][e] = nn * (e & 1 ? kj.y : kj.x);
          sq[1][n][e] = nn * q_row[h];
          sq[2][n][e] = ga * (e & 1 ? kj.y : kj.x);
          sq[3][n][e] = ga * row_k[h];
#pragma unroll
          for (int w = 0; w < 4; ++w) top[w] = fmaxf(top[w], fabsf(sq[w][n][e]));
        }
      }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const unsigned int m = __reduce_max_sync(0xffffffffu, __float_as_uint(top[w]));
      if (lane == 0) atomicMax(&s.most[w], m);
    }
    __syncthreads();
    Pow2 f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) f[w] = pow2_for(__uint_as_float(s.most[w]));
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = tile_at<kChunk>(r0 + h * 8, cg * 2 + n) + (lane & 3) * 4;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t hi, lo;
          split(sq[w][n][2 * h] * f[w].f, sq[w][n][2 * h + 1] * f[w].f, &hi, &lo);
          char* to = reinterpret_cast<char*>(s.square[w]);
          *reinterpret_cast<uint32_t*>(to + at) = hi;
          *reinterpret_cast<uint32_t*>(to + kSq + at) = lo;
        }
      }
    __syncthreads();
    // dq += N K; dk += N^T Q + beta Y + B^T K, Y = (Gamma dA) K; all lower triangular.  N's diagonal gives q . dq and
    // k . dk the same, which cancel in dG: it is added to dq and dk alone, so that no rest of a rounding stays
    {
      float b_q[NT][4] = {}, b_n[NT][4] = {}, b_y[NT][4] = {}, b_t[NT][4] = {};
      const uint32_t base = shared_u32(s.square);
      constexpr uint32_t one = kPlanes * kSq;
      const auto products = [&](auto low) {
      constexpr bool LOW = decltype(low)::value;
#pragma unroll 1
      for (int kk = 0; kk < 4; ++kk) {
        const uint32_t mk = at_mk<kChunk>(lane, rb * 16, kk * 16), km = at_km<kChunk>(lane, rb * 16, kk * 16);
        uint32_t a[kPlanes][4], g[kPlanes][4], b[IN][4];
        if (kk <= rb) {
          planes_load<kPlanes, false>(a, base + mk, kSq);
          planes_load<kPlanes, false>(g, base + 2 * one + mk, kSq);
#pragma unroll
          for (int n = 0; n < NT / 2; ++n) {
            planes_load<IN, true>(b, kt + at_kn<DK>(lane, cg * (DK / 4) + n * 16, kk * 16), L::kTile);
            planes_product<IN, LOW>(b_q[2 * n], b_q[2 * n + 1], a, b);
            planes_product<IN, LOW>(b_y[2 * n], b_y[2 * n + 1], g, b);
          }
        }
        if (kk >= rb) {
          planes_load<kPlanes, true>(a, base + one + km, kSq);
          planes_load<kPlanes, true>(g, base + 3 * one + km, kSq);
#pragma unroll
          for (int n = 0; n < NT / 2; ++n) {
            const uint32_t at = at_kn<DK>(lane, cg * (DK / 4) + n * 16, kk * 16);
            planes_load<IN, true>(b, qt + at, L::kTile);
            planes_product<IN, LOW>(b_n[2 * n], b_n[2 * n + 1], a, b);
            planes_load<IN, true>(b, kt + at, L::kTile);
            planes_product<IN, LOW>(b_t[2 * n], b_t[2 * n + 1], g, b);
          }
        }
      }
      };
      products(std::true_type{});
      products(std::false_type{});
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = r0 + h * 8;
          const uint32_t at = tile_at<DK>(i, cg * (DK / 32) + n) + (lane & 3) * 4;
          float kv[2], qv[2];
          tile_pair<IN>(s.tile[0][0], L::kTile, at, k_row[h], kv);
          tile_pair<IN>(s.tile[1][0], L::kTile, at, q_row[h], qv);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int at_e = 2 * h + e;
            const float two = b_q[n][at_e] * f[0].inverse, y = b_y[n][at_e] * f[2].inverse;
            const float three = fmaf(b_n[n][at_e], f[1].inverse, b_t[n][at_e] * f[3].inverse);
            dot[1][h] = fmaf(qv[e], two, dot[1][h]);
            dot[2][h] = fmaf(kv[e], three, dot[2][h]);
            dot[3][h] = fmaf(kv[e], y, dot[3][h]);
            dq[n][at_e] += fmaf(s.diagonal[i], kv[e], two);
            dk[n][at_e] += fmaf(beta[h], y, fmaf(s.diagonal[i], qv[e], three));
          }
        }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = r0 + h * 8;
        const float v = quad_sum(dot[w][h]);
        if ((lane & 3) == 0) s.dots[cg][w][i] = v;
      }
    // H summed over this warp's rows (a lane of each quad)
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) h_part += __shfl_xor_sync(0xffffffffu, h_part, w);
    if (lane == 0) s.warp_sum[warp] = fmaf(decay * (common[0] * common[1]), s.warp_sum[warp], h_part);
    __syncthreads();
    if (warp == 0) {  // the gates' gradients
      float dg[2], total = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w)  // quarters of Dk as in the dots: a single token's H leaves nothing
        total += (s.warp_sum[w] + s.warp_sum[4 + w]) + (s.warp_sum[8 + w] + s.warp_sum[12 + w]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 2 * lane + e;
        float v[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) v[w] = (s.dots[0][w][t] + s.dots[1][w][t]) + (s.dots[2][w][t] + s.dots[3][w][t]);
        const float with_v = ((s.xv[0][t] + s.xv[1][t]) + (s.xv[2][t] + s.xv[3][t])) + ((s.xv[4][t] + s.xv[5][t]) + (s.xv[6][t] + s.xv[7][t]));
        dg[e] = s.beta[t] * (v[0] + v[3]) + v[1] - v[2];
        const float db = (v[0] + v[3]) + with_v;
        if (t < c.len) {
          const long long at = (static_cast<long long>(c.batch) * p.tokens + c.token + t) * p.hv + vh;
          if (p.gates32)
            static_cast<float*>(p.dbeta)[at] = db;
          else
            static_cast<T*>(p.dbeta)[at] = down<T>(db);
        }
      }
      if (lane == 31) dg[1] += total;
      dg[0] += dg[1];
      float after = dg[0];  // sums from this pair to the end
#pragma unroll
      for (int w = 1; w < 32; w <<= 1) {
        const float v = __shfl_down_sync(0xffffffffu, after, w);
        if (lane + w < 32) after += v;
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
  }
  // dq, dk: dense [batch, tokens, key heads, Dk]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = r0 + h * 8, col = cg * (DK / 4) + n * 8 + (lane & 3) * 2;
      if (t >= c.len || col >= p.dk) continue;
      const long long at = ((static_cast<long long>(c.batch) * p.tokens + c.token + t) * p.hk + kh) * p.dk + col;
      const float q2[2] = {dq[n][2 * h], dq[n][2 * h + 1]}, k2[2] = {dk[n][2 * h], dk[n][2 * h + 1]};
      store_row(static_cast<T*>(p.dq) + at, q2, p.dk - col, p.pair_qk);
      store_row(static_cast<T*>(p.dk_out) + at, k2, p.dk - col, p.pair_qk);
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
