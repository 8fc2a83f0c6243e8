// delta_sweep: walks the chunks of a sequence with the state in registers
// (delta_common.cuh has the mathematics).
//
// The columns of S (one per value feature) never meet, so a warp takes 16 of
// them through the whole sequence on its own: it holds S^T [16, Dk] as the
// accumulators of m16n8k16 products.  Every product of a chunk has the value
// features as its 16 rows,
//     (K S)^T = S^T K^T,  U^T = X^T T^T,  O^T = S^T Q^T + U^T P^T,  S^T += U^T K,
// and the accumulator of one is, register for register, the left operand of
// the next: state, X and U never leave the registers.  K, Q, T and P are the
// right operands, read from shared memory by ldmatrix; the warps of a block
// share them.  They lie in the workspace as whole tiles, already in the
// shared-memory order, and come by bulk copies a few chunks ahead.
#pragma once

#include "delta_common.cuh"

namespace pla {
namespace seq {

__device__ unsigned int g_sequence_faults;  // bit 0: a wait for a copy ran out

__device__ __forceinline__ void barrier_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(shared_u32(bar)) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(shared_u32(bar)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool barrier_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(shared_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
// Waits about two seconds at most; then records the fault and lets the caller
// carry on (its results are undefined, the host sees the fault word).
__device__ __forceinline__ void barrier_wait(uint64_t* bar, uint32_t parity) {
  if (barrier_try(bar, parity)) return;
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  do {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (barrier_try(bar, parity)) return;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  } while (t - t0 < 2000000000ull);
  atomicOr(&g_sequence_faults, 1u);
}
__device__ __forceinline__ void bulk_copy(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   shared_u32(to)),
               "l"(from), "r"(bytes), "r"(shared_u32(bar))
               : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// The 64 x 16 part of v (or do, or o) that a warp works on, in its own shared
// memory: rows of 16 features, the pitch spreads eight rows over the banks.
template <typename T>
struct Slab {
  static constexpr int kPitch = 16 * sizeof(T) + 16;
  static constexpr int kBytes = kChunk * kPitch;
};

// Starts the copy of rows [0, len) of a slab; zeros elsewhere.  16-byte
// copies if the rows allow it, single elements otherwise.
template <typename T>
__device__ __forceinline__ void slab_fetch(char* to, const T* from, long long step, int len, int width, int vec, int lane) {
  constexpr int UNIT = 16 / sizeof(T), PER = 16 / UNIT;  // units of a row
  if (vec && width == 16 && len == kChunk) {
#pragma unroll
    for (int i = 0; i < kChunk * PER / 32; ++i) {
      const int at = i * 32 + lane, row = at / PER, u = at % PER;
      copy16(shared_u32(to) + row * Slab<T>::kPitch + u * 16, from + row * step + u * UNIT);
    }
  } else {
    for (int at = lane; at < kChunk * 16; at += 32) {
      const int row = at >> 4, col = at & 15;
      reinterpret_cast<T*>(to + row * Slab<T>::kPitch)[col] =
          row < len && col < width ? from[row * step + col] : down<T>(0.f);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

// A slab as accumulators of [features x tokens]: f[n][e] of token tile n.
template <typename T>
__device__ __forceinline__ void slab_read(const char* from, int lane, float (&f)[8][4]) {
  if constexpr (sizeof(T) == 2) {
    const int m = lane >> 3;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      uint32_t r[4];  // token tiles 2n, 2n + 1, features 0-7 and 8-15
      ldsm_t(r, shared_u32(from) + (n * 16 + (m >> 1) * 8 + (lane & 7)) * Slab<T>::kPitch + (m & 1) * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Vec<T, 2> v = *reinterpret_cast<const Vec<T, 2>*>(&r[i]);
        f[2 * n + (i >> 1)][(i & 1) * 2] = up(v.e[0]);
        f[2 * n + (i >> 1)][(i & 1) * 2 + 1] = up(v.e[1]);
      }
    }
  } else {
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[n][e] = up(reinterpret_cast<const T*>(from + (n * 8 + (lane & 3) * 2 + (e & 1)) *
                                                           Slab<T>::kPitch)[(lane >> 2) + (e >> 1) * 8]);
  }
}

template <typename T>
__device__ __forceinline__ void slab_write(char* to, int lane, const float (&f)[8][4]) {
  if constexpr (sizeof(T) == 2) {
    const int m = lane >> 3;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Vec<T, 2> v;
        v.e[0] = down<T>(f[2 * n + (i >> 1)][(i & 1) * 2]);
        v.e[1] = down<T>(f[2 * n + (i >> 1)][(i & 1) * 2 + 1]);
        r[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
      asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(
                       shared_u32(to) + (n * 16 + (m >> 1) * 8 + (lane & 7)) * Slab<T>::kPitch + (m & 1) * 16),
                   "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                   : "memory");
    }
  } else {
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<T*>(to + (n * 8 + (lane & 3) * 2 + (e & 1)) * Slab<T>::kPitch)[(lane >> 2) + (e >> 1) * 8] =
            down<T>(f[n][e]);
  }
}

template <typename T>
__device__ __forceinline__ void slab_store(const char* from, T* to, long long step, int len, int width, int vec, int lane) {
  constexpr int UNIT = 16 / sizeof(T), PER = 16 / UNIT;
  if (vec && width == 16) {
#pragma unroll
    for (int i = 0; i < kChunk * PER / 32; ++i) {
      const int at = i * 32 + lane, row = at / PER, u = at % PER;
      if (row < len)
        *reinterpret_cast<uint4*>(to + row * step + u * UNIT) =
            *reinterpret_cast<const uint4*>(from + row * Slab<T>::kPitch + u * 16);
    }
  } else {
    for (int at = lane; at < kChunk * 16; at += 32) {
      const int row = at >> 4, col = at & 15;
      if (row < len && col < width) to[row * step + col] = reinterpret_cast<const T*>(from + row * Slab<T>::kPitch)[col];
    }
  }
}

// Largest magnitude of each of the two accumulator rows of a lane's quad.
template <int N>
__device__ __forceinline__ void row_max(const float (&f)[N][4], float (&m)[2]) {
  m[0] = m[1] = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    m[0] = fmaxf(m[0], fmaxf(fabsf(f[n][0]), fabsf(f[n][1])));
    m[1] = fmaxf(m[1], fmaxf(fabsf(f[n][2]), fabsf(f[n][3])));
  }
  m[0] = quad_max(m[0]);
  m[1] = quad_max(m[1]);
}

// Over the quads of a warp, of what row_max gives.
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Accumulators of column tiles 2k, 2k + 1, times their rows' factors, as the
// left operand of step k of the next product.
template <int PLANES>
__device__ __forceinline__ void as_operand(const float (&x)[4], const float (&y)[4], const Pow2 (&s)[2], uint32_t (&hi)[4],
                                           uint32_t (&lo)[4]) {
  split<PLANES>(x[0] * s[0].f, x[1] * s[0].f, &hi[0], &lo[0]);
  split<PLANES>(x[2] * s[1].f, x[3] * s[1].f, &hi[1], &lo[1]);
  split<PLANES>(y[0] * s[0].f, y[1] * s[0].f, &hi[2], &lo[2]);
  split<PLANES>(y[2] * s[1].f, y[3] * s[1].f, &hi[3], &lo[3]);
}

// d0, d1 += A B for two column tiles: A in PA planes (hi, lo), B in PB planes
// `apart` bytes apart at `at`; the product of two lo planes is left out.
template <int PA, int PB, bool TRANS>
__device__ __forceinline__ void product(float (&d0)[4], float (&d1)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                        uint32_t at, uint32_t apart) {
  uint32_t b[4];
  if (TRANS) ldsm_t(b, at); else ldsm(b, at);
  mma(d0, hi, b[0], b[1]);
  mma(d1, hi, b[2], b[3]);
  if (PA > 1) {
    mma(d0, lo, b[0], b[1]);
    mma(d1, lo, b[2], b[3]);
  }
  if (PB > 1) {
    if (TRANS) ldsm_t(b, at + apart); else ldsm(b, at + apart);
    mma(d0, hi, b[0], b[1]);
    mma(d1, hi, b[2], b[3]);
  }
}

// Copies of the chunks' tiles into a ring of stages.  Thread 0 issues them; a
// stage is refilled when every warp has arrived at its `empty` barrier.
template <typename L>
struct Ring {
  char* stages;
  uint64_t *full, *empty;
  int count;
  __device__ __forceinline__ void begin(char* bytes, int n, int warps) {
    full = reinterpret_cast<uint64_t*>(bytes);
    empty = full + 8;
    stages = bytes + 128;
    count = n;
    if (threadIdx.x == 0) {
      for (int i = 0; i < n; ++i) {
        barrier_init(full + i, 1);
        barrier_init(empty + i, warps);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
  }
  __device__ __forceinline__ void fill(const DeltaParams& p, int turn, int chunk, int kh, int vh) {
    const int s = turn % count;
    if (turn >= count) barrier_wait(empty + s, (turn / count - 1) & 1);
    char* to = stages + s * L::kStage;
    barrier_expect(full + s, L::kStage);
    bulk_copy(to, p.tiles + (static_cast<long long>(chunk) * p.hk + kh) * L::kTiles, L::kTiles, full + s);
    bulk_copy(to + L::kTiles, p.heads + (static_cast<long long>(chunk) * p.hv + vh) * L::kHead, L::kHead, full + s);
  }
  __device__ __forceinline__ const char* wait(int turn) {
    barrier_wait(full + turn % count, (turn / count) & 1);
    return stages + (turn % count) * L::kStage;
  }
  __device__ __forceinline__ void done(int turn, int lane) {
    __syncwarp();
    if (lane == 0) barrier_arrive(empty + turn % count);
  }
};

// What a block of a sweep works on: value head and slabs of one sequence.
struct SweepAt {
  int sequence, vh, kh, slab, batch, lo, len, first, chunks, width;
};
__device__ __forceinline__ SweepAt sweep_at(const DeltaParams& p, int warps, int warp) {
  SweepAt a;
  const int parts = (p.slabs + warps - 1) / warps;
  int b = blockIdx.x;
  a.slab = (b % parts) * warps + warp;
  b /= parts;
  a.vh = b % p.hv;
  a.sequence = b / p.hv;
  a.kh = a.vh / (p.hv / p.hk);
  if (p.cu) {
    a.batch = 0;
    a.lo = p.plan[a.sequence];
    a.len = p.plan[p.sequences + a.sequence];
    a.first = p.plan[2 * p.sequences + a.sequence];
  } else {
    a.batch = a.sequence;
    a.lo = 0;
    a.len = p.tokens;
    a.first = a.sequence * p.row_chunks;
  }
  a.chunks = (a.len + kChunk - 1) / kChunk;
  a.width = min(16, p.dv - a.slab * 16);  // <= 0: a warp without columns only keeps the ring going
  return a;
}

// S^T of a slab from or to [Dk, Dv] fp32.
template <int DK>
__device__ __forceinline__ void state_load(const float* from, const DeltaParams& p, const SweepAt& a, int lane, float (&s)[DK / 8][4]) {
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int dk = n * 8 + (lane & 3) * 2 + (e & 1), dv = (lane >> 2) + (e >> 1) * 8;
      s[n][e] = from && dk < p.dk && dv < a.width
                    ? from[(static_cast<long long>(a.sequence) * p.hv + a.vh) * p.dk * p.dv + static_cast<long long>(dk) * p.dv +
                           a.slab * 16 + dv]
                    : 0.f;
    }
}
template <int DK>
__device__ __forceinline__ void state_store(float* to, const DeltaParams& p, const SweepAt& a, int lane, const float (&s)[DK / 8][4]) {
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int dk = n * 8 + (lane & 3) * 2 + (e & 1), dv = (lane >> 2) + (e >> 1) * 8;
      if (dk < p.dk && dv < a.width)
        to[(static_cast<long long>(a.sequence) * p.hv + a.vh) * p.dk * p.dv + static_cast<long long>(dk) * p.dv + a.slab * 16 +
           dv] = s[n][e];
    }
}
// Accumulators in fragment order: [.., column tile, lane, 4].
template <int N>
__device__ __forceinline__ void fragments_store(float* to, int lane, const float (&f)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
    *reinterpret_cast<float4*>(to + (n * 32 + lane) * 4) = make_float4(f[n][0], f[n][1], f[n][2], f[n][3]);
}

__device__ __forceinline__ float2 coef_at(const char* head, int which, int n, int lane) {
  return *reinterpret_cast<const float2*>(head + (which * kChunk + n * 8 + (lane & 3) * 2) * 4);
}

constexpr int kSweepRing = 128;  // bytes of the ring's barriers

// KEEP: store S at every chunk's start and U for the backward pass instead of O.
template <typename T, int DK, int PS, int PO, bool KEEP>
__global__ void __launch_bounds__(256) delta_sweep(DeltaParams p, int stages) {
  using L = DeltaLayout<T, DK, PS, PO>;
  constexpr int IN = L::kIn;
  extern __shared__ __align__(128) char shared_bytes[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const SweepAt a = sweep_at(p, warps, warp);
  Ring<L> ring;
  ring.begin(shared_bytes, stages, warps);
  char* slabs = shared_bytes + kSweepRing + stages * L::kStage + warp * 2 * Slab<T>::kBytes;

  const T* v = static_cast<const T*>(p.v) + a.batch * p.v_batch + a.lo * p.v_token + a.vh * p.v_head + a.slab * 16;
  const long long o_step = static_cast<long long>(p.hv) * p.dv;
  T* o = KEEP ? nullptr
              : static_cast<T*>(p.o) + (static_cast<long long>(a.batch) * p.tokens + a.lo) * o_step +
                    static_cast<long long>(a.vh) * p.dv + a.slab * 16;
  const bool mine = a.width > 0;
  if (!KEEP && p.cu && mine) {  // rows of no sequence: zero
    if (a.sequence == 0)
      for (int at = lane; at < a.lo * 16; at += 32)
        if ((at & 15) < a.width) o[((at >> 4) - a.lo) * o_step + (at & 15)] = down<T>(0.f);
    if (a.sequence == p.sequences - 1)
      for (long long at = lane; at < (p.tokens - a.lo - a.len) * 16ll; at += 32)
        if ((at & 15) < a.width) o[(a.len + (at >> 4)) * o_step + (at & 15)] = down<T>(0.f);
  }
  float s[DK / 8][4];
  state_load<DK>(mine ? p.state_in : nullptr, p, a, lane, s);
  if (threadIdx.x == 0)
    for (int i = 0; i < stages && i < a.chunks; ++i) ring.fill(p, i, a.first + i, a.kh, a.vh);
  if (mine && a.chunks) slab_fetch<T>(slabs, v, p.v_token, min(a.len, kChunk), a.width, p.vec_v, lane);

  for (int c = 0; c < a.chunks; ++c) {
    const int len = min(kChunk, a.len - c * kChunk);
    char* slab = slabs + (c & 1) * Slab<T>::kBytes;
    if (mine && c + 1 < a.chunks)
      slab_fetch<T>(slabs + (~c & 1) * Slab<T>::kBytes, v + (c + 1) * kChunk * p.v_token, p.v_token,
                    min(kChunk, a.len - (c + 1) * kChunk), a.width, p.vec_v, lane);
    const char* stage = ring.wait(c);
    if (mine) {
      const uint32_t kt = shared_u32(stage), qt = kt + IN * L::kTile, tt = kt + L::kTiles, pt = tt + L::kT;
      const char* coef = stage + L::kTiles + L::kT + L::kP;
      const long long slab_at = (static_cast<long long>(a.first + c) * p.hv + a.vh) * p.slabs + a.slab;
      if (KEEP) fragments_store(p.states + slab_at * 16 * DK, lane, s);
      float top[2];
      row_max(s, top);
      if (KEEP) {
        const float most = warp_max(fmaxf(top[0], top[1]));
        if (lane == 0) p.largest[slab_at * 4] = most;
      }
      const Pow2 ss[2] = {pow2_for(top[0]), pow2_for(top[1])};
      float x[8][4] = {}, o_acc[8][4] = {};
      // (K S)^T and (Q S)^T
#pragma unroll
      for (int kk = 0; kk < DK / 16; ++kk) {
        uint32_t hi[4], lo[4];
        as_operand<PS>(s[2 * kk], s[2 * kk + 1], ss, hi, lo);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t at = at_nk<DK>(lane, n * 16, kk * 16);
          product<PS, IN, false>(x[2 * n], x[2 * n + 1], hi, lo, kt + at, L::kTile);
          if (!KEEP) product<PO, IN, false>(o_acc[2 * n], o_acc[2 * n + 1], hi, lo, qt + at, L::kTile);
        }
      }
      // X = beta v - beta e^G K S
      if (c + 1 < a.chunks)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      else
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      {
        float vv[8][4];
        slab_read<T>(slab, lane, vv);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float2 b = coef_at(coef, kBeta, n, lane), w = coef_at(coef, kDown, n, lane);
          x[n][0] = b.x * vv[n][0] - w.x * (x[n][0] * ss[0].inverse);
          x[n][1] = b.y * vv[n][1] - w.y * (x[n][1] * ss[0].inverse);
          x[n][2] = b.x * vv[n][2] - w.x * (x[n][2] * ss[1].inverse);
          x[n][3] = b.y * vv[n][3] - w.y * (x[n][3] * ss[1].inverse);
        }
      }
      // U^T = X^T T^T, T lower triangular
      float u[8][4] = {};
      {
        row_max(x, top);
        const Pow2 sx[2] = {pow2_for(top[0]), pow2_for(top[1])};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t hi[4], lo[4];
          as_operand<PS>(x[2 * kk], x[2 * kk + 1], sx, hi, lo);
#pragma unroll
          for (int n = kk; n < 4; ++n)
            product<PS, PS, false>(u[2 * n], u[2 * n + 1], hi, lo, tt + at_nk<kChunk>(lane, n * 16, kk * 16), L::kSquare);
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float2 w = coef_at(coef, kTRow, n, lane);
          u[n][0] *= w.x * sx[0].inverse;
          u[n][1] *= w.y * sx[0].inverse;
          u[n][2] *= w.x * sx[1].inverse;
          u[n][3] *= w.y * sx[1].inverse;
        }
      }
      if (KEEP) {
        fragments_store(p.us + slab_at * 16 * kChunk, lane, u);
        row_max(u, top);
        const float most = warp_max(fmaxf(top[0], top[1]));
        if (lane == 0) p.largest[slab_at * 4 + 2] = most;
      } else {  // O^T = (Q S)^T + U^T P^T, each with its weights
        row_max(u, top);
        const Pow2 su[2] = {pow2_for(top[0]), pow2_for(top[1])};
        float pu[8][4] = {};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t hi[4], lo[4];
          as_operand<PO>(u[2 * kk], u[2 * kk + 1], su, hi, lo);
#pragma unroll
          for (int n = kk; n < 4; ++n)
            product<PO, PO, false>(pu[2 * n], pu[2 * n + 1], hi, lo, pt + at_nk<kChunk>(lane, n * 16, kk * 16), L::kSquare);
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float2 wq = coef_at(coef, kOutQ, n, lane), wp = coef_at(coef, kOutP, n, lane);
          o_acc[n][0] = wq.x * (o_acc[n][0] * ss[0].inverse) + wp.x * (pu[n][0] * su[0].inverse);
          o_acc[n][1] = wq.y * (o_acc[n][1] * ss[0].inverse) + wp.y * (pu[n][1] * su[0].inverse);
          o_acc[n][2] = wq.x * (o_acc[n][2] * ss[1].inverse) + wp.x * (pu[n][2] * su[1].inverse);
          o_acc[n][3] = wq.y * (o_acc[n][3] * ss[1].inverse) + wp.y * (pu[n][3] * su[1].inverse);
        }
        __syncwarp();
        slab_write<T>(slab, lane, o_acc);
        __syncwarp();
        slab_store<T>(slab, o + c * kChunk * o_step, o_step, len, a.width, p.vec_o, lane);
        __syncwarp();
      }
      // S^T = e^{G_C} S^T + (e^{G_C - G} U)^T K: both at one scale
      {
        const float decay = reinterpret_cast<const float*>(coef)[kDecay * kChunk];
        float su[2], sd[2];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float2 w = coef_at(coef, kTail, n, lane);
          u[n][0] *= w.x;
          u[n][1] *= w.y;
          u[n][2] *= w.x;
          u[n][3] *= w.y;
        }
        row_max(u, su);
        row_max(s, sd);
        const Pow2 sc[2] = {pow2_for(fmaxf(su[0], decay * sd[0])), pow2_for(fmaxf(su[1], decay * sd[1]))};
#pragma unroll
        for (int n = 0; n < DK / 8; ++n) {
          s[n][0] *= decay * sc[0].f;
          s[n][1] *= decay * sc[0].f;
          s[n][2] *= decay * sc[1].f;
          s[n][3] *= decay * sc[1].f;
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t hi[4], lo[4];
          as_operand<PS>(u[2 * kk], u[2 * kk + 1], sc, hi, lo);
#pragma unroll
          for (int n = 0; n < DK / 16; ++n)
            product<PS, IN, true>(s[2 * n], s[2 * n + 1], hi, lo, kt + at_kn<DK>(lane, n * 16, kk * 16), L::kTile);
        }
#pragma unroll
        for (int n = 0; n < DK / 8; ++n) {
          s[n][0] *= sc[0].inverse;
          s[n][1] *= sc[0].inverse;
          s[n][2] *= sc[1].inverse;
          s[n][3] *= sc[1].inverse;
        }
      }
    }
    ring.done(c, lane);
    if (threadIdx.x == 0 && c + stages < a.chunks) ring.fill(p, c + stages, a.first + c + stages, a.kh, a.vh);
    __syncwarp();
  }
  if (mine && p.state_out) state_store<DK>(p.state_out, p, a, lane, s);
}

}  // namespace seq
}  // namespace pla
