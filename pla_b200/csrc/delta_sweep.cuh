// delta_sweep: walks the chunks of a sequence with the state in registers
// (delta_common.cuh has the mathematics).
//
// The columns of S (one per value feature) never meet, so a block takes VB of
// them (16 or 32) through the whole sequence on its own.  Every product of
// a chunk has the value features as its rows,
//     (K S)^T = S^T K^T,  U^T = X^T T^T,  O^T = S^T Q^T + U^T P^T,  S^T += U^T K,
// so that K, Q, T and P are always the right operand, read by ldmatrix from
// tiles that lie in the workspace in shared-memory order and come by bulk
// copies a chunk or two ahead.  The chain of a chunk is three dependent
// products, and a sequence is hundreds of chunks: its time is latency.  Four
// warps share 16 value features: warp wn computes 16 of the 64 tokens of K S,
// X, U and O and a quarter of the features of S, so each step is a few dozen
// instructions a warp, and operands pass between the warps through shared
// memory as planes (one barrier a step).  One warp that kept all of S^T in
// registers instead needed no barrier, but its 400 products and 1500 other
// instructions a chunk took 8.6 us where this took 2.8 us (bf16, Dk = 128, one
// plane for the outputs; 3.1 us with two).  A chunk's 144 products a warp are
// 40 % of that; the rest is the wait for operands and barriers, which more warps
// an SM or more products at a time do not shorten.
//
// A row's planes take one scale wherever a bound gives it before the warps
// have met: |U| <= max_i sum_j |T_ij| max|X| (delta_prepare has the sums), and
// |S| <= e^{G_C} max|S0| + 64 max|e^{G_C - G} U| max|K|, the maxima being those
// of the last step, exact.  A bound a thousand times too large costs ten of
// the 26 bits that two planes have below 2^15.  X is scaled per 16 tokens, as
// each warp finds it, and its products are scaled back one by one.
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
// Waits about two seconds at most; then records the fault, which the host reads,
// and returns false: the caller's block ends without using what did not come.
__device__ __forceinline__ bool barrier_wait(uint64_t* bar, uint32_t parity) {
  if (barrier_try(bar, parity)) return true;
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  do {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (barrier_try(bar, parity)) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  } while (t - t0 < 2000000000ull);
  atomicOr(&g_sequence_faults, 1u);
  return false;
}
__device__ __forceinline__ void bulk_copy(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   shared_u32(to)),
               "l"(from), "r"(bytes), "r"(shared_u32(bar))
               : "memory");
}

// A chunk's 64 x VB part of v (or do) in shared memory; the pitch spreads
// eight rows over the banks.
template <typename T, int VB>
struct Slab {
  static constexpr int kPitch = VB * sizeof(T) + 16;
  static constexpr int kBytes = kChunk * kPitch;
};

// Starts the copy of rows [0, len) and columns [0, width) by the whole block;
// zeros elsewhere.  16-byte copies if the rows allow it, single elements otherwise.
template <typename T, int VB>
__device__ __forceinline__ void slab_fetch(char* to, const T* from, long long step, int len, int width, int vec) {
  constexpr int UNIT = 16 / sizeof(T), PER = VB / UNIT, THREADS = VB * 8;
  if (vec) {
#pragma unroll
    for (int i = 0; i < kChunk * PER / THREADS; ++i) {
      const int at = i * THREADS + threadIdx.x, row = at / PER, u = at % PER;
      const bool there = row < len && u * UNIT < width;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared_u32(to) + row * Slab<T, VB>::kPitch + u * 16),
                   "l"(there ? from + row * step + u * UNIT : from), "r"(there ? 16 : 0)
                   : "memory");
    }
  } else {
    for (int at = threadIdx.x; at < kChunk * VB; at += THREADS) {
      const int row = at / VB, col = at % VB;
      reinterpret_cast<T*>(to + row * Slab<T, VB>::kPitch)[col] =
          row < len && col < width ? from[row * step + col] : down<T>(0.f);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

// 16 tokens x 16 features of a slab as accumulators of [features x tokens].
template <typename T, int VB>
__device__ __forceinline__ void slab_read(const char* from, int t0, int f0, int lane, float (&f)[2][4]) {
  if constexpr (sizeof(T) == 2) {
    const int m = lane >> 3;
    uint32_t r[4];  // tokens 0-7, 8-15; features 0-7 and 8-15 of each
    ldsm_t(r, shared_u32(from) + (t0 + (m >> 1) * 8 + (lane & 7)) * Slab<T, VB>::kPitch + f0 * 2 + (m & 1) * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Vec<T, 2> v = *reinterpret_cast<const Vec<T, 2>*>(&r[i]);
      f[i >> 1][(i & 1) * 2] = up(v.e[0]);
      f[i >> 1][(i & 1) * 2 + 1] = up(v.e[1]);
    }
  } else {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[n][e] = up(reinterpret_cast<const T*>(from + (t0 + n * 8 + (lane & 3) * 2 + (e & 1)) *
                                                           Slab<T, VB>::kPitch)[f0 + (lane >> 2) + (e >> 1) * 8]);
  }
}

// Accumulators of [16 features x 16 tokens] to rows of a tensor, through the
// warp's own 16 x 16 part of a slab that has been read.
template <typename T, int PITCH>
__device__ __forceinline__ void strip_store(char* buffer, int lane, const float (&f)[2][4], T* to, long long step, int len,
                                            int width, int vec) {
  __syncwarp();
  if constexpr (sizeof(T) == 2) {
    const int m = lane >> 3;
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      Vec<T, 2> v;
      v.e[0] = down<T>(f[i >> 1][(i & 1) * 2]);
      v.e[1] = down<T>(f[i >> 1][(i & 1) * 2 + 1]);
      r[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(
                     shared_u32(buffer) + ((m >> 1) * 8 + (lane & 7)) * PITCH + (m & 1) * 16),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
  } else {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<T*>(buffer + (n * 8 + (lane & 3) * 2 + (e & 1)) * PITCH)[(lane >> 2) + (e >> 1) * 8] = down<T>(f[n][e]);
  }
  __syncwarp();
  constexpr int UNIT = 16 / sizeof(T), PER = 16 / UNIT;
  if (vec) {
#pragma unroll
    for (int i = 0; i < 16 * PER / 32; ++i) {
      const int at = i * 32 + lane, row = at / PER, u = at % PER;
      if (row < len && u * UNIT < width)
        *reinterpret_cast<uint4*>(to + row * step + u * UNIT) = *reinterpret_cast<const uint4*>(buffer + row * PITCH + u * 16);
    }
  } else {
    for (int at = lane; at < 256; at += 32) {
      const int row = at >> 4, col = at & 15;
      if (row < len && col < width) to[row * step + col] = reinterpret_cast<const T*>(buffer + row * PITCH)[col];
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

// Accumulators of 16 rows x 8 N columns, times a scale for each row, as planes
// of a tile of W columns.
template <int W, int N>
__device__ __forceinline__ void tile_write(char* tile, uint32_t plane, int row0, int col0, int lane, const float (&f)[N][4],
                                           const Pow2 (&s)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = row0 + (lane >> 2) + h * 8;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      uint32_t hi, lo;
      split(f[n][2 * h] * s[h].f, f[n][2 * h + 1] * s[h].f, &hi, &lo);
      const uint32_t at = tile_at<W>(row, (col0 >> 3) + n) + (lane & 3) * 4;
      *reinterpret_cast<uint32_t*>(tile + at) = hi;
      *reinterpret_cast<uint32_t*>(tile + plane + at) = lo;
    }
  }
}
// Of each row, what the four warps that share it have: [row][warp].
__device__ __forceinline__ void share(float* to, int warp, int row0, int lane, float a, float b) {
  if ((lane & 3) == 0) {
    to[(row0 + (lane >> 2)) * 4 + warp] = a;
    to[(row0 + (lane >> 2) + 8) * 4 + warp] = b;
  }
}
__device__ __forceinline__ void shared_of(const float* from, int row0, int lane, float4 (&v)[2]) {
  v[0] = *reinterpret_cast<const float4*>(from + (row0 + (lane >> 2)) * 4);
  v[1] = *reinterpret_cast<const float4*>(from + (row0 + (lane >> 2) + 8) * 4);
}
__device__ __forceinline__ float most_of(float4 v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
__device__ __forceinline__ float element(const float4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Left operand: 16 x 16 of a tile's planes.
__device__ __forceinline__ void tile_operand(uint32_t at, uint32_t plane, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  ldsm(hi, at);
  ldsm(lo, at + plane);
}

// f += g, row by row times a factor.
template <int N>
__device__ __forceinline__ void add_scaled(float (&f)[N][4], const float (&g)[N][4], float a, float b) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    f[n][0] = fmaf(g[n][0], a, f[n][0]);
    f[n][1] = fmaf(g[n][1], a, f[n][1]);
    f[n][2] = fmaf(g[n][2], b, f[n][2]);
    f[n][3] = fmaf(g[n][3], b, f[n][3]);
  }
}

// Columns (tokens) times their coefficients.
template <int N>
__device__ __forceinline__ void scale_columns(float (&f)[N][4], const float2 (&w)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    f[n][0] *= w[n].x;
    f[n][1] *= w[n].y;
    f[n][2] *= w[n].x;
    f[n][3] *= w[n].y;
  }
}

// d0, d1 (+)= A B for two column tiles: A in two planes (hi, lo), B in PB planes
// `apart` bytes apart at `at`; the product of two lo planes is left out.
template <int PB, bool TRANS>
__device__ __forceinline__ void product(float (&d0)[4], float (&d1)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                        uint32_t at, uint32_t apart, bool first) {
  uint32_t b[4];
  if (TRANS) ldsm_t(b, at); else ldsm(b, at);
  if (first) {
    mma_first(d0, hi, b[0], b[1]);
    mma_first(d1, hi, b[2], b[3]);
  } else {
    mma(d0, hi, b[0], b[1]);
    mma(d1, hi, b[2], b[3]);
  }
  mma(d0, lo, b[0], b[1]);
  mma(d1, lo, b[2], b[3]);
  if (PB > 1) {
    if (TRANS) ldsm_t(b, at + apart); else ldsm(b, at + apart);
    mma(d0, hi, b[0], b[1]);
    mma(d1, hi, b[2], b[3]);
  }
}

// Thread 0 gives `count` copies in flight their time, from stage `at` on; the
// block's shared memory is held until it returns.  (Not inlined: the sweeps need
// the registers.)
static __device__ __noinline__ void drain(uint64_t* full, int at, int filled, int stages, int count) {
  if (threadIdx.x != 0) return;
  for (int i = 0; i < count; ++i) {
    barrier_wait(full + at, filled & 1);
    if (++at == stages) at = 0, ++filled;
  }
}

// Copies of the chunks' tiles into a ring of stages.  Thread 0 issues them; a
// stage is refilled when every warp has arrived at its `empty` barrier.
template <typename L, int STAGES>
struct Ring {
  char* stages;
  uint64_t *full, *empty;
  int at, filled;             // stage and fills of it so far, of the chunk that is worked on
  __device__ __forceinline__ void begin(char* bytes, int warps) {
    full = reinterpret_cast<uint64_t*>(bytes);
    empty = full + 8;
    stages = bytes + 128;
    at = filled = 0;
    if (threadIdx.x == 0) {
      for (int i = 0; i < STAGES; ++i) {
        barrier_init(full + i, 1);
        barrier_init(empty + i, warps);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
  }
  __device__ __forceinline__ void fill(const DeltaParams& p, int stage, int chunk, int kh, int vh) {
    char* to = stages + stage * L::kStage;
    barrier_expect(full + stage, L::kStage);
    bulk_copy(to, p.tiles + (static_cast<long long>(chunk) * p.hk + kh) * L::kTiles, L::kTiles, full + stage);
    bulk_copy(to + L::kTiles, p.heads + (static_cast<long long>(chunk) * p.hv + vh) * L::kHead, L::kHead, full + stage);
  }
  __device__ __forceinline__ const char* stage() const { return stages + at * L::kStage; }
  __device__ __forceinline__ bool wait() { return barrier_wait(full + at, filled & 1); }
  // A wait ran out, `left` chunks (this one among them) are not worked on.
  __device__ __forceinline__ void give_up(int left) const { drain(full, at, filled, STAGES, min(STAGES, left)); }
  // This chunk's stage is done with; chunk `refill` (if >= 0) takes its place.
  __device__ __forceinline__ void next(const DeltaParams& p, int refill, int kh, int vh) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) barrier_arrive(empty + at);
    if (threadIdx.x == 0 && refill >= 0) {
      if (barrier_wait(empty + at, filled & 1)) fill(p, at, refill, kh, vh);  // else the wait for it runs out too
    }
    __syncwarp();
    if (++at == STAGES) {
      at = 0;
      ++filled;
    }
  }
};

// What a block of a sweep works on: VB value features of one head of one sequence.
struct SweepAt {
  int sequence, vh, kh, column, batch, lo, len, first, chunks, width;
};
__device__ __forceinline__ SweepAt sweep_at(const DeltaParams& p, int vb) {
  SweepAt a;
  const int parts = (p.dv + vb - 1) / vb;
  int b = blockIdx.x;
  a.column = (b % parts) * vb;
  b /= parts;
  a.vh = b % p.hv;
  a.sequence = b / p.hv;
  if (p.cu) a.sequence = p.plan[3 * p.sequences + 1 + a.sequence];  // the longest first
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
  a.width = min(vb, p.dv - a.column);
  return a;
}

// A warp's part of S^T, features [col0, col0 + 16) of the block and 8 N of Dk
// from dk0, from or to [Dk, Dv] fp32.
template <int N>
__device__ __forceinline__ void state_load(const float* from, const DeltaParams& p, const SweepAt& a, int col0, int dk0, int lane,
                                           float (&s)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int dk = dk0 + n * 8 + (lane & 3) * 2 + (e & 1), dv = col0 + (lane >> 2) + (e >> 1) * 8;
      s[n][e] = from && dk < p.dk && dv < a.width
                    ? from[((static_cast<long long>(a.sequence) * p.hv + a.vh) * p.dk + dk) * p.dv + a.column + dv]
                    : 0.f;
    }
}
template <int N>
__device__ __forceinline__ void state_store(float* to, const DeltaParams& p, const SweepAt& a, int col0, int dk0, int lane,
                                            const float (&s)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int dk = dk0 + n * 8 + (lane & 3) * 2 + (e & 1), dv = col0 + (lane >> 2) + (e >> 1) * 8;
      if (dk < p.dk && dv < a.width)
        to[((static_cast<long long>(a.sequence) * p.hv + a.vh) * p.dk + dk) * p.dv + a.column + dv] = s[n][e];
    }
}
// A block's planes of a tile and the inverses of their rows' scales to the
// workspace: VB rows of W columns of plane after plane.
template <int VB, int W>
__device__ __forceinline__ void keep_tile(const char* tile, const float* scale, char* to, float* scales, int rows, int column) {
  constexpr int UNITS = VB * W * 2 / 16;
  char* at = to + static_cast<long long>(column) * W * 2;
#pragma unroll
  for (int n = 0; n < kPlanes; ++n)
#pragma unroll
    for (int i = 0; i < UNITS / (VB * 8); ++i) {
      const int u = i * VB * 8 + threadIdx.x;
      reinterpret_cast<uint4*>(at + static_cast<long long>(n) * rows * W * 2)[u] =
          reinterpret_cast<const uint4*>(tile + n * VB * W * 2)[u];
    }
  if (threadIdx.x < VB) scales[column + threadIdx.x] = scale[threadIdx.x];
}
// Where a (chunk, value head) keeps what: bytes of the planes, floats of the scales.
template <int W>
__device__ __forceinline__ long long kept_at(const DeltaParams& p, long long head) {
  return head * kPlanes * p.rows * W * 2;
}

template <int N>
__device__ __forceinline__ void coef_read(const char* coef, int which, int tile, int lane, float2 (&w)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
    w[n] = *reinterpret_cast<const float2*>(coef + (which * kChunk + (tile + n) * 8 + (lane & 3) * 2) * 4);
}

constexpr int kSweepRing = 128;  // bytes of the ring's barriers

// Shared memory of a sweep behind the ring: planes of S, X, U and what else
// the steps hand on.
template <typename T, int DK, int VB, bool BACK>
struct SweepShared {
  static constexpr uint32_t kWide = VB * DK * 2, kNarrow = VB * kChunk * 2;
  alignas(128) char s[kPlanes * kWide];
  char a[kPlanes * kNarrow];  // X; back: Y
  char b[kPlanes * kNarrow];  // e^{G_C - G} U; back: beta e^G dX
  char c[kPlanes * kNarrow];  // U; back: do' with P's weights, then dX
  char d[BACK ? kPlanes * kNarrow : 128];  // back: e^G do'
  alignas(16) float most_s[VB * 4];   // largest of S's rows, by warp
  alignas(16) float scale_a[VB * 4];  // inverses of the scales of X (Y), by warp
  alignas(16) float scale_c[VB * 4];  // back: of do'
  alignas(16) float most_d[VB * 4];   // back: largest of e^G do', by warp
  float keep_s[VB], keep_c[VB];       // inverses of the scales of S and U (dX), for what is kept
  alignas(16) char slab[2][Slab<T, VB>::kBytes];
};

// |A B| over 64 tokens with one operand's planes below 2^13.
constexpr float kPlaneTop = 8192.f, kSumTop = 64.f * kPlaneTop;
// A row of T has its largest near 2^12, and at least 1 of T itself is 1: X's
// scales are handed on divided by that, so that sums of T X times them are no
// larger than U and reach the end of the float range.
constexpr float kTTop = 4096.f;
// Scale for what lies below `bound`: brings it below 2^15.
__device__ __forceinline__ Pow2 scale_below(float bound) {
  const Pow2 s = pow2_for(bound);
  return {s.f * 4.f, s.inverse * 0.25f};
}

// KEEP: store S at every chunk's start and U for the backward pass instead of O.
template <typename T, int DK, int VB, int STAGES, int PER_SM, bool KEEP>
__global__ void __launch_bounds__(VB * 8, PER_SM) delta_sweep(DeltaParams p) {
  using L = DeltaLayout<T, DK>;
  using M = SweepShared<T, DK, VB, false>;
  constexpr int IN = L::kIn, QN = DK / 32;  // column tiles of a quarter of Dk
  constexpr int kPitch = Slab<T, VB>::kPitch;
  extern __shared__ __align__(128) char shared_bytes[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = warp % (VB / 16), wn = warp / (VB / 16), m0 = wm * 16;
  const SweepAt a = sweep_at(p, VB);
  Ring<L, STAGES> ring;
  ring.begin(shared_bytes, VB / 4);
  M& m = *reinterpret_cast<M*>(shared_bytes + kSweepRing + STAGES * L::kStage);
  const uint32_t st = shared_u32(m.s), xt = shared_u32(m.a), ut = shared_u32(m.b), vt = shared_u32(m.c);

  const T* v = static_cast<const T*>(p.v) + a.batch * p.v_batch + a.lo * p.v_token + a.vh * p.v_head + a.column;
  const long long o_step = static_cast<long long>(p.hv) * p.dv;
  T* o = KEEP ? nullptr
              : static_cast<T*>(p.o) + (static_cast<long long>(a.batch) * p.tokens + a.lo) * o_step +
                    static_cast<long long>(a.vh) * p.dv + a.column;
  if (!KEEP && p.cu) {  // rows of no sequence: zero
    if (a.sequence == 0)
      for (long long at = threadIdx.x; at < a.lo * static_cast<long long>(VB); at += VB * 8)
        if (at % VB < a.width) o[(at / VB - a.lo) * o_step + at % VB] = down<T>(0.f);
    if (a.sequence == p.sequences - 1)
      for (long long at = threadIdx.x; at < (p.tokens - a.lo - a.len) * static_cast<long long>(VB); at += VB * 8)
        if (at % VB < a.width) o[(a.len + at / VB) * o_step + at % VB] = down<T>(0.f);
  }
  if (threadIdx.x == 0)
    for (int i = 0; i < STAGES && i < a.chunks; ++i) ring.fill(p, i, a.first + i, a.kh, a.vh);
  if (a.chunks) slab_fetch<T, VB>(m.slab[0], v, p.v_token, min(a.len, kChunk), a.width, p.vec_v);
  const Walk sw(st + at_mk<DK>(lane, m0, 0)), xw(xt + at_mk<kChunk>(lane, m0, 0));  // planes of S and X; U's follow X's
  const Walk kw(at_nk<DK>(lane, wn * 16, 0)), tw(at_nk<kChunk>(lane, wn * 16, 0));  // in K and Q; in T and P
  uint32_t ks[QN / 2];  // in K, for the state's update
#pragma unroll
  for (int n = 0; n < QN / 2; ++n) ks[n] = at_kn<DK>(lane, wn * (DK / 4) + n * 16, 0);
  float s[QN][4], top[2];
  Pow2 fs[2];
  state_load(p.state_in, p, a, m0, wn * (DK / 4), lane, s);
  {  // S's planes, after the four warps have met once over their rows' largest
    row_max(s, top);
    share(m.most_s, wn, m0, lane, top[0], top[1]);
    __syncthreads();
    float4 all[2];
    shared_of(m.most_s, m0, lane, all);
    fs[0] = scale_below(most_of(all[0]));
    fs[1] = scale_below(most_of(all[1]));
    tile_write<DK>(m.s, M::kWide, m0, wn * (DK / 4), lane, s, fs);
  }

  for (int c = 0; c < a.chunks; ++c) {
    const int len = min(kChunk, a.len - c * kChunk);
    const long long head_at = static_cast<long long>(a.first + c) * p.hv + a.vh;
    if (KEEP && wn == 0 && (lane & 3) == 0) {
      m.keep_s[m0 + (lane >> 2)] = fs[0].inverse;
      m.keep_s[m0 + (lane >> 2) + 8] = fs[1].inverse;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // planes of S and this chunk's v are there; the other slab is free
    if (!__syncthreads_and(ring.wait())) return ring.give_up(a.chunks - c);
    const char* stage = ring.stage();
    if (c + 1 < a.chunks)
      slab_fetch<T, VB>(m.slab[~c & 1], v + (c + 1) * kChunk * p.v_token, p.v_token, min(kChunk, a.len - (c + 1) * kChunk),
                        a.width, p.vec_v);
    if (KEEP)
      keep_tile<VB, DK>(m.s, m.keep_s, p.states + kept_at<DK>(p, head_at), p.scales + head_at * 4 * p.rows, p.rows,
                            a.column);
    const uint32_t kt = shared_u32(stage), qt = kt + IN * L::kTile, tt = kt + L::kTiles, pt = tt + L::kT;
    const char* coef = stage + L::kTiles + L::kT + L::kP;
    const float4 bounds = *reinterpret_cast<const float4*>(coef + kBounds * kChunk * 4);
    const float decay = reinterpret_cast<const float*>(coef)[kDecay * kChunk];
    float x[2][4], q[2][4];
    float2 w[2];
    // (K S)^T and (Q S)^T
#pragma unroll
    for (int kk = 0; kk < DK / 16; ++kk) {
      uint32_t hi[4], lo[4];
      tile_operand(sw[kk], M::kWide, hi, lo);
      product<IN, false>(x[0], x[1], hi, lo, kt + kw[kk], L::kTile, kk == 0);
      if (!KEEP) product<IN, false>(q[0], q[1], hi, lo, qt + kw[kk], L::kTile, kk == 0);
    }
    float4 most[2];
    shared_of(m.most_s, m0, lane, most);
    {  // X = beta v - beta e^G K S
      float vv[2][4];
      slab_read<T, VB>(m.slab[c & 1], wn * 16, m0, lane, vv);
      float2 b[2];
      coef_read(coef, kBeta, wn * 2, lane, b);
      coef_read(coef, kDown, wn * 2, lane, w);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[n][e] = (e & 1 ? b[n].y : b[n].x) * vv[n][e] - ((e & 1 ? w[n].y : w[n].x) * fs[e >> 1].inverse) * x[n][e];
    }
    {
      row_max(x, top);
      const Pow2 fx[2] = {pow2_for(top[0]), pow2_for(top[1])};
      share(m.scale_a, wn, m0, lane, fx[0].inverse / kTTop, fx[1].inverse / kTTop);
      tile_write<kChunk>(m.a, M::kNarrow, m0, wn * 16, lane, x, fx);
    }
    __syncthreads();
    // U^T = X^T T^T; T is lower triangular, but the warp with the last tokens needs every step,
    // and steps without a branch overlap
    float u[2][4] = {};
    float4 back[2];
    shared_of(m.scale_a, m0, lane, back);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4];
      float bu[2][4];
      tile_operand(xw[kk], M::kNarrow, hi, lo);
      product<kPlanes, false>(bu[0], bu[1], hi, lo, tt + tw[kk], L::kSquare, true);
      add_scaled(u, bu, element(back[0], kk), element(back[1], kk));
    }
    coef_read(coef, kTRow, wn * 2, lane, w);
#pragma unroll
    for (int n = 0; n < 2; ++n) w[n].x *= kTTop, w[n].y *= kTTop;
    scale_columns(u, w);
    const float bound_x[2] = {most_of(back[0]) * (kTTop * kPlaneTop), most_of(back[1]) * (kTTop * kPlaneTop)};
    const Pow2 fu[2] = {scale_below(bounds.x * bound_x[0]), scale_below(bounds.x * bound_x[1])};
    tile_write<kChunk>(m.c, M::kNarrow, m0, wn * 16, lane, u, fu);
    if (KEEP && wn == 0 && (lane & 3) == 0) {
      m.keep_c[m0 + (lane >> 2)] = fu[0].inverse;
      m.keep_c[m0 + (lane >> 2) + 8] = fu[1].inverse;
    }
    coef_read(coef, kTail, wn * 2, lane, w);
    scale_columns(u, w);
    const float bound_u[2] = {bounds.y * bound_x[0], bounds.y * bound_x[1]};
    const Pow2 ft[2] = {scale_below(bound_u[0]), scale_below(bound_u[1])};
    tile_write<kChunk>(m.b, M::kNarrow, m0, wn * 16, lane, u, ft);
    __syncthreads();
    if (KEEP)
      keep_tile<VB, kChunk>(m.c, m.keep_c, p.us + kept_at<kChunk>(p, head_at), p.scales + (head_at * 4 + 2) * p.rows,
                                p.rows, a.column);
    // S^T = e^{G_C} S^T + (e^{G_C - G} U)^T K
    {
      float bs[QN][4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t hi[4], lo[4];
        tile_operand(xw[kk] + (ut - xt), M::kNarrow, hi, lo);
#pragma unroll
        for (int n = 0; n < QN / 2; ++n)
          product<IN, true>(bs[2 * n], bs[2 * n + 1], hi, lo, kt + ks[n] + kk * 16 * DK * 2, L::kTile, kk == 0);
      }
#pragma unroll
      for (int n = 0; n < QN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = fmaf(bs[n][e], ft[e >> 1].inverse, decay * s[n][e]);
      const Pow2 old[2] = {fs[0], fs[1]};
#pragma unroll
      for (int h = 0; h < 2; ++h) fs[h] = scale_below(fmaf(decay, most_of(most[h]), kSumTop * bound_u[h]));
      tile_write<DK>(m.s, M::kWide, m0, wn * (DK / 4), lane, s, fs);
      row_max(s, top);
      share(m.most_s, wn, m0, lane, top[0], top[1]);
      if (!KEEP) {  // O^T = (Q S)^T + U^T P^T, each with its weights
        float pu[2][4];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t hi[4], lo[4];
          tile_operand(xw[kk] + (vt - xt), M::kNarrow, hi, lo);
          product<kPlanes, false>(pu[0], pu[1], hi, lo, pt + tw[kk], L::kSquare, kk == 0);
        }
        float2 wq[2];
        coef_read(coef, kOutQ, wn * 2, lane, wq);
        coef_read(coef, kOutP, wn * 2, lane, w);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            q[n][e] = ((e & 1 ? wq[n].y : wq[n].x) * old[e >> 1].inverse) * q[n][e] +
                      ((e & 1 ? w[n].y : w[n].x) * fu[e >> 1].inverse) * pu[n][e];
        strip_store<T, kPitch>(m.slab[c & 1] + wn * 16 * kPitch + m0 * sizeof(T), lane, q, o + (c * kChunk + wn * 16) * o_step + m0, o_step, len - wn * 16, a.width - m0,
                       p.vec_o);
      }
    }
    ring.next(p, c + STAGES < a.chunks ? a.first + c + STAGES : -1, a.kh, a.vh);
  }
  if (p.state_out) state_store(p.state_out, p, a, m0, wn * (DK / 4), lane, s);
}

}  // namespace seq
}  // namespace pla
