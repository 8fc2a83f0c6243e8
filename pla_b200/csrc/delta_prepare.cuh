// delta_prepare: everything of a chunk that does not depend on the state, for
// one (chunk, key head) a block and the value heads that share the key head:
// the fp16 planes of K and Q, T = (1 + diag(beta) M)^-1 and P as planes, and
// the per-token coefficients (delta_common.cuh).
//
// K K^T and Q K^T are one pass of tensor-core products for all value heads of
// the key head; then 128 threads a value head, two heads at a time.  The unit
// lower triangular 64 x 64 matrix is inverted in blocks, in fp32: four 16 x 16
// diagonal blocks by substitution (a thread a column, in registers), then
//     [A 0; B C]^-1 = [A^-1 0; -C^-1 B A^-1 C^-1]
// from 16 to 32 to 64.  Substitution over all 64 rows took 25 us a block's
// head, nearly all of it latency; in blocks it is some 700 multiply-adds a
// thread.
#pragma once

#include "delta_common.cuh"

namespace pla {
namespace seq {

constexpr int kPrepPitch = 68;  // floats of a row: rows 4 banks apart

struct PrepHead {
  // diag(beta) M below the diagonal, turned into T in place; the blocks above
  // the diagonal hold the products on the way
  alignas(16) float t[kChunk][kPrepPitch];
};

template <typename T, int DK, int HEADS>
struct PrepShared {
  union {
    alignas(16) __half tile[2][DeltaType<T>::kIn][kChunk * DK];  // K, Q planes, until their products are done
    PrepHead head[HEADS];
  };
  alignas(16) float kk[kChunk][kPrepPitch], qk[kChunk][kPrepPitch];
  float row[2][kChunk];               // what K / Q rows are to be multiplied by
  alignas(16) float most[2][kChunk];  // largest magnitude of the rows
  float hi[HEADS][kChunk], lo[HEADS][kChunk], beta[HEADS][kChunk];
  float rise[HEADS];                  // the largest e^{G_i - G_j}, i >= j
  unsigned int bound[HEADS][4];       // kBounds
};

// Rows of q and k as planes, in shared memory and in the workspace; a warp's
// rows of both are all in flight at once (fp32: eight at a time).
template <typename T, int DK, int HEADS, typename S>
__device__ __forceinline__ void prepare_rows(const DeltaParams& p, const T* k, const T* q, int len, int lane, int warp, S& s,
                                             char* out) {
  constexpr int IN = DeltaType<T>::kIn, E = DK / 32, ROWS = kChunk / (4 * HEADS), U = sizeof(T) == 2 ? ROWS : 8;
#pragma unroll 1
  for (int base = 0; base < ROWS; base += U) {
    Vec<T, E> raw[2][U];
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int row = warp * ROWS + base + i;
#pragma unroll
        for (int e = 0; e < E; ++e) raw[side][i].e[e] = down<T>(0.f);
        if (row < len) {
          const T* r = (side ? q + row * p.q_token : k + row * p.k_token) + lane * E;
          if (p.vec_qk) {
            if (lane * E < p.dk) raw[side][i] = *reinterpret_cast<const Vec<T, E>*>(r);
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (lane * E + e < p.dk) raw[side][i].e[e] = r[e];
          }
        }
      }
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int row = warp * ROWS + base + i;
        float f[E], m = 0.f;
        unpack(raw[side][i], f);
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, fabsf(f[e]));
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const Pow2 scale = pow2_for(m);
        if (lane == 0) {
          s.row[side][row] = scale.inverse;
          s.most[side][row] = m;
        }
        Vec<uint32_t, E / 2> plane[2];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) split<IN>(f[2 * e] * scale.f, f[2 * e + 1] * scale.f, &plane[0].e[e], &plane[1].e[e]);
        const uint32_t at = tile_at<DK>(row, lane * E / 8) + (lane * E % 8) * 2;
#pragma unroll
        for (int n = 0; n < IN; ++n) {
          *reinterpret_cast<Vec<uint32_t, E / 2>*>(reinterpret_cast<char*>(s.tile[side][n]) + at) = plane[n];
          *reinterpret_cast<Vec<uint32_t, E / 2>*>(out + (side * IN + n) * kChunk * DK * 2 + at) = plane[n];
        }
      }
  }
}

// Eight columns of a row as planes.
__device__ __forceinline__ void store_unit(char* out, int row, int unit, const float (&f)[8], float scale) {
  Vec<uint32_t, 4> plane[kPlanes];
#pragma unroll
  for (int e = 0; e < 4; ++e) split(f[2 * e] * scale, f[2 * e + 1] * scale, &plane[0].e[e], &plane[1].e[e]);
#pragma unroll
  for (int n = 0; n < kPlanes; ++n)
    *reinterpret_cast<Vec<uint32_t, 4>*>(out + n * kChunk * kChunk * 2 + tile_at<kChunk>(row, unit)) = plane[n];
}

// The four units of a row that thread id of a pair takes: the pair 16 banks
// apart and four rows 4 banks each keep eight 16-byte accesses conflict free.
__device__ __forceinline__ int unit_of(int i, int id) { return (i & 1) + 4 * (i >> 1) + 2 * (id & 1); }

__device__ __forceinline__ void head_sync(int head) { asm volatile("bar.sync %0, 128;" ::"r"(head + 1) : "memory"); }

// c = sign a b, N x N each inside the 64 x 64 matrix; a thread computes R rows
// of 4 columns.  LOWER_B / LOWER_A: that operand is lower triangular in blocks
// of 16 and holds other values above.
template <int N, int R, bool LOWER_B = false, bool LOWER_A = false>
__device__ __forceinline__ void block_product(const float* a, const float* b, float* c, float sign, int id) {
  constexpr int ACROSS = N / 4, P = kPrepPitch;
  const int col = id % ACROSS * 4, row = id / ACROSS * R;
  float4 sum[R];
#pragma unroll
  for (int r = 0; r < R; ++r) sum[r] = make_float4(0, 0, 0, 0);
#pragma unroll
  for (int k = 0; k < N; k += 4) {
    if (LOWER_B && k < (col & ~15)) continue;
    if (LOWER_A && k >= (row & ~15) + 16) continue;
    float4 bv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) bv[i] = *reinterpret_cast<const float4*>(b + (k + i) * P + col);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float4 av = *reinterpret_cast<const float4*>(a + (row + r) * P + k);
      const float v[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum[r].x = fmaf(v[i], bv[i].x, sum[r].x);
        sum[r].y = fmaf(v[i], bv[i].y, sum[r].y);
        sum[r].z = fmaf(v[i], bv[i].z, sum[r].z);
        sum[r].w = fmaf(v[i], bv[i].w, sum[r].w);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    *reinterpret_cast<float4*>(c + (row + r) * P + col) =
        make_float4(sign * sum[r].x, sign * sum[r].y, sign * sum[r].z, sign * sum[r].w);
}

// g and beta of two tokens a lane; 0 past the chunk's end.
template <typename T>
__device__ __forceinline__ void load_gates(const DeltaParams& p, const ChunkAt& c, int vh, int lane, float (&g)[2], float (&b)[2]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int t = 2 * lane + e;
    g[e] = b[e] = 0.f;
    if (t < c.len) {
      const long long gi = c.batch * p.g_batch + (c.token + t) * p.g_token + vh * p.g_head;
      const long long bi = c.batch * p.beta_batch + (c.token + t) * p.beta_token + vh * p.beta_head;
      g[e] = p.gates32 ? static_cast<const float*>(p.g)[gi] : up(static_cast<const T*>(p.g)[gi]);
      b[e] = p.gates32 ? static_cast<const float*>(p.beta)[bi] : up(static_cast<const T*>(p.beta)[bi]);
    }
  }
}

template <typename T, int DK, int HEADS>
__global__ void __launch_bounds__(128 * HEADS, 3) delta_prepare(DeltaParams p) {
  using L = DeltaLayout<T, DK>;
  extern __shared__ __align__(16) char shared_bytes[];
  PrepShared<T, DK, HEADS>& s = *reinterpret_cast<PrepShared<T, DK, HEADS>*>(shared_bytes);
  const int chunk = blockIdx.x / p.hk, kh = blockIdx.x % p.hk;
  ChunkAt c;
  if (!chunk_at(p, chunk, &c)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int id = threadIdx.x & 127, which = threadIdx.x >> 7;  // thread of a head, head of the block
  float(*t)[kPrepPitch] = s.head[which].t;
  float *hi = s.hi[which], *lo = s.lo[which], *beta = s.beta[which];
  const int group = p.hv / p.hk;
  char* tiles = p.tiles + (static_cast<long long>(chunk) * p.hk + kh) * L::kTiles;
  float gate[2], bias[2];
  if (id < 32 && which < group) load_gates<T>(p, c, kh * group + which, lane, gate, bias);
  {
    const T* k = static_cast<const T*>(p.k) + c.batch * p.k_batch + c.token * p.k_token + kh * p.k_head;
    const T* q = static_cast<const T*>(p.q) + c.batch * p.q_batch + c.token * p.q_token + kh * p.q_head;
    prepare_rows<T, DK, HEADS>(p, k, q, c.len, lane, warp, s, tiles);
  }
  __syncthreads();

  // k_i . k_j and q_i . k_j, 16 rows a warp, columns up to them
  {
    const int rb = warp & 3;
    const uint32_t kt = shared_u32(s.tile[0][0]), qt = shared_u32(s.tile[1][0]);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      if (HEADS == 2 && side != which) continue;
      float d[8][4] = {};
#pragma unroll
      for (int kk = 0; kk < DK / 16; ++kk)
#pragma unroll
        for (int pa = 0; pa < L::kIn; ++pa) {
          uint32_t a[4];
          ldsm(a, (side ? qt : kt) + pa * L::kTile + at_mk<DK>(lane, rb * 16, kk * 16));
#pragma unroll
          for (int pb = 0; pb + pa < L::kIn; ++pb)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              if (n > rb) break;
              uint32_t b[4];
              ldsm(b, kt + pb * L::kTile + at_nk<DK>(lane, n * 16, kk * 16));
              mma(d[2 * n], a, b[0], b[1]);
              mma(d[2 * n + 1], a, b[2], b[3]);
            }
        }
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = rb * 16 + (lane >> 2) + e * 8, j = n * 8 + (lane & 3) * 2;
          const float f = s.row[side][i];
          *reinterpret_cast<float2*>(&(side ? s.qk : s.kk)[i][j]) =
              make_float2(d[n][2 * e] * s.row[0][j] * f, d[n][2 * e + 1] * s.row[0][j + 1] * f);
        }
    }
  }
  float k_most = 0.f;
#pragma unroll
  for (int j = 0; j < kChunk; ++j) k_most = fmaxf(k_most, s.most[0][j]);

  __syncthreads();
  for (int sub = which; sub < group; sub += HEADS) {  // from here on the 128 threads of a head meet among themselves
    const int vh = kh * group + sub;
    char* head = p.heads + (static_cast<long long>(chunk) * p.hv + vh) * L::kHead;
    float* coef = reinterpret_cast<float*>(head + L::kT + L::kP);
    if (id < 32) {  // running sum of g in 64 bits, kept as two floats
      if (sub != which) load_gates<T>(p, c, vh, lane, gate, bias);
      double sum[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // e^-200 is 0 in fp32 already: a smaller g, -inf among them, is the same reset
        sum[e] = gate[e] < -200.f ? -200.f : gate[e];
        beta[2 * lane + e] = bias[e];
      }
      sum[1] += sum[0];
      double total = sum[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, total, o);
        if (lane >= o) total += v;
      }
      const double before = total - sum[1];
      float gf[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const double v = before + sum[e];
        gf[e] = static_cast<float>(v);
        hi[2 * lane + e] = gf[e];
        lo[2 * lane + e] = static_cast<float>(v - static_cast<double>(gf[e]));
      }
      float low = fminf(gf[0], gf[1]);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float v = __shfl_up_sync(0xffffffffu, low, o);
        if (lane >= o) low = fminf(low, v);
      }
      float earlier = __shfl_up_sync(0xffffffffu, low, 1);
      if (lane == 0) earlier = gf[0];
      float rise = fmaxf(gf[1] - low, gf[0] - fminf(earlier, gf[0]));
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) rise = fmaxf(rise, __shfl_xor_sync(0xffffffffu, rise, o));
      if (lane == 0) s.rise[which] = expf(fminf(rise, 80.f));
    }
    head_sync(which);
    // diag(beta) M below the diagonal, and P as planes at a scale from a bound:
    // |q_i . k_j| <= Dk max|q_i| max|k|
    {
      const int row = id >> 1;
      const float g_hi = hi[row], g_lo = lo[row], b = beta[row];
      const Pow2 f = pow2_for(DK * s.most[1][row] * k_most * s.rise[which]);
      if (!(id & 1)) coef[kOutP * kChunk + row] = p.scale * f.inverse;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int unit = unit_of(i, id);
        float pv[8], av[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) pv[e] = av[e] = 0.f;
        if (unit * 8 <= row) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int j = unit * 8 + e;
            const float decay = exp_fast((g_hi - hi[j]) + (g_lo - lo[j]));
            pv[e] = j <= row ? decay * s.qk[row][j] : 0.f;
            av[e] = j < row ? b * (decay * s.kk[row][j]) : 0.f;
          }
        }
        store_unit(head + L::kT, row, unit, pv, f.f);
        *reinterpret_cast<float4*>(&t[row][unit * 8]) = make_float4(av[0], av[1], av[2], av[3]);
        *reinterpret_cast<float4*>(&t[row][unit * 8 + 4]) = make_float4(av[4], av[5], av[6], av[7]);
      }
    }
    if (id < 4) s.bound[which][id] = 0;
    head_sync(which);
    float x[16];
    if (id < kChunk) {  // a column of a diagonal block's inverse
      const int base = id & ~15, col = id & 15;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float sum[4] = {};
#pragma unroll
        for (int l = 0; l < i; l += 4) {
          const float4 a = *reinterpret_cast<const float4*>(&t[base + i][base + l]);
          sum[0] = fmaf(a.x, x[l], sum[0]);
          if (l + 1 < i) sum[1] = fmaf(a.y, x[l + 1], sum[1]);
          if (l + 2 < i) sum[2] = fmaf(a.z, x[l + 2], sum[2]);
          if (l + 3 < i) sum[3] = fmaf(a.w, x[l + 3], sum[3]);
        }
        x[i] = (i == col ? 1.f : 0.f) - ((sum[0] + sum[1]) + (sum[2] + sum[3]));
      }
    }
    head_sync(which);
    if (id < kChunk)
#pragma unroll
      for (int i = 0; i < 16; ++i) t[(id & ~15) + i][id] = x[i];
    head_sync(which);
    {  // 16 -> 32, two blocks side by side
      const int b = (id >> 6) * 32, i = id & 63;
      block_product<16, 1>(&t[b + 16][b], &t[b][b], &t[b][b + 16], 1.f, i);
      head_sync(which);
      block_product<16, 1>(&t[b + 16][b + 16], &t[b][b + 16], &t[b + 16][b], -1.f, i);
      head_sync(which);
    }
    // 32 -> 64; what lies above the diagonal blocks of 32 is not T and is masked
    block_product<32, 2, true>(&t[32][0], &t[0][0], &t[0][32], 1.f, id);
    head_sync(which);
    block_product<32, 2, false, true>(&t[32][32], &t[0][32], &t[32][0], -1.f, id);
    head_sync(which);
    // T as planes, the coefficients
    {
      const int row = id >> 1;
      float v[4][8], m = 0.f, sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int unit = unit_of(i, id);
        const float4 a = *reinterpret_cast<const float4*>(&t[row][unit * 8]), b = *reinterpret_cast<const float4*>(&t[row][unit * 8 + 4]);
        v[i][0] = a.x, v[i][1] = a.y, v[i][2] = a.z, v[i][3] = a.w;
        v[i][4] = b.x, v[i][5] = b.y, v[i][6] = b.z, v[i][7] = b.w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (unit * 8 + e > row) v[i][e] = 0.f;
          m = fmaxf(m, fabsf(v[i][e]));
          sum += fabsf(v[i][e]);
        }
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      const Pow2 f = pow2_for(m);
      const float tail = expf((hi[kChunk - 1] - hi[row]) + (lo[kChunk - 1] - lo[row])) * s.row[0][row];
      const float down = fabsf(beta[row]) * exp_sum(hi[row], lo[row]) * s.row[0][row];
      // non-negative floats order as integers: the maximum does not depend on the order
      const unsigned int b0 = __reduce_max_sync(0xffffffffu, __float_as_uint(sum));
      const unsigned int b1 = __reduce_max_sync(0xffffffffu, __float_as_uint(sum * tail));
      const unsigned int b2 = __reduce_max_sync(0xffffffffu, __float_as_uint(down));
      if (lane == 0) {
        atomicMax(&s.bound[which][0], b0);
        atomicMax(&s.bound[which][1], b1);
        atomicMax(&s.bound[which][2], b2);
      }
      if (!(id & 1)) coef[kTail * kChunk + row] = tail;
#pragma unroll
      for (int i = 0; i < 4; ++i) store_unit(head, row, unit_of(i, id), v[i], f.f);
      if (!(id & 1)) coef[kTRow * kChunk + row] = f.inverse;
    }
    if (id < kChunk) {
      const float gamma = exp_sum(hi[id], lo[id]), b = beta[id];
      coef[kBeta * kChunk + id] = b;
      coef[kDown * kChunk + id] = b * gamma * s.row[0][id];
      coef[kOutQ * kChunk + id] = p.scale * gamma * s.row[1][id];
    } else {
      const int at = id - kChunk;
      coef[kSumHi * kChunk + at] = hi[at];
      coef[kSumLo * kChunk + at] = lo[at];
      coef[kKRow * kChunk + at] = s.row[0][at];
      coef[kQRow * kChunk + at] = s.row[1][at];
      coef[kDecay * kChunk + at] = exp_sum(hi[kChunk - 1], lo[kChunk - 1]);
    }
    head_sync(which);
    if (id < 4) coef[kBounds * kChunk + id] = __uint_as_float(s.bound[which][id]);
  }
}

}  // namespace seq
}  // namespace pla
