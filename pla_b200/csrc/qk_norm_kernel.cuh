// Norms of queries and keys for each head, with the position rotation in the
// same pass.  For a head x of D features at position m:
//     r = 1 / sqrt(sum x^2 / count + eps)     count = D (rms) or 1 (l2)
//     n = x r w                               w = 1 without a weight
//     the first `rot` features of n are rotated in pairs by the angle whose
//     cosine and sine the tables hold at row m:
//         (a, b) -> (a cos - b sin, b cos + a sin),
//     pairs (2i, 2i + 1) or (i, i + rot / 2); the others pass through.
// Backward, dn = dy rotated back:
//     h = dn w,  dx = r (h - xhat sum(h xhat) / count),  xhat = x r,  dw = sum dn xhat.
//
// Bound by HBM: queries and keys are read and written once (backward: read
// twice, written once), about 8 flops an element.  A group of 8, 16 or 32
// lanes owns a head; a lane holds pairs in the layout the rotation needs, so
// the partner is in the same lane and the sum of squares is the only exchange
// (shuffles).  A group keeps one set of heads (four in large calls) and walks
// tokens with their weights in registers: the set's loads are in flight
// together, the next token's while this one's are worked on, and share the
// token's cosines and sines.  All arithmetic is fp32 with one rounding at the
// end.  8192 tokens of 40 heads of 128 in bf16: 45 us, 3.7 TB/s, 57 % of the
// copy rate; what holds it there is latency (16 warps an SM at 126 registers,
// half of the issue slots), not a pipe.  One token a group without the walk and
// with 64-bit divisions took 68 us; three blocks an SM at 80 registers spill;
// asynchronous copies through shared memory two tokens ahead leave three blocks
// an SM room and still took 52 us.
#pragma once

#include "seq_common.cuh"

namespace pla {
namespace seq {

struct NormSide {
  const void* x;
  long long x_batch, x_token, x_head;
  const void* w;  // [D] or nullptr
  void* y;        // dense [batch, tokens, heads, D]; backward: the gradient of x
  const void* dy;
  long long dy_batch, dy_token, dy_head;
  int heads;
};

struct NormParams {
  NormSide side[2];        // queries, keys
  const float* cos;        // [table_rows, rot / 2]; nullptr: no rotation
  const float* sin;
  const void* positions;   // [batch, tokens] (position_batch stride), nullptr: the token's number
  long long position_batch;
  int position_bytes;      // 4 or 8
  int table_rows;
  int batch, tokens, dim, rot, interleaved, l2;
  float eps;
  int units[2];            // groups of heads of a token, per side
  int stride;              // tokens from one of a group to its next
  float* partial;          // backward: [blocks of a side][D] twice, or nullptr
  int side_blocks[2], side_stride[2];
};

// Rows whose parts are multiples of 4 pairs, at addresses that allow it: a
// lane holds 4 pairs, that is two groups of 4 features, `first` and `second`
// (2 x 4 neighbours if their pairs are adjacent).  Lanes without pairs (heads
// that do not fill the group) read what lane 0 reads and count it as 0.
struct Lane4 {
  int first, second, angle;
  bool turned, there, adjacent;
  __device__ __forceinline__ Lane4(int lane, int D, int rot, bool interleaved) {
    const int half = rot >> 1, rest_half = (D - rot) >> 1;
    there = lane * 4 < D / 2;
    const int p = there ? lane * 4 : 0, q = p - half;
    turned = p < half;
    adjacent = turned && interleaved;
    angle = p;
    first = turned ? (interleaved ? 2 * p : p) : rot + q;
    second = turned ? (interleaved ? 2 * p + 4 : p + half) : rot + rest_half + q;
  }
};
template <typename T>
struct Raw4 {
  Vec<T, 4> first, second;
};
template <typename T>
__device__ __forceinline__ Raw4<T> raw4(const T* x, const Lane4& l) {
  return {*reinterpret_cast<const Vec<T, 4>*>(x + l.first), *reinterpret_cast<const Vec<T, 4>*>(x + l.second)};
}
// Pairs (a, b) as two packed values each.  INTER: some lanes' pairs are adjacent.
template <bool INTER>
__device__ __forceinline__ void pairs_of(const float (&f)[4], const float (&s)[4], bool adjacent, Pair (&a)[2], Pair (&b)[2]) {
  a[0] = pair(f[0], INTER && adjacent ? f[2] : f[1]);
  a[1] = pair(INTER && adjacent ? s[0] : f[2], INTER && adjacent ? s[2] : f[3]);
  b[0] = pair(INTER && adjacent ? f[1] : s[0], INTER && adjacent ? f[3] : s[1]);
  b[1] = pair(INTER && adjacent ? s[1] : s[2], s[3]);
}
template <typename T, bool INTER>
__device__ __forceinline__ void unpack4(const Raw4<T>& r, const Lane4& l, Pair (&a)[2], Pair (&b)[2]) {
  float f[4], s[4];
  unpack(r.first, f);
  unpack(r.second, s);
  pairs_of<INTER>(f, s, l.adjacent, a, b);
}
template <typename T, bool INTER>
__device__ __forceinline__ void store4(T* y, const Lane4& l, const Pair (&a)[2], const Pair (&b)[2]) {
  float fa[4], fb[4], f[4], s[4];
  as_float_array(a, fa);
  as_float_array(b, fb);
  const bool adjacent = INTER && l.adjacent;
  f[0] = fa[0], f[1] = adjacent ? fb[0] : fa[1], f[2] = adjacent ? fa[1] : fa[2], f[3] = adjacent ? fb[1] : fa[3];
  s[0] = adjacent ? fa[2] : fb[0], s[1] = adjacent ? fb[2] : fb[1], s[2] = adjacent ? fa[3] : fb[2], s[3] = fb[3];
  store<T, 4>(y + l.first, f);
  store<T, 4>(y + l.second, s);
}

// Any other row: a lane of 32 holds every 32nd pair, and an odd last feature
// as the first of a pair.
struct Lane1 {
  int first[4], second[4], angle[4];
  bool turned[4], there[4], single[4];
  __device__ __forceinline__ Lane1(int lane, int D, int rot, bool interleaved) {
    const int half = rot >> 1, rest = D - rot, rest_half = rest >> 1;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int p = n * 32 + lane, q = p - half;
      turned[n] = p < half;
      angle[n] = p;
      single[n] = !turned[n] && q == rest_half && (rest & 1);
      there[n] = turned[n] || q < rest_half || single[n];
      first[n] = turned[n] ? (interleaved ? 2 * p : p) : (single[n] ? D - 1 : rot + q);
      second[n] = turned[n] ? (interleaved ? 2 * p + 1 : p + half) : rot + rest_half + q;
    }
  }
};
template <typename T>
__device__ __forceinline__ void load1(const T* x, const Lane1& l, float (&a)[4], float (&b)[4]) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    a[n] = l.there[n] ? up(x[l.first[n]]) : 0.f;
    b[n] = l.there[n] && !l.single[n] ? up(x[l.second[n]]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store1(T* y, const Lane1& l, const float (&a)[4], const float (&b)[4]) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if (l.there[n]) y[l.first[n]] = down<T>(a[n]);
    if (l.there[n] && !l.single[n]) y[l.second[n]] = down<T>(b[n]);
  }
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 1 / sqrt(v): the hardware's approximation (2^-22) and one Newton step, which
// leaves a few units of the last place.  No branch, so that the heads of a
// group overlap (1.f / sqrtf(v) has two; with them 8192 tokens of 40 heads of
// 128 in bf16 took 56 us where this took 50).
__device__ __forceinline__ float inverse_root(float v) {
  const float r = rsqrtf(v);
  const float better = r * fmaf(-0.5f * v * r, r, 1.5f);
  return v > 0.f && v < __int_as_float(0x7f800000) ? better : r;
}

// Row of the tables for a token; -1 if the position is outside them.
__device__ __forceinline__ long long table_row(const NormParams& p, int b, int t) {
  long long m = t;
  if (!p.cos) return 0;
  if (p.positions) {
    const long long at = b * p.position_batch + t;
    m = p.position_bytes == 8 ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
  }
  return m >= 0 && m < p.table_rows ? m : -1;
}

// A position outside the tables (m < 0) reads nothing: its rotated features
// are NaN.  Features that are not rotated have cosine 1 and sine 0.
__device__ __forceinline__ void angles4(const NormParams& p, const Lane4& l, long long m, float (&c)[4], float (&s)[4]) {
  const float nan = __int_as_float(0x7fc00000);
  if (l.turned && m >= 0) {
    load<float, 4>(p.cos + m * (p.rot >> 1) + l.angle, c);
    load<float, 4>(p.sin + m * (p.rot >> 1) + l.angle, s);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = l.turned ? nan : 1.f, s[i] = l.turned ? nan : 0.f;
  }
}
__device__ __forceinline__ void angles1(const NormParams& p, const Lane1& l, long long m, float (&c)[4], float (&s)[4]) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    c[n] = 1.f, s[n] = 0.f;
    if (l.turned[n]) c[n] = s[n] = __int_as_float(0x7fc00000);
    if (l.turned[n] && m >= 0) {
      c[n] = p.cos[m * (p.rot >> 1) + l.angle[n]];
      s[n] = p.sin[m * (p.rot >> 1) + l.angle[n]];
    }
  }
}

constexpr int kNormThreads = 256;

// blockIdx.y: batch row.  The groups of the grid's row are numbered; group g
// takes unit g % units (HB heads of one side) of tokens g / units,
// g / units + stride, ...  The next token's heads and angles are fetched while
// this one's are worked on.
template <typename T, int LANES, int HB, bool INTER>
__global__ void __launch_bounds__(kNormThreads) qk_norm_forward4(NormParams p) {
  const int group = (blockIdx.x * kNormThreads + threadIdx.x) / LANES;
  const int units = p.units[0] + p.units[1], b = blockIdx.y;
  int t = group / units, unit = group - t * units;
  const int which = unit >= p.units[0];
  if (which) unit -= p.units[0];
  const NormSide& side = p.side[which];
  const Lane4 lane(threadIdx.x % LANES, p.dim, p.rot, INTER);
  const int h0 = unit * HB, heads = min(HB, side.heads - h0), end = p.tokens, stride = p.stride;
  const T* x = static_cast<const T*>(side.x) + b * side.x_batch + h0 * side.x_head;
  const long long x_token = side.x_token, y_token = static_cast<long long>(side.heads) * p.dim;
  T* y = static_cast<T*>(side.y) + b * (p.tokens * y_token) + static_cast<long long>(h0) * p.dim;
  Pair wa[2], wb[2];
  {
    float f[4] = {1.f, 1.f, 1.f, 1.f}, g[4] = {1.f, 1.f, 1.f, 1.f};
    if (side.w) {
      load<T, 4>(static_cast<const T*>(side.w) + lane.first, f);
      load<T, 4>(static_cast<const T*>(side.w) + lane.second, g);
    }
    pairs_of<INTER>(f, g, lane.adjacent, wa, wb);
  }
  const float per = p.l2 ? 1.f : 1.f / p.dim;
  Raw4<T> next[HB];
  float c_next[4], s_next[4];
  // past the end the last token, and past the heads the last head, are fetched again
  const auto fetch = [&](int at, long long m) {
    const T* from = x + min(at, end - 1) * x_token;
#pragma unroll
    for (int h = 0; h < HB; ++h) next[h] = raw4(from + min(h, heads - 1) * side.x_head, lane);
    angles4(p, lane, m, c_next, s_next);
  };
  fetch(t, table_row(p, b, min(t, end - 1)));
  long long m_next = table_row(p, b, min(t + stride, end - 1));
  // a warp's groups make the same number of turns: all lanes shuffle
  for (int turn = __reduce_min_sync(0xffffffffu, t); turn < end; turn += stride, t += stride) {
    Pair ac[2], bs[2], bc[2], as[2];  // a' = r (xa (wa cos) - xb (wb sin)), b' = r (xb (wb cos) + xa (wa sin))
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Pair c = pair(c_next[2 * i], c_next[2 * i + 1]), s = pair(s_next[2 * i], s_next[2 * i + 1]);
      ac[i] = mul2(wa[i], c), bc[i] = mul2(wb[i], c), as[i] = mul2(wa[i], s);
      bs[i] = mul2(mul2(wb[i], s), pair(-1.f, -1.f));
    }
    Raw4<T> raw[HB];
#pragma unroll
    for (int h = 0; h < HB; ++h) raw[h] = next[h];
    if (turn + stride < end) {
      fetch(t + stride, m_next);
      m_next = table_row(p, b, min(t + 2 * stride, end - 1));
    }
    Pair xa[HB][2], xb[HB][2];
    float sum[HB];
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      unpack4<T, INTER>(raw[h], lane, xa[h], xb[h]);
      const float2 f = both(fma2(xa[h][0], xa[h][0], fma2(xb[h][0], xb[h][0], fma2(xa[h][1], xa[h][1], mul2(xb[h][1], xb[h][1])))));
      sum[h] = lane.there ? f.x + f.y : 0.f;  // not times 0: the sum may be infinite
    }
#pragma unroll
    for (int o = LANES / 2; o >= 1; o >>= 1)
#pragma unroll
      for (int h = 0; h < HB; ++h) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], o);
    T* to = y + t * y_token;
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      const float r = inverse_root(fmaf(sum[h], per, p.eps));
      const Pair rr = pair(r, r);
      Pair oa[2], ob[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Pair na = mul2(xa[h][i], rr), nb = mul2(xb[h][i], rr);
        Pair from_b = pair(0.f, 0.f), from_a = from_b;  // nothing without rotation: the partner may be infinite
        if (lane.turned) from_b = mul2(nb, bs[i]), from_a = mul2(na, as[i]);
        oa[i] = fma2(na, ac[i], from_b);
        ob[i] = fma2(nb, bc[i], from_a);
      }
      if (t < end && h < heads && lane.there) store4<T, INTER>(to, lane, oa, ob);
      to += p.dim;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) qk_norm_forward1(NormParams p) {
  const int group = (blockIdx.x * kNormThreads + threadIdx.x) / 32;
  const int units = p.units[0] + p.units[1], b = blockIdx.y;
  int t = group / units, unit = group - t * units;
  const int which = unit >= p.units[0];
  if (which) unit -= p.units[0];
  const NormSide& side = p.side[which];
  const Lane1 lane(threadIdx.x & 31, p.dim, p.rot, p.interleaved);
  float wa[4] = {1.f, 1.f, 1.f, 1.f}, wb[4] = {1.f, 1.f, 1.f, 1.f};
  if (side.w) load1(static_cast<const T*>(side.w), lane, wa, wb);
  const float per = p.l2 ? 1.f : 1.f / p.dim;
  for (; t < p.tokens; t += p.stride) {
    float a[4], c4[4], b4[4], s4[4];
    load1(static_cast<const T*>(side.x) + b * side.x_batch + t * side.x_token + unit * side.x_head, lane, a, b4);
    angles1(p, lane, table_row(p, b, t), c4, s4);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) sum = fmaf(a[n], a[n], fmaf(b4[n], b4[n], sum));
    const float r = inverse_root(fmaf(group_sum<32>(sum), per, p.eps));
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float na = a[n] * r * wa[n], nb = b4[n] * r * wb[n];
      a[n] = lane.turned[n] ? fmaf(na, c4[n], -nb * s4[n]) : na;
      b4[n] = lane.turned[n] ? fmaf(nb, c4[n], na * s4[n]) : nb;
    }
    store1(static_cast<T*>(side.y) + ((static_cast<long long>(b) * p.tokens + t) * side.heads + unit) * p.dim, lane, a, b4);
  }
}

// dx, and the block's sums for dw.  A block works on one side: its groups walk
// tokens with one head each and dw in registers, and are added in shared
// memory, the blocks in qk_norm_reduce, all in a fixed order.
template <int GROUPS, int LANES>
__device__ __forceinline__ void block_weight_sums(const NormParams& p, float (&ga)[4], float (&gb)[4], float (*part)[8][LANES + 1],
                                                  float (&a)[4], float (&b)[4]) {
  const int lane = threadIdx.x % LANES, in_block = threadIdx.x / LANES;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    part[in_block][2 * i][lane] = ga[i];
    part[in_block][2 * i + 1][lane] = gb[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = b[i] = 0.f;
  if (in_block) return;
  for (int g = 0; g < GROUPS; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] += part[g][2 * i][lane];
      b[i] += part[g][2 * i + 1][lane];
    }
}

template <typename T, int LANES, bool INTER>
__global__ void __launch_bounds__(kNormThreads) qk_norm_backward4(NormParams p) {
  constexpr int GROUPS = kNormThreads / LANES;
  __shared__ float part[GROUPS][8][LANES + 1];
  const int in_block = threadIdx.x / LANES;
  const int which = static_cast<int>(blockIdx.x) >= p.side_blocks[0];
  const NormSide& side = p.side[which];
  const int block = which ? blockIdx.x - p.side_blocks[0] : blockIdx.x;
  const Lane4 lane(threadIdx.x % LANES, p.dim, p.rot, INTER);
  Pair wa[2], wb[2], ga[2], gb[2];
  ga[0] = ga[1] = gb[0] = gb[1] = pair(0.f, 0.f);
  {
    float f[4] = {1.f, 1.f, 1.f, 1.f}, g[4] = {1.f, 1.f, 1.f, 1.f};
    if (side.w) {
      load<T, 4>(static_cast<const T*>(side.w) + lane.first, f);
      load<T, 4>(static_cast<const T*>(side.w) + lane.second, g);
    }
    pairs_of<INTER>(f, g, lane.adjacent, wa, wb);
  }
  const float per = p.l2 ? 1.f : 1.f / p.dim;
  const int rows = p.batch * p.tokens, stride = p.side_stride[which];  // rows below 2^30
  const int group = block * GROUPS + in_block;
  int row = group / side.heads;  // batch row and token as one number
  const int h = group - row * side.heads;
  int b = row / p.tokens, t = row - b * p.tokens;
  const int on_b = stride / p.tokens, on_t = stride - on_b * p.tokens;
  const T* x = static_cast<const T*>(side.x) + h * side.x_head;
  const T* dy = static_cast<const T*>(side.dy) + h * side.dy_head;
  // the next token's head and angles are fetched while this one's are worked on; past the end, the first's
  Raw4<T> x_next, dy_next;
  float c_next[4], s_next[4];
  const auto fetch = [&](int at_row) {
    const int bb = at_row < rows ? b : 0, tt = at_row < rows ? t : 0;
    x_next = raw4(x + bb * side.x_batch + tt * side.x_token, lane);
    dy_next = raw4(dy + bb * side.dy_batch + tt * side.dy_token, lane);
    angles4(p, lane, table_row(p, bb, tt), c_next, s_next);
    t += on_t, b += on_b;
    if (t >= p.tokens) t -= p.tokens, ++b;
  };
  fetch(row);
  // `stride` tokens on for every turn; a warp's groups make the same number of turns
  for (int turn = __reduce_min_sync(0xffffffffu, row); turn < rows; turn += stride, row += stride) {
    Pair xa[2], xb[2], ya[2], yb[2], da[2], db[2], c[2], s[2], n[2];
    unpack4<T, INTER>(x_next, lane, xa, xb);
    unpack4<T, INTER>(dy_next, lane, ya, yb);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = pair(c_next[2 * i], c_next[2 * i + 1]), s[i] = pair(s_next[2 * i], s_next[2 * i + 1]);
      n[i] = pair(-s_next[2 * i], -s_next[2 * i + 1]);
    }
    if (turn + stride < rows) fetch(row + stride);
    Pair squares = pair(0.f, 0.f), dots = pair(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // rotated back; without rotation cos is 1 and the partner left out
      Pair from_b = pair(0.f, 0.f), from_a = from_b;
      if (lane.turned) from_b = mul2(yb[i], s[i]), from_a = mul2(ya[i], n[i]);
      da[i] = fma2(ya[i], c[i], from_b);
      db[i] = fma2(yb[i], c[i], from_a);
      squares = fma2(xa[i], xa[i], fma2(xb[i], xb[i], squares));
      dots = fma2(mul2(da[i], wa[i]), xa[i], fma2(mul2(db[i], wb[i]), xb[i], dots));
    }
    const float2 q = both(squares), d = both(dots);
    const float square = group_sum<LANES>(lane.there ? q.x + q.y : 0.f);
    const float dot = group_sum<LANES>(lane.there ? d.x + d.y : 0.f);
    if (row >= rows) continue;
    const float r = inverse_root(fmaf(square, per, p.eps));
    const Pair back = pair(-dot * r * r * per, -dot * r * r * per), rr = pair(r, r);  // - sum(h xhat) r / count
    Pair oa[2], ob[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      oa[i] = mul2(rr, fma2(back, xa[i], mul2(da[i], wa[i])));
      ob[i] = mul2(rr, fma2(back, xb[i], mul2(db[i], wb[i])));
      ga[i] = fma2(da[i], mul2(xa[i], rr), ga[i]);
      gb[i] = fma2(db[i], mul2(xb[i], rr), gb[i]);
    }
    if (lane.there)
      store4<T, INTER>(static_cast<T*>(side.y) + (static_cast<long long>(row) * side.heads + h) * p.dim, lane, oa, ob);
  }
  if (!p.partial || !side.w) return;
  float fa[4], fb[4], a[4], b2[4];
  as_float_array(ga, fa);
  as_float_array(gb, fb);
  block_weight_sums<GROUPS, LANES>(p, fa, fb, part, a, b2);
  if (in_block || !lane.there) return;
  Pair pa[2], pb[2];
  as_pair_array(a, pa);
  as_pair_array(b2, pb);
  store4<float, INTER>(p.partial + static_cast<long long>(blockIdx.x) * p.dim, lane, pa, pb);
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) qk_norm_backward1(NormParams p) {
  constexpr int GROUPS = kNormThreads / 32;
  __shared__ float part[GROUPS][8][33];
  const int in_block = threadIdx.x / 32;
  const int which = static_cast<int>(blockIdx.x) >= p.side_blocks[0];
  const NormSide& side = p.side[which];
  const int block = which ? blockIdx.x - p.side_blocks[0] : blockIdx.x;
  const Lane1 lane(threadIdx.x & 31, p.dim, p.rot, p.interleaved);
  float wa[4] = {1.f, 1.f, 1.f, 1.f}, wb[4] = {1.f, 1.f, 1.f, 1.f}, ga[4] = {}, gb[4] = {};
  if (side.w) load1(static_cast<const T*>(side.w), lane, wa, wb);
  const float per = p.l2 ? 1.f : 1.f / p.dim;
  const int rows = p.batch * p.tokens, stride = p.side_stride[which];
  const int group = block * GROUPS + in_block;
  int row = group / side.heads;
  const int h = group - row * side.heads;
  for (; row < rows; row += stride) {
    const int b = row / p.tokens, t = row - b * p.tokens;
    float xa[4], xb[4], da[4], db[4], c[4], s[4];
    load1(static_cast<const T*>(side.x) + b * side.x_batch + t * side.x_token + h * side.x_head, lane, xa, xb);
    load1(static_cast<const T*>(side.dy) + b * side.dy_batch + t * side.dy_token + h * side.dy_head, lane, da, db);
    angles1(p, lane, table_row(p, b, t), c, s);
    float square = 0.f, dot = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (lane.turned[n]) {
        const float ya = da[n], yb = db[n];
        da[n] = fmaf(ya, c[n], yb * s[n]);
        db[n] = fmaf(yb, c[n], -ya * s[n]);
      }
      square = fmaf(xa[n], xa[n], fmaf(xb[n], xb[n], square));
      dot = fmaf(da[n] * wa[n], xa[n], fmaf(db[n] * wb[n], xb[n], dot));
    }
    square = group_sum<32>(square);
    dot = group_sum<32>(dot);
    const float r = inverse_root(fmaf(square, per, p.eps));
    const float back = dot * r * r * per;  // sum(h xhat) r / count
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      ga[n] = fmaf(da[n], xa[n] * r, ga[n]);
      gb[n] = fmaf(db[n], xb[n] * r, gb[n]);
      da[n] = r * fmaf(-back, xa[n], da[n] * wa[n]);
      db[n] = r * fmaf(-back, xb[n], db[n] * wb[n]);
    }
    store1(static_cast<T*>(side.y) + (static_cast<long long>(row) * side.heads + h) * p.dim, lane, da, db);
  }
  if (!p.partial || !side.w) return;
  float a[4], b2[4];
  block_weight_sums<GROUPS, 32>(p, ga, gb, part, a, b2);
  if (!in_block) store1(p.partial + static_cast<long long>(blockIdx.x) * p.dim, lane, a, b2);
}

// dw of one side: blocks' sums in 32 interleaved parts, the parts in order.
template <typename T>
__global__ void __launch_bounds__(1024) qk_norm_reduce(const float* partial, int blocks_q, int blocks_k, int dim, T* dwq, T* dwk) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  const int blocks = blockIdx.y ? blocks_k : blocks_q;
  const float* from = partial + (blockIdx.y ? static_cast<long long>(blocks_q) * dim : 0);
  T* to = blockIdx.y ? dwk : dwq;
  if (!to) return;
  float sum = 0.f;
  if (d < dim)
#pragma unroll 8
    for (int i = row; i < blocks; i += 32) sum += from[static_cast<long long>(i) * dim + d];
  part[row][lane] = sum;
  __syncthreads();
  if (row || d >= dim) return;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) sum += part[i][lane];
  to[d] = down<T>(sum);
}

}  // namespace seq
}  // namespace pla
