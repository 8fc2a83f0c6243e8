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
// together and share the token's cosines and sines, and a token costs no
// division and no set-up (with a set-up per token the kernel was bound by
// instructions, 68 us for 8192 tokens of 40 heads of 128 in bf16, against
// NORMFWD).  All arithmetic is fp32 with one rounding at the end.
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

// A lane's NC chunks of CH pairs of a head's features.  CH = 4 needs rot / 2
// and (D - rot) / 2 to be multiples of 4 and 16-byte rows; CH = 1 takes any D.
template <int CH, int NC>
struct PairMap {
  int first[NC], second[NC];  // first feature of each chunk's a and b parts
  bool turned[NC], there[NC], adjacent[NC], single[NC];
  int angle[NC];
  __device__ __forceinline__ PairMap(int lane, int lanes, int D, int rot, int interleaved) {
    const int half = rot >> 1, rest = D - rot, rest_half = rest >> 1;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int p = (n * lanes + lane) * CH;  // pair number
      turned[n] = p < half;
      adjacent[n] = turned[n] && interleaved;
      angle[n] = p;
      const int q = p - half;
      single[n] = CH == 1 && !turned[n] && q == rest_half && (rest & 1);  // CH = 4: never
      there[n] = turned[n] || q < rest_half || single[n];
      first[n] = turned[n] ? (interleaved ? 2 * p : p) : (single[n] ? D - 1 : rot + q);
      second[n] = turned[n] ? (interleaved ? 2 * p + CH : p + half) : rot + rest_half + q;
    }
  }
};

// The two chunks of a lane as they lie in memory, and as pairs.
template <typename T, int CH>
struct RawPairs {
  Vec<T, CH> first, second;
};
template <typename T, int CH>
__device__ __forceinline__ RawPairs<T, CH> raw_pairs(const T* x, int first, int second, bool there, bool single) {
  RawPairs<T, CH> r;
#pragma unroll
  for (int i = 0; i < CH; ++i) r.first.e[i] = r.second.e[i] = down<T>(0.f);
  if (there) r.first = *reinterpret_cast<const Vec<T, CH>*>(x + first);
  if (there && !single) r.second = *reinterpret_cast<const Vec<T, CH>*>(x + second);
  return r;
}
template <typename T, int CH>
__device__ __forceinline__ void as_pairs(const RawPairs<T, CH>& r, bool adjacent, float (&a)[CH], float (&b)[CH]) {
  float f[CH], s[CH];
  unpack(r.first, f);
  unpack(r.second, s);
#pragma unroll
  for (int i = 0; i < CH; ++i) {  // adjacent: 2 CH neighbours, even ones are a, odd ones b
    a[i] = CH > 1 && adjacent ? (2 * i < CH ? f[(2 * i) % CH] : s[(2 * i) % CH]) : f[i];
    b[i] = CH > 1 && adjacent ? (2 * i < CH ? f[(2 * i + 1) % CH] : s[(2 * i + 1) % CH]) : s[i];
  }
}
template <typename T, int CH>
__device__ __forceinline__ void load_pairs(const T* x, int first, int second, bool adjacent, bool single, float (&a)[CH],
                                           float (&b)[CH]) {
  as_pairs(raw_pairs<T, CH>(x, first, second, true, single), adjacent, a, b);
}

template <typename T, int CH>
__device__ __forceinline__ void store_pairs(T* y, int first, int second, bool adjacent, bool single, const float (&a)[CH],
                                            const float (&b)[CH]) {
  float f[CH], s[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (CH > 1 && adjacent) {
      f[i] = i % 2 == 0 ? a[i / 2] : b[i / 2];
      s[i] = i % 2 == 0 ? a[(CH + i) / 2] : b[(CH + i) / 2];
    } else {
      f[i] = a[i];
      s[i] = b[i];
    }
  }
  store<T, CH>(y + first, f);
  if (!single) store<T, CH>(y + second, s);
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
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
template <int CH, int NC>
__device__ __forceinline__ void load_angles(const NormParams& p, const PairMap<CH, NC>& map, long long m, float (&c)[NC][CH],
                                            float (&s)[NC][CH]) {
  const float nan = __int_as_float(0x7fc00000);
#pragma unroll
  for (int n = 0; n < NC; ++n) {
#pragma unroll
    for (int i = 0; i < CH; ++i) c[n][i] = map.turned[n] ? nan : 1.f, s[n][i] = map.turned[n] ? nan : 0.f;
    if (map.turned[n] && m >= 0) {
      load<float, CH>(p.cos + m * (p.rot >> 1) + map.angle[n], c[n]);
      load<float, CH>(p.sin + m * (p.rot >> 1) + map.angle[n], s[n]);
    }
  }
}

constexpr int kNormThreads = 256;

// A lane's parts of a weight; ones without.
template <typename T, int CH, int NC>
__device__ __forceinline__ void load_weight(const NormSide& side, const PairMap<CH, NC>& map, float (&wa)[NC][CH], float (&wb)[NC][CH]) {
#pragma unroll
  for (int n = 0; n < NC; ++n) {
#pragma unroll
    for (int i = 0; i < CH; ++i) wa[n][i] = wb[n][i] = 1.f;
    if (side.w && map.there[n])
      load_pairs<T, CH>(static_cast<const T*>(side.w), map.first[n], map.second[n], map.adjacent[n], map.single[n], wa[n],
                        wb[n]);
  }
}

// blockIdx.y: batch row.  The groups of the grid's row are numbered; group g
// takes unit g % units of tokens g / units, g / units + stride, ...
template <typename T, int CH, int NC, int LANES, int HB>
__global__ void __launch_bounds__(kNormThreads) qk_norm_forward(NormParams p) {
  constexpr int H = (CH + 1) / 2;
  const int lane = threadIdx.x % LANES;
  const int group = (blockIdx.x * kNormThreads + threadIdx.x) / LANES;
  const int units = p.units[0] + p.units[1], b = blockIdx.y;
  int t = group / units, unit = group - t * units;
  const int which = unit >= p.units[0];
  if (which) unit -= p.units[0];
  const NormSide& side = p.side[which];
  const PairMap<CH, NC> map(lane, LANES, p.dim, p.rot, p.interleaved);
  const int h0 = unit * HB, heads = min(HB, side.heads - h0);
  const T* x = static_cast<const T*>(side.x) + b * side.x_batch + h0 * side.x_head;
  T* y = static_cast<T*>(side.y) + (static_cast<long long>(b) * p.tokens * side.heads + h0) * p.dim;
  float wa[NC][CH], wb[NC][CH];
  load_weight<T, CH, NC>(side, map, wa, wb);
  const float per = p.l2 ? 1.f : 1.f / p.dim;
  using Raw = RawPairs<T, CH>;
  // heads and angles of the next token are fetched while this one's are worked on
  Raw next[HB][NC];
  float c_next[NC][CH], s_next[NC][CH];
  const auto fetch = [&](int at, long long m) {
    const T* from = x + at * side.x_token;
#pragma unroll
    for (int h = 0; h < HB; ++h) {
#pragma unroll
      for (int n = 0; n < NC; ++n)
        next[h][n] = raw_pairs<T, CH>(from, map.first[n], map.second[n], at < p.tokens && h < heads && map.there[n],
                                      map.single[n]);
      from += side.x_head;
    }
    load_angles<CH, NC>(p, map, m, c_next, s_next);
  };
  const auto position = [&](int at) { return at < p.tokens ? table_row(p, b, at) : -1ll; };
  fetch(t, position(t));
  long long m_next = position(t + p.stride);
  // a warp's groups make the same number of turns: all lanes shuffle
  for (int turn = __reduce_min_sync(0xffffffffu, t); turn < p.tokens; turn += p.stride, t += p.stride) {
    const bool live = t < p.tokens;
    Raw raw[HB][NC];
    float c[NC][CH], s[NC][CH];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
      for (int h = 0; h < HB; ++h) raw[h][n] = next[h][n];
#pragma unroll
      for (int i = 0; i < CH; ++i) c[n][i] = c_next[n][i], s[n][i] = s_next[n][i];
    }
    if (turn + p.stride < p.tokens) {
      fetch(t + p.stride, m_next);
      m_next = position(t + 2 * p.stride);
    }
    // weights and angles together: a' = r (xa (wa cos) - xb (wb sin)), b' = r (xb (wb cos) + xa (wa sin))
    Pair ac[NC][H], bs[NC][H], bc[NC][H], as[NC][H];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float f[4][CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        f[0][i] = wa[n][i] * c[n][i];
        f[1][i] = -wb[n][i] * s[n][i];
        f[2][i] = wb[n][i] * c[n][i];
        f[3][i] = wa[n][i] * s[n][i];
      }
      as_pair_array(f[0], ac[n]);
      as_pair_array(f[1], bs[n]);
      as_pair_array(f[2], bc[n]);
      as_pair_array(f[3], as[n]);
    }
    T* to = y + static_cast<long long>(t) * side.heads * p.dim;
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      Pair xa[NC][H], xb[NC][H], sums = pair(0.f, 0.f);
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        float fa[CH], fb[CH];
        as_pairs(raw[h][n], map.adjacent[n], fa, fb);
        as_pair_array(fa, xa[n]);
        as_pair_array(fb, xb[n]);
#pragma unroll
        for (int i = 0; i < H; ++i) sums = fma2(xa[n][i], xa[n][i], fma2(xb[n][i], xb[n][i], sums));
      }
      const float2 sum = both(sums);
      const float r = 1.f / sqrtf(fmaf(group_sum<LANES>(sum.x + sum.y), per, p.eps));
      if (live && h < heads) {
        const Pair rr = pair(r, r);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          if (!map.there[n]) continue;
          Pair oa[H], ob[H];
          float fa[CH], fb[CH];
#pragma unroll
          for (int i = 0; i < H; ++i) {
            const Pair na = mul2(xa[n][i], rr), nb = mul2(xb[n][i], rr);
            oa[i] = fma2(na, ac[n][i], mul2(nb, bs[n][i]));
            ob[i] = fma2(nb, bc[n][i], mul2(na, as[n][i]));
          }
          as_float_array(oa, fa);
          as_float_array(ob, fb);
          store_pairs<T, CH>(to, map.first[n], map.second[n], map.adjacent[n], map.single[n], fa, fb);
        }
      }
      to += p.dim;
    }
  }
}

// dx, and the block's sums for dw.  A block works on one side: its groups walk
// tokens with one head each and dw in registers, and are added in shared
// memory, the blocks in qk_norm_reduce, all in a fixed order.
template <typename T, int CH, int NC, int LANES>
__global__ void __launch_bounds__(kNormThreads) qk_norm_backward(NormParams p) {
  constexpr int GROUPS = kNormThreads / LANES;
  __shared__ float part[GROUPS][2 * CH * NC][LANES + 1];
  const int lane = threadIdx.x % LANES, in_block = threadIdx.x / LANES;
  const int which = static_cast<int>(blockIdx.x) >= p.side_blocks[0];
  const NormSide& side = p.side[which];
  const int block = which ? blockIdx.x - p.side_blocks[0] : blockIdx.x;
  const PairMap<CH, NC> map(lane, LANES, p.dim, p.rot, p.interleaved);
  float wa[NC][CH], wb[NC][CH], ga[NC][CH] = {}, gb[NC][CH] = {};
  load_weight<T, CH, NC>(side, map, wa, wb);
  const float per = p.l2 ? 1.f : 1.f / p.dim;
  const int rows = p.batch * p.tokens;  // below 2^31
  const int group = block * GROUPS + in_block;
  int row = group / side.heads;  // batch row and token as one number
  const int h = group - row * side.heads;
  int b = row / p.tokens, t = row - b * p.tokens;
  using Raw = RawPairs<T, CH>;
  // the next token's head and angles are fetched while this one's are worked on
  Raw x_next[NC], dy_next[NC];
  float c_next[NC][CH], s_next[NC][CH];
  const int stride = p.side_stride[which];
  const auto fetch = [&](int at_row) {
    while (t >= p.tokens) t -= p.tokens, ++b;
    const bool in = at_row < rows;
    const T* x = static_cast<const T*>(side.x) + b * side.x_batch + t * side.x_token + h * side.x_head;
    const T* dy = static_cast<const T*>(side.dy) + b * side.dy_batch + t * side.dy_token + h * side.dy_head;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      x_next[n] = raw_pairs<T, CH>(x, map.first[n], map.second[n], in && map.there[n], map.single[n]);
      dy_next[n] = raw_pairs<T, CH>(dy, map.first[n], map.second[n], in && map.there[n], map.single[n]);
    }
    load_angles<CH, NC>(p, map, in ? table_row(p, b, t) : -1, c_next, s_next);
    t += stride;
  };
  fetch(row);
  // `stride` tokens on for every turn; a warp's groups make the same number of turns
  for (int turn = __reduce_min_sync(0xffffffffu, row); turn < rows; turn += stride, row += stride) {
    const bool live = row < rows;
    float xa[NC][CH], xb[NC][CH], da[NC][CH], db[NC][CH], c[NC][CH], s[NC][CH];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      as_pairs(x_next[n], map.adjacent[n], xa[n], xb[n]);
      as_pairs(dy_next[n], map.adjacent[n], da[n], db[n]);
#pragma unroll
      for (int i = 0; i < CH; ++i) c[n][i] = c_next[n][i], s[n][i] = s_next[n][i];
    }
    if (turn + stride < rows) fetch(row + stride);
    float square = 0.f, dot = 0.f;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const float ya = da[n][i], yb = db[n][i];  // rotated back; cos 1, sin 0 where there is no rotation
        da[n][i] = fmaf(ya, c[n][i], yb * s[n][i]);
        db[n][i] = fmaf(yb, c[n][i], -ya * s[n][i]);
        square = fmaf(xa[n][i], xa[n][i], fmaf(xb[n][i], xb[n][i], square));
        dot = fmaf(da[n][i] * wa[n][i], xa[n][i], fmaf(db[n][i] * wb[n][i], xb[n][i], dot));
      }
    square = group_sum<LANES>(square);
    dot = group_sum<LANES>(dot);
    if (!live) continue;
    const float r = 1.f / sqrtf(fmaf(square, per, p.eps));
    const float back = dot * r * r * per;  // sum(h xhat) r / count
    T* dx = static_cast<T*>(side.y) + (static_cast<long long>(row) * side.heads + h) * p.dim;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      if (!map.there[n]) continue;
      float oa[CH], ob[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        oa[i] = r * fmaf(-back, xa[n][i], da[n][i] * wa[n][i]);
        ob[i] = r * fmaf(-back, xb[n][i], db[n][i] * wb[n][i]);
        ga[n][i] = fmaf(da[n][i], xa[n][i] * r, ga[n][i]);
        gb[n][i] = fmaf(db[n][i], xb[n][i] * r, gb[n][i]);
      }
      store_pairs<T, CH>(dx, map.first[n], map.second[n], map.adjacent[n], map.single[n], oa, ob);
    }
  }
  if (!p.partial || !side.w) return;
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      part[in_block][2 * (n * CH + i)][lane] = ga[n][i];
      part[in_block][2 * (n * CH + i) + 1][lane] = gb[n][i];
    }
  __syncthreads();
  if (in_block) return;
  float* out = p.partial + static_cast<long long>(blockIdx.x) * p.dim;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    if (!map.there[n]) continue;
    float a[CH] = {}, b2[CH] = {};
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        a[i] += part[g][2 * (n * CH + i)][lane];
        b2[i] += part[g][2 * (n * CH + i) + 1][lane];
      }
    store_pairs<float, CH>(out, map.first[n], map.second[n], map.adjacent[n], map.single[n], a, b2);
  }
}

// dw of one side: blocks' sums in eight interleaved parts, the parts pairwise.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_reduce(const float* partial, int blocks_q, int blocks_k, int dim, T* dwq, T* dwk) {
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  const int blocks = blockIdx.y ? blocks_k : blocks_q;
  const float* from = partial + (blockIdx.y ? static_cast<long long>(blocks_q) * dim : 0);
  T* to = blockIdx.y ? dwk : dwq;
  if (!to) return;
  float sum = 0.f;
  if (d < dim)
    for (int i = row; i < blocks; i += 8) sum += from[static_cast<long long>(i) * dim + d];
  part[row][lane] = sum;
  __syncthreads();
  if (row || d >= dim) return;
  sum = ((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane])) +
        ((part[4][lane] + part[5][lane]) + (part[6][lane] + part[7][lane]));
  to[d] = down<T>(sum);
}

}  // namespace seq
}  // namespace pla
