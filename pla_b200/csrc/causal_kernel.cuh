// Causal depthwise convolution along time (the short convolution of a
// sequence block), channels last: x [batch, tokens, C], filter [C, K], K <= 4,
//     p[t] = b + sum_{j<K} w[j] x[t - K + 1 + j],   y = p  or  p * sigmoid(p).
// Tokens before a sequence's first one are the K - 1 rows of its state
// (oldest first) or zero.
//
// Bound by HBM: x is read and y written once, 2 K flops an element.  A thread
// owns four neighbouring channels of a strip of tokens and walks it with the
// last K - 1 inputs in registers, so an input is fetched once plus
// (K - 1) / strip of overlap that neighbouring strips leave in L2; a ring of
// eight rows is in flight, each refilled as soon as it is used.  Four channels
// (8 bytes a 16-bit load) and not eight: eight took 148 registers a thread,
// which left 8 warps an SM and too few bytes in flight (140 us for 8191 x 8192
// bf16, against 59).  The products are summed in fp32 in tap
// order, two channels an instruction, and rounded once.
//
// Backward, with dp[t] = dy[t] act'(p[t]) recomputed from x:
//     dx[t] = sum_j w[j] dp[t + K - 1 - j],  dw[j] = sum_t dp[t] x[t - K + 1 + j],  db = sum_t dp[t].
// A thread walks its strip and K - 1 tokens past it, adds each dp[t] to the
// K pending dx it reaches inside the same sequence, and keeps dw / db of its
// own strip in registers.  The strips of a block are added in shared memory,
// the blocks' partial sums in a second kernel, both in a fixed order: no
// atomics, so the same inputs give the same bits.  2 x 4096 x 4096 bf16: 74 us,
// 2.7 TB/s (three passes over the data); two channels a thread, because it
// holds five times the forward's registers.
#pragma once

#include "seq_common.cuh"

namespace pla {
namespace seq {

struct CausalParams {
  const void* x;
  long long x_batch, x_token;
  const void* w;
  const void* b;           // nullptr: none
  const int* cu;           // nullptr: every batch row is one sequence
  const void* state_in;    // [sequences, K - 1, C] or nullptr (zeros)
  void* state_out;         // likewise, or nullptr
  void* y;                 // dense
  int batch, tokens, channels, sequences, silu;
  int strip, strips;       // tokens of a strip, strips of a batch row
  // backward
  const void* dy;
  long long dy_batch, dy_token;
  const void* dstate_out;
  void* dx;                // dense
  void* dstate_in;
  float* partial;          // [blocks, K + 1, C]
};

// Walks the sequences of one batch row from a token on.
struct SequenceWalk {
  int index, start, end;
  __device__ __forceinline__ void begin(const CausalParams& p, int batch, int t) {
    if (!p.cu) {
      index = batch;
      start = 0;
      end = p.tokens;
      return;
    }
    index = find_sequence(p.cu, p.sequences, t);
    if (index >= 0) {
      start = max(p.cu[index], 0);
      end = p.cu[index + 1];
    } else {  // before the first sequence or behind the last one
      start = t;
      end = t < p.cu[0] ? p.cu[0] : 0x7fffffff;
    }
  }
  // t == end: the next sequence that holds t.
  __device__ __forceinline__ void next(const CausalParams& p, int batch, int t) {
    begin(p, batch, t);
    if (end <= t) end = t + 1;  // entries that do not ascend: stay in bounds and go on
  }
};

// Input row `back` tokens before t (back < K): the tensor's, the state's or zero.
template <typename T, int V, int K>
__device__ __forceinline__ void input_before(const CausalParams& p, const T* x, const SequenceWalk& s, int t, int back,
                                             int c, float (&f)[V]) {
  const int at = t - back;
  if (s.index >= 0 && at >= s.start) {
    load<T, V>(x + at * p.x_token + c, f);
    return;
  }
  const int row = K - 1 - (s.start - at);
  if (s.index >= 0 && p.state_in && row >= 0) {
    load<T, V>(static_cast<const T*>(p.state_in) + (static_cast<long long>(s.index) * (K - 1) + row) * p.channels + c, f);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = 0.f;
}

template <typename T, int V, int K>
__device__ __forceinline__ void load_filter(const CausalParams& p, int c, float (&w)[K][V], float (&b)[V]) {
  const T* wt = static_cast<const T*>(p.w) + static_cast<long long>(c) * K;  // V filters of K taps
  float flat[V * K];
#pragma unroll
  for (int i = 0; i < K; ++i) load<T, V>(wt + i * V, *reinterpret_cast<float(*)[V]>(&flat[i * V]));
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][i] = flat[i * K + j];
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = 0.f;
  if (p.b) load<T, V>(static_cast<const T*>(p.b) + c, b);
}

// The K - 1 inputs behind a sequence's last token: rows len .. len + K - 2 of [state; x].
template <typename T, int V, int K>
__device__ __forceinline__ void copy_state(const CausalParams& p, long long item) {
  const int nvec = p.channels / V;
  const int c = static_cast<int>(item % nvec) * V;
  const long long at = item / nvec;
  const int row = static_cast<int>(at % (K - 1)), n = static_cast<int>(at / (K - 1));
  if (n >= p.sequences) return;
  int lo = 0, len = p.tokens;
  if (p.cu) {
    lo = clamp_token(p.cu[n], p.tokens);
    len = max(clamp_token(p.cu[n + 1], p.tokens) - lo, 0);
  }
  const T* x = static_cast<const T*>(p.x) + (p.cu ? 0 : n * p.x_batch);
  SequenceWalk s{n, lo, lo + len};
  float f[V];
  input_before<T, V, K>(p, x, s, lo + len, K - 1 - row, c, f);
  store<T, V>(static_cast<T*>(p.state_out) + (static_cast<long long>(n) * (K - 1) + row) * p.channels + c, f);
}

constexpr int kCausalThreads = 256;

template <typename T, int V, int K>
__global__ void __launch_bounds__(kCausalThreads, 3) causal_forward(CausalParams p, int main_blocks) {
  if (static_cast<int>(blockIdx.x) >= main_blocks) {
    copy_state<T, V, K>(p, static_cast<long long>(blockIdx.x - main_blocks) * kCausalThreads + threadIdx.x);
    return;
  }
  const long long item = static_cast<long long>(blockIdx.x) * kCausalThreads + threadIdx.x;
  const int nvec = p.channels / V;
  const int c = static_cast<int>(item % nvec) * V;
  const long long strip = item / nvec;
  const int batch = static_cast<int>(strip / p.strips);
  if (batch >= p.batch) return;
  const int t0 = static_cast<int>(strip % p.strips) * p.strip;
  const int t1 = min(t0 + p.strip, p.tokens);
  const T* x = static_cast<const T*>(p.x) + batch * p.x_batch;
  T* y = static_cast<T*>(p.y) + (static_cast<long long>(batch) * p.tokens + t0) * p.channels + c;

  constexpr int U = 8, H = (V + 1) / 2;
  using Row = Vec<T, V>;
  const T* from = x + t0 * p.x_token + c;
  Row ring[U];
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (t0 + i < t1) ring[i] = *reinterpret_cast<const Row*>(from + i * p.x_token);
  from += U * p.x_token;
  Pair w[K][H], b[H], seen[K - 1][H];
  SequenceWalk s;
  s.begin(p, batch, t0);
  {
    float wf[K][V], bf[V];
    load_filter<T, V, K>(p, c, wf, bf);
#pragma unroll
    for (int j = 0; j < K; ++j) as_pair_array(wf[j], w[j]);
    as_pair_array(bf, b);
  }
  const auto refill = [&](int t) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      float f[V];
      input_before<T, V, K>(p, x, s, t, K - 1 - j, c, f);
      as_pair_array(f, seen[j]);
    }
  };
  const auto one = [&](const Row& row) {
    float in[V], out[V];
    unpack(row, in);
    Pair now[H], a[H];
    as_pair_array(in, now);
#pragma unroll
    for (int v = 0; v < H; ++v) {
      a[v] = b[v];
#pragma unroll
      for (int j = 0; j < K - 1; ++j) a[v] = fma2(w[j][v], seen[j][v], a[v]);
      a[v] = fma2(w[K - 1][v], now[v], a[v]);
#pragma unroll
      for (int j = 0; j + 1 < K - 1; ++j) seen[j][v] = seen[j + 1][v];
      seen[K - 2][v] = now[v];
    }
    as_float_array(a, out);
    if (p.silu)
#pragma unroll
      for (int v = 0; v < V; ++v) out[v] *= sigmoid<T>(out[v]);
    store<T, V>(y, out);
    y += p.channels;
  };
  refill(t0);
  for (int t = t0; t < t1; t += U) {
    if (t + 2 * U <= t1 && t + U <= s.end && s.index >= 0) {  // eight tokens of one sequence, and eight more to fetch
#pragma unroll
      for (int i = 0; i < U; ++i) {
        one(ring[i]);
        ring[i] = *reinterpret_cast<const Row*>(from);
        from += p.x_token;
      }
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (t + i >= t1) break;
        if (t + i >= s.end) {
          s.next(p, batch, t + i);
          refill(t + i);
        }
        if (s.index >= 0) {
          one(ring[i]);
        } else {
          const float none[V] = {};
          store<T, V>(y, none);
          y += p.channels;
        }
        if (t + U + i < t1) ring[i] = *reinterpret_cast<const Row*>(from);
        from += p.x_token;
      }
    }
  }
}

// act'(p) for dp = dy act'(p).
template <typename T>
__device__ __forceinline__ float act_slope(float a) {
  const float z = sigmoid<T>(a);
  return z * fmaf(a, 1.f - z, 1.f);
}

constexpr int kCausalRows = 8;  // strips of a block in the backward pass

template <typename T, int V, int K>
__global__ void __launch_bounds__(kCausalThreads, V > 1 ? 2 : 3) causal_backward(CausalParams p) {
  __shared__ float part[kCausalRows / 2][K + 1][32 * V];
  constexpr int H = (V + 1) / 2, U = 8;
  using Row = Vec<T, V>;
  const int nvec = p.channels / V;
  const int across = (nvec + 31) / 32;
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int cv = static_cast<int>(blockIdx.x % across) * 32 + lane;
  const int block_row = blockIdx.x / across;
  const long long strip = static_cast<long long>(block_row) * kCausalRows + row;
  const int batch = static_cast<int>(strip / p.strips);
  const int c = cv * V;
  float dw[K][V] = {}, db[V] = {};
  if (cv < nvec && batch < p.batch) {
    const int t0 = static_cast<int>(strip % p.strips) * p.strip;
    const int t1 = min(t0 + p.strip, p.tokens);
    const int last = t1 + K - 1, there = min(last, p.tokens);  // tokens past the strip only finish its last dx
    const T* x = static_cast<const T*>(p.x) + batch * p.x_batch;
    const T* x_at = x + t0 * p.x_token + c;
    const T* dy_at = static_cast<const T*>(p.dy) + batch * p.dy_batch + t0 * p.dy_token + c;
    T* dx = static_cast<T*>(p.dx) + (static_cast<long long>(batch) * p.tokens + t0) * p.channels + c;
    Row ring[U], dy_ring[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (t0 + i < there) {
        ring[i] = *reinterpret_cast<const Row*>(x_at);
        dy_ring[i] = *reinterpret_cast<const Row*>(dy_at);
      }
      x_at += p.x_token;
      dy_at += p.dy_token;
    }
    Pair w[K][H], b[H], seen[K][H], ahead[K][H], gw[K][H], gb[H];  // ahead[j]: dx of token t - K + 1 + j so far
    const Pair zero = pair(0.f, 0.f), ones = pair(1.f, 1.f);
    {
      float wf[K][V], bf[V];
      load_filter<T, V, K>(p, c, wf, bf);
      as_pair_array(bf, b);
#pragma unroll
      for (int j = 0; j < K; ++j) as_pair_array(wf[j], w[j]);
#pragma unroll
      for (int v = 0; v < H; ++v) {
        gb[v] = zero;
#pragma unroll
        for (int j = 0; j < K; ++j) seen[j][v] = ahead[j][v] = gw[j][v] = zero;
      }
    }
    SequenceWalk s;
    s.begin(p, batch, t0);
    const auto refill = [&](int t) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        float f[V];
        input_before<T, V, K>(p, x, s, t, K - 1 - j, c, f);
        as_pair_array(f, seen[j + 1]);
      }
    };
    // gradient of one token that is in a sequence, without what the state after it gives
    const auto one = [&](const Row& row, const Row& grad, bool own, int reach) {
      float in[V], up_in[V];
      unpack(row, in);
      unpack(grad, up_in);
      as_pair_array(in, seen[K - 1]);
      if (p.silu) {
        Pair a[H];
        float f[V];
#pragma unroll
        for (int v = 0; v < H; ++v) {
          a[v] = b[v];
#pragma unroll
          for (int j = 0; j < K; ++j) a[v] = fma2(w[j][v], seen[j][v], a[v]);
        }
        as_float_array(a, f);
#pragma unroll
        for (int v = 0; v < V; ++v) up_in[v] *= act_slope<T>(f[v]);
      }
      Pair g[H];
      as_pair_array(up_in, g);
#pragma unroll
      for (int v = 0; v < H; ++v) {
        if (own) {
#pragma unroll
          for (int j = 0; j < K; ++j) gw[j][v] = fma2(g[v], seen[j][v], gw[j][v]);
          gb[v] = fma2(g[v], ones, gb[v]);
        }
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (K - 1 - j <= reach) ahead[j][v] = fma2(w[j][v], g[v], ahead[j][v]);
      }
    };
    const auto shift = [&](const float (&give)[V]) {
#pragma unroll
      for (int v = 0; v < H; ++v)
#pragma unroll
        for (int j = 0; j < K - 1; ++j) seen[j][v] = seen[j + 1][v], ahead[j][v] = ahead[j + 1][v];
      as_pair_array(give, ahead[K - 1]);
    };
    const auto emit = [&]() {
      float out[V];
      as_float_array(ahead[0], out);
      store<T, V>(dx, out);
      dx += p.channels;
    };
    const float none[V] = {};
    refill(t0);
    for (int t = t0; t < last; t += U) {
      if (s.index >= 0 && t >= t0 + K - 1 && t >= s.start + K - 1 && t + U <= t1 && t + U + K - 1 <= s.end && t + 2 * U <= there) {
#pragma unroll
        for (int i = 0; i < U; ++i) {  // eight tokens well inside a sequence and the strip, and eight more to fetch
          shift(none);
          one(ring[i], dy_ring[i], true, K - 1);
          emit();
          ring[i] = *reinterpret_cast<const Row*>(x_at);
          dy_ring[i] = *reinterpret_cast<const Row*>(dy_at);
          x_at += p.x_token;
          dy_at += p.dy_token;
        }
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int now = t + i;
          if (now >= last) break;
          if (now < p.tokens && now >= s.end) {
            s.next(p, batch, now);
            refill(now);
          }
          const bool live = now < p.tokens && s.index >= 0;
          float give[V] = {};
          if (live && p.dstate_out) {  // the state after the sequence holds this token's input
            const int r = K - 1 + now - min(s.end, p.tokens);
            if (r >= 0)
              load<T, V>(static_cast<const T*>(p.dstate_out) +
                             (static_cast<long long>(s.index) * (K - 1) + r) * p.channels + c, give);
          }
          shift(give);
          if (live) one(ring[i], dy_ring[i], now < t1, now - s.start);
          if (now - (K - 1) >= t0) emit();
          if (now + U < there) {
            ring[i] = *reinterpret_cast<const Row*>(x_at);
            dy_ring[i] = *reinterpret_cast<const Row*>(dy_at);
          }
          x_at += p.x_token;
          dy_at += p.dy_token;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < K; ++j) as_float_array(gw[j], dw[j]);
    as_float_array(gb, db);
  }
  if (!p.partial) return;
  // the block's eight strips, added pairwise in a fixed order
#pragma unroll
  for (int half = kCausalRows / 2; half >= 1; half >>= 1) {
    if (row >= half && row < 2 * half)
#pragma unroll
      for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int j = 0; j < K; ++j) part[row - half][j][lane + 32 * v] = dw[j][v];
        part[row - half][K][lane + 32 * v] = db[v];
      }
    __syncthreads();
    if (row < half)
#pragma unroll
      for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int j = 0; j < K; ++j) dw[j][v] += part[row][j][lane + 32 * v];
        db[v] += part[row][K][lane + 32 * v];
      }
    __syncthreads();
  }
  if (row == 0 && cv < nvec) {
    float* out = p.partial + static_cast<long long>(block_row) * (K + 1) * p.channels + c;
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) out[static_cast<long long>(j) * p.channels + v] = dw[j][v];
#pragma unroll
    for (int v = 0; v < V; ++v) out[static_cast<long long>(K) * p.channels + v] = db[v];
  }
}

// dw [C, K] and db [C] from the blocks' partial sums, in block order within
// each of eight interleaved parts, the parts pairwise.
template <typename T>
__global__ void __launch_bounds__(256) causal_reduce(const float* partial, int blocks, int channels, int K, T* dw, T* db) {
  __shared__ float part[8][33];
  const long long at = static_cast<long long>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const long long count = static_cast<long long>(K + 1) * channels;
  const int row = threadIdx.x >> 5;
  float sum = 0.f;
  if (at < count)
    for (int i = row; i < blocks; i += 8) sum += partial[i * count + at];
  part[row][threadIdx.x & 31] = sum;
  __syncthreads();
  if (row || at >= count) return;
  const int l = threadIdx.x;
  sum = ((part[0][l] + part[1][l]) + (part[2][l] + part[3][l])) + ((part[4][l] + part[5][l]) + (part[6][l] + part[7][l]));
  const int j = static_cast<int>(at / channels), c = static_cast<int>(at % channels);
  if (j < K) {
    if (dw) dw[static_cast<long long>(c) * K + j] = down<T>(sum);
  } else if (db) {
    db[c] = down<T>(sum);
  }
}

// Gradient of the state before a sequence: its rows are the inputs of the
// first K - 1 tokens' taps, and stay in the state after it where fewer than
// K - 1 tokens follow.
template <typename T, int K>
__global__ void __launch_bounds__(256) causal_state_gradient(CausalParams p) {
  const long long item = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int n = static_cast<int>(item / p.channels), c = static_cast<int>(item % p.channels);
  if (n >= p.sequences) return;
  int lo = 0, len = p.tokens;
  if (p.cu) {
    lo = clamp_token(p.cu[n], p.tokens);
    len = max(clamp_token(p.cu[n + 1], p.tokens) - lo, 0);
  }
  const T* x = static_cast<const T*>(p.x) + (p.cu ? 0 : n * p.x_batch);
  const T* dy = static_cast<const T*>(p.dy) + (p.cu ? 0 : n * p.dy_batch);
  SequenceWalk s{n, lo, lo + len};
  float w[K][1], b[1], grad[K - 1] = {};
  load_filter<T, 1, K>(p, c, w, b);
#pragma unroll
  for (int l = 0; l < K - 1; ++l) {
    if (l >= len) break;
    float g = up(dy[(lo + l) * p.dy_token + c]);
    if (p.silu) {
      float a = b[0];
#pragma unroll
      for (int j = 0; j < K; ++j) {
        float f[1];
        input_before<T, 1, K>(p, x, s, lo + l, K - 1 - j, c, f);
        a = fmaf(w[j][0], f[0], a);
      }
      g *= act_slope<T>(a);
    }
#pragma unroll
    for (int i = 0; i < K - 1; ++i)
      if (i >= l) grad[i] = fmaf(w[i - l][0], g, grad[i]);
  }
#pragma unroll
  for (int i = 0; i < K - 1; ++i) {
    const long long row = static_cast<long long>(n) * (K - 1);
    if (p.dstate_out && i >= len)
      grad[i] += up(static_cast<const T*>(p.dstate_out)[(row + i - len) * p.channels + c]);
    static_cast<T*>(p.dstate_in)[(row + i) * p.channels + c] = down<T>(grad[i]);
  }
}

// One more token: y from the state's K - 1 rows and x, then the state moves up
// by one row in place.  One thread holds all rows of its channels, so the
// shift needs no second buffer.  x [n, C], state [n, K - 1, C].
template <typename T, int V, int K>
__global__ void __launch_bounds__(128) causal_step(const T* x, long long x_row, T* state, long long state_row, CausalParams p) {
  const int nvec = p.channels / V;
  const long long item = static_cast<long long>(blockIdx.x) * 128 + threadIdx.x;
  const long long n = item / nvec;
  if (n >= p.batch) return;
  const int c = static_cast<int>(item % nvec) * V;
  Vec<T, V> rows[K];
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
    rows[j] = *reinterpret_cast<const Vec<T, V>*>(state + n * state_row + static_cast<long long>(j) * p.channels + c);
  rows[K - 1] = *reinterpret_cast<const Vec<T, V>*>(x + n * x_row + c);
  float w[K][V], b[V], out[V];
  load_filter<T, V, K>(p, c, w, b);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float a = b[v];
#pragma unroll
    for (int j = 0; j < K; ++j) a = fmaf(w[j][v], up(rows[j].e[v]), a);
    out[v] = p.silu ? a * sigmoid<T>(a) : a;
  }
  store<T, V>(static_cast<T*>(p.y) + n * p.channels + c, out);
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
    *reinterpret_cast<Vec<T, V>*>(state + n * state_row + static_cast<long long>(j) * p.channels + c) = rows[j + 1];
}

}  // namespace seq
}  // namespace pla
