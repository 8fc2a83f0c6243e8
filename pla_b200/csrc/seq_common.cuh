// Shared device helpers of the sequence operators (causal depthwise
// convolution, query / key norm with rotation, gated delta rule).
//
// Tensors are addressed as base + batch * stride + token * stride + ..., with
// 64-bit element offsets.  A ragged batch is one row of `tokens` tokens cut
// by cu_seqlens[0 .. sequences]; the entries come from device memory, so the
// kernels clamp them to [0, tokens] and never index by an unchecked one.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace pla {
namespace seq {

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }

// One rounding to the nearest value of the output type.
template <typename T> __device__ __forceinline__ T down(float v);
template <> __device__ __forceinline__ float down<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half down<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements moved by one access (V * sizeof(T) <= 16 bytes, a power of two).
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};
template <typename T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V>& v, float (&f)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {  // two at a time, from whole registers
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const uint32_t r = reinterpret_cast<const uint32_t*>(v.e)[i];
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[2 * i] = __uint_as_float(r << 16);
        f[2 * i + 1] = __uint_as_float(r & 0xffff0000u);
      } else {
        const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&r));
        f[2 * i] = g.x;
        f[2 * i + 1] = g.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = up(v.e[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&f)[V]) {
  unpack(*reinterpret_cast<const Vec<T, V>*>(p), f);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  Vec<T, V> v;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value)
        reinterpret_cast<__nv_bfloat162*>(v.e)[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      else
        reinterpret_cast<__half2*>(v.e)[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v.e[i] = down<T>(f[i]);
  }
  *reinterpret_cast<Vec<T, V>*>(p) = v;
}

// Two fp32 values in one register pair, and their fused multiply-add in one
// instruction (sm_100), each rounded once.
struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ float2 both(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
  return f;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}

__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
// V values as (V + 1) / 2 pairs (a zero behind an odd one) and back.
template <int V>
__device__ __forceinline__ void as_pair_array(const float (&f)[V], Pair (&p)[(V + 1) / 2]) {
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) p[i] = pair(f[2 * i], 2 * i + 1 < V ? f[(2 * i + 1) % V] : 0.f);
}
template <int V>
__device__ __forceinline__ void as_float_array(const Pair (&p)[(V + 1) / 2], float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) {
    const float2 g = both(p[i]);
    f[2 * i] = g.x;
    if (2 * i + 1 < V) f[(2 * i + 1) % V] = g.y;
  }
}

// 1 / (1 + e^-p).  16-bit results take the hardware's 2^x and reciprocal (2^-22
// relative each, their own rounding is 2^-12 at best; subnormal values of
// either count as 0, that is |p| above 87).
template <typename T> __device__ __forceinline__ float sigmoid(float p) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(p * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}
template <> __device__ __forceinline__ float sigmoid<float>(float p) { return 1.f / (1.f + expf(-p)); }

__device__ __forceinline__ int clamp_token(int v, int tokens) { return v < 0 ? 0 : (v > tokens ? tokens : v); }

// The sequence a token belongs to: cu[i] <= t < cu[i + 1], by bisection; -1 if none.
__device__ __forceinline__ int find_sequence(const int* cu, int sequences, int t) {
  int lo = 0, hi = sequences;  // first index in (0, sequences] with cu > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > t) hi = mid; else lo = mid + 1;
  }
  return lo < sequences && cu[lo] <= t ? lo : -1;
}

}  // namespace seq
}  // namespace pla
