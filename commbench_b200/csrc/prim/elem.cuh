// Element types of the row operators (norm, rotary positions): vectors of up to 16 bytes in memory, fp32 in
// registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace cb {

enum ElemType : int { ELEM_BF16 = 0, ELEM_F16 = 1, ELEM_F32 = 2 };

__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }

// V consecutive elements, aligned to their size together: as 32-bit words while they wait (an array of 16-bit
// elements takes a register each), as fp32 for arithmetic.
template <class T, int V, bool kWords = (sizeof(T) * V >= 4)>
struct Vec;
template <class T, int V>
struct alignas(sizeof(T) * V) Vec<T, V, true> {
  uint32_t w[sizeof(T) * V / 4];
};
template <class T, int V>
struct alignas(sizeof(T) * V) Vec<T, V, false> {
  T e[V];
};
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (__is_same(T, __nv_bfloat16))
      return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else
      return __half22float2(*reinterpret_cast<const __half2*>(&w));
  } else {
    return make_float2(0.f, 0.f);
  }
}
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (__is_same(T, __nv_bfloat16)) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <class T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V>& v, float (&x)[V]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = __uint_as_float(v.w[i]);
  } else if constexpr (V == 1) {
    x[0] = to_f32(v.e[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 f = unpack2<T>(v.w[i / 2]);
      x[i] = f.x;
      x[i + 1] = f.y;
    }
  }
}
template <class T, int V>
__device__ __forceinline__ void pack(const float (&x)[V], Vec<T, V>& v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) v.w[i] = __float_as_uint(x[i]);
  } else if constexpr (V == 1) {
    v.e[0] = from_f32<T>(x[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) v.w[i / 2] = pack2<T>(x[i], x[i + 1]);
  }
}
template <class T, int V>
__device__ __forceinline__ void clear(Vec<T, V>& v) {
  if constexpr (sizeof(T) * V >= 4) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) * V / 4; ++i) v.w[i] = 0u;
  } else {
    v.e[0] = from_f32<T>(0.f);
  }
}
template <class T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[V]) {
  unpack(*reinterpret_cast<const Vec<T, V>*>(p), x);
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[V]) {
  Vec<T, V> v;
  pack(x, v);
  *reinterpret_cast<Vec<T, V>*>(p) = v;
}

// Two fp32 numbers in one register pair: half the instructions of kernels that are bound by issuing them.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 f2_parts(uint64_t a) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(a));
  return f;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Two sums over a warp in six shuffles: the lower lanes go on with the first, the upper ones with the second.
__device__ __forceinline__ float2 warp_sum2(float a, float b) {
  const bool up = (threadIdx.x & 16u) != 0u;
  float x = (up ? b : a) + __shfl_xor_sync(0xffffffffu, up ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  const float y = __shfl_xor_sync(0xffffffffu, x, 16);
  return up ? make_float2(y, x) : make_float2(x, y);
}

}  // namespace cb
