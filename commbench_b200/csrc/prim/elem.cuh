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

// V consecutive elements, aligned to their size together.
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};
template <class T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[V]) {
  const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to_f32(v.e[i]);
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[V]) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.e[i] = from_f32<T>(x[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = v;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

}  // namespace cb
