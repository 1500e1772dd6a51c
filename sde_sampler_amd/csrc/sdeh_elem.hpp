// Elements of fp32 / bf16 / fp16 tensors in registers, and sums over a workgroup: shared by the kernels that stream caller tensors
// (sdeh_policy.hip, sdeh_adamw.hip).
#pragma once
#include "sdeh_common.hpp"

namespace sdeh {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// V neighbours, loaded and stored as one access (V * sizeof(T) = 16 bytes, or less)
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* __restrict__ p, float (&x)[V]) {
  const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = static_cast<float>(k.v[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* __restrict__ p, const float (&x)[V]) {
  Pack<T, V> k;
#pragma unroll
  for (int i = 0; i < V; ++i) k.v[i] = static_cast<T>(x[i]);  // (to nearest even: the one rounding of an output)
  *reinterpret_cast<Pack<T, V>*>(p) = k;
}

// 16 bytes as they were loaded, and their values: loads that run ahead of their use stay in this form (a value unpacked where it is loaded is waited for
// there)
typedef unsigned Raw __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ Raw load_raw(const T* p) {
  return *reinterpret_cast<const Raw*>(p);
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw& r, float (&x)[V]) {
  const Pack<T, V> k = __builtin_bit_cast(Pack<T, V>, r);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = static_cast<float>(k.v[i]);
}

// the same past the caches, for tensors that are read and written once a pass and do not fit them
template <int B>
struct Bits;
template <>
struct Bits<16> {
  typedef Raw type;
};
template <>
struct Bits<8> {
  typedef unsigned type __attribute__((ext_vector_type(2)));
};
template <typename T, int V>
__device__ __forceinline__ void stream_in(const T* __restrict__ p, float (&x)[V]) {
  typedef typename Bits<V * sizeof(T)>::type B;
  const Pack<T, V> k = __builtin_bit_cast(Pack<T, V>, __builtin_nontemporal_load(reinterpret_cast<const B*>(p)));
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = static_cast<float>(k.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void stream_out(T* __restrict__ p, const float (&x)[V]) {
  typedef typename Bits<V * sizeof(T)>::type B;
  Pack<T, V> k;
#pragma unroll
  for (int i = 0; i < V; ++i) k.v[i] = static_cast<T>(x[i]);
  __builtin_nontemporal_store(__builtin_bit_cast(B, k), reinterpret_cast<B*>(p));
}

// one element of a tensor whose type is known at run time
__device__ __forceinline__ float load_as(const void* p, int dtype, long long i) {
  if (dtype == SDEH_F32) return static_cast<const float*>(p)[i];
  if (dtype == SDEH_BF16) return static_cast<float>(static_cast<const bf16_t*>(p)[i]);
  return static_cast<float>(static_cast<const f16_t*>(p)[i]);
}

template <typename A>
__device__ __forceinline__ A wave_sum(A x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// the sum over a workgroup of NT threads, in every thread and in an order that does not change from call to call
template <int NT, typename A>
__device__ __forceinline__ A block_sum(A x) {
  __shared__ A part[NT / 64];
  x = wave_sum(x);
  __syncthreads();  // (an earlier sum's readers are done)
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  A s = part[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) s += part[w];
  return s;
}

inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace sdeh
