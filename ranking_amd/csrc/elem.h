// Element types and vector accesses of the kernels that take fp32, bf16 and fp16 tensors (embedding.hip,
// token_logprob.hip, adamw.hip).  Arithmetic is fp32 throughout: values are widened as they are read and rounded once,
// to nearest even, as they are written.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/tfr_hip.h"

namespace tfr {

template <int DTYPE> struct ElemOf;
template <> struct ElemOf<TFR_DTYPE_F32> { typedef float type; };
template <> struct ElemOf<TFR_DTYPE_BF16> { typedef __bf16 type; };
template <> struct ElemOf<TFR_DTYPE_F16> { typedef _Float16 type; };

inline int elem_bytes(int dtype) { return dtype == TFR_DTYPE_F32 ? 4 : 2; }
inline bool elem_known(int dtype) { return dtype == TFR_DTYPE_F32 || dtype == TFR_DTYPE_BF16 || dtype == TFR_DTYPE_F16; }

// E consecutive elements; E * sizeof(T) is 2, 4, 8 or 16 bytes and the address a multiple of it.
template <typename T, int E> struct Pack { typedef T type __attribute__((ext_vector_type(E))); };
template <typename T> struct Pack<T, 1> { typedef T type; };

template <typename T, int E>
__device__ __forceinline__ typename Pack<T, E>::type load_raw(const T* __restrict__ p) {
  return *reinterpret_cast<const typename Pack<T, E>::type*>(p);
}

// The same of what is read once and is larger than the caches.
template <typename T, int E>
__device__ __forceinline__ typename Pack<T, E>::type load_raw_stream(const T* __restrict__ p) {
  return __builtin_nontemporal_load(reinterpret_cast<const typename Pack<T, E>::type*>(p));
}

template <typename T, int E>
__device__ __forceinline__ void widen(const typename Pack<T, E>::type x, float (&v)[E]) {
  if constexpr (E == 1) {
    v[0] = (float)x;
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = (float)x[i];
  }
}

template <typename T, int E>
__device__ __forceinline__ void load_pack(const T* __restrict__ p, float (&v)[E]) {
  widen<T, E>(load_raw<T, E>(p), v);
}

template <typename T, int E>
__device__ __forceinline__ typename Pack<T, E>::type narrow(const float (&v)[E]) {
  typename Pack<T, E>::type x;
  if constexpr (E == 1) {
    x = (T)v[0];
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = (T)v[i];
  }
  return x;
}

template <typename T, int E>
__device__ __forceinline__ void store_pack(T* __restrict__ p, const float (&v)[E]) {
  *reinterpret_cast<typename Pack<T, E>::type*>(p) = narrow<T, E>(v);
}

// The same past the caches, for results that are larger than them.
template <typename T, int E>
__device__ __forceinline__ void store_pack_stream(T* __restrict__ p, const float (&v)[E]) {
  __builtin_nontemporal_store(narrow<T, E>(v), reinterpret_cast<typename Pack<T, E>::type*>(p));
}

}  // namespace tfr
