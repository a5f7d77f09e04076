// Element types of the size-generic operators (linear, policy loss, AdamW): float32, bfloat16,
// float16, with arithmetic in float32.  Conversions round to nearest even in hardware
// (v_cvt_pk_bf16_f32, v_cvt_f16_f32).
#pragma once

#include "dz_common.h"

namespace {

typedef __bf16 dz_bf16;
typedef _Float16 dz_f16;

template <typename T>
__device__ __forceinline__ float dz_to_f32(T x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T dz_from_f32(float x) { return (T)x; }

// N elements at any address the element type allows: the unaligned forms of the wide vector
// loads and stores (the hardware takes them at any alignment; an aligned address costs nothing).
template <typename T, int N>
struct DzPack { T v[N]; };

template <typename T, int N>
__device__ __forceinline__ DzPack<T, N> dz_load(const T* p) {
  DzPack<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void dz_store(T* p, const DzPack<T, N>& x) {
  __builtin_memcpy(p, &x, sizeof(x));
}

template <typename T, int N>
__device__ __forceinline__ DzPack<T, N> dz_round(const float (&x)[N]) {
  DzPack<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = (T)x[i];
  return r;
}

// Runs body(T{}) for the element type `dtype` (DZ_F32 / DZ_BF16 / DZ_F16); false if it is none.
template <class F>
bool dz_for_dtype(int dtype, F&& body) {
  switch (dtype) {
    case DZ_F32: body(float{}); return true;
    case DZ_BF16: body(dz_bf16{}); return true;
    case DZ_F16: body(dz_f16{}); return true;
    default: return false;
  }
}

inline bool dz_is_dtype(int dtype) { return dtype == DZ_F32 || dtype == DZ_BF16 || dtype == DZ_F16; }
inline int64_t dz_elem_bytes(int dtype) { return dtype == DZ_F32 ? 4 : 2; }

}  // namespace
