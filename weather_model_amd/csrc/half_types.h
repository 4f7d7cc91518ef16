// half_types.h -- 16-bit element types and their conversions (round to nearest even), vector views that
// need no more than the element's alignment (the hardware takes such global accesses at any address).
#pragma once

#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <class T> struct Vec4 { typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T)))); };

template <class T> __device__ __forceinline__ float to_float(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T from_float(float v) { return (T)v; }

// four consecutive elements from float32, one rounding each
template <class T> __device__ __forceinline__ void store4(T *p, f32x4 v)
{
    *reinterpret_cast<typename Vec4<T>::type *>(p) = __builtin_convertvector(v, typename Vec4<T>::type);
}
