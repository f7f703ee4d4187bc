// 16-bit types, the matrix instructions on them and the layouts those leave their results in (gfx950).
#pragma once
#include "wave.hpp"

namespace gearhip {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <typename T>
using vec4 = T __attribute__((ext_vector_type(4)));
template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

// 8 elements of a row, as 32-bit floats and back (rounded to nearest)
template <typename T>
struct Row8 {
  vec8<T> v;
  __device__ __forceinline__ void load(const T *p) { v = *reinterpret_cast<const vec8<T> *>(p); }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<vec8<T> *>(p) = v; }
  __device__ __forceinline__ f32x8 floats() const { return __builtin_convertvector(v, f32x8); }
  __device__ __forceinline__ void set(f32x8 x) { v = __builtin_convertvector(x, vec8<T>); }
};
template <>
struct Row8<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float *p) {
    a = *reinterpret_cast<const f32x4 *>(p);
    b = *reinterpret_cast<const f32x4 *>(p + 4);
  }
  __device__ __forceinline__ void store(float *p) const {
    *reinterpret_cast<f32x4 *>(p) = a;
    *reinterpret_cast<f32x4 *>(p + 4) = b;
  }
  __device__ __forceinline__ f32x8 floats() const { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
  __device__ __forceinline__ void set(f32x8 x) {
    a = __builtin_shufflevector(x, x, 0, 1, 2, 3);
    b = __builtin_shufflevector(x, x, 4, 5, 6, 7);
  }
};

}  // namespace gearhip
