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

}  // namespace gearhip
