// Rows of any width, stride and alignment, 16 bytes a lane, and sums and maxima over the lanes of a row (gfx950).
#pragma once
#include <type_traits>

#include "half.hpp"

namespace gearhip {

template <typename T>
constexpr int kPer = 16 / sizeof(T);  // elements of a vector
template <typename T>
using Raw = T __attribute__((ext_vector_type(16 / sizeof(T))));
template <typename T>
using Vals = float __attribute__((ext_vector_type(16 / sizeof(T))));

// A vector at any element's address: still one load of 16 bytes (unaligned access is enabled).
template <typename T>
struct __attribute__((packed, aligned(alignof(T)))) AnyRaw {
  Raw<T> v;
};

// Where vector v of a row lies, if the row begins `shift` elements behind a multiple of 16 bytes and vectors lie at such
// multiples.  Those at both ends, partial in general, are moved inside the row, so that each is one load: the elements
// [skip, end) are a vector's own, the others another one's.
template <typename T>
struct Slot {
  int col, skip, end;
  Slot() = default;
  __device__ __forceinline__ Slot(int c, int s, int e) : col(c), skip(s), end(e) {}
  __device__ __forceinline__ Slot(int v, int width) {
    const int at = v * kPer<T>;
    col = at + kPer<T> <= width ? at : width - kPer<T> < 0 ? 0 : width - kPer<T>;
    skip = at < width ? at - col : kPer<T>;
    end = width - col < kPer<T> ? width - col : kPer<T>;
    if (at >= width) col = 0;
  }
  static __device__ __forceinline__ Slot shifted(int v, int width, int shift) {
    const int at = v * kPer<T> - shift, lo = max(at, 0), hi = min(at + kPer<T>, width);
    const int c = max(min(at, width - kPer<T>), 0);
    return lo < hi ? Slot(c, lo - c, hi - c) : none();
  }
  static __device__ __forceinline__ Slot none() { return Slot(0, kPer<T>, 0); }
  __device__ __forceinline__ bool any() const { return skip < kPer<T>; }
  __device__ __forceinline__ bool whole() const { return skip == 0 && end == kPer<T>; }
  __device__ __forceinline__ bool own(int e) const { return e >= skip && e < end; }
};
// elements from the multiple of 16 bytes before
template <typename T>
__device__ __forceinline__ int misaligned(const T *p) {
  return (int)(reinterpret_cast<uintptr_t>(p) / sizeof(T)) & (kPer<T> - 1);
}

// tiny: the row is narrower than a vector
template <typename T>
__device__ __forceinline__ Raw<T> load_slot(const T *row, const Slot<T> &s, bool tiny) {
  if (tiny) {
    Raw<T> x = {};
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e)
      if (e < s.end) x[e] = row[s.col + e];
    return x;
  }
  return reinterpret_cast<const AnyRaw<T> *>(row + s.col)->v;
}
template <typename T>
__device__ __forceinline__ void store_slot(T *row, const Slot<T> &s, const Vals<T> &x) {
  const Raw<T> y = __builtin_convertvector(x, Raw<T>);
  if (s.whole()) {
    reinterpret_cast<AnyRaw<T> *>(row + s.col)->v = y;
  } else {
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e)
      if (s.own(e)) row[s.col + e] = y[e];
  }
}

// The same for rows whose width is a multiple of a vector (kWhole): nothing of theirs is partial.
template <bool kWhole, typename T>
struct Place : Slot<T> {
  __device__ __forceinline__ Place(int v, int width) : Slot<T>(v, width) {}
};
template <typename T>
struct Place<true, T> {
  int col;
  bool here;
  __device__ __forceinline__ Place(int v, int width) : col(v * kPer<T>), here(v * kPer<T> < width) {}
  __device__ __forceinline__ bool any() const { return here; }
  __device__ __forceinline__ bool whole() const { return true; }
  __device__ __forceinline__ bool own(int) const { return here; }
};
template <typename T>
__device__ __forceinline__ Raw<T> load_slot(const T *row, const Place<true, T> &s, bool) {
  return reinterpret_cast<const AnyRaw<T> *>(row + s.col)->v;
}
template <typename T>
__device__ __forceinline__ void store_slot(T *row, const Place<true, T> &s, const Vals<T> &x) {
  reinterpret_cast<AnyRaw<T> *>(row + s.col)->v = __builtin_convertvector(x, Raw<T>);
}

// A vector as it came, from here on: the compiler may not keep what it made of it earlier in its place (which takes two to
// four times the registers).
template <typename T>
__device__ __forceinline__ void as_it_came(Raw<T> &x) {
  u32x4 y = __builtin_bit_cast(u32x4, x);
  asm volatile("" : "+v"(y));
  x = __builtin_bit_cast(Raw<T>, y);
}

// kOnce: data that nobody reads again soon, passed by the caches (a load or store of 16 bytes at any element's address).
template <bool kOnce, typename T>
__device__ __forceinline__ Raw<T> load_raw(const T *p) {
  if (kOnce) return __builtin_bit_cast(Raw<T>, __builtin_nontemporal_load(reinterpret_cast<const u32x4_a1 *>(p)));
  return reinterpret_cast<const AnyRaw<T> *>(p)->v;
}
template <bool kOnce, typename T>
__device__ __forceinline__ void store_raw(T *p, const Raw<T> &x) {
  if (kOnce)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, x), reinterpret_cast<u32x4_a1 *>(p));
  else
    reinterpret_cast<AnyRaw<T> *>(p)->v = x;
}

// Its elements in 32 bits.  (bfloat16 by its bits: a maximum of two numbers that the compiler knows to have been bfloat16 is
// taken in that type, which gfx950 has no instruction for, and costs a conversion back and forth.)
template <typename T>
__device__ __forceinline__ Vals<T> values_of(const Raw<T> &x) {
  if constexpr (std::is_same<T, bf16>::value) {
    const u32x4 y = __builtin_bit_cast(u32x4, x);
    Vals<T> v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(y[i] << 16), v[2 * i + 1] = __uint_as_float(y[i] & 0xffff0000u);
    return v;
  } else {
    return __builtin_convertvector(x, Vals<T>);
  }
}

// ---- over the kLanes lanes of a row (a power of two, at most 64), the result in all of them ----------------------
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int kLanes, typename F>
__device__ __forceinline__ float over_lanes(float x, const F &f) {
  if (kLanes > 1) x = f(x, dpp_f32<0xB1>(x));   // lanes 1 apart
  if (kLanes > 2) x = f(x, dpp_f32<0x4E>(x));   // 2 apart
  if (kLanes > 4) x = f(x, dpp_f32<0x141>(x));  // the other half of 8
  if (kLanes > 8) x = f(x, dpp_f32<0x140>(x));  // the other half of 16
  if (kLanes > 16) {
    const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(y[0]), __uint_as_float(y[1]));
  }
  if (kLanes > 32) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(y[0]), __uint_as_float(y[1]));
  }
  return x;
}
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float x) {
  return over_lanes<kLanes>(x, [](float a, float b) __attribute__((always_inline)) { return a + b; });
}
template <int kLanes>
__device__ __forceinline__ float lanes_max(float x) {
  return over_lanes<kLanes>(x, [](float a, float b) __attribute__((always_inline)) { return fmaxf(a, b); });
}

__device__ __forceinline__ float sum_of(const f32x4 &x) { return (x[0] + x[1]) + (x[2] + x[3]); }
__device__ __forceinline__ float sum_of(const f32x8 &x) {
  return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

// Tokens come in 32 or 64 bits; what is outside [0, vocab) is none: -1.
__device__ __forceinline__ int64_t token_at(const void *tokens, int wide, int64_t i, int64_t vocab) {
  const int64_t t = wide ? static_cast<const int64_t *>(tokens)[i] : static_cast<const int32_t *>(tokens)[i];
  return t >= 0 && t < vocab ? t : -1;
}

// f(T()) for an element type of the C ABI
template <typename F>
inline void by_type(int dtype, const F &f) {
  if (dtype == GEAR_HIP_F32)
    f(float());
  else if (dtype == GEAR_HIP_F16)
    f(f16());
  else
    f(bf16());
}
inline int element_bytes(int dtype) { return dtype == GEAR_HIP_F32 ? 4 : dtype == GEAR_HIP_F16 || dtype == GEAR_HIP_BF16 ? 2 : 0; }
inline bool aligned_to(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

}  // namespace gearhip
