// Rows one by one, for results that are not finite.
//
// A matrix product takes in every key of a tile: one that a row does not see has p = 0, but 0 times a NaN or an infinity in
// that key's V is NaN.  Testing every tile for that would cost each call what nearly none needs, so the results are
// tested: a row whose sums are not finite though its inputs are is worked out again from what it sees and nothing else.
// Where something that the row does see is not finite, the result is left as it is: that search ends at the
// first such element, so a model that has diverged costs little more than one that has not.
// Lane l holds the elements 2l, 2l + 1 of a row.
#pragma once
#include "attention.hpp"

namespace gearhip {

struct Pair {
  float x, y;
};

template <typename T>
__device__ __forceinline__ Pair load_pair(const T *row, int dim) {
  typedef T two __attribute__((ext_vector_type(2)));
  const int d = 2 * lane_id();
  if (d >= dim) return Pair{0.f, 0.f};
  const two v = *reinterpret_cast<const two *>(row + d);
  return Pair{(float)v[0], (float)v[1]};
}
template <typename T>
__device__ __forceinline__ void store_pair(T *row, Pair v, int dim) {
  typedef T two __attribute__((ext_vector_type(2)));
  const int d = 2 * lane_id();
  if (d < dim) *reinterpret_cast<two *>(row + d) = two{(T)v.x, (T)v.y};
}
__device__ __forceinline__ bool finite_pair(Pair v) {
  return wave_ballot(!(fabsf(v.x) < INFINITY) || !(fabsf(v.y) < INFINITY)) == 0;
}
__device__ __forceinline__ float dot(Pair a, Pair b) {
  float s = a.x * b.x + a.y * b.y;
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) s += __shfl_xor(s, m);
  return s;
}
__device__ __forceinline__ float lane_value(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// Whether any of a lane's sums is not finite.
template <int N>
__device__ __forceinline__ bool not_finite(const f32x16 (&x)[N]) {
  float t = 0;
#pragma unroll
  for (int b = 0; b < N; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) t = fmaf(x[b][r], 0.f, t);
  return t != 0.f || t != t;
}
// The same of a wave whose lanes l and l + 32 share a column: a bit a column.
template <int N>
__device__ __forceinline__ uint32_t columns_not_finite(const f32x16 (&x)[N], bool count) {
  const uint64_t bad = wave_ballot(count && not_finite(x));
  return (uint32_t)bad | (uint32_t)(bad >> 32);
}

// Whether rows [lo, hi) are finite, 16 loads at a time.
template <typename T>
__device__ __forceinline__ bool rows_finite(const T *rows, int64_t stride, int lo, int hi, int dim) {
  for (int j = lo; j < hi; j += 16) {
    Pair sum = {0.f, 0.f};
#pragma unroll
    for (int y = 0; y < 16; ++y) {
      const Pair x = load_pair(rows + min(j + y, hi - 1) * stride, dim);
      sum.x = fmaf(x.x, 0.f, sum.x), sum.y = fmaf(x.y, 0.f, sum.y);
    }
    if (!finite_pair(sum)) return false;
  }
  return true;
}

// One row of the forward pass.  lse_log2: of the row.  False: left alone.
template <typename T, int MODE>
__device__ __forceinline__ bool exact_out(Pair &out, const T *q, const T *k, int64_t k_stride, const T *v, int64_t v_stride, int lo,
                                          int hi, int dim, int place, float lse_log2, const Scores<MODE> &scores) {
  if (!(fabsf(lse_log2) < INFINITY) || !rows_finite(v, v_stride, lo, hi, dim)) return false;
  const Pair own = load_pair(q, dim);
  out = Pair{0.f, 0.f};
  for (int j = lo; j < hi; ++j) {
    const float z = scores.z(scores.capped(dot(own, load_pair(k + j * k_stride, dim))), (float)(place - j));
    const float p = exp2_fast(fmaf(z, scores.factor, scores.offset - lse_log2));
    const Pair x = load_pair(v + j * v_stride, dim);
    out.x += p * x.x, out.y += p * x.y;
  }
  return true;
}

// p and the gradient of the score of one pair
template <int MODE>
__device__ __forceinline__ float2 exact_pair(float product, float dp, int distance, float lse_log2, float delta, const Scores<MODE> &scores) {
  const float x = scores.capped(product);
  const float p = exp2_fast(fmaf(scores.z(x, (float)distance), scores.factor, scores.offset - lse_log2));
  return make_float2(p, p * (dp - delta) * scores.shrink(x));
}

// One row of dq, without the scale.
template <typename T, int MODE>
__device__ __forceinline__ bool exact_dq(Pair &dq, const T *q, const T *dout, const T *k, int64_t k_stride, const T *v, int64_t v_stride,
                                         int lo, int hi, int dim, int place, float lse_log2, float delta, const Scores<MODE> &scores) {
  if (!(fabsf(lse_log2) < INFINITY) || !(fabsf(delta) < INFINITY) || !rows_finite(k, k_stride, lo, hi, dim)) return false;
  const Pair own = load_pair(q, dim), g = load_pair(dout, dim);
  dq = Pair{0.f, 0.f};
  for (int j = lo; j < hi; ++j) {
    const Pair x = load_pair(k + j * k_stride, dim);
    const float ds = exact_pair(dot(own, x), dot(g, load_pair(v + j * v_stride, dim)), place - j, lse_log2, delta, scores).y;
    dq.x += ds * x.x, dq.y += ds * x.y;
  }
  return true;
}

}  // namespace gearhip
