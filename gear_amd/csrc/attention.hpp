// What the attention kernels share: arguments, tiles of rows in LDS, fragments, scores.
//
// The matrix instruction is 32x32x16: lane l holds of A the row l%32, of B the column l%32, in both the 8
// elements of the contracted axis that begin at 8*(l/32); of the result the column l%32 and, in element r
// of 16, the row 8*(r/4) + 4*(l/32) + r%4.
//
// Every product here is arranged so that the softmax axis of one product is the contracted axis of the
// next without a lane exchange.  Scores are worked out transposed, keys by queries, so a lane holds
// one query and 16 of 32 keys.  Which 16 contracted elements an instruction calls 0..15 is free as long
// as both operands agree: the next product takes its keys in the order 4*(l/32) + e (e < 4) and
// 8 + 4*(l/32) + e - 4, which is the order in which the lane already has them.  The other
// operand, rows of V by key, comes from LDS through the transposing read: a group of 16 lanes reads 4 rows of
// 16 elements and each lane gets a column.
//
// Rows lie in LDS as 16-byte pieces; piece c of row r at c ^ swizzle(r), so that both the reads of a
// piece of 8 consecutive rows and the transposing read of 2 pieces of 4 rows touch every bank once.
#pragma once
#include <limits.h>

#include <type_traits>

#include "half.hpp"

namespace gearhip {

struct Strides {
  int64_t batch, token, head;
};

struct AttentionArgs {
  const void *q, *k, *v;
  Strides qs, ks, vs;
  int batch, queries, keys, heads, kv_heads, dim;
  const int32_t *lo, *hi;
  const float *slopes;
  float scale;       // of the scores
  float scale_log2;  // scale * log2(e): scores are exponents of 2
  float cap;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRows = 32;  // rows (queries or keys) of a wave

__device__ __forceinline__ f32x16 mfma(vec8<f16> a, vec8<f16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(vec8<bf16> a, vec8<bf16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <int D>
__device__ __forceinline__ int swizzle(int row) {
  return D >= 64 ? ((row & 3) << 1) | ((row >> 2) & 1) : (((row >> 1) & 1) << 1) | ((row >> 2) & 1);
}
// element offset of piece c (8 elements) of a row
template <int D>
__device__ __forceinline__ int piece_at(int row, int c) {
  return row * D + ((c ^ swizzle<D>(row)) << 3);
}

// The operand whose row (or column) l%32 is row `first` + l%32 of the tile, contracted elements 16*s...
template <typename T, int D>
__device__ __forceinline__ vec8<T> rows_frag(const T *tile, int first, int s) {
  const int l = lane_id();
  return *reinterpret_cast<const vec8<T> *>(tile + piece_at<D>(first + (l & 31), 2 * s + (l >> 5)));
}

// The operand whose row l%32 is column 32*block + l%32 of the tile, contracted over the rows first..first+15
// in the order above.
template <typename T, int D>
__device__ __forceinline__ vec8<T> columns_frag(const T *tile, int first, int block) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  const int l = lane_id(), t = l & 15;
  const int row = first + 4 * (l >> 5) + (t >> 2), column = 32 * block + 16 * ((l >> 4) & 1) + 4 * (t & 3);
  auto read = [&](int r) {
    const T *p = tile + piece_at<D>(r, column >> 3) + (column & 7);
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(const_cast<T *>(p)));
  };
  const s16x4 a = read(row), b = read(row + 8);
  return __builtin_bit_cast(vec8<T>, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// 8 neighbouring results as an operand of the next product
template <typename T, int U>
__device__ __forceinline__ vec8<T> packed(const f32x16 &x) {
  const f32x8 y = U == 0 ? __builtin_shufflevector(x, x, 0, 1, 2, 3, 4, 5, 6, 7)
                         : __builtin_shufflevector(x, x, 8, 9, 10, 11, 12, 13, 14, 15);
  return __builtin_convertvector(y, vec8<T>);
}

// row of the result that element r of this lane holds
__device__ __forceinline__ int result_row(int r) { return 8 * (r >> 2) + 4 * (lane_id() >> 5) + (r & 3); }

// A 16-byte piece of a row in memory, or zeros.
template <typename T>
__device__ __forceinline__ vec8<T> piece_or_zero(const T *row, int c, bool there) {
  vec8<T> x = {};
  if (there) x = *reinterpret_cast<const vec8<T> *>(row + 8 * c);
  return x;
}

// The lane's fragments of its own row (l%32): D/16 pieces; zeros beyond `dim` and where the row is not there.
template <typename T, int D>
__device__ __forceinline__ void own_row_frags(vec8<T> (&f)[D / 16], const T *row, int dim, bool there) {
  const int h = lane_id() >> 5;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) f[s] = piece_or_zero(row, 2 * s + h, there && (2 * s + h) * 8 < dim);
}

// Rows first.. of a tile of ROWS rows on their way from memory to LDS through the registers of a
// workgroup of THREADS threads.
template <typename T, int D, int ROWS, int THREADS>
struct TileLoad {
  static constexpr int kPieces = ROWS * D / 8 / THREADS;
  vec8<T> x[kPieces];
  // there(row): whether the row is read
  template <typename F>
  __device__ __forceinline__ void load(const T *base, int64_t stride, int thread, int dim, const F &there) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int at = thread + i * THREADS, row = at / (D / 8), c = at % (D / 8);
      x[i] = piece_or_zero(base + row * stride, c, c * 8 < dim && there(row));
    }
  }
  __device__ __forceinline__ void store(T *tile, int thread) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int at = thread + i * THREADS, row = at / (D / 8), c = at % (D / 8);
      *reinterpret_cast<vec8<T> *>(tile + piece_at<D>(row, c)) = x[i];
    }
  }
};

// The value of the lane 32 further (or before): the other half of the same result column.
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

template <typename F>
__device__ __forceinline__ int wave_reduce(int x, const F &f) {
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) x = f(x, __shfl_xor(x, m));
  return __builtin_amdgcn_readfirstlane(x);
}

// The keys that the rows of a wave see: row `lane%32` those in [lo, hi).
struct Seen {
  int lo, hi;            // of the lane's row; 0, 0 if it sees nothing
  int first, end;        // of all rows together; INT_MAX, 0 if none sees anything
  int all_from, all_to;  // every row that sees something sees [all_from, all_to)
  __device__ __forceinline__ bool empty() const { return hi <= lo; }
  __device__ __forceinline__ void set(int l, int h, int keys) {
    lo = max(l, 0), hi = min(h, keys);
    const bool none = hi <= lo;
    if (none) lo = hi = 0;
    first = wave_reduce(none ? INT_MAX : lo, [](int a, int b) { return min(a, b); });
    end = wave_reduce(none ? 0 : hi, [](int a, int b) { return max(a, b); });
    all_from = wave_reduce(none ? 0 : lo, [](int a, int b) { return max(a, b); });
    all_to = wave_reduce(none ? INT_MAX : hi, [](int a, int b) { return min(a, b); });
  }
  __device__ __forceinline__ bool touches(int k0, int k1) const { return k0 < end && k1 > first; }
  __device__ __forceinline__ bool covers(int k0, int k1) const { return k0 >= all_from && k1 <= all_to; }
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh by 1 - 2 / (1 + e^2x): within 2e-7 of 1, which the cap scales like its scores
__device__ __forceinline__ float tanh_of(float x) {
  return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + exp2_fast(x * (2 * kLog2e)));
}

// A score as an exponent of 2, from the product of the rows; `shrink`: the cap's derivative there.
struct Shape {
  float scale_log2, over_cap, cap_log2, slope_log2;
  bool capped;
  __device__ __forceinline__ Shape(const AttentionArgs &a, int head)
      : scale_log2(a.scale_log2), over_cap(a.cap > 0 ? a.scale / a.cap : 0), cap_log2(a.cap * kLog2e),
        slope_log2(a.slopes ? a.slopes[head] * kLog2e : 0), capped(a.cap > 0) {}
  __device__ __forceinline__ float score(float x, int distance, float &shrink) const {
    float y = x * scale_log2;
    shrink = 1.f;
    if (capped) {
      const float t = tanh_of(x * over_cap);
      y = t * cap_log2;
      shrink = 1.f - t * t;
    }
    return y - slope_log2 * (float)abs(distance);
  }
};

// f(std::integral_constant<int, D>(), element, std::bool_constant<shaped>()) for the call's type and sizes
template <typename F>
void by_attention_type(const AttentionArgs &a, int dtype, const F &f) {
  auto shape = [&](auto dim, auto type) {
    if (a.cap > 0 || a.slopes != nullptr)
      f(dim, type, std::true_type());
    else
      f(dim, type, std::false_type());
  };
  auto dims = [&](auto type) {
    if (a.dim <= 32)
      shape(std::integral_constant<int, 32>(), type);
    else if (a.dim <= 64)
      shape(std::integral_constant<int, 64>(), type);
    else
      shape(std::integral_constant<int, 128>(), type);
  };
  if (dtype == GEAR_HIP_F16)
    dims(f16());
  else
    dims(bf16());
}

// Checks of what every attention call takes.  0: go on; 1: no queries; else the error.
int attention_args(const gear_hip_attention_desc *d, AttentionArgs &a);
// base and strides are multiples of 16 bytes
bool rows_aligned(const void *p, const int64_t *stride, int element);

}  // namespace gearhip
