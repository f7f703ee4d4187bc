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
// Rows lie in LDS as 16-byte pieces; piece c of row r at c ^ swizzle(r), so that the pieces of 8 consecutive rows, and
// the transposing read of 2 pieces of 4 rows, lie in different banks (rows of 128 elements: in half of all banks).
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

// Which column of a tile the row r of operand `block` is.  With rows of 128 elements a block is two runs of 16 columns 64 apart: 32
// next to each other lie in half of the banks.
template <int D>
constexpr int column_of(int block, int r) {
  return D == 128 ? 16 * block + r % 16 + 64 * (r / 16) : 32 * block + r;
}
// Operands out of a tile, by offsets that a lane works out once: what remains of an address is a constant of the
// instruction.  (swizzle() of a row is the same for rows a multiple of 8 apart, and changes the lower 3 bits of a
// piece only.)
//   rows     the operand whose row (or column) l%32 is row first + l%32 of the tile, contracted over the elements 16 s..
//   columns  the operand whose row l%32 is column `column_of<D>(block, l%32)`, contracted over the rows
//            first..first + 15 in the order above
template <typename T, int D>
struct TileReader {
  static constexpr int kRowOffsets = D / 16 < 4 ? D / 16 : 4, kColumnOffsets = D / 32, kColumnPieces = D == 128 ? 2 : 4;
  int row[kRowOffsets], column[kColumnOffsets];  // elements
  __device__ __forceinline__ TileReader() {
    const int l = lane_id(), half = l >> 5, t = l & 15;
#pragma unroll
    for (int s = 0; s < kRowOffsets; ++s) row[s] = piece_at<D>(l & 31, 2 * s + half);
#pragma unroll
    for (int b = 0; b < kColumnOffsets; ++b)
      column[b] = piece_at<D>(4 * half + (t >> 2), kColumnPieces * b + (D == 128 ? 8 : 2) * ((l >> 4) & 1) + ((t & 3) >> 1)) + 4 * (t & 1);
  }
  // (first: a multiple of 8)
  __device__ __forceinline__ vec8<T> rows(const T *tile, int first, int s) const {
    return *reinterpret_cast<const vec8<T> *>(tile + row[s % kRowOffsets] + first * D + s / kRowOffsets * 64);
  }
  // (first: a multiple of 16)
  __device__ __forceinline__ vec8<T> columns(const T *tile, int first, int block) const {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    auto read = [&](int r) {
      const T *p = tile + column[block] + r * D;
      return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(const_cast<T *>(p)));
    };
    const s16x4 a = read(first), b = read(first + 8);
    return __builtin_bit_cast(vec8<T>, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// 8 neighbouring results as an operand of the next product (in pairs: one instruction rounds two)
template <typename T, int U>
__device__ __forceinline__ vec8<T> packed(const f32x16 &x) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef T pair __attribute__((ext_vector_type(2)));
  vec8<T> y;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const pair z = __builtin_convertvector((f32x2){x[8 * U + 2 * e], x[8 * U + 2 * e + 1]}, pair);
    y[2 * e] = z[0], y[2 * e + 1] = z[1];
  }
  return y;
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

// Rows of a tile of ROWS rows straight from memory into LDS, 64 pieces an instruction, the instructions dealt
// out to the waves of a workgroup.  Rows outside [first, end) are replaced by the nearest inside, pieces
// beyond `dim` by the last: what a tile holds there is finite wherever the rows in range are, and multiplied
// by zeros only.  A tile is complete after staged_wait() in every wave and a barrier.
// ONCE: what nobody reads again is loaded past the caches.
// KEYS: pieces beyond `dim` are left as clear_beyond() made them, once for all that the tile is asked for: a key's last piece may
// be infinite, and that times the zeros of a query would be NaN where the score is -inf.
// The instruction is written out because the compiler, which cannot tell the tile that is asked for from
// the one that is read meanwhile, has every read of LDS behind its builtin wait for the memory.
template <typename T, int D, int ROWS, bool ONCE = false, bool KEYS = false>
struct Stage {
  static constexpr int kPieces = D / 8, kRowsEach = kWave / kPieces, kCount = ROWS / kRowsEach;
  const T *base;
  int64_t stride;
  int first, end, dim, lane;
  int64_t offset[2];  // of the lane's piece within an even and an odd instruction's rows

  __device__ __forceinline__ Stage(const T *base, int64_t stride, int first, int end, int dim, int lane = lane_id())
      : base(base), stride(stride), first(first), end(end), dim(dim), lane(lane) {
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) offset[odd] = (lane / kPieces) * stride + piece(odd) * 8;
  }
  // (rows of an instruction differ from those of the next but one by a multiple of 8: the same swizzle)
  __device__ __forceinline__ int own_piece(int x) const { return (lane % kPieces) ^ swizzle<D>(x * kRowsEach + lane / kPieces); }
  __device__ __forceinline__ int piece(int x) const { return min(own_piece(x), dim / 8 - 1); }
  __device__ __forceinline__ void one(const T *from, uint32_t at, int x) const {
    if (KEYS && own_piece(x & 1) >= dim / 8) return;
    const uint32_t m0 = __builtin_amdgcn_readfirstlane(at);
    if (ONCE)
      asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" : : "v"(from), "s"(m0) : "memory", "m0");
    else
      asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(m0) : "memory", "m0");
  }
  // pieces beyond dim made zeros, by one wave: for the operand that has to be (once complete, or with KEYS before it is asked for)
  __device__ __forceinline__ void clear_beyond(T *tile) const {
    const int extra = kPieces - dim / 8;
    for (int x = lane_id(); x < ROWS * extra; x += kWave)
      *reinterpret_cast<vec8<T> *>(tile + piece_at<D>(x / extra, dim / 8 + x % extra)) = vec8<T>{};
  }
  // the share of wave `wave` of WAVES
  template <int WAVES>
  __device__ __forceinline__ void ask(T *tile, int row0, int wave) const {
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) T *)tile + wave * 1024;
    constexpr int kNext = WAVES * 1024;  // bytes of LDS that the waves' instructions fill together
    if (row0 >= first && row0 + ROWS <= end) {
#pragma unroll
      for (int y = 0; y < (kCount + WAVES - 1) / WAVES; ++y) {
        const int x = wave + y * WAVES;
        if ((y + 1) * WAVES > kCount && x >= kCount) break;
        one(base + (int64_t)(row0 + x * kRowsEach) * stride + ((x & 1) ? offset[1] : offset[0]), at + y * kNext, x);
      }
    } else {
#pragma unroll 1
      for (int x = wave, to = at; x < kCount; x += WAVES, to += kNext) {
        const int row = row0 + x * kRowsEach + lane / kPieces;
        one(base + (int64_t)min(max(row, first), end - 1) * stride + piece(x) * 8, to, x);
      }
    }
  }
};
// 4 bytes a lane into LDS, in the same way: lane l's to `to` + 4 l.
__device__ __forceinline__ void stage_words(const void *from, const void *to) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)const_cast<void *>(to));
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(from), "s"(m0) : "memory", "m0");
}

// All but the last `LEFT` instructions of the wave (of this kind, and the compiler's own loads and stores) are complete.
// (the builtin: the compiler then knows that its own loads have arrived too, and waits for none of them, and with
// them for what is asked for next, inside the loop)
template <int LEFT = 0>
__device__ __forceinline__ void staged_wait() {
  static_assert(LEFT < 64, "");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (LEFT & 15) | (LEFT >> 4 << 14));  // vmcnt
  asm volatile("" ::: "memory");
}

// The maximum and the sum of a lane's value and that of the lane 32 further (or before): the other half of the
// same result column.
__device__ __forceinline__ float max_of_halves(float x) {
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float sum_of_halves(float x) {
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}

// f over the 64 lanes, for an f with f(x, x) == x (lanes without a partner are given their own value)
template <typename F>
__device__ __forceinline__ int wave_reduce(int x, const F &f) {
  x = f(x, __builtin_amdgcn_update_dpp(x, x, kDppRowShr1, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, kDppRowShr2, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, kDppRowShr4, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, kDppRowShr8, 0xf, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, kDppRowBcast15, 0xa, 0xf, false));
  x = f(x, __builtin_amdgcn_update_dpp(x, x, kDppRowBcast31, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, kWave - 1);
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

// Scores as exponents of 2: factor * z + offset, where z comes from the product x of the rows.
//   plain       z = x
//   kCap        cap tanh(u), u = x scale / cap: z = -1 / (1 + e^2u), in [-1, 0], from tanh(u) = 1 - 2 / (1 + e^2u)
//   with kFar   z = tanh(u)
//   kBias       z = x scale log2(e) - slope |distance|, and with the cap the same of the capped score
// so that a plain or capped score costs no instruction for its scale: it is part of the exponent's
// multiply-add.
// The first form of the cap is off by up to 2^-22 cap however small the score is, so it is for caps up to kNearCap: 1.6e-5 at
// most, which moves p by a thirtieth of its own rounding to fp16.  kFar, for larger caps, takes tanh up to |u| = kSmall
// as u + u^3 P(u^2), with P fitted to be least off relative to tanh (0.7 units of 2^-24 at most): a score is within a few units of
// itself whatever the cap.  A tile whose arguments are all that small, as they are where the cap is far above the scores, takes
// only that.  32 x 1470: 478 + 690 + 1022 us in the three kernels at a cap of 100, 439 + 683 + 946 of the first form at 30; at a cap of 5,
// whose tiles hold both kinds of arguments, kFar took 580 forward against 431.
constexpr int kCap = 1, kBias = 2, kFar = 4;
constexpr float kNearCap = 64.f;
template <int MODE>
struct Scores {
  static constexpr float kSmall = 0.35f;
  float factor, offset, inner, outer, slope;
  // (UNIFORM: one head for the whole wave, its slope in a scalar register)
  template <bool UNIFORM = true>
  __device__ __forceinline__ Scores(const AttentionArgs &a, int head, std::bool_constant<UNIFORM> = {}) {
    const float cap_log2 = a.cap * kLog2e;
    inner = MODE & kFar ? a.scale / a.cap : MODE & kCap ? a.scale / a.cap * (2 * kLog2e) : a.scale_log2;
    outer = MODE & kFar ? cap_log2 : 2 * cap_log2;
    slope = MODE & kBias && a.slopes ? a.slopes[head] * kLog2e : 0.f;
    if (MODE & kBias && UNIFORM) slope = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(slope)));
    factor = !(MODE & kCap) ? a.scale_log2 : outer;
    if (MODE & kBias) factor = 1.f;
    offset = MODE & kCap && !(MODE & kFar) ? cap_log2 : 0.f;
  }
  static __device__ __forceinline__ float tanh_small(float u) {
    const float w = u * u;
    return fmaf(u * w, fmaf(fmaf(w, -0.0491485037f, 0.132998258f), w, -0.333326638f), u);
  }
  static __device__ __forceinline__ float tanh_any(float u) {
    const float large = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + exp2_fast(u * (2 * kLog2e))), 1.f);
    return fabsf(u) <= kSmall ? tanh_small(u) : large;
  }
  // a product made what z() and shrink() take; with kFar those of a tile before all else
  __device__ __forceinline__ float capped(float x) const {
    if (!(MODE & kCap)) return x;
    return MODE & kFar ? tanh_any(x * inner) : __builtin_amdgcn_rcpf(-1.f - exp2_fast(x * inner));
  }
  __device__ __forceinline__ void cap_far(f32x16 &x) const {
    if (!(MODE & kFar)) return;
    float most = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] *= inner;
      most = fmaxf(most, fabsf(x[r]));
    }
    if (__builtin_expect(wave_ballot(most > kSmall) == 0, 1)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = tanh_small(x[r]);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = tanh_any(x[r]);
    }
  }
  // (of an element of a tile)
  __device__ __forceinline__ float in_tile(float x) const { return MODE & kFar ? x : capped(x); }
  __device__ __forceinline__ float z(float c, float distance) const {
    if (!(MODE & kBias)) return c;
    return fmaf(c, MODE & kCap ? outer : inner, -slope * fabsf(distance));
  }
  // the derivative of the cap: 1 - tanh^2 = -4 z (1 + z)
  __device__ __forceinline__ float shrink(float c) const {
    return !(MODE & kCap) ? 1.f : MODE & kFar ? fmaf(-c, c, 1.f) : -4.f * fmaf(c, c, c);
  }
};

// The sum of p along a row: a tile's first, then with what the sum so far has no bits for carried on, so that a key with most of
// the weight does not swallow thousands that have little.
struct Sum {
  float x = 0, over = 0;
  __device__ __forceinline__ void add(float y) {
    y -= over;
    const float to = x + y;
    over = (to - x) - y;
    x = to;
  }
  __device__ __forceinline__ void scale(float by) { x *= by, over *= by; }
};

// What p is times, in exponents of 2, where it is rounded for its product with V: a maximum that is up to 2^8 behind leaves fp16 room
// for 2^7, and what is below 2^-25 of that, 2^-32 of the largest p, is lost, not 2^-25 of it: over 131071 keys 2^-15 of the weight
// at most.  (It is taken off again by the sum, which has it too.)
template <typename T>
constexpr float kLevel = std::is_same<T, f16>::value ? 7.f : 0.f;

// Workgroups go round the 8 dies: neighbours in this numbering share a die, and its cache.
__device__ __forceinline__ int same_die_index() {
  const int n = gridDim.x, per = n / 8, rest = n % 8, die = blockIdx.x % 8;
  return die * per + min(die, rest) + blockIdx.x / 8;
}

// The 32 rows of 32 * (D / 32) results that a wave holds by columns (column l%32: row l%32 of the output), rounded, to
// memory through a piece of LDS of 32 * D elements of the wave's own, 16 bytes a lane.  to(row): where a row begins, or null.
template <typename T, int D, typename F>
__device__ __forceinline__ void store_packed(T *piece, const vec8<T> (&x)[D / 32][2], int dim, const F &to) {
  const int l = lane_id(), half = l >> 5;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const vec8<T> &y = x[db][g >> 1];
      *reinterpret_cast<vec4<T> *>(piece + piece_at<D>(l & 31, column_of<D>(db, 8 * g) / 8) + 4 * half) =
          (g & 1) ? __builtin_shufflevector(y, y, 4, 5, 6, 7) : __builtin_shufflevector(y, y, 0, 1, 2, 3);
    }
  wave_lds_sync();
#pragma unroll
  for (int y = 0; y < D / 16; ++y) {
    const int at = y * kWave + l, row = at / (D / 8), c = at % (D / 8);
    T *p = to(row);
    if (p != nullptr && c * 8 < dim)
      *reinterpret_cast<vec8<T> *>(p + c * 8) = *reinterpret_cast<const vec8<T> *>(piece + piece_at<D>(row, c));
  }
}
// The same from sums, times `factor` of the column; zeros where `zero`.
template <typename T, int D, typename F>
__device__ __forceinline__ void store_rows(T *piece, f32x16 (&x)[D / 32], float factor, bool zero, int dim, const F &to) {
  vec8<T> y[D / 32][2];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[db][r] = zero ? 0.f : x[db][r] * factor;
    y[db][0] = packed<T, 0>(x[db]), y[db][1] = packed<T, 1>(x[db]);
  }
  store_packed<T, D>(piece, y, dim, to);
}

// f(std::integral_constant<int, D>(), element, std::integral_constant<int, MODE>()) for the call's type and sizes
template <typename F>
void by_attention_type(const AttentionArgs &a, int dtype, const F &f) {
  auto shape = [&](auto dim, auto type) {
    auto with = [&](auto bias) {
      constexpr int kWith = decltype(bias)::value;
      if (!(a.cap > 0))
        f(dim, type, std::integral_constant<int, kWith>());
      else if (a.cap <= kNearCap)
        f(dim, type, std::integral_constant<int, kWith | kCap>());
      else
        f(dim, type, std::integral_constant<int, kWith | kCap | kFar>());
    };
    if (a.slopes == nullptr)
      with(std::integral_constant<int, 0>());
    else
      with(std::integral_constant<int, kBias>());
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

// f(std::integral_constant<int, waves>()), 1 to 4 waves
template <typename F>
void by_waves(int waves, const F &f) {
  if (waves == 1)
    f(std::integral_constant<int, 1>());
  else if (waves == 2)
    f(std::integral_constant<int, 2>());
  else if (waves == 3)
    f(std::integral_constant<int, 3>());
  else
    f(std::integral_constant<int, 4>());
}

// Checks of what every attention call takes.  0: go on; 1: no queries; else the error.
int attention_args(const gear_hip_attention_desc *d, AttentionArgs &a);
// Whether a launch of so many workgroups can be.
inline bool launchable(int64_t workgroups, int waves) { return workgroups <= kMostItems / (waves * kWave); }
// base and strides are multiples of 16 bytes
bool rows_aligned(const void *p, const int64_t *stride, int element);

}  // namespace gearhip
