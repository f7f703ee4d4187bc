// Gradients of attention over ranges of keys (gear_hip_attention_backward).
//
// With p = exp(s - lse), dp_ij = dout_i . v_j and delta_i = dout_i . out_i:
//   ds_ij = p_ij (dp_ij - delta_i) (1 - tanh^2);  dq = scale ds k;  dk = scale ds^T q;  dv = p^T dout
// Two launches, each of which works p out again, so that no sum is shared between workgroups and the same bits
// come out on every run: seven matrix products in place of five, for no atomics.
//   1. by queries (the layout of the forward pass): delta, dq, and the range that each 32 queries see
//   2. by keys: a wave holds 32 keys and passes over all queries (of all heads that share them) whose ranges
//      reach them; scores are not transposed here, a lane holds one key
// dq's delta is dout . out, which starts from out as it was stored, rounded; on the way sum_j p_ij dp_ij is summed in 32 bits for the
// second launch, which costs it next to nothing.  The difference matters where dp - delta is a small one, in rows of which one key has
// most of the weight (dq off by 1.7 % in bf16 where all rows are such): tiles where some p is above 1/2 are gone through once more
// at the end, with two products, for what they owe to it.  dq and dk are then within 0.0024 of the exact ones in bf16 (norm of the difference
// over the norm; packed, dq 0.0029 without), where the rounding of the results alone leaves 0.0017.  us of the launch with / without:
// 2 x 8193 with a bias, in half of whose heads nearly all rows are such, 450 / 413, without a bias 377 / 367, 32 x 1470 684 / 671; from 1/16 on
// 483 and 945.  The exact delta for all tiles takes a third pass, 2/7 more work.  Short windows, whose probabilities stay in
// registers, have it for nothing: one launch (below).
// p and ds are rounded to the type for their products, the sums are held in 32 bits.
// Bound by the matrix unit, the exponentials and LDS together: 2 x 8193, 16 heads of 128 over 8, packed, with a bias: 1. 432 us (three
// products), 2. 671 us (four products of twice the loads); 32 x 1470, 16 over 4, frames, a cap: 683 and 946 us.  Tiles of 32
// keys in 1., which the forward pass gains by, changed nothing here: 404 against 407, 697 against 686 us.
#include <type_traits>

#include "attention_exact.hpp"

namespace gearhip {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kTile = 64;

struct GradArgs {
  AttentionArgs a;
  const void *dout, *out;
  Strides gs;
  const float *lse;
  // left by the first launch for the second, padded to `padded` queries (those see nothing):
  float *lse_log2, *delta;  // [batch][heads][padded]; infinite and 0 where a row sees nothing
  int *lo, *hi;             // [batch][padded]; 0, 0 there
  i32x4 *bounds;            // [batch][padded / 32]: first, end, all_from, all_to (0 where a row sees nothing)
  int padded;
  void *dq, *dk, *dv;
  int blocks;      // workgroups of a head
};

// Rows i0 + r of dq, r a bit of `bad`, worked out alone (lse and delta: of the lane's row).
template <typename T, int MODE>
__device__ __forceinline__ void mend_dq(const GradArgs &g, uint32_t bad, int b, int head, int kv_head, int i0, const Seen &seen,
                                        float lse_log2, float delta, const Scores<MODE> &scores) {
  const AttentionArgs &a = g.a;
  staged_wait();  // (what was stored, before it is stored again)
  for (; bad != 0; bad &= bad - 1) {
    const int r = __builtin_ctz(bad), i = i0 + r;
    Pair x;
    if (exact_dq<T, MODE>(x, static_cast<const T *>(a.q) + b * a.qs.batch + i * a.qs.token + head * a.qs.head,
                          static_cast<const T *>(g.dout) + b * g.gs.batch + i * g.gs.token + head * g.gs.head,
                          static_cast<const T *>(a.k) + b * a.ks.batch + kv_head * a.ks.head, a.ks.token,
                          static_cast<const T *>(a.v) + b * a.vs.batch + kv_head * a.vs.head, a.vs.token, wave_read_lane(seen.lo, r),
                          wave_read_lane(seen.hi, r), a.dim, i + a.keys - a.queries, lane_value(lse_log2, r), lane_value(delta, r), scores))
      store_pair(static_cast<T *>(g.dq) + (((int64_t)b * a.queries + i) * a.heads + head) * a.dim, Pair{x.x * a.scale, x.y * a.scale}, a.dim);
  }
}

// Keys first_key + c of dk and dv, c a bit of `bad`, worked out alone, over all heads that share them.  known(head, i, lse, delta,
// lo, hi): what is known of a query.
template <typename T, int MODE, typename F>
__device__ __forceinline__ void mend_dkv(const GradArgs &g, uint32_t bad, int b, int kv_head, int first_key, const F &known) {
  const AttentionArgs &a = g.a;
  const int shared = a.heads / a.kv_heads;
  staged_wait();
  for (; bad != 0; bad &= bad - 1) {
    const int key = first_key + __builtin_ctz(bad);
    if (key >= a.keys) break;
    const Pair k = load_pair(static_cast<const T *>(a.k) + b * a.ks.batch + key * a.ks.token + kv_head * a.ks.head, a.dim);
    const Pair v = load_pair(static_cast<const T *>(a.v) + b * a.vs.batch + key * a.vs.token + kv_head * a.vs.head, a.dim);
    bool fine = finite_pair(k) && finite_pair(v);
    // (64 queries at a time by what is known of them: a gradient or a score that is not finite shows there)
    for (int head = kv_head * shared; head < (kv_head + 1) * shared && fine; ++head)
      for (int i0 = 0; i0 < a.queries && fine; i0 += kWave) {
        float lse_log2, delta;
        int lo, hi;
        known(head, min(i0 + lane_id(), a.queries - 1), lse_log2, delta, lo, hi);
        fine = wave_ballot(key >= lo && key < hi && !(fabsf(lse_log2) < INFINITY && fabsf(delta) < INFINITY)) == 0;
      }
    Pair dk = {0.f, 0.f}, dv = {0.f, 0.f};
    for (int pass = 0; pass < 2; ++pass)  // whether all that sees the key is finite; then the sums
      for (int head = kv_head * shared; head < (kv_head + 1) * shared && fine; ++head) {
        const Scores<MODE> scores(a, head);
        for (int i = 0; i < a.queries && fine; ++i) {
          float lse_log2, delta;
          int lo, hi;
          known(head, i, lse_log2, delta, lo, hi);
          if (key < lo || key >= hi) continue;
          const Pair q = load_pair(static_cast<const T *>(a.q) + b * a.qs.batch + i * a.qs.token + head * a.qs.head, a.dim);
          const Pair d = load_pair(static_cast<const T *>(g.dout) + b * g.gs.batch + i * g.gs.token + head * g.gs.head, a.dim);
          if (pass == 0) {
            fine = finite_pair(q) && finite_pair(d);
          } else {
            const float2 y = exact_pair(dot(q, k), dot(d, v), i + a.keys - a.queries - key, lse_log2, delta, scores);
            dv.x += y.x * d.x, dv.y += y.x * d.y;
            dk.x += y.y * q.x, dk.y += y.y * q.y;
          }
        }
      }
    if (!fine) continue;
    const int64_t to = (((int64_t)b * a.keys + key) * a.kv_heads + kv_head) * a.dim;
    store_pair(static_cast<T *>(g.dk) + to, Pair{dk.x * a.scale, dk.y * a.scale}, a.dim);
    store_pair(static_cast<T *>(g.dv) + to, dv, a.dim);
  }
}

// ds = p (dp - delta) is as large as the gradients that come in, and those may be anywhere: below 2^-24, where fp16 ends, or beyond
// 2^16.  So each column of sums (a lane's query, or its key) has ds rounded to fp16 times a power of two of its own, by which
// |dp - delta| lies below 2^15 and its largest began at 2^8..2^9 (p is at most 1): where a later tile goes beyond that, the power
// is lowered and the sums with it.  A ds is off by 2^-33 of the largest |dp - delta| at most, which does not depend on the
// gradients' size.  fp16, 2 x 8193 with a bias: 429 + 725 us, 416 + 704 without; 2048 windows of 90: 369, 366.  bf16 has the
// exponents of 32 bits: there this is nothing.
template <typename T>
struct Lift {
  static constexpr bool kOn = std::is_same<T, f16>::value;
  int e = 0;          // the power is 2^e
  float limit = 0.f;  // of |dp - delta|
  __device__ __forceinline__ float power() const { return kOn ? __builtin_ldexpf(1.f, e) : 1.f; }
  __device__ __forceinline__ float back() const { return kOn ? __builtin_ldexpf(1.f, -e) : 1.f; }
  static __device__ __forceinline__ int power_of(float top) { return min(9 - __builtin_amdgcn_frexp_expf(top), 100); }
  // top: the largest of a tile's that the lane has
  __device__ __forceinline__ bool beyond(float top) const { return kOn && wave_ballot(top > limit) != 0; }
  template <int N>
  __device__ __forceinline__ void lower(float top, f32x16 (&sums)[N]) {
    top = max_of_halves(top);
    const bool beyond = top > limit && top < INFINITY;
    const int to = beyond ? power_of(top) : e;
    const float by = __builtin_ldexpf(1.f, to - e);
    limit = beyond ? __builtin_ldexpf(1.f, 15 - to) : limit;
    e = to;
#pragma unroll
    for (int x = 0; x < N; ++x) sums[x] *= by;
  }
};
__device__ __forceinline__ float largest(const f32x16 &x) {
  float top = 0;
#pragma unroll
  for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
  return top;
}

// A key that has this much of a row's weight: the launch by queries goes through its tile again.
constexpr float kHeavy = 1.f / 2;

// What by_query() does with what a row sees of a tile: its probabilities, and the largest |dp|, which the row's sums follow or
// which is kept.
template <typename T, int N>
struct Follow {
  Lift<T> &lift;
  f32x16 (&sums)[N];
  float delta;  // its size
  bool &heavy;  // whether a row of the wave has much of its weight in one key of the tile
  __device__ __forceinline__ void weights(const f32x16 &p) const { heavy = wave_ballot(largest(p) > kHeavy) != 0; }
  __device__ __forceinline__ void saw(float top) const {
    if (__builtin_expect(lift.beyond(top + delta), 0)) lift.lower(top + delta, sums);
  }
};
struct Keep {
  float &most;
  __device__ __forceinline__ void weights(const f32x16 &) const {}
  __device__ __forceinline__ void saw(float top) const { most = fmaxf(most, top); }
};

// 32 keys (rows `row0`.. of the tiles, kk.. in memory) by the wave's 32 queries, a lane a query: s, the probabilities times
// the cap's derivative, and dp; `delta` gains the lane's share of sum p dp.
template <typename T, int D, int MODE, typename F>
__device__ __forceinline__ void by_query(f32x16 &s, f32x16 &dp, float &delta, const F &of_row, const T *k_tile, const T *v_tile, int row0, int kk,
                                         const vec8<T> (&q)[D / 16], const vec8<T> (&dout)[D / 16], const TileReader<T, D> &reader,
                                         const Scores<MODE> &scores, const Seen &seen, int place, float less) {
  const int half = lane_id() >> 5;
  s = dp = f32x16{};
#pragma unroll
  for (int x = 0; x < D / 16; ++x) s = mfma(reader.rows(k_tile, row0, x), q[x], s);
#pragma unroll
  for (int x = 0; x < D / 16; ++x) dp = mfma(reader.rows(v_tile, row0, x), dout[x], dp);
  const float ahead = (float)(place - kk - 4 * half);
  f32x16 shrink;
  scores.cap_far(s);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const float c = scores.in_tile(s[r]), z = scores.z(c, ahead - (float)(8 * (r >> 2) + (r & 3)));
    shrink[r] = scores.shrink(c);
    s[r] = exp2_fast(fmaf(z, scores.factor, less));
  }
  float top = Lift<T>::kOn ? largest(dp) : 0;
  if (__builtin_expect(!seen.covers(kk, kk + 32), 0)) {
    const uint32_t from_lo = (uint32_t)(kk + 4 * half - seen.lo), count = (uint32_t)(seen.hi - seen.lo);
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (from_lo + (uint32_t)(8 * (r >> 2) + (r & 3)) >= count) s[r] = dp[r] = shrink[r] = 0;
    if (Lift<T>::kOn) top = largest(dp);
    asm volatile("");  // (keeps this a branch of its own: whole tiles pay nothing)
  }
  of_row.weights(s);
  of_row.saw(top);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    delta += s[r] * dp[r];
    if (MODE & kCap) s[r] *= shrink[r];
  }
}

// x += (rows row0.. of the tile, transposed) times the 32 x 32 block y
template <typename T, int D>
__device__ __forceinline__ void add_columns(f32x16 (&x)[D / 32], const T *tile, int row0, const f32x16 &y, const TileReader<T, D> &reader) {
  const vec8<T> y0 = packed<T, 0>(y), y1 = packed<T, 1>(y);
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
    x[db] = mfma(reader.columns(tile, row0, db), y0, x[db]);
    x[db] = mfma(reader.columns(tile, row0 + 16, db), y1, x[db]);
  }
}

// p is at most 1 and often far below the smallest normal f16, so it is multiplied with dout 2^10 times as large.
template <typename T>
constexpr float kRaise = std::is_same<T, f16>::value ? 10.f : 0.f;

// What the keys' side needs of `N` queries, in LDS.
template <int N>
struct __attribute__((aligned(16))) QueryRows {
  float lse[N], delta[N];  // lse in exponents of 2, infinite where a row sees nothing
  int lo[N], hi[N];        // 0, 0 there
};

// 32 queries (rows `row0`.. of the tiles and of `rows`, i0.. in memory) by the wave's 32 keys, a lane a key: dv += p^T dout,
// dk += ds^T q.
// KEEP_V: V's operands are in v, else in LDS, the wave's 32 rows at own_v.
template <bool KEEP_V, typename T, int D, int MODE, int N>
__device__ __forceinline__ void add_by_key(f32x16 (&dk)[D / 32], f32x16 (&dv)[D / 32], Lift<T> &lift, const T *q_tile, const T *g_tile, int row0,
                                           const QueryRows<N> &rows, const vec8<T> (&k)[D / 16], const vec8<T> (&v)[D / 16],
                                           const T *own_v, const TileReader<T, D> &reader, const Scores<MODE> &scores, int ahead, int key,
                                           bool whole) {
  const int half = lane_id() >> 5;
  f32x16 s = {}, dp = {};
#pragma unroll
  for (int y = 0; y < D / 16; ++y) s = mfma(reader.rows(q_tile, row0, y), k[y], s);
#pragma unroll
  for (int y = 0; y < D / 16; ++y) dp = mfma(reader.rows(g_tile, row0, y), KEEP_V ? v[y] : reader.rows(own_v, 0, y), dp);
  const float distance = (float)(ahead + 4 * half - key);
  scores.cap_far(s);
#pragma unroll
  for (int z = 0; z < 4; ++z) {
    const int r0 = row0 + 8 * z + 4 * half;
    const f32x4 lse = *reinterpret_cast<const f32x4 *>(rows.lse + r0), delta = *reinterpret_cast<const f32x4 *>(rows.delta + r0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 4 * z + e;
      const float c = scores.in_tile(s[r]), y = scores.z(c, distance + (float)(8 * z + e)), shrink = scores.shrink(c);
      const float p = exp2_fast(fmaf(y, scores.factor, scores.offset + kRaise<T> - lse[e]));
      float ds = dp[r] - delta[e];
      if (!Lift<T>::kOn) ds *= p;
      if (MODE & kCap) ds *= shrink;
      s[r] = p, dp[r] = ds;
    }
  }
  float top = Lift<T>::kOn ? largest(dp) : 0;
  if (__builtin_expect(!whole, 0)) {
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      const int r0 = row0 + 8 * z + 4 * half;
      const i32x4 lo = *reinterpret_cast<const i32x4 *>(rows.lo + r0), hi = *reinterpret_cast<const i32x4 *>(rows.hi + r0);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((uint32_t)(key - lo[e]) >= (uint32_t)(hi[e] - lo[e])) s[4 * z + e] = dp[4 * z + e] = 0;
    }
    if (Lift<T>::kOn) top = largest(dp);
    asm volatile("");  // (keeps this a branch of its own: whole tiles pay nothing)
  }
  if (__builtin_expect(lift.beyond(top), 0)) lift.lower(top, dk);
  if (Lift<T>::kOn) {
    const float power = __builtin_ldexpf(1.f, lift.e - (int)kRaise<T>);
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] *= power * s[r];
  }
  add_columns<T, D>(dv, g_tile, row0, s, reader);
  add_columns<T, D>(dk, q_tile, row0, dp, reader);
}

template <typename T, int D, int MODE, int WAVES>
__global__ __launch_bounds__(WAVES *kWave, 2) void attention_dq_kernel(GradArgs g) {
  __shared__ __attribute__((aligned(16))) T k_tile[2][kTile * D];  // (at the end: the rows of dq)
  __shared__ __attribute__((aligned(16))) T v_tile[2][kTile * D];
  __shared__ int ranges[WAVES][2];
  __shared__ uint64_t heavy_of[WAVES];
  const AttentionArgs &a = g.a;
  const int tid = threadIdx.x, l = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = l >> 5;
  const int at = same_die_index(), block = g.blocks - 1 - at % g.blocks, bh = at / g.blocks, head = bh % a.heads, b = bh / a.heads;
  const int kv_head = head / (a.heads / a.kv_heads);
  const int i0 = (block * WAVES + wave) * kRows, i = i0 + (l & 31);
  const bool row_there = i < a.queries;

  Seen seen;
  const int64_t row = (int64_t)b * a.queries + i;
  seen.set(row_there ? a.lo[row] : 0, row_there ? a.hi[row] : 0, a.keys);
  if (l == 0) ranges[wave][0] = seen.first, ranges[wave][1] = seen.end;
  const bool some_empty = wave_ballot(seen.empty()) != 0;
  if (head == 0 && i < g.padded) {
    if (half == 0) g.lo[(int64_t)b * g.padded + i] = seen.lo, g.hi[(int64_t)b * g.padded + i] = seen.hi;
    if (l == 0)
      g.bounds[((int64_t)b * g.padded + i0) / kRows] = i32x4{seen.first, seen.end, seen.all_from, some_empty ? 0 : seen.all_to};
  }

  vec8<T> q[D / 16], dout[D / 16];
  own_row_frags<T, D>(q, static_cast<const T *>(a.q) + b * a.qs.batch + i * a.qs.token + head * a.qs.head, a.dim, !seen.empty());
  own_row_frags<T, D>(dout, static_cast<const T *>(g.dout) + b * g.gs.batch + i * g.gs.token + head * g.gs.head, a.dim,
                      !seen.empty());
  float delta = 0;
  {
    vec8<T> out[D / 16];
    own_row_frags<T, D>(out, static_cast<const T *>(g.out) + (row * a.heads + head) * a.dim, a.dim, !seen.empty());
#pragma unroll
    for (int x = 0; x < D / 16; ++x)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)dout[x][e] * (float)out[x][e];
    delta = sum_of_halves(delta);
  }
  float lse_log2 = INFINITY;  // a row that sees nothing: p = 0
  if (!seen.empty()) lse_log2 = g.lse[((int64_t)b * a.heads + head) * a.queries + i] * kLog2e;
  __syncthreads();
  int first = INT_MAX, end = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) first = min(first, ranges[w][0]), end = max(end, ranges[w][1]);
  first = __builtin_amdgcn_readfirstlane(first), end = __builtin_amdgcn_readfirstlane(end);

  const Scores<MODE> scores(a, head);
  const TileReader<T, D> reader;
  const float less = scores.offset - lse_log2;
  const int place = i + a.keys - a.queries;
  f32x16 dq[D / 32] = {};
  Lift<T> lift;
  float summed = 0;  // sum p dp: what delta is, without the rounding of out
  const Stage<T, D, kTile, false, true> k_rows(static_cast<const T *>(a.k) + b * a.ks.batch + kv_head * a.ks.head, a.ks.token, first, end, a.dim);
  const Stage<T, D, kTile> v_rows(static_cast<const T *>(a.v) + b * a.vs.batch + kv_head * a.vs.head, a.vs.token, first, end, a.dim);
  auto load = [&](int k0, int to) __attribute__((always_inline)) {
    k_rows.template ask<WAVES>(k_tile[to], k0, wave);
    v_rows.template ask<WAVES>(v_tile[to], k0, wave);
  };
  const int k_first = first < end ? first / kTile * kTile : 0;
  int k0 = k_first, buffer = 0;
  // the tiles in which a key has much of a row's weight, a bit for each of 64 (or 128, 256 .. keys, where there are more tiles)
  uint64_t heavy_tiles = 0;
  int keys_a_bit = 6;
  while ((end - 1 - k_first) >> keys_a_bit >= 64) ++keys_a_bit;
  for (int x = wave; x < 2; x += WAVES) k_rows.clear_beyond(k_tile[x]);
  if (k0 < end) load(k0, 0);
  for (; k0 < end; k0 += kTile, buffer ^= 1) {
    staged_wait();
    __syncthreads();
    if (k0 + kTile < end) load(k0 + kTile, buffer ^ 1);
    const T *k_here = k_tile[buffer], *v_here = v_tile[buffer];
#pragma unroll 1
    for (int kb = 0; kb < 2; ++kb) {
      const int kk = k0 + kb * 32;
      if (!seen.touches(kk, kk + 32)) continue;
      f32x16 s, dp;
      bool heavy = false;
      by_query<T, D, MODE>(s, dp, summed, Follow<T, D / 32>{lift, dq, fabsf(delta), heavy}, k_here, v_here, kb * 32, kk, q, dout, reader,
                           scores, seen, place, less);
      if (heavy) heavy_tiles |= 1ull << ((k0 - k_first) >> keys_a_bit);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= Lift<T>::kOn ? fmaf(dp[r], lift.power(), -delta * lift.power()) : dp[r] - delta;
      add_columns<T, D>(dq, k_here, kb * 32, s, reader);
    }
  }
  summed = seen.empty() ? 0.f : sum_of_halves(summed);
  if (half == 0 && i < g.padded) {
    const int64_t stats = ((int64_t)b * a.heads + head) * g.padded + i;
    g.lse_log2[stats] = lse_log2, g.delta[stats] = summed;
  }
  if (l == 0) heavy_of[wave] = heavy_tiles;
  __syncthreads();
  // those tiles again, by what their sums owe to the difference of both deltas: p (dout . out - sum p dp) (1 - tanh^2) k
  const float owed = seen.empty() ? 0.f : (delta - summed) * lift.power();
  uint64_t any_heavy = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) any_heavy |= heavy_of[w];
  any_heavy = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(any_heavy >> 32)) << 32 |
              (uint32_t)__builtin_amdgcn_readfirstlane((int)any_heavy);
  auto heavy_from = [&](int k) __attribute__((always_inline)) {
    while (k < end && !((any_heavy >> ((k - k_first) >> keys_a_bit)) & 1)) k += kTile;
    return k;
  };
  k0 = heavy_from(k_first), buffer = 0;
  if (k0 < end) k_rows.template ask<WAVES>(k_tile[0], k0, wave);
  while (k0 < end) {
    staged_wait();
    __syncthreads();
    const int next = heavy_from(k0 + kTile);
    if (next < end) k_rows.template ask<WAVES>(k_tile[buffer ^ 1], next, wave);
#pragma unroll 1
    for (int kb = 0; kb < 2; ++kb) {
      const int kk = k0 + kb * 32;
      if (!seen.touches(kk, kk + 32)) continue;
      f32x16 s = {};
#pragma unroll
      for (int x = 0; x < D / 16; ++x) s = mfma(reader.rows(k_tile[buffer], kb * 32, x), q[x], s);
      scores.cap_far(s);
      const float ahead = (float)(place - kk - 4 * half);
      const uint32_t from_lo = (uint32_t)(kk + 4 * half - seen.lo), count = (uint32_t)(seen.hi - seen.lo);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float c = scores.in_tile(s[r]), z = scores.z(c, ahead - (float)(8 * (r >> 2) + (r & 3)));
        const float ds = exp2_fast(fmaf(z, scores.factor, less)) * scores.shrink(c) * owed;
        s[r] = from_lo + (uint32_t)(8 * (r >> 2) + (r & 3)) < count ? ds : 0.f;
      }
      add_columns<T, D>(dq, k_tile[buffer], kb * 32, s, reader);
    }
    k0 = next, buffer ^= 1;
  }
  __syncthreads();
  const uint32_t bad = columns_not_finite(dq, !seen.empty());
  store_rows<T, D>(k_tile[0] + wave * kRows * D, dq, a.scale * lift.back(), seen.empty(), a.dim, [&](int r) {
    return i0 + r < a.queries ? static_cast<T *>(g.dq) + (((int64_t)b * a.queries + i0 + r) * a.heads + head) * a.dim : nullptr;
  });
  if (__builtin_expect(bad != 0, 0)) mend_dq<T, MODE>(g, bad, b, head, kv_head, i0, seen, lse_log2, summed, scores);
}

// Rows of 128 elements leave no registers for V beside K, dk and dv at two waves a SIMD (spilled, they would be waited for
// together with the tiles to come): V stays in LDS, and to make room for it a tile is 32 queries.
// (Rows of 64 with a bias are a few registers above what three waves a SIMD may have: held there, both gradients of 2 x 8193 take
// 598 us in bf16 and 645 in fp16, in place of 631 and 676.)
template <typename T, int D, int MODE>
__global__ __launch_bounds__(kThreads, D == 64 && MODE == kBias ? 3 : 2) void attention_dkv_kernel(GradArgs g) {
  constexpr bool kKeepV = D < 128;  // in registers
  constexpr int kTile = kKeepV ? 64 : 32, kSides = kTile / kRows;
  __shared__ __attribute__((aligned(16))) T q_tile[2][kTile * D];  // (at the end: the rows of dk and dv)
  __shared__ __attribute__((aligned(16))) T g_tile[2][kTile * D];
  __shared__ __attribute__((aligned(16))) T v_rows[kKeepV ? 8 : kWaves * kRows * D];
  __shared__ QueryRows<kTile> rows[2];
  const AttentionArgs &a = g.a;
  const int l = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int at = same_die_index(), block = at % g.blocks, bh = at / g.blocks, kv_head = bh % a.kv_heads, b = bh / a.kv_heads;
  const int shared = a.heads / a.kv_heads;
  const int block_key = block * (kWaves * kRows), wave_key = block_key + wave * kRows, key = wave_key + (l & 31);
  const bool key_there = key < a.keys;

  vec8<T> k[D / 16], v[D / 16];
  own_row_frags<T, D>(k, static_cast<const T *>(a.k) + b * a.ks.batch + key * a.ks.token + kv_head * a.ks.head, a.dim, key_there);
  T *own_v = v_rows + wave * kRows * D;
  const T *v_base = static_cast<const T *>(a.v) + b * a.vs.batch + kv_head * a.vs.head;
  if (kKeepV) {
    own_row_frags<T, D>(v, v_base + key * a.vs.token, a.dim, key_there);
  } else {
    const Stage<T, D, kRows> v_stage(v_base, a.vs.token, 0, a.keys, a.dim);
    v_stage.template ask<1>(own_v, wave_key, 0);
    staged_wait();
    v_stage.clear_beyond(own_v);
    wave_lds_sync();
  }
  f32x16 dk[D / 32] = {}, dv[D / 32] = {};
  Lift<T> lift;
  const int groups = g.padded / kRows, tiles = (a.queries + kTile - 1) / kTile;
  // (read through the scalar cache: the launch before wrote them)
  typedef const __attribute__((address_space(4))) i32x4 *Bounds;
  const Bounds bounds = (Bounds)(uintptr_t)(g.bounds + (int64_t)b * groups);
  const TileReader<T, D> reader;

  // The tiles of queries that see any of the workgroup's keys, head after head: 64 are looked at at a time.
  int head = kv_head * shared, base = -kWave;
  uint64_t left = 0;
  auto next_tile = [&]() __attribute__((always_inline)) -> int {  // or -1
    while (left == 0) {
      base += kWave;
      if (base >= tiles) {
        base = 0;
        if (++head == (kv_head + 1) * shared || tiles == 0) return -1;
      }
      bool reaches = false;
      if (base + l < tiles) {
        const i32x4 *mine = g.bounds + (int64_t)b * groups + (base + l) * kSides;
#pragma unroll
        for (int y = 0; y < kSides; ++y) reaches |= mine[y][0] < block_key + kWaves * kRows && mine[y][1] > block_key;
      }
      left = wave_ballot(reaches);
    }
    const int tile = base + (int)__builtin_ctzll(left);
    left &= left - 1;
    return tile;
  };
  // A tile is asked for while the one before it is worked on: rows of q and dout, and (an array a wave) what is known of them.
  auto ask = [&](int tile, int to) __attribute__((always_inline)) {
    const int i0 = tile * kTile;
    int lane = l;
    // with a bias there are too few registers to keep what Stage works out between the tiles (2 x 8193: 725 us spilled, 675
    // worked out again; without, 961 kept, 1028 worked out again)
    if (MODE & kBias) asm volatile("" : "+v"(lane));
    const Stage<T, D, kTile> q_rows(static_cast<const T *>(a.q) + b * a.qs.batch + head * a.qs.head, a.qs.token, 0, a.queries, a.dim, lane);
    const Stage<T, D, kTile> g_rows(static_cast<const T *>(g.dout) + b * g.gs.batch + head * g.gs.head, g.gs.token, 0, a.queries, a.dim, lane);
    q_rows.template ask<kWaves>(q_tile[to], i0, wave);
    g_rows.template ask<kWaves>(g_tile[to], i0, wave);
    static_assert(kWaves == 4, "");
    const int64_t stats = ((int64_t)b * a.heads + head) * g.padded + i0, of_batch = (int64_t)b * g.padded + i0;
    const void *from = wave == 0 ? (const void *)(g.lse_log2 + stats) : wave == 1 ? (const void *)(g.delta + stats)
                       : wave == 2 ? (const void *)(g.lo + of_batch) : (const void *)(g.hi + of_batch);
    if (l < kTile) stage_words(static_cast<const int *>(from) + l, reinterpret_cast<const int *>(&rows[to]) + wave * kTile);
  };

  int tile = tiles > 0 ? next_tile() : -1, tile_head = -1, buffer = 0;
  Scores<MODE> scores(a, kv_head * shared);
  if (tile >= 0) ask(tile, 0);
  for (; tile >= 0; buffer ^= 1) {
    const int i0 = tile * kTile;
    i32x4 reach[kSides];
#pragma unroll
    for (int y = 0; y < kSides; ++y) reach[y] = bounds[tile * kSides + y];
    if (MODE & kBias && head != tile_head) scores = Scores<MODE>(a, head), tile_head = head;
    staged_wait();
    __syncthreads();
    if (reach[0][3] == 0 || reach[kSides - 1][3] == 0) {  // rows that see nothing may hold anything: zeros in their place
      for (int x = threadIdx.x; x < kTile * D / 8; x += kThreads)
        if (rows[buffer].hi[x / (D / 8)] == 0) {
          *reinterpret_cast<vec8<T> *>(q_tile[buffer] + x * 8) = vec8<T>{};
          *reinterpret_cast<vec8<T> *>(g_tile[buffer] + x * 8) = vec8<T>{};
        }
      __syncthreads();
    }
    tile = next_tile();
    if (tile >= 0) ask(tile, buffer ^ 1);
#pragma unroll
    for (int y = 0; y < kSides; ++y) {
      if (reach[y][0] >= wave_key + kRows || reach[y][1] <= wave_key) continue;
      add_by_key<kKeepV, T, D, MODE>(dk, dv, lift, q_tile[buffer], g_tile[buffer], y * kRows, rows[buffer], k, v, own_v, reader, scores,
                                     i0 + y * kRows + a.keys - a.queries, key,
                                     reach[y][2] <= wave_key && reach[y][3] >= wave_key + kRows);
    }
  }
  __syncthreads();
  const auto to = [&](void *p) {
    return [=](int r) {
      return wave_key + r < a.keys ? static_cast<T *>(p) + (((int64_t)b * a.keys + wave_key + r) * a.kv_heads + kv_head) * a.dim : nullptr;
    };
  };
  const uint32_t bad = columns_not_finite(dk, key_there) | columns_not_finite(dv, key_there);
  // (the 4 x 32 rows of dk fill both tiles of q, those of dv the tiles of dout or what was V)
  store_rows<T, D>(kKeepV ? q_tile[0] + wave * kRows * D : own_v, dk, a.scale * lift.back(), false, a.dim, to(g.dk));
  wave_lds_sync();
  store_rows<T, D>(kKeepV ? g_tile[0] + wave * kRows * D : own_v, dv, 1.f / (1 << (int)kRaise<T>), false, a.dim, to(g.dv));
  if (__builtin_expect(bad != 0, 0))
    mend_dkv<T, MODE>(g, bad, b, kv_head, wave_key, [&](int of_head, int i, float &lse_log2, float &delta, int &lo, int &hi) {
      const int64_t stats = ((int64_t)b * a.heads + of_head) * g.padded + i, of_batch = (int64_t)b * g.padded + i;
      lse_log2 = g.lse_log2[stats], delta = g.delta[stats], lo = g.lo[of_batch], hi = g.hi[of_batch];
    });
}

// ---- short windows: one launch ----------------------------------------------------------------------------
// Where all queries and all keys of a window are at most 128 (and a row at most 64 elements, and no heads share keys),
// a workgroup holds queries, keys, values and dout of a window and head in LDS: each is read once, out not at all, because delta
// can be summed from the probabilities themselves -- in 32 bits, where dout . out begins from the rounded out.
// us in one launch / two: 2048 x 90, 8 heads of 64, causal, bf16: 361 / 527; 64 x 60, 4 of 32, bf16: 8.7 / 12.0.  The first is 1.3 GB at
// 3.7 TB/s: loads, products and stores of a workgroup follow each other, and 200 registers leave two waves a SIMD to
// overlap them (three: 28 registers spilled, 490 us).
// A wave is responsible for 32 queries (delta, dq) and for 32 keys (dk, dv) in turn.
template <typename T, int D, int MODE, int WAVES>
__global__ __launch_bounds__(WAVES *kWave, 2) void attention_window_grad_kernel(GradArgs g) {
  constexpr int kMost = WAVES * kRows;
  __shared__ __attribute__((aligned(16))) T q_tile[kMost * D], g_tile[kMost * D], k_tile[kMost * D], v_tile[kMost * D];
  __shared__ QueryRows<kMost> rows;
  __shared__ i32x4 bounds[WAVES];
  const AttentionArgs &a = g.a;
  const int tid = threadIdx.x, l = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = l >> 5;
  const int unit = same_die_index(), head = unit % a.heads, b = unit / a.heads;
  const int own = wave * kRows, mine = own + (l & 31);
  const int64_t row = (int64_t)b * a.queries + mine, stats = ((int64_t)b * a.heads + head) * a.queries + mine;
  const bool row_there = mine < a.queries;
  const TileReader<T, D> reader;

  // (asked for before anything is known of the ranges; rows beyond the last are copies of it)
  const Stage<T, D, kRows> q_rows(static_cast<const T *>(a.q) + b * a.qs.batch + head * a.qs.head, a.qs.token, 0, a.queries, a.dim);
  const Stage<T, D, kRows> g_rows(static_cast<const T *>(g.dout) + b * g.gs.batch + head * g.gs.head, g.gs.token, 0, a.queries, a.dim);
  const int lo = row_there ? a.lo[row] : 0, hi = row_there ? a.hi[row] : 0;
  const float lse = row_there ? g.lse[stats] : 0;
  q_rows.template ask<1>(q_tile + own * D, own, 0);
  g_rows.template ask<1>(g_tile + own * D, own, 0);
  Seen seen;
  seen.set(lo, hi, a.keys);
  const float lse_log2 = seen.empty() ? INFINITY : lse * kLog2e;
  const uint64_t empties = wave_ballot(seen.empty());
  if (half == 0) rows.lo[mine] = seen.lo, rows.hi[mine] = seen.hi, rows.lse[mine] = lse_log2;
  if (l == 0) bounds[wave] = i32x4{seen.first, seen.end, seen.all_from, empties != 0 ? 0 : seen.all_to};
  __syncthreads();
  int first = INT_MAX, end = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) first = min(first, bounds[w][0]), end = max(end, bounds[w][1]);
  first = __builtin_amdgcn_readfirstlane(first), end = __builtin_amdgcn_readfirstlane(end);
  if (first < end) {
    const Stage<T, D, kRows, false, true> k_rows(static_cast<const T *>(a.k) + b * a.ks.batch + head * a.ks.head, a.ks.token, first, end, a.dim);
    const Stage<T, D, kRows> v_rows(static_cast<const T *>(a.v) + b * a.vs.batch + head * a.vs.head, a.vs.token, first, end, a.dim);
    k_rows.clear_beyond(k_tile + own * D);
    k_rows.template ask<1>(k_tile + own * D, own, 0);
    v_rows.template ask<1>(v_tile + own * D, own, 0);
  }
  staged_wait();
  if (empties != 0) {  // rows that see nothing may hold anything: zeros in their place
    wave_lds_sync();
    for (int y = l; y < kRows * D / 8; y += kWave)
      if ((empties >> (y / (D / 8))) & 1) {
        *reinterpret_cast<vec8<T> *>(q_tile + own * D + y * 8) = vec8<T>{};
        *reinterpret_cast<vec8<T> *>(g_tile + own * D + y * 8) = vec8<T>{};
      }
  }
  __syncthreads();
  const Scores<MODE> scores(a, head);
  vec8<T> u[D / 16], w[D / 16];  // rows of the wave: of q and dout, then of k and v
  auto take = [&](const T *p, const T *r) __attribute__((always_inline)) {
#pragma unroll
    for (int y = 0; y < D / 16; ++y) u[y] = reader.rows(p, own, y), w[y] = reader.rows(r, own, y);
    if (a.dim < D) {  // the tiles repeat a piece there
#pragma unroll
      for (int y = 0; y < D / 16; ++y)
        if ((2 * y + half) * 8 >= a.dim) u[y] = w[y] = vec8<T>{};
      asm volatile("");
    }
  };
  vec8<T> dq_kept[D / 32][2];
  uint32_t bad_dq;
  float own_delta;
  {
    const float less = scores.offset - lse_log2;
    const int place = mine + a.keys - a.queries;
    float delta = 0, most = 0;
    f32x16 s[WAVES], dp[WAVES];
    take(q_tile, g_tile);
#pragma unroll
    for (int x = 0; x < WAVES; ++x)
      if (seen.touches(x * kRows, x * kRows + kRows))
        by_query<T, D, MODE>(s[x], dp[x], delta, Keep{most}, k_tile, v_tile, x * kRows, x * kRows, u, w, reader, scores, seen, place, less);
    delta = seen.empty() ? 0.f : sum_of_halves(delta);
    if (half == 0) rows.delta[mine] = delta;
    f32x16 dq[D / 32] = {};
    Lift<T> lift;  // (all of the row's dp are known)
    lift.e = Lift<T>::power_of(max_of_halves(most) + fabsf(delta));
#pragma unroll
    for (int x = 0; x < WAVES; ++x)
      if (seen.touches(x * kRows, x * kRows + kRows)) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[x][r] *= Lift<T>::kOn ? fmaf(dp[x][r], lift.power(), -delta * lift.power()) : dp[x][r] - delta;
        add_columns<T, D>(dq, k_tile, x * kRows, s[x], reader);
      }
    bad_dq = columns_not_finite(dq, !seen.empty()), own_delta = delta;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      dq[db] *= a.scale * lift.back();
      if (empties != 0) {  // (p = 0 is not enough where a key that others see is not finite)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[db][r] = seen.empty() ? 0.f : dq[db][r];
        asm volatile("");
      }
      dq_kept[db][0] = packed<T, 0>(dq[db]), dq_kept[db][1] = packed<T, 1>(dq[db]);
    }
  }
  __syncthreads();
  const auto to = [&](void *p, int count) {
    return [=](int r) {
      return own + r < count ? static_cast<T *>(p) + (((int64_t)b * count + own + r) * a.heads + head) * a.dim : nullptr;
    };
  };
  take(k_tile, v_tile);
  wave_lds_sync();  // nobody reads the wave's rows of K any more
  store_packed<T, D>(k_tile + own * D, dq_kept, a.dim, to(g.dq, a.queries));
  f32x16 dk[D / 32] = {}, dv[D / 32] = {};
  Lift<T> lift;
#pragma unroll 1
  for (int qb = 0; qb < WAVES; ++qb) {
    const i32x4 reach = bounds[qb];
    if (__builtin_amdgcn_readfirstlane(reach[0]) >= own + kRows || __builtin_amdgcn_readfirstlane(reach[1]) <= own) continue;
    const bool whole = __builtin_amdgcn_readfirstlane(reach[2]) <= own && __builtin_amdgcn_readfirstlane(reach[3]) >= own + kRows;
    add_by_key<true, T, D, MODE>(dk, dv, lift, q_tile, g_tile, qb * kRows, rows, u, w, nullptr, reader, scores, qb * kRows + a.keys - a.queries, mine, whole);
  }
  const uint32_t bad = columns_not_finite(dk, mine < a.keys) | columns_not_finite(dv, mine < a.keys);
  wave_lds_sync();
  store_rows<T, D>(k_tile + own * D, dk, a.scale * lift.back(), false, a.dim, to(g.dk, a.keys));
  store_rows<T, D>(v_tile + own * D, dv, 1.f / (1 << (int)kRaise<T>), false, a.dim, to(g.dv, a.keys));
  if (__builtin_expect(bad_dq != 0, 0)) mend_dq<T, MODE>(g, bad_dq, b, head, head, own, seen, lse_log2, own_delta, scores);
  if (__builtin_expect(bad != 0, 0))
    mend_dkv<T, MODE>(g, bad, b, head, own, [&](int, int i, float &lse_of, float &delta, int &lo_of, int &hi_of) {
      lse_of = rows.lse[i], delta = rows.delta[i], lo_of = rows.lo[i], hi_of = rows.hi[i];
    });
}

// Queries in the statistics: whole tiles.
int64_t padded(int64_t queries) { return ceil_div64(queries, 64) * 64; }

}  // namespace
}  // namespace gearhip

using namespace gearhip;

extern "C" size_t gear_hip_attention_backward_workspace_bytes(int64_t batch, int64_t queries, int64_t heads) {
  if (batch <= 0 || queries <= 0 || heads <= 0) return 0;
  const size_t rows = (size_t)(batch * padded(queries));
  return rows * heads * 2 * sizeof(float) + rows * 2 * sizeof(int) + rows / kRows * sizeof(i32x4);
}

extern "C" int gear_hip_attention_backward(const gear_hip_attention_desc *desc, const void *dout,
                                           const int64_t *dout_stride, const void *out, const float *lse, void *dq,
                                           void *dk, void *dv, void *workspace, size_t workspace_bytes, void *stream) {
  GradArgs g = {};
  const int rc = attention_args(desc, g.a);
  if (rc < 0) return rc;
  if (rc == 1) return 0;
  const AttentionArgs &a = g.a;
  if (a.queries > 0 && (dout == nullptr || dout_stride == nullptr || out == nullptr || lse == nullptr || dq == nullptr))
    return GEAR_HIP_EINVAL;
  if (a.keys > 0 && (dk == nullptr || dv == nullptr)) return GEAR_HIP_EINVAL;
  const size_t want = gear_hip_attention_backward_workspace_bytes(a.batch, a.queries, a.heads);
  if (want > 0 && (workspace == nullptr || workspace_bytes < want)) return GEAR_HIP_EWORKSPACE;
  for (const void *p : {out, (const void *)dq, (const void *)dk, (const void *)dv, (const void *)workspace})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return GEAR_HIP_EALIGN;
  if (a.queries > 0) {
    if (!rows_aligned(dout, dout_stride, 2)) return GEAR_HIP_EALIGN;
    g.gs = Strides{dout_stride[0], dout_stride[1], dout_stride[2]};
  }
  g.dout = dout, g.out = out, g.lse = lse;
  g.padded = (int)padded(a.queries);
  const int64_t rows = (int64_t)a.batch * g.padded;
  g.bounds = static_cast<i32x4 *>(workspace);
  g.lse_log2 = reinterpret_cast<float *>(g.bounds + rows / kRows);
  g.delta = g.lse_log2 + rows * a.heads;
  g.lo = reinterpret_cast<int *>(g.delta + rows * a.heads);
  g.hi = g.lo + rows;
  g.dq = dq, g.dk = dk, g.dv = dv;
  const int longest = a.queries > a.keys ? a.queries : a.keys;
  if (longest <= 4 * kRows && a.dim <= 64 && a.heads == a.kv_heads && a.queries > 0) {
    if (!launchable((int64_t)a.heads * a.batch, (longest + kRows - 1) / kRows)) return GEAR_HIP_ERANGE;
    by_attention_type(a, desc->dtype, [&](auto dim, auto type, auto mode) {
      if constexpr (decltype(dim)::value <= 64)
        by_waves((longest + kRows - 1) / kRows, [&](auto w) {
          hipLaunchKernelGGL((attention_window_grad_kernel<decltype(type), decltype(dim)::value, decltype(mode)::value, decltype(w)::value>),
                             dim3((unsigned)a.heads * a.batch), dim3(decltype(w)::value * kWave), 0, as_stream(stream), g);
        });
    });
    GEARHIP_RETURN_IF_LAUNCH_FAILED();
    return 0;
  }
  const int groups = g.padded / kRows;  // (padding included: its statistics are written too)
  const int query_blocks = (groups + kWaves - 1) / kWaves, waves = query_blocks > 0 ? (groups + query_blocks - 1) / query_blocks : 1;
  const int key_blocks = (int)ceil_div64(a.keys, kWaves * kRows);
  if (!launchable((int64_t)query_blocks * a.heads * a.batch, waves) || !launchable((int64_t)key_blocks * a.kv_heads * a.batch, kWaves))
    return GEAR_HIP_ERANGE;
  by_attention_type(a, desc->dtype, [&](auto dim, auto type, auto mode) {
    typedef decltype(type) T;
    constexpr int D = decltype(dim)::value;
    constexpr int kMode = decltype(mode)::value;
    if (query_blocks > 0) {
      g.blocks = query_blocks;
      by_waves(waves, [&](auto w) {
        hipLaunchKernelGGL((attention_dq_kernel<T, D, kMode, decltype(w)::value>),
                           dim3((unsigned)g.blocks * a.heads * a.batch), dim3(decltype(w)::value * kWave), 0,
                           as_stream(stream), g);
      });
    }
    g.blocks = key_blocks;
    if (g.blocks > 0)
      hipLaunchKernelGGL((attention_dkv_kernel<T, D, kMode>), dim3((unsigned)g.blocks * a.kv_heads * a.batch),
                         dim3(kThreads), 0, as_stream(stream), g);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
