// Attention over ranges of keys, forward (gear_hip_attention).
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(z_ij - lse_i),  lse_i = log sum_j exp z_ij,  j in [lo_i, hi_i)
// A workgroup takes up to 128 queries of one head, 32 a wave; tiles of 32 keys pass through LDS, two deep, the next asked for
// while one is worked on.  The softmax runs along: a lane holds its query's maximum m and sum l so far, in exponents of 2,
// and the sums of p v are rescaled when m grows.  Tiles outside a wave's ranges are passed over, tiles that all its rows
// see in full need no comparison.  p is rounded to the type for its product (the matrix unit takes nothing wider at this
// rate), its sum is of the values before that.
// bf16: 2048 windows of 90, 8 heads of 64, causal: 134 us, bound by memory (755 MB, 5.7 TB/s).  2 x 8193, 16 heads of 128 over 8,
// packed, a bias: 327 us; 32 x 1470, 16 over 4, frames, a cap: 439 us, 400 TFLOP/s of the pairs that are seen.  There the
// exponentials (and the tanh of the cap) and the matrix unit take about the same time and do not overlap in full.
#include <type_traits>

#include "attention_exact.hpp"

namespace gearhip {

bool rows_aligned(const void *p, const int64_t *stride, int element) {
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (stride[i] * element % 16 != 0) return false;
  return true;
}

int attention_args(const gear_hip_attention_desc *d, AttentionArgs &a) {
  if (d == nullptr || d->batch < 0 || d->queries < 0 || d->keys < 0 || d->heads < 1 || d->kv_heads < 1) return GEAR_HIP_EINVAL;
  if (d->dtype != GEAR_HIP_F16 && d->dtype != GEAR_HIP_BF16) return GEAR_HIP_EINVAL;
  if (d->heads % d->kv_heads != 0 || d->head_dim < 16 || d->head_dim % 16 != 0) return GEAR_HIP_EINVAL;
  if (!(d->scale > 0) || !(d->scale < 1e30f) || !(d->cap >= 0) || !(d->cap < 1e30f) ||
      (d->cap > 0 && !(d->scale / d->cap < 1e30f)))
    return GEAR_HIP_EINVAL;
  if (d->head_dim > 128 || d->queries >= (1 << 30) || d->keys >= (1 << 30) || d->batch >= (1 << 30)) return GEAR_HIP_ERANGE;
  // workgroups of a launch, and rows of the statistics
  if (d->batch * ceil_div64(d->queries, kRows) > INT_MAX / d->heads || d->batch * ceil_div64(d->keys, kRows) > INT_MAX / d->heads)
    return GEAR_HIP_ERANGE;
  if (d->batch == 0 || (d->queries == 0 && d->keys == 0)) return 1;
  if ((d->queries > 0 && (d->q == nullptr || d->lo == nullptr || d->hi == nullptr)) ||
      (d->keys > 0 && (d->k == nullptr || d->v == nullptr)))
    return GEAR_HIP_EINVAL;
  if (!rows_aligned(d->q, d->q_stride, 2) || !rows_aligned(d->k, d->k_stride, 2) || !rows_aligned(d->v, d->v_stride, 2))
    return GEAR_HIP_EALIGN;
  auto strides = [](const int64_t *s) { return Strides{s[0], s[1], s[2]}; };
  a = AttentionArgs{d->q, d->k, d->v, strides(d->q_stride), strides(d->k_stride), strides(d->v_stride),
                    (int)d->batch, (int)d->queries, (int)d->keys, d->heads, d->kv_heads, d->head_dim, d->lo, d->hi,
                    d->slopes, d->scale, d->scale * kLog2e, d->cap};
  return 0;
}

namespace {

constexpr int kMostWaves = 4;
// Keys of a tile.  With 32, three waves a SIMD have the registers and the LDS they need with rows of 128, and less is passed
// over at the edges of ranges: us with 32 / 64, 2048 windows of 90 (64) 133 / 150, 32 x 1470 with a cap (128) 429 / 487,
// 2 x 8193 with a bias 334 / 326.
constexpr int kTile = 32;

// (At least three waves a SIMD, where LDS has room for them: rows of 128 without a cap or a bias came out with 170 registers, two
// waves and 326 us for 2 x 8193 in place of 296.)
template <typename T, int D, int MODE, int WAVES>
__global__ __launch_bounds__(WAVES *kWave, WAVES >= 3 ? 3 : 2) void attention_kernel(AttentionArgs a, T *__restrict__ out,
                                                                    float *__restrict__ lse, int blocks) {
  __shared__ __attribute__((aligned(16))) T k_tile[2][kTile * D];  // (at the end, with those of V: the rows of the output)
  __shared__ __attribute__((aligned(16))) T v_tile[2][kTile * D];
  __shared__ int ranges[WAVES][2];
  const int tid = threadIdx.x, l = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = l >> 5;
  // a head's workgroups share its keys: next to each other on one die; the last first, where causal rows see most
  const int at = same_die_index(), block = blocks - 1 - at % blocks, bh = at / blocks, head = bh % a.heads, b = bh / a.heads;
  const int kv_head = head / (a.heads / a.kv_heads);
  const int i = (block * WAVES + wave) * kRows + (l & 31);
  const bool row_there = i < a.queries;

  Seen seen;
  const int64_t row = (int64_t)b * a.queries + i;
  seen.set(row_there ? a.lo[row] : 0, row_there ? a.hi[row] : 0, a.keys);
  if (l == 0) ranges[wave][0] = seen.first, ranges[wave][1] = seen.end;
  vec8<T> q[D / 16];
  own_row_frags<T, D>(q, static_cast<const T *>(a.q) + b * a.qs.batch + i * a.qs.token + head * a.qs.head, a.dim, !seen.empty());
  __syncthreads();
  int first = INT_MAX, end = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) first = min(first, ranges[w][0]), end = max(end, ranges[w][1]);
  first = __builtin_amdgcn_readfirstlane(first), end = __builtin_amdgcn_readfirstlane(end);

  const Scores<MODE> scores(a, head);
  const TileReader<T, D> reader;
  const int place = i + a.keys - a.queries;
  f32x16 o[D / 32] = {};
  float m = -INFINITY;  // of z
  Sum sums;

  const Stage<T, D, kTile, false, true> k_rows(static_cast<const T *>(a.k) + b * a.ks.batch + kv_head * a.ks.head, a.ks.token, first, end, a.dim);
  const Stage<T, D, kTile> v_rows(static_cast<const T *>(a.v) + b * a.vs.batch + kv_head * a.vs.head, a.vs.token, first, end, a.dim);
  auto load = [&](int k0, T *k_to, T *v_to) {
    k_rows.template ask<WAVES>(k_to, k0, wave);
    v_rows.template ask<WAVES>(v_to, k0, wave);
  };
  auto tile = [&](int k0, const T *k_here, const T *v_here) __attribute__((always_inline)) {
    if (!seen.touches(k0, k0 + kTile)) return;
    f32x16 s = {};
#pragma unroll
    for (int x = 0; x < D / 16; ++x) s = mfma(reader.rows(k_here, 0, x), q[x], s);
    const float ahead = (float)(place - k0 - 4 * half);
    scores.cap_far(s);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = scores.z(scores.in_tile(s[r]), ahead - (float)(8 * (r >> 2) + (r & 3)));
    if (__builtin_expect(!seen.covers(k0, k0 + kTile), 0)) {
      const uint32_t from_lo = (uint32_t)(k0 + 4 * half - seen.lo), count = (uint32_t)(seen.hi - seen.lo);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (from_lo + (uint32_t)(8 * (r >> 2) + (r & 3)) >= count) s[r] = -INFINITY;
      asm volatile("");  // (keeps this a branch of its own: whole tiles pay nothing)
    }
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
    top = max_of_halves(top);
    // the sums are rescaled only where a maximum grows by more than 2^8: p stays below that
    if (wave_ballot((top - m) * scores.factor > 8.f) != 0) {
      const float grown = fmaxf(m, top);
      const float rescale = grown == -INFINITY ? 1.f : exp2_fast((m - grown) * scores.factor);
      m = grown;
      sums.scale(rescale);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] *= rescale;
    }
    const float from = m == -INFINITY ? 0.f : kLevel<T> - m * scores.factor;  // (no key seen yet)
    float of_tile = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = exp2_fast(fmaf(s[r], scores.factor, from));
      of_tile += s[r];
    }
    sums.add(of_tile);
    const vec8<T> p0 = packed<T, 0>(s), p1 = packed<T, 1>(s);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      o[db] = mfma(reader.columns(v_here, 0, db), p0, o[db]);
      o[db] = mfma(reader.columns(v_here, 16, db), p1, o[db]);
    }
  };
  int k0 = first < end ? first / kTile * kTile : 0;
  for (int x = wave; x < 2; x += WAVES) k_rows.clear_beyond(k_tile[x]);
  if (k0 < end) load(k0, k_tile[0], v_tile[0]);
  for (; k0 < end; k0 += 2 * kTile) {
    staged_wait();
    __syncthreads();
    if (k0 + kTile < end) load(k0 + kTile, k_tile[1], v_tile[1]);
    tile(k0, k_tile[0], v_tile[0]);
    if (k0 + kTile >= end) break;
    staged_wait();
    __syncthreads();
    if (k0 + 2 * kTile < end) load(k0 + 2 * kTile, k_tile[0], v_tile[0]);
    tile(k0 + kTile, k_tile[1], v_tile[1]);
  }

  const float sum = sum_of_halves(sums.x);
  const bool empty = seen.empty();
  const float lse_log2 = m * scores.factor + scores.offset + __builtin_log2f(sum * (1.f / (1 << (int)kLevel<T>)));
  if (lse != nullptr && half == 0 && row_there)
    lse[((int64_t)b * a.heads + head) * a.queries + i] = empty ? -INFINITY : lse_log2 * kLn2;
  uint32_t bad = columns_not_finite(o, !empty);
  __syncthreads();  // the tiles are free
  const int i0 = (block * WAVES + wave) * kRows;
  T *piece = (wave < 2 ? k_tile[wave] : v_tile[wave - 2]);
  store_rows<T, D>(piece, o, 1.f / sum, empty, a.dim, [&](int r) {
    return i0 + r < a.queries ? out + (((int64_t)b * a.queries + i0 + r) * a.heads + head) * a.dim : nullptr;
  });
  if (__builtin_expect(bad == 0, 1)) return;
  staged_wait();  // (what is stored above, before it is stored again)
  for (; bad != 0; bad &= bad - 1) {
    const int r = __builtin_ctz(bad), at_row = i0 + r;
    Pair x;
    if (exact_out<T, MODE>(x, static_cast<const T *>(a.q) + b * a.qs.batch + at_row * a.qs.token + head * a.qs.head, k_rows.base,
                           a.ks.token, v_rows.base, a.vs.token, wave_read_lane(seen.lo, r), wave_read_lane(seen.hi, r), a.dim,
                           at_row + a.keys - a.queries, lane_value(lse_log2, r), scores))
      store_pair(out + (((int64_t)b * a.queries + at_row) * a.heads + head) * a.dim, x, a.dim);
  }
}

}  // namespace
}  // namespace gearhip

using namespace gearhip;

extern "C" int gear_hip_attention(const gear_hip_attention_desc *desc, void *out, float *lse, void *stream) {
  AttentionArgs a;
  const int rc = attention_args(desc, a);
  if (rc < 0) return rc;
  if (rc == 1 || a.queries == 0) return 0;
  if (out == nullptr) return GEAR_HIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(out) % 16 != 0) return GEAR_HIP_EALIGN;
  // as few workgroups as hold all rows, and in each no more waves than the rows need
  const int groups = (int)ceil_div64(a.queries, kRows), blocks = (groups + kMostWaves - 1) / kMostWaves;
  const int waves = (groups + blocks - 1) / blocks;
  if (!launchable((int64_t)blocks * a.heads * a.batch, waves)) return GEAR_HIP_ERANGE;
  by_attention_type(a, desc->dtype, [&](auto dim, auto type, auto mode) {
    typedef decltype(type) T;
    by_waves(waves, [&](auto w) {
      constexpr int kWaves = decltype(w)::value;
      hipLaunchKernelGGL((attention_kernel<T, decltype(dim)::value, decltype(mode)::value, kWaves>),
                         dim3((unsigned)blocks * a.heads * a.batch), dim3(kWaves * kWave), 0, as_stream(stream), a,
                         static_cast<T *>(out), lse, blocks);
    });
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
