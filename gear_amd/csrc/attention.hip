// Attention over ranges of keys, forward (gear_hip_attention).
//
// A workgroup takes 128 queries of one head, 32 a wave; tiles of 64 keys pass through LDS.  The softmax runs
// along: a lane holds its query's maximum m and sum l so far, in exponents of 2, and the sums of p v are
// rescaled when m grows.  Tiles outside a wave's ranges are passed over, tiles that all its rows see
// in full need no comparison.
#include <type_traits>

#include "attention.hpp"

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
  if (!(d->scale > 0) || !(d->scale < 1e30f) || !(d->cap >= 0) || !(d->cap < 1e30f)) return GEAR_HIP_EINVAL;
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

constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kTile = 64;  // keys of a tile

template <typename T, int D, bool SHAPED>
__global__ __launch_bounds__(kThreads) void attention_kernel(AttentionArgs a, T *__restrict__ out,
                                                             float *__restrict__ lse, int blocks) {
  __shared__ __attribute__((aligned(16))) T k_tile[kTile * D];
  __shared__ __attribute__((aligned(16))) T v_tile[kTile * D];
  __shared__ int ranges[kWaves][2];
  const int tid = threadIdx.x, l = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = l >> 5;
  const int block = blockIdx.x % blocks, bh = blockIdx.x / blocks, head = bh % a.heads, b = bh / a.heads;
  const int kv_head = head / (a.heads / a.kv_heads);
  const int i = block * (kWaves * kRows) + wave * kRows + (l & 31);
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
  for (int w = 0; w < kWaves; ++w) first = min(first, ranges[w][0]), end = max(end, ranges[w][1]);

  const Shape shape(a, head);
  const int place = i + a.keys - a.queries;
  f32x16 o[D / 32] = {};
  float m = -INFINITY, sum = 0;

  const T *k_rows = static_cast<const T *>(a.k) + b * a.ks.batch + kv_head * a.ks.head;
  const T *v_rows = static_cast<const T *>(a.v) + b * a.vs.batch + kv_head * a.vs.head;
  TileLoad<T, D, kTile, kThreads> k_load, v_load;
  auto load = [&](int k0) {
    auto there = [&](int r) { return k0 + r >= first && k0 + r < end; };
    k_load.load(k_rows + k0 * a.ks.token, a.ks.token, tid, a.dim, there);
    v_load.load(v_rows + k0 * a.vs.token, a.vs.token, tid, a.dim, there);
  };
  int k0 = first < end ? first / kTile * kTile : 0;
  if (k0 < end) load(k0);
  for (; k0 < end; k0 += kTile) {
    __syncthreads();
    k_load.store(k_tile, tid);
    v_load.store(v_tile, tid);
    __syncthreads();
    if (k0 + kTile < end) load(k0 + kTile);
    if (!seen.touches(k0, k0 + kTile)) continue;
    const bool whole = seen.covers(k0, k0 + kTile);

    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = f32x16{};
#pragma unroll
      for (int x = 0; x < D / 16; ++x) s[kb] = mfma(rows_frag<T, D>(k_tile, kb * 32, x), q[x], s[kb]);
    }
    float top = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = k0 + kb * 32 + result_row(r);
        float shrink, y = SHAPED ? shape.score(s[kb][r], place - key, shrink) : s[kb][r] * a.scale_log2;
        if (!whole && (uint32_t)(key - seen.lo) >= (uint32_t)(seen.hi - seen.lo)) y = -INFINITY;
        s[kb][r] = y;
        top = fmaxf(top, y);
      }
    top = fmaxf(m, fmaxf(top, other_half(top)));
    const float from = top == -INFINITY ? 0.f : top;  // (no key seen yet)
    const float rescale = exp2_fast(m - from);
    m = top;
    sum *= rescale;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) o[db] *= rescale;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[kb][r] = exp2_fast(s[kb][r] - from);
        sum += s[kb][r];
      }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const vec8<T> p0 = packed<T, 0>(s[kb]), p1 = packed<T, 1>(s[kb]);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        o[db] = mfma(columns_frag<T, D>(v_tile, kb * 32, db), p0, o[db]);
        o[db] = mfma(columns_frag<T, D>(v_tile, kb * 32 + 16, db), p1, o[db]);
      }
    }
  }

  sum += other_half(sum);
  if (!row_there) return;
  const bool empty = seen.empty();
  const float over = 1.f / sum;
  if (lse != nullptr && half == 0)
    lse[((int64_t)b * a.heads + head) * a.queries + i] = empty ? -INFINITY : (m + __builtin_log2f(sum)) * kLn2;
  T *to = out + (row * a.heads + head) * a.dim;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + 8 * g + 4 * half;
      vec4<T> x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (T)(empty ? 0.f : o[db][4 * g + e] * over);
      if (d < a.dim) *reinterpret_cast<vec4<T> *>(to + d) = x;
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
  const int blocks = (int)ceil_div64(a.queries, kWaves * kRows);
  by_attention_type(a, desc->dtype, [&](auto dim, auto type, auto shaped) {
    typedef decltype(type) T;
    hipLaunchKernelGGL((attention_kernel<T, decltype(dim)::value, decltype(shaped)::value>),
                       dim3((unsigned)blocks * a.heads * a.batch), dim3(kThreads), 0, as_stream(stream), a,
                       static_cast<T *>(out), lse, blocks);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
