// Gradients of attention over ranges of keys (gear_hip_attention_backward).
//
// With p = exp(s - lse), dp_ij = dout_i . v_j and delta_i = dout_i . out_i:
//   ds_ij = p_ij (dp_ij - delta_i) (1 - tanh^2);  dq = scale ds k;  dk = scale ds^T q;  dv = p^T dout
// Two launches, each of which works p out again, so that no sum is shared between workgroups and the same bits
// come out on every run: seven matrix products in place of five, for no atomics.
//   1. by queries (the layout of the forward pass): delta, dq, and the range that each 32 queries see
//   2. by keys: a wave holds 32 keys and passes over all queries (of all heads that share them) whose ranges
//      reach them; scores are not transposed here, a lane holds one key
#include <type_traits>

#include "attention.hpp"

namespace gearhip {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kTile = 64;

struct GradArgs {
  AttentionArgs a;
  const void *dout, *out;
  Strides gs;
  const float *lse;
  float *delta;    // [batch][heads][queries]
  i32x4 *bounds;   // [batch][ceil(queries/32)]: first, end, all_from, all_to
  void *dq, *dk, *dv;
  int blocks;      // workgroups of a head
};

template <typename T, int D, int MODE>
__global__ __launch_bounds__(kThreads) void attention_dq_kernel(GradArgs g) {
  __shared__ __attribute__((aligned(16))) T k_tile[kTile * D];
  __shared__ __attribute__((aligned(16))) T v_tile[kTile * D];
  __shared__ int ranges[kWaves][2];
  const AttentionArgs &a = g.a;
  const int tid = threadIdx.x, l = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = l >> 5;
  const int block = blockIdx.x % g.blocks, bh = blockIdx.x / g.blocks, head = bh % a.heads, b = bh / a.heads;
  const int kv_head = head / (a.heads / a.kv_heads);
  const int i = block * (kWaves * kRows) + wave * kRows + (l & 31);
  const bool row_there = i < a.queries;

  Seen seen;
  const int64_t row = (int64_t)b * a.queries + i;
  seen.set(row_there ? a.lo[row] : 0, row_there ? a.hi[row] : 0, a.keys);
  if (l == 0) ranges[wave][0] = seen.first, ranges[wave][1] = seen.end;
  const int group = block * kWaves + wave, groups = (a.queries + kRows - 1) / kRows;
  if (head == 0 && l == 0 && group < groups)
    g.bounds[(int64_t)b * groups + group] = i32x4{seen.first, seen.end, seen.all_from, seen.all_to};

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
  if (row_there) {
    const int64_t at = ((int64_t)b * a.heads + head) * a.queries + i;
    if (half == 0) g.delta[at] = delta;
    if (!seen.empty()) lse_log2 = g.lse[at] * kLog2e;
  }
  __syncthreads();
  int first = INT_MAX, end = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) first = min(first, ranges[w][0]), end = max(end, ranges[w][1]);

  const Scores<MODE> scores(a, head);
  const int place = i + a.keys - a.queries;
  f32x16 dq[D / 32] = {};
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
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int kk = k0 + kb * 32;
      if (!seen.touches(kk, kk + 32)) continue;
      const bool whole = seen.covers(kk, kk + 32);
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int x = 0; x < D / 16; ++x) s = mfma(rows_frag<T, D>(k_tile, kb * 32, x), q[x], s);
#pragma unroll
      for (int x = 0; x < D / 16; ++x) dp = mfma(rows_frag<T, D>(v_tile, kb * 32, x), dout[x], dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = kk + result_row(r);
        float shrink;
        const float z = scores.z(s[r], (float)(place - key), shrink);
        float ds = exp2_fast(fmaf(z, scores.factor, scores.offset - lse_log2)) * (dp[r] - delta);
        if (MODE & kCap) ds *= shrink;
        if (!whole && (uint32_t)(key - seen.lo) >= (uint32_t)(seen.hi - seen.lo)) ds = 0;
        s[r] = ds;
      }
      const vec8<T> d0 = packed<T, 0>(s), d1 = packed<T, 1>(s);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        dq[db] = mfma(columns_frag<T, D>(k_tile, kb * 32, db), d0, dq[db]);
        dq[db] = mfma(columns_frag<T, D>(k_tile, kb * 32 + 16, db), d1, dq[db]);
      }
    }
  }
  if (!row_there) return;
  T *to = static_cast<T *>(g.dq) + (row * a.heads + head) * a.dim;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = db * 32 + 8 * x + 4 * half;
      vec4<T> y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(seen.empty() ? 0.f : dq[db][4 * x + e] * a.scale);
      if (d < a.dim) *reinterpret_cast<vec4<T> *>(to + d) = y;
    }
}

// p is at most 1 and often far below the smallest normal f16, so it is multiplied with dout 2^10 times as large.
template <typename T>
constexpr float kRaise = std::is_same<T, f16>::value ? 10.f : 0.f;

template <typename T, int D, int MODE>
__global__ __launch_bounds__(kThreads) void attention_dkv_kernel(GradArgs g) {
  __shared__ __attribute__((aligned(16))) T q_tile[kTile * D];
  __shared__ __attribute__((aligned(16))) T g_tile[kTile * D];
  __shared__ __attribute__((aligned(16))) float row_lse[kTile], row_delta[kTile];
  __shared__ __attribute__((aligned(16))) int row_lo[kTile], row_hi[kTile];
  const AttentionArgs &a = g.a;
  const int tid = threadIdx.x, l = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kWave), half = l >> 5;
  const int block = blockIdx.x % g.blocks, bh = blockIdx.x / g.blocks, kv_head = bh % a.kv_heads, b = bh / a.kv_heads;
  const int shared = a.heads / a.kv_heads;
  const int block_key = block * (kWaves * kRows), wave_key = block_key + wave * kRows, key = wave_key + (l & 31);
  const bool key_there = key < a.keys;

  vec8<T> k[D / 16], v[D / 16];
  own_row_frags<T, D>(k, static_cast<const T *>(a.k) + b * a.ks.batch + key * a.ks.token + kv_head * a.ks.head, a.dim, key_there);
  own_row_frags<T, D>(v, static_cast<const T *>(a.v) + b * a.vs.batch + key * a.vs.token + kv_head * a.vs.head, a.dim, key_there);
  f32x16 dk[D / 32] = {}, dv[D / 32] = {};
  const int groups = (a.queries + kRows - 1) / kRows, tiles = (a.queries + kTile - 1) / kTile;
  const i32x4 *bounds = g.bounds + (int64_t)b * groups;
  const i32x4 nothing = {INT_MAX, 0, 0, 0};

  for (int x = 0; x < shared; ++x) {
    const int head = kv_head * shared + x;
    const Scores<MODE> scores(a, head);
    const T *q_rows = static_cast<const T *>(a.q) + b * a.qs.batch + head * a.qs.head;
    const T *g_rows = static_cast<const T *>(g.dout) + b * g.gs.batch + head * g.gs.head;
    const int64_t stats = ((int64_t)b * a.heads + head) * a.queries;
    for (int tile_base = 0; tile_base < tiles; tile_base += kWave) {
      // which of the next 64 tiles of queries see any of the workgroup's keys
      bool reaches = false;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int group = 2 * (tile_base + l) + y;
        if (group < groups) reaches |= bounds[group][0] < block_key + kWaves * kRows && bounds[group][1] > block_key;
      }
      for (uint64_t left = wave_ballot(reaches); left != 0; left &= left - 1) {
        const int tile = tile_base + (int)__builtin_ctzll(left), i0 = tile * kTile;
        __syncthreads();
        {
          auto there = [&](int r) {
            const int64_t row = (int64_t)b * a.queries + i0 + r;
            return i0 + r < a.queries && min(a.hi[row], a.keys) > max(a.lo[row], 0);
          };
          TileLoad<T, D, kTile, kThreads> q_load, g_load;
          q_load.load(q_rows + i0 * a.qs.token, a.qs.token, tid, a.dim, there);
          g_load.load(g_rows + i0 * g.gs.token, g.gs.token, tid, a.dim, there);
          if (tid < kTile) {
            const bool ok = there(tid);
            const int64_t row = (int64_t)b * a.queries + i0 + tid;
            row_lse[tid] = ok ? g.lse[stats + i0 + tid] * kLog2e : INFINITY;
            row_delta[tid] = ok ? g.delta[stats + i0 + tid] : 0;
            row_lo[tid] = ok ? max(a.lo[row], 0) : 0;
            row_hi[tid] = ok ? min(a.hi[row], a.keys) : 0;
          }
          q_load.store(q_tile, tid);
          g_load.store(g_tile, tid);
        }
        __syncthreads();
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const i32x4 reach = 2 * tile + qb < groups ? bounds[2 * tile + qb] : nothing;
          if (reach[0] >= wave_key + kRows || reach[1] <= wave_key) continue;
          const bool whole = reach[2] <= wave_key && reach[3] >= wave_key + kRows;
          f32x16 s = {}, dp = {};
#pragma unroll
          for (int y = 0; y < D / 16; ++y) s = mfma(rows_frag<T, D>(q_tile, qb * 32, y), k[y], s);
#pragma unroll
          for (int y = 0; y < D / 16; ++y) dp = mfma(rows_frag<T, D>(g_tile, qb * 32, y), v[y], dp);
          constexpr float lower = 1.f / (1 << (int)kRaise<T>);
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const int r0 = qb * 32 + 8 * z + 4 * half;
            const f32x4 lse = *reinterpret_cast<const f32x4 *>(row_lse + r0), delta = *reinterpret_cast<const f32x4 *>(row_delta + r0);
            i32x4 lo = {}, hi = {};
            if (!whole) lo = *reinterpret_cast<const i32x4 *>(row_lo + r0), hi = *reinterpret_cast<const i32x4 *>(row_hi + r0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 4 * z + e;
              float shrink;
              const float z = scores.z(s[r], (float)(i0 + r0 + e + a.keys - a.queries - key), shrink);
              float p = exp2_fast(fmaf(z, scores.factor, scores.offset + kRaise<T> - lse[e]));
              float ds = p * (lower * dp[r] - lower * delta[e]);
              if (MODE & kCap) ds *= shrink;
              if (!whole && (uint32_t)(key - lo[e]) >= (uint32_t)(hi[e] - lo[e])) p = ds = 0;
              s[r] = p, dp[r] = ds;
            }
          }
          const vec8<T> p0 = packed<T, 0>(s), p1 = packed<T, 1>(s), d0 = packed<T, 0>(dp), d1 = packed<T, 1>(dp);
#pragma unroll
          for (int db = 0; db < D / 32; ++db) {
            dv[db] = mfma(columns_frag<T, D>(g_tile, qb * 32, db), p0, dv[db]);
            dv[db] = mfma(columns_frag<T, D>(g_tile, qb * 32 + 16, db), p1, dv[db]);
            dk[db] = mfma(columns_frag<T, D>(q_tile, qb * 32, db), d0, dk[db]);
            dk[db] = mfma(columns_frag<T, D>(q_tile, qb * 32 + 16, db), d1, dk[db]);
          }
        }
      }
    }
  }
  if (!key_there) return;
  const int64_t to = (((int64_t)b * a.keys + key) * a.kv_heads + kv_head) * a.dim;
  constexpr float lower = 1.f / (1 << (int)kRaise<T>);
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = db * 32 + 8 * x + 4 * half;
      vec4<T> y, z;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = (T)(dk[db][4 * x + e] * a.scale);
        z[e] = (T)(dv[db][4 * x + e] * lower);
      }
      if (d < a.dim) {
        *reinterpret_cast<vec4<T> *>(static_cast<T *>(g.dk) + to + d) = y;
        *reinterpret_cast<vec4<T> *>(static_cast<T *>(g.dv) + to + d) = z;
      }
    }
}

size_t delta_bytes(int64_t batch, int64_t queries, int64_t heads) {
  return align_up((size_t)(batch * heads * queries) * sizeof(float), 256);
}

}  // namespace
}  // namespace gearhip

using namespace gearhip;

extern "C" size_t gear_hip_attention_backward_workspace_bytes(int64_t batch, int64_t queries, int64_t heads) {
  if (batch <= 0 || queries <= 0 || heads <= 0) return 0;
  return delta_bytes(batch, queries, heads) + (size_t)(batch * ceil_div64(queries, kRows)) * sizeof(i32x4);
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
  g.delta = static_cast<float *>(workspace);
  g.bounds = reinterpret_cast<i32x4 *>(static_cast<char *>(workspace) + delta_bytes(a.batch, a.queries, a.heads));
  g.dq = dq, g.dk = dk, g.dv = dv;
  by_attention_type(a, desc->dtype, [&](auto dim, auto type, auto mode) {
    typedef decltype(type) T;
    constexpr int D = decltype(dim)::value;
    constexpr int kMode = decltype(mode)::value;
    g.blocks = (int)ceil_div64(a.queries, kWaves * kRows);
    if (g.blocks > 0)
      hipLaunchKernelGGL((attention_dq_kernel<T, D, kMode>), dim3((unsigned)g.blocks * a.heads * a.batch),
                         dim3(kThreads), 0, as_stream(stream), g);
    g.blocks = (int)ceil_div64(a.keys, kWaves * kRows);
    if (g.blocks > 0)
      hipLaunchKernelGGL((attention_dkv_kernel<T, D, kMode>), dim3((unsigned)g.blocks * a.kv_heads * a.batch),
                         dim3(kThreads), 0, as_stream(stream), g);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
