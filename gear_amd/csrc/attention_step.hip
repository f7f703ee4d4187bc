// Attention of the newest tokens of rollouts over their caches (gear_hip_attention_step).
//
// Few queries, many keys: what counts is reading the caches once, at the rate of memory.  The queries of
// all heads that share a key head are the rows of one matrix operand (32 at a time; most calls have fewer, the
// unused rows cost nothing that memory would not), so every key is read once for 32 of them; with more, each 32 read the keys
// again, past the caches.  A rollout's
// keys are split over `splits` workgroups and within one over its waves, 32 keys at a time.  A wave has two tiles of K and
// V in a piece of LDS of its own, filled past the caches (nobody reads a key again) while the one before is worked on, so no
// wave waits for another before the end.  What the parts of a split have -- maximum, sum, sums of p v -- is joined by a second
// launch, in a fixed order.
// Bound by memory.  bf16: 256 rollouts of up to 3000 keys, 8 heads of 64: 142 us, 5.3 TB/s of the keys that are seen; 3 of up to 131071,
// 16 heads of 128 over 2: 66 us (3.1 TB/s; 49 at best) and 6 for the join.  There a workgroup fills a CU's LDS alone, and its start
// and end are time in which the CU asks for little: two waves a workgroup 63 us, 64 parts 62, 256 parts 84, parts of
// one size 75.
#include <type_traits>

#include "attention_exact.hpp"

namespace gearhip {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kMaxSplits = 128;

struct StepArgs {
  AttentionArgs a;
  int row_blocks, splits;
  float *part_o;   // [batch][kv_heads][row_blocks][splits][32][dim]
  float2 *part_ml; // [batch][kv_heads][row_blocks][splits][32]
  void *out;
};

// Row r of a key head's rows, worked out alone (max_log2: maximum and sum of its scores, without the offset).
template <typename T, int MODE>
__device__ __forceinline__ void mend_row(const StepArgs &g, int64_t b, int r, int kv_head, float max_log2) {
  const AttentionArgs &a = g.a;
  const int shared = a.heads / a.kv_heads, t = r / shared, head = kv_head * shared + r % shared;
  const int64_t row = b * a.queries + t;
  const int lo = max(a.lo[row], 0), hi = min(a.hi[row], a.keys);
  const Scores<MODE> scores(a, head);
  Pair x;
  if (hi > lo && exact_out<T, MODE>(x, static_cast<const T *>(a.q) + b * a.qs.batch + t * a.qs.token + head * a.qs.head,
                                    static_cast<const T *>(a.k) + b * a.ks.batch + kv_head * a.ks.head, a.ks.token,
                                    static_cast<const T *>(a.v) + b * a.vs.batch + kv_head * a.vs.head, a.vs.token, lo, hi, a.dim,
                                    hi - 1, max_log2 + scores.offset, scores))
    store_pair(static_cast<T *>(g.out) + (row * a.heads + head) * a.dim, x, a.dim);
}

// WHOLE: rows have D elements.  (Chosen inside the kernel, that costs a wave that is alone on its SIMD 5 %: 3 rollouts of up to 131071
// keys 68 us for 64.)
template <typename T, int D, int MODE, bool WHOLE>
__global__ __launch_bounds__(kThreads, 1) void attention_step_kernel(StepArgs g) {
  constexpr int kAsks = D / 8;  // instructions that ask for a tile of K and V
  constexpr size_t kTileBytes = sizeof(T) * kRows * D, kJoinBytes = sizeof(float) * kRows * D;
  constexpr size_t kOwnBytes = 4 * kTileBytes > kJoinBytes ? 4 * kTileBytes : kJoinBytes;
  __shared__ __attribute__((aligned(16))) char memory[kWaves][kOwnBytes];  // two tiles of K and V a wave; its sums
  __shared__ float2 joined_ml[kWaves][kRows];
  const AttentionArgs &a = g.a;
  const int l = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = l >> 5;
  // Workgroups go round the 8 dies: the key heads of a part, whose rows alternate in memory, run on one die (256 rollouts,
  // 8 heads of 64: 142 us, against 161 on any die), the parts go round, so that no die has the short rollouts only.
  const int die_index = blockIdx.x / 8, kv_head = die_index % a.kv_heads;
  const int part_index = die_index / a.kv_heads * 8 + blockIdx.x % 8;
  if (part_index >= a.batch * g.row_blocks * g.splits) return;
  const int split = part_index % g.splits, block = part_index / g.splits % g.row_blocks, b = part_index / g.splits / g.row_blocks;
  const int shared = a.heads / a.kv_heads, rows = a.queries * shared;
  const int r_own = block * kRows + (l & 31), i = r_own / shared, head = kv_head * shared + r_own % shared;
  const bool row_there = r_own < rows;
  T *k_tile[2], *v_tile[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    k_tile[x] = reinterpret_cast<T *>(memory[wave] + x * 2 * kTileBytes);
    v_tile[x] = reinterpret_cast<T *>(memory[wave] + (x * 2 + 1) * kTileBytes);
  }

  Seen seen;
  const int64_t row = (int64_t)b * a.queries + i;
  seen.set(row_there ? a.lo[row] : 0, row_there ? a.hi[row] : 0, a.keys);
  vec8<T> q[D / 16];
  own_row_frags<T, D>(q, static_cast<const T *>(a.q) + b * a.qs.batch + i * a.qs.token + head * a.qs.head, a.dim, !seen.empty());
  // this workgroup's part of the keys that the rows see, [first, end)
  const int length = seen.first < seen.end ? seen.end - seen.first : 0;
  const int part = ((length + g.splits - 1) / g.splits + kRows - 1) / kRows * kRows;
  const int first = (int)min((int64_t)seen.end, (length > 0 ? seen.first : 0) + (int64_t)split * part);
  const int end = (int)min((int64_t)seen.end, (int64_t)first + part);

  const Scores<MODE> scores(a, row_there ? head : 0, std::false_type());
  const TileReader<T, D> reader;
  f32x16 o[D / 32] = {};
  float m = -INFINITY;  // of z
  Sum sums;
  const Stage<T, D, kRows, true, !WHOLE> k_rows(static_cast<const T *>(a.k) + b * a.ks.batch + kv_head * a.ks.head, a.ks.token, first, end, a.dim);
  const Stage<T, D, kRows, true> v_rows(static_cast<const T *>(a.v) + b * a.vs.batch + kv_head * a.vs.head, a.vs.token, first, end, a.dim);
  constexpr int kStep = kWaves * kRows;
  auto ask = [&](int k0, int to) __attribute__((always_inline)) {
    k_rows.template ask<1>(k_tile[to], k0, 0);
    v_rows.template ask<1>(v_tile[to], k0, 0);
  };
  auto tile = [&](int k0, int from_buffer) __attribute__((always_inline)) {
    f32x16 s = {};
#pragma unroll
    for (int x = 0; x < D / 16; ++x) s = mfma(reader.rows(k_tile[from_buffer], 0, x), q[x], s);
    const float ahead = (float)(seen.hi - 1 - k0 - 4 * half);
    scores.cap_far(s);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = scores.z(scores.in_tile(s[r]), ahead - (float)(8 * (r >> 2) + (r & 3)));
    if (__builtin_expect(k0 + kRows > end || !seen.covers(k0, k0 + kRows), 0)) {
      const uint32_t from_lo = (uint32_t)(k0 + 4 * half - seen.lo), count = (uint32_t)(min(seen.hi, end) - seen.lo);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (from_lo + (uint32_t)(8 * (r >> 2) + (r & 3)) >= count || seen.lo >= end) s[r] = -INFINITY;
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
    const float from = m == -INFINITY ? 0.f : kLevel<T> - m * scores.factor;
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
      o[db] = mfma(reader.columns(v_tile[from_buffer], 0, db), p0, o[db]);
      o[db] = mfma(reader.columns(v_tile[from_buffer], 16, db), p1, o[db]);
    }
  };
  int k0 = first + wave * kRows;
  if (!WHOLE)
    for (int x = 0; x < 2; ++x) k_rows.clear_beyond(k_tile[x]);
  if (k0 < end) ask(k0, 0);
  if (k0 + kStep < end) ask(k0 + kStep, 1);
  for (int buffer = 0; k0 < end; k0 += kStep, buffer ^= 1) {
    if (k0 + kStep < end)
      staged_wait<kAsks>();  // the next tile may still be on its way
    else
      staged_wait<0>();
    tile(k0, buffer);
    if (k0 + 2 * kStep < end) ask(k0 + 2 * kStep, buffer);
  }
  const float sum = sum_of_halves(sums.x);

  // join the waves (each reads and writes its own memory until here)
  m = m == -INFINITY ? m : m * scores.factor - kLevel<T>;
  float *own_sums = reinterpret_cast<float *>(memory[wave]);
  wave_lds_sync();
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      *reinterpret_cast<f32x4 *>(own_sums + (l & 31) * D + column_of<D>(db, 8 * x) + 4 * half) =
          f32x4{o[db][4 * x], o[db][4 * x + 1], o[db][4 * x + 2], o[db][4 * x + 3]};
  if (half == 0) joined_ml[wave][l & 31] = make_float2(m, sum);
  __syncthreads();
  const int here = min(kRows, rows - block * kRows);
  bool bad = false;
  for (int x = threadIdx.x; x < here * a.dim; x += kThreads) {
    const int r = x / a.dim, d = x - r * a.dim;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, joined_ml[w][r].x);
    const float from = top == -INFINITY ? 0.f : top;
    float total = 0, y = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float share = exp2_fast(joined_ml[w][r].x - from);
      total += share * joined_ml[w][r].y;
      y += share * reinterpret_cast<const float *>(memory[w])[r * D + d];
    }
    if (g.splits == 1) {
      const int at = block * kRows + r, t = at / shared, h = kv_head * shared + at % shared;
      const int64_t q_row = (int64_t)b * a.queries + t;
      const bool none = min(a.hi[q_row], a.keys) <= max(a.lo[q_row], 0);
      static_cast<T *>(g.out)[(q_row * a.heads + h) * a.dim + d] = (T)(none ? 0.f : y / total);
      bad = bad || (!none && !(fabsf(y) < INFINITY));
    } else {
      const int64_t at = ((((int64_t)b * a.kv_heads + kv_head) * g.row_blocks + block) * g.splits + split) * kRows + r;
      g.part_o[at * a.dim + d] = y;
      if (d == 0) g.part_ml[at] = make_float2(top, total);
    }
  }
  if (g.splits > 1 || __builtin_expect(!__syncthreads_or(bad), 1)) return;
  for (int r = wave; r < here; r += kWaves) {  // (which rows it is was not kept: all of them are looked at)
    float top = -INFINITY, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, joined_ml[w][r].x);
    const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += exp2_fast(joined_ml[w][r].x - from) * joined_ml[w][r].y;
    mend_row<T, MODE>(g, b, block * kRows + r, kv_head, top + __builtin_log2f(total));
  }
}

// One workgroup a query and head: the parts of its split, joined.  Every thread takes 4 elements of each eighth part (or
// more often, with shorter rows), so that the loads of a row's parts are in flight together.
template <typename T, int MODE>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(StepArgs g) {
  __shared__ float share[kMaxSplits];
  __shared__ f32x4 sums[kThreads];
  const AttentionArgs &a = g.a;
  const int shared = a.heads / a.kv_heads;
  const int64_t q_row = blockIdx.x / a.heads;
  const int head = blockIdx.x % a.heads, kv_head = head / shared;
  const int64_t b = q_row / a.queries;
  const int r = (int)(q_row - b * a.queries) * shared + head % shared;
  const int64_t unit = (b * a.kv_heads + kv_head) * g.row_blocks + r / kRows;
  const int64_t first = unit * g.splits * kRows + r % kRows;  // part p: first + p * kRows
  // (every wave works the shares out for itself)
  const int l = lane_id();
  float top = -INFINITY, total = 0;
  for (int p = l; p < g.splits; p += kWave) top = fmaxf(top, g.part_ml[first + (int64_t)p * kRows].x);
#pragma unroll
  for (int x = 1; x < kWave; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
  const float from = top == -INFINITY ? 0.f : top;
  for (int p = l; p < g.splits; p += kWave) {
    const float2 ml = g.part_ml[first + (int64_t)p * kRows];
    const float s = exp2_fast(ml.x - from);
    total += s * ml.y;
    share[p] = s;
  }
#pragma unroll
  for (int x = 1; x < kWave; x *= 2) total += __shfl_xor(total, x);
  __syncthreads();
  const int lanes = a.dim / 4, groups = kThreads / lanes, group = threadIdx.x / lanes, d = threadIdx.x % lanes * 4;
  f32x4 y = {};
  if (group < groups)
#pragma unroll 4
    for (int p = group; p < g.splits; p += groups)
      y += share[p] * *reinterpret_cast<const f32x4 *>(g.part_o + (first + (int64_t)p * kRows) * a.dim + d);
  sums[threadIdx.x] = y;
  __syncthreads();
  bool bad = false;
  if (group == 0) {
    for (int x = 1; x < groups; ++x) y += sums[x * lanes + threadIdx.x];
    const bool none = min(a.hi[q_row], a.keys) <= max(a.lo[q_row], 0);
    vec4<T> z;
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = (T)(none ? 0.f : y[e] / total), bad = bad || (!none && !(fabsf(y[e]) < INFINITY));
    *reinterpret_cast<vec4<T> *>(static_cast<T *>(g.out) + (q_row * a.heads + head) * a.dim + d) = z;
  }
  if (__builtin_expect(__syncthreads_or(bad), 0) && threadIdx.x < kWave)
    mend_row<T, MODE>(g, b, r, kv_head, top + __builtin_log2f(total));
}

int64_t row_blocks_of(int64_t queries, int64_t heads, int64_t kv_heads) {
  return ceil_div64(queries * (heads / kv_heads), kRows);
}

// Parts of a rollout's keys: enough workgroups for the GPU, at least 256 keys each.
int splits_of(int64_t units, int64_t keys) {
  int64_t n = ceil_div64(1024, units < 1 ? 1 : units);
  const int64_t most = ceil_div64(keys, 256);
  if (n > most) n = most;
  return (int)(n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : n);
}

}  // namespace
}  // namespace gearhip

using namespace gearhip;

extern "C" size_t gear_hip_attention_step_workspace_bytes(int64_t batch, int64_t queries, int64_t keys, int64_t heads,
                                                          int64_t kv_heads, int64_t head_dim) {
  if (batch <= 0 || queries <= 0 || keys < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0) return 0;
  const int64_t units = batch * kv_heads * row_blocks_of(queries, heads, kv_heads);
  const int splits = splits_of(units, keys);
  return splits == 1 ? 0 : (size_t)(units * splits * kRows) * (head_dim * sizeof(float) + sizeof(float2));
}

extern "C" int gear_hip_attention_step(const gear_hip_attention_desc *desc, void *out, void *workspace,
                                       size_t workspace_bytes, void *stream) {
  StepArgs g = {};
  const int rc = attention_args(desc, g.a);
  if (rc < 0) return rc;
  const AttentionArgs &a = g.a;
  if (rc == 1 || a.queries == 0) return 0;
  if (out == nullptr) return GEAR_HIP_EINVAL;
  if (a.queries > (1 << 20) || (int64_t)a.queries * a.heads * a.batch > INT_MAX) return GEAR_HIP_ERANGE;
  const size_t want = gear_hip_attention_step_workspace_bytes(a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.dim);
  if (want > 0 && (workspace == nullptr || workspace_bytes < want)) return GEAR_HIP_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(out) % 16 != 0 || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return GEAR_HIP_EALIGN;
  g.row_blocks = (int)row_blocks_of(a.queries, a.heads, a.kv_heads);
  const int64_t units = (int64_t)a.batch * a.kv_heads * g.row_blocks;
  g.splits = splits_of(units, a.keys);
  const int64_t workgroups = ceil_div64((int64_t)a.batch * g.row_blocks * g.splits, 8) * 8 * a.kv_heads;
  if (!launchable(workgroups, kWaves)) return GEAR_HIP_ERANGE;  // (the join is for fewer than 1024 blocks of 32 rows)
  g.part_o = static_cast<float *>(workspace);
  g.part_ml = reinterpret_cast<float2 *>(g.part_o + units * g.splits * kRows * a.dim);
  g.out = out;
  by_attention_type(a, desc->dtype, [&](auto dim, auto type, auto mode) {
    typedef decltype(type) T;
    constexpr int D = decltype(dim)::value, kMode = decltype(mode)::value;
    auto step = [&](auto whole) {
      hipLaunchKernelGGL((attention_step_kernel<T, D, kMode, decltype(whole)::value>), dim3((unsigned)workgroups), dim3(kThreads), 0,
                         as_stream(stream), g);
    };
    if (a.dim == D)
      step(std::true_type());
    else
      step(std::false_type());
    if (g.splits > 1)
      hipLaunchKernelGGL((attention_join_kernel<T, decltype(mode)::value>), dim3((unsigned)(a.queries * a.heads * a.batch)), dim3(kThreads), 0,
                         as_stream(stream), g);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
