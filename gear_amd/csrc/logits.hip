// What is asked of rows of logits: log probabilities of given tokens, entropies, the best tokens, the divergence from a
// teacher's best tokens, and the gradients (gear_hip_token_log_probs, gear_hip_distill and the calls beside them).
//
// With x a row, m its maximum, d_j = scale (x_j - m), S = sum exp d, A = sum d exp d:
//   lse = scale m + log S,  log p_t = d_t - log S,  entropy = log S - A / S
// which leaves no difference of large numbers.  A logit of -inf is a probability of 0 and has no part in A.  The
// gradient is p_j (alpha + beta log p_j), with p as exact as lse is in 32 bits, plus what the given token (+dlogp) or the
// teacher's entries (-dloss q) add: after the row is written the few columns concerned are written again.
//
// All are bound by memory: a row is read once and held in registers as it came, its maximum is taken before any exponential
// (an element costs six instructions of 4 cycles and an exponential of 16, which leaves room for 9 TB/s of bfloat16).
// Rows of up to 256 vectors of 16 bytes: a wave or a part of one.  Wider ones: a workgroup of 256 threads for every part of a
// row of at most 17 vectors a thread, or of 1024 where rows are few; parts are joined by a second launch.
//
// The best k: groups of lanes have a maximum each, 64 in all; the k-th largest of those is a bound below which none of
// the best k lies, so that few elements are left to be put in order.  Where more are left than a list holds (rows of equal
// logits, or of fewer that are allowed than are asked for), or a row holds NaN or infinity, the bound is taken once more of
// pairs of logit and column, which all differ; where that leaves too many as well, they are taken one after the other.
// The best one alone is the row's maximum, of which only the column is looked for.
//
// Measured: 16384 x 33025 bf16 155-190 us forward (with how memory lies; 5.6-6.8 TB/s), 366 backward (5.8 TB/s), rows of 20001 and
// 50001 of as much memory 187 and 179 + 20, 377 and 375; 8191 x 33025 against 32
// entries 100 and 191; 184320 x 1024 bf16 95 and 117 (4.0 and 6.5 TB/s); 184320 x 18 in 32 bits 8 and 8; 64 x 65537 fp16 with the best
// eight 11; 4096 x 33024 bf16 46, 54 where no cache has any of it, with the best 32 76 and 79 (64: 180; of equal logits 283 and 345,
// one after the other 2230 and 4350).
// The wide rows' forward with 128, 512 or 1024 threads of 34, 9 or 5 vectors in place of 256 of 17: 16384 x 33025 220, 219 and 394 for
// 185, 4096 x 33024 with the best 32 106, 107 and 165 for 75-84.
#include <algorithm>

#include "rows.hpp"

namespace gearhip {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxTop = 64;     // best tokens, and a teacher's entries
constexpr int kHeld = 17;       // vectors of a thread
constexpr int kHeldFew = 12;    // ... of a workgroup of 1024
constexpr int kJoined = 4096;   // entries that a join puts in order
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kLow = -1e30f;   // below any logit that is allowed
constexpr float kLeast = -1e4f;  // below any exponent that counts

struct LogitsArgs {
  const void *logits;
  int64_t stride, rows;
  int vocab;
  float scale, scale2;  // scale2: scale log2 e
  // log probabilities
  const void *tokens;  // or null
  int wide;            // tokens (and entries) in 64 bits
  int top;
  float *log_probs, *entropy, *lse, *top_log_probs;
  int64_t *top_tokens;
  // distillation
  const void *entries;
  const float *teacher;
  int count;
  float *loss;
  bool once;  // the logits are more than the caches hold
  // rows in parts
  int parts, part_vecs;
  float *stats;     // [rows][parts][4]: m, S, A
  uint64_t *lists;  // [rows][parts][top]
  // gradients
  const float *dlog_probs, *dentropy, *dloss, *lse_in, *entropy_in;
  void *dlogits;
};

enum { kLogProbs, kDistill };
enum { kNoBest, kOneBest, kSomeBest };

// ---- order: larger first, the lower index first among equals, NaN before all --------------------------------------
__device__ __forceinline__ uint64_t entry_of(float x, int column) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 is 0)
  const uint32_t key = x != x ? ~1u : (int32_t)b < 0 ? ~b : b | 0x80000000u;
  return (uint64_t)key << 32 | (uint32_t)~column;
}
__device__ __forceinline__ float entry_value(uint64_t e) {
  const uint32_t key = (uint32_t)(e >> 32);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ int entry_column(uint64_t e) { return (int)~(uint32_t)e; }

template <int kLanes>
__device__ __forceinline__ uint64_t lanes_max64(uint64_t x) {
#pragma unroll
  for (int by = 1; by < kLanes; by *= 2) {
    const uint64_t y = __shfl_xor((unsigned long long)x, by);
    x = y > x ? y : x;
  }
  return x;
}

// ---- the statistics of a row ------------------------------------------------------------------------------------
struct Stats {
  float m, s, a;  // maximum, S, A / ln 2 (or 0)
};
// (a row without a finite logit has S = 0 that way round, not NaN)
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.f : m; }

template <typename T>
__device__ __forceinline__ Raw<T> nothing() {
  Raw<T> x;
#pragma unroll
  for (int e = 0; e < kPer<T>; ++e) x[e] = (T)-INFINITY;
  return x;
}
// a vector of a row, -inf where it has no elements of its own
template <typename T>
__device__ __forceinline__ Raw<T> load_logits(const T *row, const Slot<T> &s, bool tiny) {
  if (!s.any()) return nothing<T>();
  Raw<T> x = load_slot<T>(row, s, tiny);
  if (!s.whole()) {
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e)
      if (!s.own(e)) x[e] = (T)-INFINITY;
  }
  return x;
}
// A row of more than a vector, cut where addresses are multiples of 16 bytes: elements before the first such place, whole
// vectors, elements behind the last.  (16384 odd rows of 66 KB, read at any address 213 us, cut so 170.)
template <typename T>
struct Cut {
  int head, vecs, tail;
  __device__ __forceinline__ Cut(const T *row, int width) {
    head = (kPer<T> - misaligned(row)) & (kPer<T> - 1);
    vecs = (width - head) / kPer<T>;
    tail = width - head - vecs * kPer<T>;
  }
  __device__ __forceinline__ Slot<T> whole(int v) const { return Slot<T>(head + v * kPer<T>, 0, kPer<T>); }
  // both ends, of lanes 0 and 1 of a workgroup that has them
  __device__ __forceinline__ Slot<T> edge(int id, int width, bool first, bool last) const {
    if (id == 0 && first && head > 0) return Slot<T>(0, 0, head);
    if (id == 1 && last && tail > 0) return Slot<T>(width - kPer<T>, kPer<T> - tail, kPer<T>);
    return Slot<T>::none();
  }
};
template <typename T>
__device__ __forceinline__ float max_of(const Raw<T> &x) {
  const Vals<T> v = values_of<T>(x);
  float m = v[0];
#pragma unroll
  for (int e = 1; e < kPer<T>; ++e) m = fmaxf(m, v[e]);
  return m;
}
// Exponents are in base 2.  Those of x scale2 - m2, with m2 = m scale2 as it is rounded, take one operation an element;
// what m2 is off by is the same for all of them and taken out of the sums.  Where m2 is so large that this would not
// do, x less m comes first.
struct Shift {
  float m, m2, rest;
  __device__ __forceinline__ Shift(float maximum, float scale2) : m(shift_of(maximum)), m2(m * scale2), rest(fmaf(m, scale2, -m2)) {}
  __device__ __forceinline__ bool huge() const { return !(fabsf(m2) < 0x1p29f); }
  __device__ __forceinline__ void settle(Stats &t) const {
    const float by = __builtin_amdgcn_exp2f(-rest);
    t.a = fmaf(-rest, t.s, t.a) * by, t.s *= by;
  }
};
template <bool kEntropy, bool kHuge, typename T>
__device__ __forceinline__ void add_to(Stats &t, const Raw<T> &x, const Shift &m, float scale2) {
  const Vals<T> v = values_of<T>(x);
#pragma unroll
  for (int e = 0; e < kPer<T>; ++e) {
    const float d = kHuge ? (v[e] - m.m) * scale2 : fmaf(v[e], scale2, -m.m2), p = __builtin_amdgcn_exp2f(d);
    t.s += p;
    if (kEntropy) t.a = fmaf(fmaxf(d, kLeast), p, t.a);
  }
}

// ---- what is made of them ---------------------------------------------------------------------------------------
struct Result {
  float shift, log_s;
  // Nothing is allowed, and nothing is NaN: maxima pass NaN by, S does not.  (The lowest numbers of 32 bits and of bfloat16 are as good a
  // mask as -inf; -65504, fp16's, is a logit like any other.)
  bool none;
  __device__ __forceinline__ Result(const Stats &t)
      : shift(shift_of(t.m)), log_s(__builtin_amdgcn_logf(t.s) * kLn2), none(t.m < kLow && t.s == t.s) {}
  __device__ __forceinline__ float log_p(float x, float scale) const {
    return none ? -INFINITY : x == -INFINITY ? x + (log_s - log_s) : (x - shift) * scale - log_s;  // (NaN: all of the row)
  }
  __device__ __forceinline__ float lse(const Stats &t, float scale) const { return none ? -INFINITY : fmaf(scale, t.m, log_s); }
};

template <typename T>
__device__ __forceinline__ float logit_at(const LogitsArgs &a, int64_t row, int64_t column) {
  return (float)static_cast<const T *>(a.logits)[row * a.stride + column];
}

// by one lane; x: the token's logit
__device__ __forceinline__ void finish_log_probs(const LogitsArgs &a, int64_t row, float x, const Stats &t) {
  const Result r(t);
  if (a.log_probs) a.log_probs[row] = r.log_p(x, a.scale);
  a.lse[row] = r.lse(t, a.scale);
  a.entropy[row] = r.none ? 0.f : r.log_s - t.a / t.s * kLn2;
}
__device__ __forceinline__ void pass_over(const LogitsArgs &a, int64_t row) {
  if (a.log_probs) a.log_probs[row] = 0;
  if (a.entropy) a.entropy[row] = 0;
  if (a.loss) a.loss[row] = 0;
  a.lse[row] = 0;
}
__device__ __forceinline__ void put_best(const LogitsArgs &a, int64_t row, int at, uint64_t e, const Stats &t) {
  a.top_log_probs[row * a.top + at] = e == 0 ? -INFINITY : Result(t).log_p(entry_value(e), a.scale);
  a.top_tokens[row * a.top + at] = e == 0 ? -1 : entry_column(e);
}

// The teacher's entries of a row: entry k is held by lane k % kLanes.  `count` 0: the lanes have no row.
template <int kLanes>
struct Teacher {
  static constexpr int kHeldEntries = kMaxTop / kLanes;
  int column[kHeldEntries];                       // -1: none
  float l[kHeldEntries], q[kHeldEntries], log_sum;  // logits less their maximum, weights
  bool some;
  __device__ __forceinline__ Teacher(const LogitsArgs &a, int64_t row, int count, int lane) {
    float top = -INFINITY, any = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) {
      column[i] = -1, l[i] = -INFINITY, q[i] = 0;
      const int k = lane + i * kLanes;
      if (k < count) {
        column[i] = (int)token_at(a.entries, a.wide, row * a.count + k, a.vocab);
        if (column[i] >= 0) l[i] = a.teacher[row * a.count + k];
      }
    }
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) {
      top = fmaxf(top, l[i]);
      if (!(l[i] == -INFINITY)) any = 1;
    }
    top = shift_of(lanes_max<kLanes>(top));
    some = lanes_max<kLanes>(any) > 0;
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) {
      l[i] -= top;
      q[i] = __builtin_amdgcn_exp2f(l[i] * kLog2e);
      sum += q[i];
    }
    sum = lanes_sum<kLanes>(sum);
    log_sum = __builtin_amdgcn_logf(sum) * kLn2;
    const float over = 1.f / sum;
#pragma unroll
    for (int i = 0; i < kHeldEntries; ++i) q[i] *= over;
  }
};
template <typename T, int kLanes>
__device__ __forceinline__ void finish_distill(const LogitsArgs &a, int64_t row, bool here, int lane, const Teacher<kLanes> &q,
                                               const Stats &t) {
  const Result r(t);
  float x[Teacher<kLanes>::kHeldEntries], loss = 0;
#pragma unroll
  for (int i = 0; i < Teacher<kLanes>::kHeldEntries; ++i) x[i] = here && q.column[i] >= 0 ? logit_at<T>(a, row, q.column[i]) : 0.f;
#pragma unroll
  for (int i = 0; i < Teacher<kLanes>::kHeldEntries; ++i)
    if (here && q.column[i] >= 0 && !(q.q[i] == 0)) loss += q.q[i] * (q.l[i] - q.log_sum - r.log_p(x[i], a.scale));
  loss = lanes_sum<kLanes>(loss);
  if (here && lane == 0) {
    a.loss[row] = loss;
    a.lse[row] = r.lse(t, a.scale);
  }
}

// ---- the best tokens ----------------------------------------------------------------------------------------------
template <int kThreads>
__device__ __forceinline__ void group_sync() {
  if (kThreads == kWave)
    wave_lds_sync();
  else
    __syncthreads();
}

template <typename T, int kThreads, int kVecs>
struct BestSmem {
  static constexpr int kList = kThreads < 256 ? 512 : 1024;  // candidates: for 64 of the best there are about 300
  static constexpr int kOwners = 40;                         // threads that have some: for 16 of the best about 25
  uint32_t groups[kWave];
  uint64_t best[2][kThreads / kWave];
  uint64_t list[kList];
  u32x4 held[kOwners][kVecs];
  uint16_t owner[kOwners];
  int owners, listed;
};

__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return (int32_t)b < 0 ? ~b : b | 0x80000000u;
}

// The best `top` of what kThreads threads hold, put(place, entry) for each; entries that are not there are 0.  slot(id, i): where
// vector i of a thread lies; mine: the largest of a thread's elements; finite: whether the row holds no NaN or infinity.
template <typename T, int kThreads, int kVecs, typename At, typename Put>
__device__ __forceinline__ void best_of(const T *row, bool tiny, Raw<T> (&x)[kVecs], const At &slot, float mine, bool finite, int top,
                                        BestSmem<T, kThreads, kVecs> &sm, const Put &put) {
  constexpr int kGroup = kThreads / kWave;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) as_it_came<T>(x[i]);
  const int lane = threadIdx.x % kWave, id = threadIdx.x % kThreads;
  // 64 maxima; the lowest bits make them differ, and leave the bound a little low
  const float g = lanes_max<(kGroup > 1 ? kGroup : 1)>(mine);
  if (id % kGroup == 0) sm.groups[id / kGroup] = (order_of(g) & ~63u) | (id / kGroup);
  if (id == 0) sm.owners = sm.listed = 0;
  group_sync<kThreads>();
  const uint32_t key = sm.groups[lane];
  int before = 0;
#pragma unroll
  for (int j = 0; j < kWave; j += 4) {
    const u32x4 other = *reinterpret_cast<const u32x4 *>(&sm.groups[j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) before += other[i] > key;
  }
  const uint32_t kth = __builtin_amdgcn_readlane(key, __builtin_ctzll(__ballot(before == top - 1))) & ~63u;
  const float bound = __uint_as_float(kth & 0x80000000u ? kth & 0x7fffffffu : ~kth);
  const bool listing = finite && kth > 0x007fffffu;  // (-inf is no bound)
  // What the few threads hold that have some goes where all threads look at it; where they are not few, each looks at its own
  // (4096 x 33024, the best 8: 59 us so, 60 each its own; the best 32: 73 and 69; 64 rows, the best 8: 9.5 and 15.7).
  const bool few = listing && top <= 16;
  if (few && mine >= bound) {
    const int at = atomicAdd(&sm.owners, 1);
    if (at < sm.kOwners) {
      sm.owner[at] = (uint16_t)id;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) sm.held[at][i] = __builtin_bit_cast(u32x4, x[i]);
    }
  }
  if (few) group_sync<kThreads>();
  auto add = [&](float value, int column) __attribute__((always_inline)) {
    const int at = atomicAdd(&sm.listed, 1);
    if (at < sm.kList) sm.list[at] = entry_of(value, column);
  };
  const int owners = sm.owners;
  if (few && owners <= sm.kOwners) {
    constexpr int kEach = kVecs * kPer<T>;
    for (int c = id; c < owners * kEach; c += kThreads) {
      const int o = c / kEach, e = c - o * kEach;
      const float value = (float)reinterpret_cast<const T *>(&sm.held[o][0])[e];
      if (value >= bound) add(value, slot(sm.owner[o], e / kPer<T>).col + e % kPer<T>);
    }
  } else if (listing && mine >= bound) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      if (max_of<T>(x[i]) >= bound) {
        const Vals<T> value = values_of<T>(x[i]);
#pragma unroll
        for (int e = 0; e < kPer<T>; ++e)
          if (value[e] >= bound) add(value[e], slot(id, i).col + e);
      }
  }
  group_sync<kThreads>();
  auto listed = [&](int count) __attribute__((always_inline)) {
    for (int c = id; c < count || c < top; c += kThreads) {
      if (c < count) {
        const uint64_t w = sm.list[c];
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < count; ++j) place += sm.list[j] > w;
        if (place < top) put(place, w);
      } else {
        put(c, 0ull);
      }
    }
    group_sync<kThreads>();
  };
  // what is given for each element of a thread, from where it lies (nothing of this is kept in registers for it)
  auto each = [&](const auto &f) __attribute__((always_inline)) {
#pragma unroll 1
    for (int i = 0; i < kVecs; ++i) {
      const Slot<T> s = slot(id, i);
      if (!s.any()) continue;
      const Vals<T> y = values_of<T>(load_slot<T>(row, s, tiny));
#pragma unroll
      for (int e = 0; e < kPer<T>; ++e)
        if (s.own(e)) f(entry_of(y[e], s.col + e));
    }
  };
  int count = sm.listed;
  if (listing && count <= sm.kList) return listed(count);
  // Once more with entries in place of values, so that equal logits differ; now the groups are of threads 64 apart: of equal
  // logits the lowest columns are asked for, which then lie in as many groups as can be.
  uint64_t own = 0;
  each([&](uint64_t w) { own = w > own ? w : own; });
  group_sync<kThreads>();
  sm.list[id] = own;
  if (id == 0) sm.listed = 0;
  group_sync<kThreads>();
#pragma unroll
  for (int w = 0; w < kGroup; ++w) own = w == 0 || sm.list[lane + w * kWave] > own ? sm.list[lane + w * kWave] : own;
  uint64_t least = 0;
  int above = 0;
#pragma unroll 4
  for (int j = 0; j < kWave; ++j) above += __shfl((unsigned long long)own, j) > own;
  const uint64_t kth_lane = __ballot(above == top - 1);  // (none where fewer groups than that have elements)
  if (kth_lane) least = __shfl((unsigned long long)own, __builtin_ctzll(kth_lane));
  group_sync<kThreads>();
  each([&](uint64_t w) {
    if (w >= least) {
      const int at = atomicAdd(&sm.listed, 1);
      if (at < sm.kList) sm.list[at] = w;
    }
  });
  group_sync<kThreads>();
  count = sm.listed;
  if (count <= sm.kList) return listed(count);
  uint64_t limit = ~0ull;
#pragma unroll 1
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    each([&](uint64_t w) {
      if (w < limit && w > best) best = w;
    });
    limit = lanes_max64<kWave>(best);
    if (kThreads > kWave) {
      if (lane == 0) sm.best[k & 1][id / kWave] = limit;
      __syncthreads();
      limit = sm.best[k & 1][0];
#pragma unroll
      for (int w = 1; w < kThreads / kWave; ++w) limit = sm.best[k & 1][w] > limit ? sm.best[k & 1][w] : limit;
    }
    if (id == 0) put(k, limit);
  }
}

// The best one alone, as an entry in the lanes of its row (all threads of a workgroup come here): where the largest logit is known,
// and finite, its lowest column is looked for, in the few vectors that hold it (184320 x 1024 92 us, as one of many 140; 4096 x 33024
// 50 and 55; 64 x 65537 8.5 and 9.9).
template <typename T, int kThreads, int kLanes, int kVecs, typename At>
__device__ __forceinline__ uint64_t best_one(const T *row, bool tiny, Raw<T> (&x)[kVecs], const At &slot, bool here, float mine, float most,
                                             bool finite, uint64_t *share) {
  const int id = threadIdx.x % (kThreads > kWave ? kThreads : kLanes);
  const bool known = finite && most > -INFINITY;
  float column = -INFINITY;  // less than 0
#pragma unroll
  for (int i = 0; i < kVecs; ++i) as_it_came<T>(x[i]);
  if (known && mine == most) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      if (max_of<T>(x[i]) == most) {
        const Vals<T> value = values_of<T>(x[i]);
        const int first = slot(id, i).col;
#pragma unroll
        for (int e = 0; e < kPer<T>; ++e)
          if (value[e] == most) column = fmaxf(column, -(float)(first + e));
      }
  }
  column = lanes_max<kLanes>(column);
  uint64_t best = column > -INFINITY ? entry_of(most, (int)-column) : 0ull;
  if (__ballot(here && !known)) {
    if (here && !known) {
#pragma unroll 1
      for (int i = 0; i < kVecs; ++i) {
        const Slot<T> s = slot(id, i);
        if (!s.any()) continue;
        const Vals<T> y = values_of<T>(load_slot<T>(row, s, tiny));
#pragma unroll
        for (int e = 0; e < kPer<T>; ++e)
          if (s.own(e) && entry_of(y[e], s.col + e) > best) best = entry_of(y[e], s.col + e);
      }
    }
    best = lanes_max64<kLanes>(best);
  }
  if (kThreads > kWave) {
    if (threadIdx.x % kWave == 0) share[threadIdx.x / kWave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) best = share[w] > best ? share[w] : best;
  }
  return best;
}

// ---- rows of a wave or less -------------------------------------------------------------------------------------
template <typename T, int kLanes, int kVecs, int kKind, int kTop>
__global__ __launch_bounds__(kBlock) void narrow_kernel(LogitsArgs a) {
  constexpr int kRows = kBlock / kLanes;
  __shared__ BestSmem<T, kWave, kTop == kSomeBest && kLanes == kWave ? kVecs : 1> best[kTop == kSomeBest && kLanes == kWave ? kRows : 1];
  const int lane = threadIdx.x % kLanes;
  const bool tiny = kLanes == 4 && a.vocab < kPer<T>;
  // (the lanes of a wave go round alike: they exchange sums)
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.rows; base += (int64_t)gridDim.x * kRows) {
    const int64_t row = base + threadIdx.x / kLanes;
    bool here = row < a.rows;
    // (asked for before it is known whether the row is passed over)
    Raw<T> x[kVecs];
    const T *from = static_cast<const T *>(a.logits) + row * a.stride;
    const int shift = kLanes * kVecs < 64 || tiny ? 0 : misaligned(from);  // (short rows share their lines anyway)
    auto slot = [&](int id, int i) { return Slot<T>::shifted(id + i * kLanes, a.vocab, shift); };
#pragma unroll
    for (int i = 0; i < kVecs; ++i) x[i] = here ? load_logits<T>(from, slot(lane, i), tiny) : nothing<T>();
    float at_token = 0;
    if (kKind == kLogProbs && a.tokens) {
      const int64_t token = here ? token_at(a.tokens, a.wide, row, a.vocab) : -1;
      if (here && token < 0) {
        if (lane == 0) pass_over(a, row);
        if (kTop)
          for (int k = lane; k < a.top; k += kLanes) put_best(a, row, k, 0, Stats{});
      }
      here = token >= 0;
      if constexpr (kLanes * kVecs <= 32) {  // (from where it is: another load would wait for the token)
        float found = -INFINITY;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const Slot<T> s = slot(lane, i);
          const Vals<T> value = values_of<T>(x[i]);
#pragma unroll
          for (int e = 0; e < kPer<T>; ++e)
            if (s.col + e == (int)token && s.own(e)) found = value[e];
        }
        at_token = lanes_max<kLanes>(found);
      } else if (here) {
        at_token = logit_at<T>(a, row, token);
      }
    }
    auto stats = [&](Stats &t) __attribute__((always_inline)) {
      const float mine = t.m;
      t.m = lanes_max<kLanes>(mine);
      const Shift m(t.m, a.scale2);
      if (m.huge()) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) add_to<kKind == kLogProbs, true, T>(t, x[i], m, a.scale2);
      } else {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) add_to<kKind == kLogProbs, false, T>(t, x[i], m, a.scale2);
      }
      t.s = lanes_sum<kLanes>(t.s);
      if (kKind == kLogProbs) t.a = lanes_sum<kLanes>(t.a);
      if (!m.huge()) m.settle(t);
    };
    Stats t{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kVecs; ++i) t.m = fmaxf(t.m, max_of<T>(x[i]));
    const float mine = t.m;
    if constexpr (kKind == kDistill) {
      const Teacher<kLanes> q(a, row, here ? a.count : 0, lane);
      if (here && !q.some && lane == 0) pass_over(a, row);
      stats(t);
      finish_distill<T, kLanes>(a, row, here && q.some, lane, q, t);
    } else {
      stats(t);
      if (here && lane == 0) finish_log_probs(a, row, at_token, t);
      if constexpr (kTop == kOneBest) {
        const uint64_t e = best_one<T, kWave, kLanes, kVecs>(from, tiny, x, slot, here, mine, t.m, t.s == t.s, nullptr);
        if (here && lane == 0) put_best(a, row, 0, e, t);
      } else if constexpr (kTop == kSomeBest && kLanes == kWave) {
        if (here)
          best_of<T, kWave, kVecs>(from, tiny, x, slot, mine, t.s == t.s, a.top, best[threadIdx.x / kWave],
                                   [&](int place, uint64_t e) { put_best(a, row, place, e, t); });
      } else if constexpr (kTop == kSomeBest) {
        uint64_t entry[kVecs * kPer<T>], last = 0;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const Slot<T> s = slot(lane, i);
#pragma unroll
          for (int e = 0; e < kPer<T>; ++e) entry[i * kPer<T> + e] = s.own(e) ? entry_of((float)x[i][e], s.col + e) : 0;
        }
        for (int k = 0; k < a.top; ++k) {
          uint64_t best = 0;
#pragma unroll
          for (int e = 0; e < kVecs * kPer<T>; ++e) {
            if (entry[e] == last) entry[e] = 0;  // (it was the last one's)
            best = entry[e] > best ? entry[e] : best;
          }
          last = lanes_max64<kLanes>(best);
          if (here && lane == k % kLanes) put_best(a, row, k, last, t);
        }
      }
    }
  }
}

// ---- rows, or parts of them, of a workgroup ---------------------------------------------------------------------
template <int kThreads, typename F>
__device__ __forceinline__ float block_reduce(float x, float *part, const F &f) {  // (x: of the wave)
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = x;
  __syncthreads();
  x = part[0];
#pragma unroll
  for (int w = 1; w < kThreads / kWave; ++w) x = f(x, part[w]);
  return x;
}

template <typename T, int kThreads, int kVecs, int kKind, int kTop>
__global__ __launch_bounds__(kThreads, kThreads == kBlock && kVecs == kHeld ? (kTop ? 4 : 5) : 1) void wide_kernel(LogitsArgs a) {
  __shared__ float part_max[kThreads / kWave], part_sum[2][kThreads / kWave];
  __shared__ BestSmem<T, kTop == kSomeBest ? kThreads : kWave, kTop == kSomeBest ? kVecs + 1 : 1> best;
  __shared__ uint64_t share[kTop == kOneBest ? kThreads / kWave : 1];
  for (int64_t unit = blockIdx.x; unit < a.rows * a.parts; unit += gridDim.x) {
    const int64_t row = unit / a.parts;
    const int part = (int)(unit - row * a.parts);
    const T *from = static_cast<const T *>(a.logits) + row * a.stride;
    const Cut<T> cut(from, a.vocab);
    const int first = part * a.part_vecs, last = min(first + a.part_vecs, cut.vecs);
    auto slot = [&](int id, int i) {  // (the last one is an end of the row)
      const int v = first + id + i * kThreads;
      return i == kVecs ? cut.edge(id, a.vocab, part == 0, part == a.parts - 1) : v < last ? cut.whole(v) : Slot<T>::none();
    };
    float at_token = 0;
    if (kKind == kLogProbs && a.tokens) {
      const int64_t token = token_at(a.tokens, a.wide, row, a.vocab);
      if (token < 0) {  // (with several parts the launch that joins them sees to the row)
        if (a.parts == 1) {
          if (threadIdx.x == 0) pass_over(a, row);
          if (kTop && (int)threadIdx.x < a.top) put_best(a, row, threadIdx.x, 0, Stats{});
        }
        continue;
      }
      at_token = logit_at<T>(a, row, token);
    }
    Raw<T> x[kVecs + 1];
    auto load = [&]() __attribute__((always_inline)) {
      const T *at = from + cut.head + (int64_t)(first + threadIdx.x) * kPer<T>;
      auto vectors = [&](auto once) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          x[i] = nothing<T>();
          if (first + (int)threadIdx.x + i * kThreads < last) x[i] = load_raw<decltype(once)::value>(at + i * kThreads * kPer<T>);
        }
      };
      if (a.once)
        vectors(std::true_type());
      else
        vectors(std::false_type());
      x[kVecs] = nothing<T>();
      if (threadIdx.x < 2) x[kVecs] = load_logits<T>(from, slot(threadIdx.x, kVecs), false);
    };
    if (kKind == kLogProbs) load();
    // (whether a wave has anything of round i)
    auto some = [&](int i) __attribute__((always_inline)) { return i < kVecs ? first + i * kThreads < last : threadIdx.x < kWave; };
    auto stats = [&](float &mine) __attribute__((always_inline)) {
      mine = -INFINITY;
#pragma unroll
      for (int i = 0; i <= kVecs; ++i)
        if (some(i)) mine = fmaxf(mine, max_of<T>(x[i]));
#pragma unroll
      for (int i = 0; i <= kVecs; ++i) as_it_came<T>(x[i]);
      __syncthreads();  // (of the unit before: its shared memory)
      Stats t{block_reduce<kThreads>(lanes_max<kWave>(mine), part_max, [](float p, float r) { return fmaxf(p, r); }), 0.f, 0.f};
      const Shift m(t.m, a.scale2);
      if (__builtin_expect(m.huge(), 0)) {
#pragma unroll 1
        for (int i = 0; i <= kVecs; ++i)
          add_to<kKind == kLogProbs, true, T>(t, load_logits<T>(from, slot(threadIdx.x, i), false), m, a.scale2);
      } else {
#pragma unroll
        for (int i = 0; i <= kVecs; ++i)
          if (some(i)) add_to<kKind == kLogProbs, false, T>(t, x[i], m, a.scale2);
      }
      auto plus = [](float p, float r) { return p + r; };
      const float s = lanes_sum<kWave>(t.s);
      if (kKind == kLogProbs) {
        const float a2 = lanes_sum<kWave>(t.a);
        if (threadIdx.x % kWave == 0) part_sum[1][threadIdx.x / kWave] = a2;
      }
      t.s = block_reduce<kThreads>(s, part_sum[0], plus);
      if (kKind == kLogProbs) {
        t.a = part_sum[1][0];
#pragma unroll
        for (int w = 1; w < kThreads / kWave; ++w) t.a += part_sum[1][w];
      }
      if (!m.huge()) m.settle(t);
      return t;
    };
    float mine;
    if constexpr (kKind == kDistill) {
      const Teacher<kWave> q(a, row, a.count, threadIdx.x % kWave);
      if (!q.some) {
        if (a.parts == 1 && threadIdx.x == 0) pass_over(a, row);
        continue;
      }
      load();
      const Stats t = stats(mine);
      if (a.parts > 1) {
        if (threadIdx.x == 0) *reinterpret_cast<f32x4 *>(a.stats + unit * 4) = f32x4{t.m, t.s, t.a, 0.f};
      } else if (threadIdx.x < kWave) {
        finish_distill<T, kWave>(a, row, true, threadIdx.x, q, t);
      }
    } else {
      const Stats t = stats(mine);
      const bool alone = a.parts == 1;
      if (threadIdx.x == 0) {
        if (alone)
          finish_log_probs(a, row, at_token, t);
        else
          *reinterpret_cast<f32x4 *>(a.stats + unit * 4) = f32x4{t.m, t.s, t.a, 0.f};
      }
      auto put = [&](int place, uint64_t e) __attribute__((always_inline)) {
        if (alone)
          put_best(a, row, place, e, t);
        else
          a.lists[unit * a.top + place] = e;
      };
      if constexpr (kTop == kOneBest) {
        const uint64_t e = best_one<T, kThreads, kWave, kVecs + 1>(from, false, x, slot, true, mine, t.m, t.s == t.s, share);
        if (threadIdx.x == 0) put(0, e);
      } else if constexpr (kTop == kSomeBest) {
        best_of<T, kThreads, kVecs + 1>(from, false, x, slot, mine, t.s == t.s, a.top, best, put);
      }
    }
  }
}

// Rows in several parts: a workgroup each, a part a lane.
template <typename T, int kKind>
__global__ __launch_bounds__(kBlock) void join_kernel(LogitsArgs a) {
  __shared__ uint64_t lists[kKind == kLogProbs ? kJoined : 1];
  const int lane = threadIdx.x % kWave;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    auto stats = [&]() __attribute__((always_inline)) {
      f32x4 p = {-INFINITY, 0.f, 0.f, 0.f};
      if (lane < a.parts) p = *reinterpret_cast<const f32x4 *>(a.stats + (row * a.parts + lane) * 4);
      Stats t{lanes_max<kWave>(p[0]), 0.f, 0.f};
      const float d = fmaxf((p[0] - shift_of(t.m)) * a.scale2, kLeast), e = __builtin_amdgcn_exp2f(d);
      t.s = lanes_sum<kWave>(p[1] * e), t.a = lanes_sum<kWave>(fmaf(d, p[1], p[2]) * e);
      return t;
    };
    if constexpr (kKind == kDistill) {
      const Teacher<kWave> q(a, row, a.count, lane);
      if (threadIdx.x < kWave) {
        if (q.some)
          finish_distill<T, kWave>(a, row, true, lane, q, stats());
        else if (lane == 0)
          pass_over(a, row);
      }
    } else {
      const int all = a.parts * a.top;
      __syncthreads();  // (of the row before)
      for (int i = threadIdx.x; i < all; i += kBlock) lists[i] = a.lists[row * all + i];
      float at_token = 0;
      if (a.tokens) {
        const int64_t token = token_at(a.tokens, a.wide, row, a.vocab);
        if (token < 0) {
          if (threadIdx.x == 0) pass_over(a, row);
          if ((int)threadIdx.x < a.top) put_best(a, row, threadIdx.x, 0, Stats{});
          continue;
        }
        at_token = logit_at<T>(a, row, token);
      }
      const Stats t = stats();
      if (threadIdx.x == 0) finish_log_probs(a, row, at_token, t);
      if (a.top == 0) continue;
      __syncthreads();
      // an entry's place: how many of every part's, each in order, come before it
      for (int i = threadIdx.x; i < all; i += kBlock) {
        const uint64_t w = lists[i];
        if (w == 0) continue;
        int place = 0;
        for (int p = 0; p < a.parts && place < a.top; ++p) {
          int lo = 0, hi = a.top;
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (lists[p * a.top + mid] > w)
              lo = mid + 1;
            else
              hi = mid;
          }
          place += lo;
        }
        if (place < a.top) put_best(a, row, place, w, t);
      }
    }
  }
}

// ---- gradients --------------------------------------------------------------------------------------------------
// p (alpha + beta log2 p) of a logit, times the scale; kBeta: beta is not 0.  The difference from lse is taken before anything is
// rounded: with scale2 and lse2 in its place, one operation less, p at logits of 500 was off by 1e-5 and at 70000 by 3e-3.
struct Slope {
  float lse, scale, alpha, beta;
  template <bool kBeta>
  __device__ __forceinline__ float at(float x) const {
    // (above 0 only by what lse lost when it was rounded, where logits are huge)
    const float l = __builtin_amdgcn_fmed3f(fmaf(x, scale, -lse) * kLog2e, kLeast, 0.f), p = __builtin_amdgcn_exp2f(l);
    return p * (kBeta ? fmaf(beta, l, alpha) : alpha);
  }
};

// What a row's slope is made of, asked for before anything of it is looked at.
template <int kKind>
struct Given {
  float lse, by, de = 0, entropy = 0;
  __device__ __forceinline__ Given(const LogitsArgs &a, int64_t row) {
    lse = a.lse_in[row];
    if (kKind == kDistill) {
      by = a.dloss[row];
    } else {
      by = a.dlog_probs ? a.dlog_probs[row] : 0.f;
      if (a.dentropy) de = a.dentropy[row], entropy = a.entropy_in[row];
    }
  }
  // whether there is anything to write but zeros; more: what is added at the given token, or taken at an entry
  __device__ __forceinline__ bool slope(const LogitsArgs &a, bool some, Slope &s, float &more) const {
    if (!some || lse == -INFINITY) return false;  // (nothing was allowed)
    s.lse = lse, s.scale = a.scale;
    const float nan = lse - lse;  // 0, or NaN for a row of NaN
    s.alpha = (kKind == kDistill ? a.scale * by : -a.scale * (by + de * entropy)) + nan;
    s.beta = -a.scale * de * kLn2;
    more = kKind == kDistill ? -s.alpha : a.scale * by;
    return true;
  }
};

template <bool kBeta, typename T>
__device__ __forceinline__ Vals<T> grad_of(const Raw<T> &x, bool live, const Slope &slope) {
  Vals<T> y = {};
  if (live) {
    y = values_of<T>(x);
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e) y[e] = slope.template at<kBeta>(y[e]);
  }
  return y;
}

struct Fix {
  int column;  // or -1
  float q;
};
// The teacher's entries with their weights, where the lanes of a row find them all.
template <int kLanes>
__device__ __forceinline__ bool put_entries(const LogitsArgs &a, int64_t row, int count, int lane, bool write, Fix *fix) {
  const Teacher<kLanes> q(a, row, count, lane);
#pragma unroll
  for (int i = 0; i < Teacher<kLanes>::kHeldEntries; ++i)
    if (write && lane + i * kLanes < count) fix[lane + i * kLanes] = Fix{q.column[i], q.column[i] < 0 ? 0.f : q.q[i]};
  return q.some;
}
// An entry that stands for its column, with the weights of all that name it.
__device__ __forceinline__ Fix fix_of(const Fix *fix, int k, int count) {
  Fix f = fix[k];
  for (int j = 0; j < count && f.column >= 0; ++j) {
    if (j == k || fix[j].column != f.column) continue;
    if (j < k) f.column = -1;
    f.q += fix[j].q;
  }
  return f;
}

template <typename T, int kLanes, int kVecs, int kKind, bool kBeta>
__global__ __launch_bounds__(kBlock) void narrow_grad_kernel(LogitsArgs a) {
  constexpr int kRows = kBlock / kLanes;
  __shared__ Fix fixes[kKind == kDistill ? kRows : 1][kMaxTop];
  const int lane = threadIdx.x % kLanes;
  const bool tiny = kLanes == 4 && a.vocab < kPer<T>;
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.rows; base += (int64_t)gridDim.x * kRows) {
    const int64_t row = base + threadIdx.x / kLanes;
    const bool here = row < a.rows;
    Fix *fix = fixes[kKind == kDistill ? threadIdx.x / kLanes : 0];
    const T *from = static_cast<const T *>(a.logits) + row * a.stride;
    T *to = static_cast<T *>(a.dlogits) + row * a.vocab;
    const int shift = kLanes * kVecs < 64 || tiny ? 0 : misaligned(to);
    auto slot = [&](int i) { return Slot<T>::shifted(lane + i * kLanes, a.vocab, shift); };
    // (asked for before it is known whether the row is passed over)
    Raw<T> x[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      x[i] = Raw<T>{};
      if (here && slot(i).any()) x[i] = load_slot<T>(from, slot(i), tiny);
    }
    const Given<kKind> given(a, here ? row : 0);
    int token = -1;
    bool some = here;
    if (kKind == kDistill) {
      __syncthreads();  // (of the rows before)
      some = put_entries<kLanes>(a, row, here ? a.count : 0, lane, true, fix) && here;
    } else if (here && a.tokens) {
      token = (int)token_at(a.tokens, a.wide, row, a.vocab);
      some = token >= 0;
    }
    Slope slope{};
    float more = 0;
    const bool live = given.slope(a, some, slope, more);
    if (here) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const Slot<T> s = slot(i);
        Vals<T> y = grad_of<kBeta, T>(x[i], live, slope);
        if (kKind == kLogProbs && kLanes * kVecs <= 32 && live) {
#pragma unroll
          for (int e = 0; e < kPer<T>; ++e)
            if (s.col + e == token) y[e] += more;
        }
        if (s.any()) store_slot(to, s, y);
      }
      // (the lane that wrote the token's column writes it again)
      if (kKind == kLogProbs && kLanes * kVecs > 32 && live && token >= 0 && (token + shift) / kPer<T> % kLanes == lane)
        to[token] = (T)(slope.at<kBeta>((float)from[token]) + more);
    }
    if (kKind == kDistill) {
      __syncthreads();  // the entries are there, and the row is written
      if (live)
        for (int k = lane; k < a.count; k += kLanes) {
          const Fix f = fix_of(fix, k, a.count);
          if (f.column >= 0) to[f.column] = (T)fmaf(more, f.q, slope.at<false>((float)from[f.column]));
        }
    }
  }
}

template <typename T, int kVecs, int kKind, bool kBeta, bool kOnce>
__global__ __launch_bounds__(kBlock) void wide_grad_kernel(LogitsArgs a) {
  __shared__ Fix fix[kMaxTop];
  for (int64_t unit = blockIdx.x; unit < a.rows * a.parts; unit += gridDim.x) {
    const int64_t row = (uint32_t)unit / (uint32_t)a.parts;
    const int part = (int)(unit - row * a.parts);
    const T *from = static_cast<const T *>(a.logits) + row * a.stride;
    T *to = static_cast<T *>(a.dlogits) + row * a.vocab;
    const Cut<T> cut(to, a.vocab);  // (where logits and gradients lie differently, it is for the stores)
    const int first = part * a.part_vecs, last = min(first + a.part_vecs, cut.vecs);
    const Slot<T> edge = cut.edge(threadIdx.x, a.vocab, part == 0, part == a.parts - 1);
    // (asked for before it is known whether the row is passed over)
    Raw<T> x[kVecs], end = {};
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = first + threadIdx.x + i * kBlock;
      if (v < last) x[i] = load_raw<kOnce>(from + cut.head + v * kPer<T>);
    }
    if (threadIdx.x < 2 && edge.any()) end = load_slot<T>(from, edge, false);
    const Given<kKind> given(a, row);
    int token = -1;
    bool some = true;
    if (kKind == kDistill) {
      __syncthreads();  // (of the unit before)
      some = put_entries<kWave>(a, row, a.count, threadIdx.x % kWave, threadIdx.x < kWave, fix);
    } else if (a.tokens) {
      token = (int)token_at(a.tokens, a.wide, row, a.vocab);
      some = token >= 0;
    }
    Slope slope{};
    float more = 0;
    const bool live = given.slope(a, some, slope, more);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = first + threadIdx.x + i * kBlock;
      if (v < last)
        store_raw<kOnce>(to + cut.head + v * kPer<T>, __builtin_convertvector((grad_of<kBeta, T>(x[i], live, slope)), Raw<T>));
    }
    if (threadIdx.x < 2 && edge.any()) store_slot(to, edge, grad_of<kBeta, T>(end, live, slope));
    if (kKind == kLogProbs && live && token >= 0) {
      // (the thread that wrote the token's column writes it again)
      const int at = token - cut.head, v = at / kPer<T>;
      const int writer = at < 0 ? (part == 0 ? 0 : -1) : v >= cut.vecs ? (part == a.parts - 1 ? 1 : -1) :
                         v >= first && v < last ? (v - first) % kBlock : -1;
      if ((int)threadIdx.x == writer) to[token] = (T)(slope.at<kBeta>((float)from[token]) + more);
    }
    if (kKind == kDistill) {
      __syncthreads();  // the entries are there, and the part is written
      if (live && (int)threadIdx.x < a.count) {
        const Fix f = fix_of(fix, threadIdx.x, a.count);
        // (parts are cut from as many vectors as a row can have, so that the last one may begin behind this row's and have only its end)
        const int begin = part == 0 ? 0 : cut.head + min(first, cut.vecs) * kPer<T>, end = part == a.parts - 1 ? a.vocab : cut.head + last * kPer<T>;
        if (f.column >= begin && f.column < end)
          to[f.column] = (T)fmaf(more, f.q, slope.at<false>((float)from[f.column]));
      }
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------------------
constexpr int kWaveVecs = 256;  // widest row of a wave
constexpr int kLarge = 1024;    // threads of a workgroup where rows are few and one of 256 would not hold them
// Rows for which there is a CU each, in workgroups of 1024 threads, and the rest in parts that are joined: 64 rows of 65537 fp16
// 7.4 us and 8.6, 128 of 33024 in 32 bits 5.9 and 8.2, 400 of them 12.9 and 13.9; rows of 33024 bf16 fit 256 threads, 6.3 and 6.2.
constexpr int kFewRows = 256;
bool few(int64_t rows, int vecs) { return rows <= kFewRows && vecs > kHeld * kBlock && vecs <= kHeldFew * kLarge; }
// Parts of a row: what a workgroup holds at most.
void split(int64_t rows, int vecs, int &parts, int &part_vecs) {
  const int most = few(rows, vecs) ? vecs : kHeld * kBlock, n = (vecs + most - 1) / most;
  part_vecs = (vecs + n - 1) / n;
  parts = (vecs + part_vecs - 1) / part_vecs;
}
static_assert(kMaxVocab / 4 / (kHeld * kBlock) < kWave && (kMaxVocab / 4 / (kHeld * kBlock) + 1) * kMaxTop <= kJoined,
              "a part a lane, and all their best tokens in shared memory");
// (of the type with most vectors: the workspace does not go by the type)
size_t split_bytes(int64_t rows, int64_t vocab, int64_t top) {
  if (rows <= 0 || vocab <= 0 || vocab > kMaxVocab || top < 0 || top > kMaxTop) return 0;
  size_t most = 0;
  for (const int per : {4, 8}) {
    int parts, each;
    split(rows, (int)((vocab + per - 1) / per), parts, each);
    if (parts > 1) most = std::max(most, align_up((size_t)rows * parts * 16, 256) + (size_t)rows * parts * (size_t)top * 8);
  }
  return most;
}

// f(lanes of a row, vectors of a lane) for rows of a wave or less.  With few lanes and many vectors each, more rows of a wave
// share what is done once a row: 184320 rows of 50 vectors, 16 lanes with four against 32 with two, 44 + 51 us against 52 + 53; of 128,
// 32 with four against 64 with two (16 with eight), 94 + 117 against 101 + 118 (98 + 127), but against a teacher's 16 entries 110 +
// 188 against 105 + 175.  The best tokens, if more than one, are looked for by whole waves.
template <int kKind, int kTop, typename F>
void by_lanes(int vecs, const F &f) {
  using two = std::integral_constant<int, 2>;
  using four = std::integral_constant<int, 4>;
  constexpr bool kWaves64 = kTop == kSomeBest, kWaves128 = kWaves64 || kKind != kLogProbs;
  if (vecs <= 4)
    f(std::integral_constant<int, 4>(), std::integral_constant<int, 1>());
  else if (vecs <= 8)
    f(std::integral_constant<int, 4>(), two());
  else if (vecs <= 16)
    f(std::integral_constant<int, 8>(), two());
  else if (vecs <= 32)
    f(std::integral_constant<int, 16>(), two());
  else if (vecs <= 64)
    f(std::integral_constant<int, kWaves64 ? 64 : 16>(), std::integral_constant<int, kWaves64 ? 2 : 4>());
  else if (vecs <= 128)
    f(std::integral_constant<int, kWaves128 ? 64 : 32>(), std::integral_constant<int, kWaves128 ? 2 : 4>());
  else
    f(std::integral_constant<int, 64>(), four());
}

// vectors of a row at most (one that is partial at both ends has one more)
template <typename T>
int vecs_of(const LogitsArgs &a) {
  const bool same = aligned_to(a.logits, 16) && (a.rows == 1 || a.stride % kPer<T> == 0) &&
                    aligned_to(a.dlogits, 16) && (a.dlogits == nullptr || a.rows == 1 || a.vocab % kPer<T> == 0);
  return a.vocab < kPer<T> ? 1 : (a.vocab + (same ? 0 : kPer<T> - 1) + kPer<T> - 1) / kPer<T>;
}

// Logits that no cache holds until they are read again are read past it, and their gradients written so: from 512 MB on
// forward (16384 x 33025 bf16, 1.08 GB, 207 -> 155 us; with what is left of 0.3 GB the gradient's launch is the faster one: 30000 x 5000
// 174 in both, 181 read past the caches), from 256 MB on backward, where they are read for the last time (391 -> 370; 8191 x 33025
// against 32 entries 207 -> 193).
constexpr int64_t kOnceForward = (int64_t)1 << 29, kOnceBackward = (int64_t)1 << 28;
template <typename T>
int64_t bytes_of(const LogitsArgs &a) {
  return a.rows * a.vocab * (int64_t)sizeof(T);
}

int64_t grid_of(int64_t blocks) { return std::min(blocks, kMostItems / kBlock); }

template <int kKind>
int forward(LogitsArgs &a, int dtype, char *ws, hipStream_t st) {
  by_type(dtype, [&](auto type) {
    using T = decltype(type);
    const int vecs = vecs_of<T>(a);
    if (vecs <= kWaveVecs) {
      auto narrow = [&](auto top) {
        constexpr int kTop = decltype(top)::value;
        by_lanes<kKind, kTop>(vecs, [&](auto lanes, auto held) {
          constexpr int kLanes = decltype(lanes)::value;
          const dim3 grid((unsigned)grid_of(ceil_div64(a.rows, kBlock / kLanes)));
          hipLaunchKernelGGL((narrow_kernel<T, kLanes, decltype(held)::value, kKind, kTop>), grid, dim3(kBlock), 0, st, a);
        });
      };
      if constexpr (kKind == kLogProbs) {
        if (a.top > 0) {
          if (a.top == 1)
            narrow(std::integral_constant<int, kOneBest>());
          else
            narrow(std::integral_constant<int, kSomeBest>());
          return;
        }
      }
      narrow(std::integral_constant<int, kNoBest>());
      return;
    }
    split(a.rows, (a.vocab + kPer<T> - 1) / kPer<T>, a.parts, a.part_vecs);
    a.once = bytes_of<T>(a) >= kOnceForward;
    a.stats = reinterpret_cast<float *>(ws);
    a.lists = reinterpret_cast<uint64_t *>(ws + align_up((size_t)a.rows * a.parts * 16, 256));
    auto launch = [&](auto size, auto held) {
      constexpr int kThreads = decltype(size)::value, kVecs = decltype(held)::value;
      const dim3 grid((unsigned)std::min(a.rows * a.parts, kMostItems / kThreads)), block(kThreads);
      if (kKind == kLogProbs && a.top == 1)
        hipLaunchKernelGGL((wide_kernel<T, kThreads, kVecs, kKind, kKind == kLogProbs ? kOneBest : kNoBest>), grid, block, 0, st, a);
      else if (kKind == kLogProbs && a.top > 0)
        hipLaunchKernelGGL((wide_kernel<T, kThreads, kVecs, kKind, kKind == kLogProbs ? kSomeBest : kNoBest>), grid, block, 0, st, a);
      else
        hipLaunchKernelGGL((wide_kernel<T, kThreads, kVecs, kKind, kNoBest>), grid, block, 0, st, a);
    };
    using small = std::integral_constant<int, kBlock>;
    using large = std::integral_constant<int, kLarge>;
    if (few(a.rows, (a.vocab + kPer<T> - 1) / kPer<T>))
      launch(large(), std::integral_constant<int, kHeldFew>());
    else if (a.part_vecs <= 4 * kBlock)
      launch(small(), std::integral_constant<int, 4>());
    else if (a.part_vecs <= 8 * kBlock)
      launch(small(), std::integral_constant<int, 8>());
    else
      launch(small(), std::integral_constant<int, kHeld>());
    if (a.parts > 1)
      hipLaunchKernelGGL((join_kernel<T, kKind>), dim3((unsigned)grid_of(a.rows)), dim3(kBlock), 0, st, a);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}

template <int kKind>
int backward(LogitsArgs &a, int dtype, hipStream_t st) {
  if (a.rows > (((int64_t)1 << 32) - 1) / ceil_div64(a.vocab, 1024)) return GEAR_HIP_ERANGE;  // (parts are numbered in 32 bits)
  by_type(dtype, [&](auto type) {
    using T = decltype(type);
    const int vecs = vecs_of<T>(a);
    auto launch = [&](auto beta) {
      constexpr bool kBeta = decltype(beta)::value;
      if (vecs <= kWaveVecs) {
        by_lanes<kKind, kNoBest>(vecs, [&](auto lanes, auto held) {
          constexpr int kLanes = decltype(lanes)::value;
          const dim3 grid((unsigned)grid_of(ceil_div64(a.rows, kBlock / kLanes)));
          hipLaunchKernelGGL((narrow_grad_kernel<T, kLanes, decltype(held)::value, kKind, kBeta>), grid, dim3(kBlock), 0, st, a);
        });
      } else {
        // Few vectors a thread, so that what is read and written lies close together at any time (a plain copy of rows of
        // 66 KB: 1, 2, 4, 8 vectors a thread 332, 348, 360, 390 us), but what a workgroup finds out about its row costs as
        // much for each part: 16384 x 33025 with 1, 2, 4, 6 vectors 398, 371, 388, 381 us; against a teacher's 32 entries,
        // 8191 rows, with 2, 4, 8 205, 190, 192.  Rows of four rounds at most are not cut (30000 x 5000: 112 -> 87).
        const int rounds = (vecs + kBlock - 1) / kBlock;
        auto parts = [&](auto held) {
          constexpr int kVecs = decltype(held)::value;
          const int n = (rounds + kVecs - 1) / kVecs;
          a.part_vecs = (rounds + n - 1) / n * kBlock, a.parts = (vecs + a.part_vecs - 1) / a.part_vecs;
          const dim3 grid((unsigned)grid_of(a.rows * a.parts));
          if (bytes_of<T>(a) >= kOnceBackward)
            hipLaunchKernelGGL((wide_grad_kernel<T, kVecs, kKind, kBeta, true>), grid, dim3(kBlock), 0, st, a);
          else
            hipLaunchKernelGGL((wide_grad_kernel<T, kVecs, kKind, kBeta, false>), grid, dim3(kBlock), 0, st, a);
        };
        if (kKind == kDistill || rounds <= 4)
          parts(std::integral_constant<int, 4>());
        else
          parts(std::integral_constant<int, 2>());
      }
    };
    if constexpr (kKind == kLogProbs) {
      if (a.dentropy) {
        launch(std::true_type());
        return;
      }
    }
    launch(std::false_type());
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}

// 0: go on; 1: nothing to do; else the error
int prepare(const gear_hip_logits_desc *d, LogitsArgs &a) {
  if (d == nullptr || d->rows < 0 || d->vocab < 1 || element_bytes(d->dtype) == 0 || !(d->scale > 0) || !(d->scale < 1e30f))
    return GEAR_HIP_EINVAL;
  if (d->vocab > kMaxVocab || d->rows >= (int64_t)1 << 31) return GEAR_HIP_ERANGE;
  if (d->rows == 0) return 1;
  if (d->logits == nullptr) return GEAR_HIP_EINVAL;
  if (!aligned_to(d->logits, element_bytes(d->dtype))) return GEAR_HIP_EALIGN;
  a.logits = d->logits, a.stride = d->row_stride, a.rows = d->rows, a.vocab = (int)d->vocab;
  a.scale = d->scale, a.scale2 = d->scale * kLog2e;
  return 0;
}
int enough(void *workspace, size_t bytes, size_t need) {
  if (need > 0 && (workspace == nullptr || bytes < need)) return GEAR_HIP_EWORKSPACE;
  if (need > 0 && !aligned_to(workspace, 256)) return GEAR_HIP_EALIGN;
  return 0;
}

}  // namespace
}  // namespace gearhip

using namespace gearhip;

extern "C" size_t gear_hip_token_log_probs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top) {
  return split_bytes(rows, vocab, top);
}

extern "C" int gear_hip_token_log_probs(const gear_hip_logits_desc *desc, const void *tokens, int tokens_i64, int64_t top,
                                        float *log_probs, float *entropy, float *lse, float *top_log_probs, int64_t *top_tokens,
                                        void *workspace, size_t workspace_bytes, void *stream) {
  LogitsArgs a = {};
  const int rc = prepare(desc, a);
  if (rc < 0) return rc;
  if (top < 0 || top > desc->vocab) return GEAR_HIP_EINVAL;
  if (top > kMaxTop) return GEAR_HIP_ERANGE;
  if (rc == 1) return 0;
  if ((tokens == nullptr) != (log_probs == nullptr)) return GEAR_HIP_EINVAL;
  if (entropy == nullptr || lse == nullptr || (top > 0 && (top_log_probs == nullptr || top_tokens == nullptr))) return GEAR_HIP_EINVAL;
  if (!aligned_to(tokens, tokens_i64 ? 8 : 4) || !aligned_to(log_probs, 4) || !aligned_to(entropy, 4) || !aligned_to(lse, 4) ||
      !aligned_to(top_log_probs, 4) || !aligned_to(top_tokens, 8))
    return GEAR_HIP_EALIGN;
  const int ws = enough(workspace, workspace_bytes, split_bytes(a.rows, a.vocab, top));
  if (ws != 0) return ws;
  a.tokens = tokens, a.wide = tokens_i64 != 0, a.top = (int)top;
  a.log_probs = log_probs, a.entropy = entropy, a.lse = lse, a.top_log_probs = top_log_probs, a.top_tokens = top_tokens;
  return forward<kLogProbs>(a, desc->dtype, static_cast<char *>(workspace), as_stream(stream));
}

extern "C" int gear_hip_token_log_probs_backward(const gear_hip_logits_desc *desc, const float *dlog_probs, const float *dentropy,
                                                 const void *tokens, int tokens_i64, const float *lse, const float *entropy,
                                                 void *dlogits, void *stream) {
  LogitsArgs a = {};
  const int rc = prepare(desc, a);
  if (rc != 0) return rc < 0 ? rc : 0;
  if (lse == nullptr || dlogits == nullptr || (dlog_probs != nullptr && tokens == nullptr) || (dentropy != nullptr && entropy == nullptr))
    return GEAR_HIP_EINVAL;
  if (!aligned_to(tokens, tokens_i64 ? 8 : 4) || !aligned_to(dlogits, element_bytes(desc->dtype)) || !aligned_to(dlog_probs, 4) ||
      !aligned_to(dentropy, 4) || !aligned_to(lse, 4) || !aligned_to(entropy, 4))
    return GEAR_HIP_EALIGN;
  a.tokens = tokens, a.wide = tokens_i64 != 0;
  a.dlog_probs = dlog_probs, a.dentropy = dentropy, a.lse_in = lse, a.entropy_in = entropy, a.dlogits = dlogits;
  return backward<kLogProbs>(a, desc->dtype, as_stream(stream));
}

extern "C" size_t gear_hip_distill_workspace_bytes(int64_t rows, int64_t vocab) { return split_bytes(rows, vocab, 0); }

namespace {
int entries(LogitsArgs &a, const void *top_tokens, int tokens_i64, const float *top_logits, int64_t count) {
  if (count < 1 || top_tokens == nullptr || top_logits == nullptr) return GEAR_HIP_EINVAL;
  if (count > kMaxTop) return GEAR_HIP_ERANGE;
  if (!aligned_to(top_tokens, tokens_i64 ? 8 : 4) || !aligned_to(top_logits, 4)) return GEAR_HIP_EALIGN;
  a.entries = top_tokens, a.wide = tokens_i64 != 0, a.teacher = top_logits, a.count = (int)count;
  return 0;
}
}  // namespace

extern "C" int gear_hip_distill(const gear_hip_logits_desc *desc, const void *top_tokens, int tokens_i64, const float *top_logits,
                                int64_t count, float *loss, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
  LogitsArgs a = {};
  int rc = prepare(desc, a);
  if (rc != 0) return rc < 0 ? rc : 0;
  rc = entries(a, top_tokens, tokens_i64, top_logits, count);
  if (rc != 0) return rc;
  if (loss == nullptr || lse == nullptr) return GEAR_HIP_EINVAL;
  if (!aligned_to(loss, 4) || !aligned_to(lse, 4)) return GEAR_HIP_EALIGN;
  rc = enough(workspace, workspace_bytes, split_bytes(a.rows, a.vocab, 0));
  if (rc != 0) return rc;
  a.loss = loss, a.lse = lse;
  return forward<kDistill>(a, desc->dtype, static_cast<char *>(workspace), as_stream(stream));
}

extern "C" int gear_hip_distill_backward(const gear_hip_logits_desc *desc, const float *dloss, const void *top_tokens, int tokens_i64,
                                         const float *top_logits, int64_t count, const float *lse, void *dlogits, void *stream) {
  LogitsArgs a = {};
  int rc = prepare(desc, a);
  if (rc != 0) return rc < 0 ? rc : 0;
  rc = entries(a, top_tokens, tokens_i64, top_logits, count);
  if (rc != 0) return rc;
  if (dloss == nullptr || lse == nullptr || dlogits == nullptr) return GEAR_HIP_EINVAL;
  if (!aligned_to(dloss, 4) || !aligned_to(lse, 4) || !aligned_to(dlogits, element_bytes(desc->dtype))) return GEAR_HIP_EALIGN;
  a.dloss = dloss, a.lse_in = lse, a.dlogits = dlogits;
  return backward<kDistill>(a, desc->dtype, as_stream(stream));
}
