// Ranges of keys and positions of a batch of windows (gear_hip_token_ranges).
//
// A document is a maximal run of valid steps without a done before its last step, so all that a token
// needs is the nearest start at or below its step and, for documents and prefixes, the nearest end.
// A wave takes 64 steps of one window: both are ballots and bit scans of a 64-bit word.  A document
// that began before the wave's steps (or ends behind them) is looked for there, 1024 steps a look;
// nothing passes between waves, so any number of windows and any length is one launch.
// Two bytes a step are read, 12 (20 with a grid) a token written: launch-bound for the sizes of a batch.
#include "wave.hpp"

namespace gearhip {
namespace {

constexpr int kWaves = 4;

struct RangesArgs {
  const uint8_t *mask, *done;
  int64_t batch, steps, chunks;
  int tokens, mode, cols;
  int64_t prefix;
  int32_t *lo, *hi, *pos;
};

struct Steps {
  const uint8_t *mask, *done;  // of one window
  int64_t steps;
  __device__ __forceinline__ bool valid(int64_t s) const { return s >= 0 && s < steps && (mask == nullptr || mask[s] != 0); }
  __device__ __forceinline__ bool ends(int64_t s) const { return done != nullptr && s >= 0 && s < steps && done[s] != 0; }
  // whether the document of step s, if it has one, ends with it or before the next
  __device__ __forceinline__ bool breaks(int64_t s) const { return !valid(s) || ends(s); }
};

// The largest step below `top` that breaks, or -1.  All lanes of the wave, `top` the same in all.
__device__ __forceinline__ int64_t last_break_below(const Steps &w, int64_t top) {
  constexpr int kEach = 16;
  const int lane = lane_id();
  for (; top > 0; top -= kWave * kEach) {
    const int64_t mine = top - (int64_t)(lane + 1) * kEach;  // this lane looks at [mine, mine + kEach)
    int64_t found = -1;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (mine + e >= 0 && w.breaks(mine + e)) found = mine + e;
    const uint64_t any = wave_ballot(found >= 0);
    if (any) return wave_read_lane(found, (int)__builtin_ctzll(any));
  }
  return -1;
}

// The smallest step from `from` on that breaks, or steps.
__device__ __forceinline__ int64_t first_break_from(const Steps &w, int64_t from) {
  constexpr int kEach = 16;
  const int lane = lane_id();
  for (; from < w.steps; from += kWave * kEach) {
    const int64_t mine = from + (int64_t)lane * kEach;
    int64_t found = -1;
#pragma unroll
    for (int e = kEach - 1; e >= 0; --e)
      if (mine + e < w.steps && w.breaks(mine + e)) found = mine + e;
    const uint64_t any = wave_ballot(found >= 0);
    if (any) return wave_read_lane(found, (int)__builtin_ctzll(any));
  }
  return w.steps;
}

__global__ __launch_bounds__(kWaves *kWave) void token_ranges_kernel(RangesArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (unit >= a.batch * a.chunks) return;
  const int lane = lane_id();
  const int64_t b = unit / a.chunks, base = (unit % a.chunks) * kWave, s = base + lane;
  const Steps w{a.mask ? a.mask + b * a.steps : nullptr, a.done ? a.done + b * a.steps : nullptr, a.steps};

  const bool valid = w.valid(s), ends = w.ends(s);
  const uint64_t valids = wave_ballot(valid), goes_on = wave_ballot(valid && !ends);
  const bool from_before = base > 0 && !w.breaks(base - 1), to_next = w.valid(base + kWave);
  const uint64_t starts = valids & ~((goes_on << 1) | (from_before ? 1u : 0u));
  const uint64_t lasts = valids & (~goes_on | ~((valids >> 1) | (to_next ? 1ull << 63 : 0ull)));
  const bool want_end = a.mode == GEAR_HIP_RANGE_DOCUMENT || a.prefix > 0;

  const int64_t start_before = (valids & 1) && from_before ? last_break_below(w, base - 1) + 1 : 0;
  int64_t end_behind = 0;
  if (want_end && (valids >> 63) != 0 && (lasts >> 63) == 0) {
    end_behind = first_break_from(w, base + kWave);
    if (w.valid(end_behind)) end_behind += 1;  // a done ends its document behind itself
  }
  const uint64_t upto = starts & (~0ull >> (63 - lane)), from = lasts & (~0ull << lane);
  const int64_t s0 = upto ? base + 63 - __builtin_clzll(upto) : start_before;
  const int64_t s1 = from ? base + __builtin_ctzll(from) + 1 : end_behind;

  // what a token needs of its step: fits 32 bits, since steps * tokens does
  const int n = a.tokens;
  const int lo = valid ? (int)(s0 * n) : 0, time = valid ? (int)(s - s0) : 0;
  int hi = 0;  // (causal: filled in per token, at least this)
  if (valid) {
    if (a.mode == GEAR_HIP_RANGE_STEP) hi = (int)((s + 1) * n);
    if (a.mode == GEAR_HIP_RANGE_DOCUMENT) hi = (int)(s1 * n);
    if (a.prefix > 0) hi = max(hi, (int)(min(s0 + a.prefix, s1) * n));
  }
  const int here = (int)min((int64_t)kWave, a.steps - base) * n;
  const int64_t first = (b * a.steps + base) * n;
  for (uint32_t x = 0; x < (uint32_t)here; x += kWave) {  // (all lanes go round alike: the shuffles need them all)
    const uint32_t i = x + lane;
    const int step = i / (uint32_t)n, u = i - (uint32_t)step * n;
    const int t_lo = __shfl(lo, step & 63), t_hi = __shfl(hi, step & 63), t_time = __shfl(time, step & 63);
    const bool ok = (valids >> (step & 63)) & 1;
    if (i >= (uint32_t)here) continue;
    a.lo[first + i] = t_lo;
    const int own = (int)(base * n) + (int)i + 1;
    a.hi[first + i] = ok && a.mode == GEAR_HIP_RANGE_CAUSAL ? max(t_hi, own) : t_hi;
    if (a.cols == 0) {
      a.pos[first + i] = t_time;
    } else {
      int32_t *p = a.pos + (first + i) * 3;
      p[0] = t_time;
      p[1] = ok ? u / a.cols : 0;
      p[2] = ok ? u % a.cols : 0;
    }
  }
}

}  // namespace
}  // namespace gearhip

using namespace gearhip;

extern "C" int gear_hip_token_ranges(const uint8_t *mask, const uint8_t *done, int64_t batch, int64_t steps,
                                     int64_t tokens_per_step, int mode, int64_t prefix, int64_t grid_rows,
                                     int64_t grid_cols, int32_t *lo, int32_t *hi, int32_t *pos, void *stream) {
  if (batch < 0 || steps < 0 || tokens_per_step < 1 || prefix < 0 || grid_rows < 0 || grid_cols < 0)
    return GEAR_HIP_EINVAL;
  if (mode != GEAR_HIP_RANGE_CAUSAL && mode != GEAR_HIP_RANGE_STEP && mode != GEAR_HIP_RANGE_DOCUMENT)
    return GEAR_HIP_EINVAL;
  constexpr int64_t kMost = ((int64_t)1 << 31) - 1;
  if (steps > kMost || tokens_per_step > kMost || grid_rows > kMost || grid_cols > kMost ||
      steps * tokens_per_step > kMost)
    return GEAR_HIP_ERANGE;
  if ((grid_rows > 0) != (grid_cols > 0) || (grid_cols > 0 && grid_rows * grid_cols != tokens_per_step))
    return GEAR_HIP_EINVAL;
  if (batch == 0 || steps == 0) return 0;
  if (lo == nullptr || hi == nullptr || pos == nullptr) return GEAR_HIP_EINVAL;
  RangesArgs a{mask, done, batch, steps, ceil_div64(steps, kWave), (int)tokens_per_step, mode, (int)grid_cols,
               prefix < steps ? prefix : steps, lo, hi, pos};
  if (batch > ((int64_t)kMost * kWaves) / a.chunks) return GEAR_HIP_ERANGE;
  const int64_t blocks = ceil_div64(batch * a.chunks, kWaves);
  hipLaunchKernelGGL(token_ranges_kernel, dim3((unsigned)blocks), dim3(kWaves * kWave), 0, as_stream(stream), a);
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
