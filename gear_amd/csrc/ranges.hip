// Ranges of keys and positions of a batch of windows (gear_hip_token_ranges).
//
// A document is a maximal run of valid steps without a done before its last step, so all that a token
// needs is the nearest start at or below its step and, for documents and prefixes, the nearest end.
// A wave takes 64 steps of one window: both are ballots and bit scans of a 64-bit word.  A document
// that began before the wave's steps (or ends behind them) is looked for there, 1024 steps a look;
// nothing passes between waves, so any number of windows and any length is one launch.  Where 64 steps are many
// tokens, several waves find the same ranges and each writes kWrite tokens of them (8 x 1000 steps of 49 tokens: 22 us by
// one wave, 7 by several).
// Two bytes a step are read, 12 (20 with a grid) a token written: launch-bound for the sizes of a batch.
#include "wave.hpp"

namespace gearhip {
namespace {

constexpr int kWaves = 4;
constexpr int kWrite = 256;  // tokens a wave writes

struct RangesArgs {
  const uint8_t *mask, *done;
  int64_t batch, steps;
  uint32_t chunks, slices;  // of 64 steps of a window; of a chunk's tokens
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

// Which of the 16 steps from s on break, a bit each; steps outside the window do not.
__device__ __forceinline__ uint32_t breaks16(const Steps &w, int64_t s) {
  if (s <= -16 || s >= w.steps) return 0;
  uint32_t found = 0;
  if (w.steps < 16) {
    for (int e = 0; e < 16; ++e)
      if (s + e >= 0 && s + e < w.steps && w.breaks(s + e)) found |= 1u << e;
    return found;
  }
  const int64_t at = min(max(s, (int64_t)0), w.steps - 16);  // the nearest 16 inside, shifted into place
  u32x4 m = {~0u, ~0u, ~0u, ~0u}, d = {};
  if (w.mask != nullptr) m = reinterpret_cast<const u32x4_any *>(w.mask + at)->v;
  if (w.done != nullptr) d = reinterpret_cast<const u32x4_any *>(w.done + at)->v;
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (((m[e / 4] >> (e % 4 * 8)) & 0xff) == 0 || ((d[e / 4] >> (e % 4 * 8)) & 0xff) != 0) found |= 1u << e;
  return s < at ? (found << (int)(at - s)) & 0xffff : found >> (int)(s - at);
}

// The largest step below `top` that breaks, or -1.  All lanes of the wave, `top` the same in all.
__device__ __forceinline__ int64_t last_break_below(const Steps &w, int64_t top) {
  const int lane = lane_id();
  for (; top > 0; top -= kWave * 16) {
    const int64_t mine = top - (int64_t)(lane + 1) * 16;
    const uint32_t found = breaks16(w, mine);
    const uint64_t any = wave_ballot(found != 0);
    if (any) return wave_read_lane(mine + 31 - __builtin_clz(found | 1), (int)__builtin_ctzll(any));
  }
  return -1;
}

// The smallest step from `from` on that breaks, or steps.
__device__ __forceinline__ int64_t first_break_from(const Steps &w, int64_t from) {
  const int lane = lane_id();
  for (; from < w.steps; from += kWave * 16) {
    const int64_t mine = from + (int64_t)lane * 16;
    const uint32_t found = breaks16(w, mine);
    const uint64_t any = wave_ballot(found != 0);
    if (any) return wave_read_lane(mine + __builtin_ctz(found | 1u << 31), (int)__builtin_ctzll(any));
  }
  return w.steps;
}

__global__ __launch_bounds__(kWaves *kWave) void token_ranges_kernel(RangesArgs a) {
  const uint32_t unit = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t chunk = unit / a.slices, slice = unit - chunk * a.slices, window = chunk / a.chunks;
  if (window >= a.batch) return;
  const int lane = lane_id();
  const int64_t b = window, base = (int64_t)(chunk - window * a.chunks) * kWave, s = base + lane;
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
  const uint32_t here = (uint32_t)min((int64_t)kWave, a.steps - base) * n;
  const uint32_t from_token = slice * kWrite, to_token = min(here, from_token + kWrite);
  const int64_t first = (b * a.steps + base) * n;
  for (uint32_t x = from_token; x < to_token; x += kWave) {  // (all lanes go round alike: the shuffles need them all)
    const uint32_t i = x + lane;
    const int step = i / (uint32_t)n, u = i - (uint32_t)step * n;
    const int t_lo = __shfl(lo, step & 63), t_hi = __shfl(hi, step & 63), t_time = __shfl(time, step & 63);
    const bool ok = (valids >> (step & 63)) & 1;
    if (i >= to_token) continue;
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
  const int64_t longest = steps < kWave ? steps : kWave;
  RangesArgs a{mask, done, batch, steps, (uint32_t)ceil_div64(steps, kWave), (uint32_t)ceil_div64(longest * tokens_per_step, kWrite), (int)tokens_per_step, mode, (int)grid_cols,
               prefix < steps ? prefix : steps, lo, hi, pos};
  // a launch has less than 2^32 work items; a window needs at most 2^25 waves
  const int64_t waves = (int64_t)a.chunks * a.slices, most = (kMostItems / kWave - kWaves) / waves;
  for (int64_t from = 0; from < batch; from += most) {
    a.batch = batch - from < most ? batch - from : most;
    hipLaunchKernelGGL(token_ranges_kernel, dim3((unsigned)ceil_div64(a.batch * waves, kWaves)), dim3(kWaves * kWave), 0,
                       as_stream(stream), a);
    GEARHIP_RETURN_IF_LAUNCH_FAILED();
    const int64_t tokens = a.batch * steps * tokens_per_step;
    if (a.mask != nullptr) a.mask += a.batch * steps;
    if (a.done != nullptr) a.done += a.batch * steps;
    a.lo += tokens, a.hi += tokens, a.pos += tokens * (grid_cols > 0 ? 3 : 1);
  }
  return 0;
}
