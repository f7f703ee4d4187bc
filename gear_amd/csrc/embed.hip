// Rows of a table by token, scaled, and the gradient of the table (gear_hip_embed and the call beside it).
//
// out[n] = scale * table[token[n]];  dtable[v] = scale * sum over n with token[n] = v of dout[n].  Tokens outside the
// vocabulary give rows of zeros and take part in no sum.
//
// Both are bound by memory.  The gradient has no atomics on results, so that it is the same on every run: positions are
// sorted by token (stable), and the sorted list is cut into chunks of equal length whatever the tokens are.  A group of
// lanes, each with 16 bytes of columns, goes through a chunk's rows in order and adds up runs of one token in 32 bits.
// A run inside its chunk goes straight to the table; a run that a border cuts leaves a partial sum on each side of it,
// and a last launch adds those up.  So a token that is half of the batch costs no more than one that is rare.
//
// The sort: a batch of 4096 positions or less is ranked in one launch.  More of them, in a vocabulary of less than 4096:
// one pass by counting, tiles' counts, their prefixes, and a workgroup a tile that ranks its positions in order (184320
// positions, 1025 tokens: 5 + 6 + 10 us, where two digits of 8 bits take 30).  Else digits of 8 bits (radix_sort.hpp), or, for
// three of them and up to 32768 positions, one launch (range_sort.hpp; two digits of 16016 words take 18 us, one launch 23,
// because some words are everywhere).
//
// Measured, us: 184320 x 512 bf16 of 1025 rows: look-up 31 (6.1 TB/s), gradient 68, of which 39 for the rows (4.8 TB/s: 1 KB each, in
// no order); 16016 x 768 in 32 bits of 33025 rows: 13 and 54, of which 14 to clear the table (7.2 TB/s) and 18 for the sort.
#include <algorithm>

#include "range_sort.hpp"
#include "rows.hpp"

namespace gearhip {
namespace {

constexpr int kBlock = 256;
constexpr int kAhead = 16;  // rows in flight

struct EmbedArgs {
  const void *tokens;
  int wide;
  int64_t n, vocab;
  int width;
  const void *rows;  // table, or dout
  int64_t stride;
  void *to;          // out, or dtable: contiguous
  float scale;
  bool once;
};

// Two rows a group of lanes (184320 x 512 bf16 from 1025 rows: 1, 2, 4, 8 rows 52, 29, 30, 34 us).  Rows of more than the L2
// caches hold are written past them (300000 x 512 from 33025 rows: 91 -> 57 us).
constexpr int kRowsEach = 2;
constexpr int64_t kOnceBytes = 32 << 20;

// kRows rows a group of lanes
template <typename T, int kLanes, int kRows>
__global__ __launch_bounds__(kBlock) void embed_kernel(EmbedArgs a) {
  constexpr int kGroups = kBlock / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool tiny = kLanes == 4 && a.width < kPer<T>;  // (a row of a vector has few lanes)
  for (int64_t base = ((int64_t)blockIdx.x * kGroups + threadIdx.x / kLanes) * kRows; base < a.n;
       base += (int64_t)gridDim.x * kGroups * kRows) {
    int64_t token[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) token[r] = base + r < a.n ? token_at(a.tokens, a.wide, base + r, a.vocab) : -1;
    for (int v = lane; v * kPer<T> < a.width; v += kLanes) {
      const Slot<T> s(v, a.width);
      Raw<T> x[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        x[r] = Raw<T>{};
        if (token[r] >= 0) x[r] = load_slot<T>(static_cast<const T *>(a.rows) + token[r] * a.stride, s, tiny);
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (base + r < a.n) {
          T *to = static_cast<T *>(a.to) + (base + r) * a.width;
          const Vals<T> y = values_of<T>(x[r]) * a.scale;
          if (a.once && s.whole())
            store_raw<true>(to + s.col, __builtin_convertvector(y, Raw<T>));
          else
            store_slot(to, s, y);
        }
    }
  }
}

// ---- the gradient: positions by token -----------------------------------------------------------------------------
// The table begins as zeros, for the rows that nothing is added to (`threads` threads, i0 the first).
__device__ __forceinline__ void clear(char *table, int64_t bytes, int64_t i0, int64_t threads) {
  // (it may begin and end at any element)
  const int64_t head = (16 - (int64_t)(reinterpret_cast<uintptr_t>(table) & 15)) & 15, whole = bytes > head ? (bytes - head) / 16 : 0;
  for (int64_t i = i0; i < whole; i += threads) reinterpret_cast<u32x4 *>(table + head)[i] = u32x4{0, 0, 0, 0};
  const int64_t edge = bytes - whole * 16;  // bytes before and behind
  for (int64_t i = i0 * 2; i < edge; i += threads * 2) *reinterpret_cast<uint16_t *>(table + (i < head ? i : i + whole * 16)) = 0;
}
// What a position is sorted by; none comes last.
__device__ __forceinline__ uint32_t key_of(const EmbedArgs &a, int64_t i) {
  const int64_t token = token_at(a.tokens, a.wide, i, a.vocab);
  return token < 0 ? (uint32_t)a.vocab : (uint32_t)token;
}

__global__ __launch_bounds__(kBlock) void embed_keys_kernel(EmbedArgs a, uint32_t *keys, uint32_t *places, char *table,
                                                            int64_t bytes) {
  const int64_t threads = (int64_t)gridDim.x * kBlock, i0 = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (keys != nullptr)
    for (int64_t i = i0; i < a.n; i += threads) keys[i] = key_of(a, i), places[i] = (uint32_t)i;
  clear(table, bytes, i0, threads);
}

// One launch for up to 20 000 or so: reads the tokens, writes keys and places in order.
struct TokenKeys {
  EmbedArgs a;
  __device__ __forceinline__ void begin() {}
  __device__ __forceinline__ uint32_t key(int j) const { return key_of(a, j); }
};
struct EmitPlaces {
  EmbedArgs a;
  uint32_t *keys, *places;
  __device__ __forceinline__ void put(uint32_t place, int j) const { keys[place] = key_of(a, j), places[place] = (uint32_t)j; }
  template <typename L>
  __device__ __forceinline__ void list(const L &list, const uint32_t *rank, int n, uint32_t base) const {
    const int e = threadIdx.x;
    if (e < n) put(base + rank[e], list.pos(e));
  }
  __device__ __forceinline__ void equal(const uint32_t *at, int n, uint32_t base) const {
    const int e = threadIdx.x;
    if (e < n) put(base + (uint32_t)e, (int)at[e]);
  }
};

// By counting: tiles of kTile positions, bins of one token.
constexpr int kTile = 1024, kMostBins = 4096, kMostTiles = 1024;
struct CountArgs {
  EmbedArgs e;
  int tiles, bins;
  uint32_t *table, *totals;  // [tiles][bins]: counts, then how many of a bin lie in tiles before; [bins]
  uint32_t *keys, *places;
};
__global__ __launch_bounds__(kBlock) void embed_count_kernel(CountArgs a, char *table, int64_t bytes) {
  if ((int)blockIdx.x >= a.tiles) {
    clear(table, bytes, (int64_t)(blockIdx.x - a.tiles) * kBlock + threadIdx.x, (int64_t)(gridDim.x - a.tiles) * kBlock);
    return;
  }
  __shared__ uint32_t count[kMostBins];
  for (int b = threadIdx.x; b < a.bins; b += kBlock) count[b] = 0;
  const int64_t first = (int64_t)blockIdx.x * kTile;
  uint32_t key[kTile / kBlock];
#pragma unroll
  for (int i = 0; i < kTile / kBlock; ++i) {
    const int64_t at = first + threadIdx.x + i * kBlock;
    key[i] = at < a.e.n ? key_of(a.e, at) : ~0u;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kTile / kBlock; ++i)
    if (key[i] < (uint32_t)a.bins) atomicAdd(&count[key[i]], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < a.bins; b += kBlock) a.table[(int64_t)blockIdx.x * a.bins + b] = count[b];
}
// 64 bins a workgroup, the tiles in 16 stretches
constexpr int kStretches = 16;
__global__ __launch_bounds__(kWave *kStretches) void embed_prefix_kernel(CountArgs a) {
  __shared__ uint32_t sums[kStretches][kWave];
  const int lane = threadIdx.x % kWave, stretch = threadIdx.x / kWave, bin = blockIdx.x * kWave + lane;
  const int each = (a.tiles + kStretches - 1) / kStretches, t0 = stretch * each, t1 = min(t0 + each, a.tiles);
  uint32_t sum = 0;
  if (bin < a.bins)
#pragma unroll 8
    for (int t = t0; t < t1; ++t) sum += a.table[(int64_t)t * a.bins + bin];
  sums[stretch][lane] = sum;
  __syncthreads();
  if (bin >= a.bins) return;
  uint32_t run = 0, total = 0;
#pragma unroll
  for (int s = 0; s < kStretches; ++s) {
    run += s < stretch ? sums[s][lane] : 0u;
    total += sums[s][lane];
  }
  if (stretch == 0) a.totals[bin] = total;
#pragma unroll 8
  for (int t = t0; t < t1; ++t) {
    const uint32_t c = a.table[(int64_t)t * a.bins + bin];
    a.table[(int64_t)t * a.bins + bin] = run;
    run += c;
  }
}
// Four waves a tile: each ranks a quarter of it in order, and begins where the quarters before end.
__global__ __launch_bounds__(kBlock) void embed_place_kernel(CountArgs a) {
  constexpr int kQuarters = kBlock / kWave, kRounds = kTile / kBlock;
  __shared__ uint32_t next[kMostBins];
  __shared__ uint16_t count[kQuarters][kMostBins];
  __shared__ uint32_t sums[kQuarters];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t first = (int64_t)blockIdx.x * kTile + wave * (kTile / kQuarters);
  uint32_t key[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int64_t at = first + i * kWave + lane;
    key[i] = at < a.e.n ? key_of(a.e, at) : ~0u;
  }
  // bins below a wave's own, and where each begins
  constexpr int kMostLoads = kMostBins / kBlock;
  const int each = (a.bins + kBlock - 1) / kBlock, loads = min(each, kMostLoads);
  const int bin0 = wave * loads * kWave;
  uint32_t total[kMostLoads], before[kMostLoads], sum = 0;
#pragma unroll
  for (int i = 0; i < kMostLoads; ++i) {
    const int b = bin0 + i * kWave + lane;
    const bool here = i < loads && b < a.bins;
    total[i] = here ? a.totals[b] : 0u, before[i] = here ? a.table[(int64_t)blockIdx.x * a.bins + b] : 0u;
    sum += total[i];
  }
  for (int b = threadIdx.x; b < a.bins; b += kBlock)
#pragma unroll
    for (int q = 0; q < kQuarters; ++q) count[q][b] = 0;
  sum = (uint32_t)wave_sum((int)sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  uint32_t carry = 0;
  for (int w = 0; w < wave; ++w) carry += sums[w];
#pragma unroll
  for (int i = 0; i < kMostLoads; ++i)
    if (i < loads) {
      const int b = bin0 + i * kWave + lane;
      const uint32_t upto = (uint32_t)wave_inclusive_sum((int)total[i]);
      if (b < a.bins) next[b] = carry + upto - total[i] + before[i];
      carry += (uint32_t)wave_read_lane((int)upto, kWave - 1);
    }
  const int bits = 32 - __builtin_clz((uint32_t)a.bins);
  const uint64_t lower = lane == 0 ? 0ull : ~0ull >> (64 - lane);
  uint32_t rank[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const bool valid = key[i] < (uint32_t)a.bins;
    uint64_t peers = __ballot(valid);
    for (int b = 0; b < bits; ++b) {
      const bool bit = (key[i] >> b) & 1u;
      const uint64_t with = __ballot(bit);
      peers &= bit ? with : ~with;
    }
    const uint32_t seen = valid ? count[wave][key[i]] : 0u;
    wave_lds_sync();
    const uint32_t mine = (uint32_t)__popcll(peers & lower);
    if (valid && mine == 0) count[wave][key[i]] = (uint16_t)(seen + (uint32_t)__popcll(peers));
    wave_lds_sync();
    rank[i] = seen + mine;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    if (key[i] >= (uint32_t)a.bins) continue;
    uint32_t at = next[key[i]] + rank[i];
    for (int w = 0; w < wave; ++w) at += count[w][key[i]];
    a.keys[at] = key[i], a.places[at] = (uint32_t)(first + i * kWave + lane);
  }
}

// ---- the gradient: sums -------------------------------------------------------------------------------------------
struct SumArgs {
  EmbedArgs e;
  const uint32_t *keys, *places;  // sorted
  int64_t chunks;
  int chunk, tiles;
  float *parts;  // [chunks][2][tiles * kLanes * kPer]: of the run that a chunk begins in, of the run that it ends in
};

// x of lane `from` of a group
template <int kLanes>
__device__ __forceinline__ uint32_t of_lane(uint32_t x, int from) {
  return kLanes == kWave ? (uint32_t)__builtin_amdgcn_readlane((int)x, from) : (uint32_t)__shfl((int)x, from, kLanes);
}

template <typename T, int kLanes>
__global__ __launch_bounds__(kBlock) void embed_sums_kernel(SumArgs a) {
  constexpr int kHeld = kLanes < kAhead ? kAhead / kLanes : 1;  // positions of a lane
  constexpr int kStep = kLanes * kHeld;
  const int64_t unit = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / kLanes, chunk = unit / a.tiles;
  const int lane = threadIdx.x % kLanes;
  const bool here = chunk < a.chunks;  // (the lanes of a wave exchange positions)
  const int v = (int)(unit - chunk * a.tiles) * kLanes + lane;
  const Slot<T> s(v, a.e.width);
  const bool tiny = kLanes == 4 && a.e.width < kPer<T>;
  const int64_t begin = chunk * a.chunk, end = here ? min(begin + a.chunk, a.e.n) : begin, pitch = (int64_t)a.tiles * kLanes * kPer<T>;
  const uint32_t none = (uint32_t)a.e.vocab;
  const uint32_t before = here && begin > 0 ? a.keys[begin - 1] : ~0u, after = here && end < a.e.n ? a.keys[end] : ~0u;
  uint32_t current = none;
  bool first = true, any = false;
  Vals<T> sum = {};
  auto flush = [&](bool last) __attribute__((always_inline)) {
    if (current == none || !s.any()) return;
    if (first && before == current)
      *reinterpret_cast<Vals<T> *>(a.parts + chunk * 2 * pitch + v * kPer<T>) = sum;
    else if (last && after == current)
      *reinterpret_cast<Vals<T> *>(a.parts + (chunk * 2 + 1) * pitch + v * kPer<T>) = sum;
    else
      store_slot(static_cast<T *>(a.e.to) + (int64_t)current * a.e.width, s, sum * a.e.scale);
  };
  for (int at = 0; at < a.chunk; at += kStep) {
    uint32_t keys[kHeld], places[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int64_t p = begin + at + i * kLanes + lane;
      keys[i] = p < end ? a.keys[p] : ~0u, places[i] = p < end ? a.places[p] : 0u;
    }
#pragma unroll 1
    for (int b = 0; b < kStep && at + b < a.chunk; b += kAhead) {
      uint32_t key[kAhead];
      Raw<T> row[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        key[i] = kHeld > 1 ? of_lane<kLanes>(keys[i / kLanes], i % kLanes) : of_lane<kLanes>(keys[0], b + i);
        const uint32_t place = kHeld > 1 ? of_lane<kLanes>(places[i / kLanes], i % kLanes) : of_lane<kLanes>(places[0], b + i);
        row[i] = Raw<T>{};
        if (key[i] < none) {  // (lanes without columns read the first ones)
          const T *from = static_cast<const T *>(a.e.rows) + (int64_t)place * a.e.stride;
          row[i] = tiny ? load_slot<T>(from, s, true) : load_raw<true>(from + s.col);  // (read once)
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (key[i] == ~0u) continue;  // (behind the last position)
        if (key[i] != current) {
          flush(false);
          first = !any;
          current = key[i];
          sum = Vals<T>{};
        }
        any = true;
        sum += values_of<T>(row[i]);
      }
    }
  }
  flush(true);
}

// The runs that borders cut: a wave for every chunk (and tile of columns) that such a run may begin in; a run of very many
// chunks is added up by all waves of a workgroup.
constexpr int kJoinBlock = 1024, kJoinWaves = kJoinBlock / kWave;
constexpr int kLongRun = 64;
template <typename T, int kLanes>
__global__ __launch_bounds__(kJoinBlock) void embed_join_kernel(SumArgs a) {
  constexpr int kGroups = kWave / kLanes;
  __shared__ Vals<T> pile[kJoinWaves][kLanes];
  __shared__ int64_t runs[kJoinWaves];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, column = lane % kLanes, group = lane / kLanes;
  const int64_t units = a.chunks * a.tiles, pitch = (int64_t)a.tiles * kLanes * kPer<T>;
  // the sum of the partial ones of chunks from + group, ..., `by` apart, over the groups of a wave
  auto total = [&](int64_t from, int64_t upto, int64_t by, int v) __attribute__((always_inline)) {
    Vals<T> sum = {};
#pragma unroll 8
    for (int64_t c = from + group; c <= upto; c += by)
      sum += *reinterpret_cast<const Vals<T> *>(a.parts + c * 2 * pitch + v * kPer<T>);
#pragma unroll
    for (int x = kLanes; x < kWave; x *= 2)
#pragma unroll
      for (int e = 0; e < kPer<T>; ++e) sum[e] += __shfl_xor(sum[e], x);
    return sum;
  };
  for (int64_t base = (int64_t)blockIdx.x * kJoinWaves; base < units; base += (int64_t)gridDim.x * kJoinWaves) {
    const int64_t unit = base + wave, chunk = unit / a.tiles, begin = chunk * a.chunk, end = begin + a.chunk;
    const int v = (int)(unit - chunk * a.tiles) * kLanes + column;
    const Slot<T> s(v, a.e.width);
    uint32_t key = ~0u;
    if (unit < units && end < a.e.n) {
      key = a.keys[end - 1];
      if (key == (uint32_t)a.e.vocab || a.keys[end] != key) key = ~0u;
      // (a run that began before is another chunk's)
      if (key != ~0u && a.keys[begin] == key && begin > 0 && a.keys[begin - 1] == key) key = ~0u;
    }
    int64_t last = chunk;  // the last chunk that begins with it
    if (key != ~0u) {
      for (;;) {
        const int64_t c = last + 1 + lane;
        const uint64_t other = __ballot(!(c < a.chunks && a.keys[c * a.chunk] == key));
        const int more = other == 0 ? kWave : __builtin_ctzll(other);
        last += more;
        if (more < kWave) break;
      }
    }
    const bool is_long = last - chunk > kLongRun;
    auto put = [&](const Vals<T> &sum, const Slot<T> &at, uint32_t token) __attribute__((always_inline)) {
      if (group == 0 && at.any()) store_slot(static_cast<T *>(a.e.to) + (int64_t)token * a.e.width, at, sum * a.e.scale);
    };
    auto begun = [&](int64_t c, int at) __attribute__((always_inline)) {
      return *reinterpret_cast<const Vals<T> *>(a.parts + (c * 2 + 1) * pitch + at * kPer<T>);
    };
    if (key != ~0u && !is_long) put(total(chunk + 1, last, kGroups, v) + begun(chunk, v), s, key);
    __syncthreads();  // (of the units before)
    if (lane == 0) runs[wave] = is_long ? last : -1;
    __syncthreads();
    for (int w = 0; w < kJoinWaves; ++w) {
      const int64_t upto = runs[w];
      if (upto < 0) continue;
      const int64_t c = (base + w) / a.tiles;
      const int at = (int)(base + w - c * a.tiles) * kLanes + column;
      const Vals<T> mine = total(c + 1 + wave * kGroups, upto, kJoinWaves * kGroups, at);
      if (group == 0) pile[wave][column] = mine;
      __syncthreads();
      if (wave == 0) {
        Vals<T> sum = begun(c, at);
        for (int k = 0; k < kJoinWaves; ++k) sum += pile[k][column];
        put(sum, Slot<T>(at, a.e.width), a.keys[(c + 1) * a.chunk]);
      }
      __syncthreads();
    }
  }
}

// f(T(), lanes of a row)
template <typename F>
void by_type_and_lanes(int dtype, int width, const F &f) {
  by_type(dtype, [&](auto type) {
    const int vecs = (width + kPer<decltype(type)> - 1) / kPer<decltype(type)>;
    if (vecs <= 4)
      f(type, std::integral_constant<int, 4>());
    else if (vecs <= 16)
      f(type, std::integral_constant<int, 16>());
    else
      f(type, std::integral_constant<int, 64>());
  });
}

constexpr int kColumns = 64 * 8;  // most columns of a group of lanes
struct Plan {
  int chunk, pitch;
  int64_t chunks;
  size_t keys, places, keys_tmp, places_tmp, sorted_keys, sorted_places, hist, parts, total;
};
// Chunks of 16 to 256 positions: short ones where there are few (4096 groups of lanes fill the GPU), long ones for fewer borders.
// The workspace goes by the number of tokens and the width, whatever the vocabulary.
Plan plan_of(int64_t n, int width) {
  Plan p;
  p.chunk = 16;
  while (p.chunk < 256 && ceil_div64(n, p.chunk) > 4096) p.chunk *= 2;
  p.chunks = ceil_div64(n, p.chunk);
  p.pitch = (width + kColumns - 1) / kColumns * kColumns;  // at least what a group of lanes covers, in any type
  const size_t list = align_up((size_t)n * 4, 256);
  p.keys = 0, p.places = list, p.keys_tmp = 2 * list, p.places_tmp = 3 * list, p.sorted_keys = 4 * list, p.sorted_places = 5 * list;
  p.hist = 6 * list;
  const size_t counts = ceil_div64(n, kTile) <= kMostTiles ? (size_t)(ceil_div64(n, kTile) + 1) * kMostBins * 4 : 0;
  p.parts = align_up(p.hist + std::max(radix::hist_bytes(n), counts), 256);
  p.total = p.parts + (size_t)p.chunks * 2 * (size_t)p.pitch * 4;
  return p;
}

constexpr int64_t kMostTokens = (int64_t)1 << 31;
constexpr int kMaxWidth = 1 << 20;

int check(int64_t n, int64_t vocab, int64_t width, int dtype, float scale) {
  if (n < 0 || vocab < 0 || width < 1 || element_bytes(dtype) == 0 || !(scale - scale == 0)) return GEAR_HIP_EINVAL;
  if (n >= kMostTokens || vocab >= kMostTokens - 1 || width > kMaxWidth) return GEAR_HIP_ERANGE;
  return 0;
}
}  // namespace
}  // namespace gearhip

using namespace gearhip;

extern "C" int gear_hip_embed(const void *tokens, int tokens_i64, int64_t n, const void *table, int64_t table_stride,
                              int64_t vocab, int64_t width, int dtype, float scale, void *out, void *stream) {
  const int rc = check(n, vocab, width, dtype, scale);
  if (rc != 0) return rc;
  if (n == 0) return 0;
  if (tokens == nullptr || out == nullptr || (vocab > 0 && table == nullptr)) return GEAR_HIP_EINVAL;
  const int element = element_bytes(dtype);
  if (!aligned_to(tokens, tokens_i64 ? 8 : 4) || !aligned_to(table, element) || !aligned_to(out, element)) return GEAR_HIP_EALIGN;
  const EmbedArgs a{tokens, tokens_i64 != 0, n, vocab, (int)width, table, table_stride, out, scale, n * width * element >= kOnceBytes};
  by_type_and_lanes(dtype, (int)width, [&](auto type, auto lanes) {
    constexpr int kLanes = decltype(lanes)::value;
    constexpr int kRows = kRowsEach;
    const int64_t blocks = ceil_div64(n, kBlock / kLanes * kRows), most = kMostItems / kBlock;
    hipLaunchKernelGGL((embed_kernel<decltype(type), kLanes, kRows>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(kBlock), 0,
                       as_stream(stream), a);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}

extern "C" size_t gear_hip_embed_backward_workspace_bytes(int64_t n, int64_t width) {
  if (n <= 0 || n >= kMostTokens || width < 1 || width > kMaxWidth) return 0;
  return plan_of(n, (int)width).total;
}

extern "C" int gear_hip_embed_backward(const void *dout, int64_t dout_stride, const void *tokens, int tokens_i64, int64_t n,
                                       int64_t vocab, int64_t width, int dtype, float scale, void *dtable, void *workspace,
                                       size_t workspace_bytes, void *stream) {
  const int rc = check(n, vocab, width, dtype, scale);
  if (rc != 0) return rc;
  if (vocab == 0) return 0;
  if (dtable == nullptr || (n > 0 && (tokens == nullptr || dout == nullptr))) return GEAR_HIP_EINVAL;
  const int element = element_bytes(dtype);
  if (!aligned_to(tokens, tokens_i64 ? 8 : 4) || !aligned_to(dout, element) || !aligned_to(dtable, element)) return GEAR_HIP_EALIGN;
  const Plan p = plan_of(n, (int)width);
  if (p.chunks * (p.pitch / 256) > kMostItems / kWave) return GEAR_HIP_ERANGE;
  if (n > 0 && (workspace == nullptr || workspace_bytes < p.total)) return GEAR_HIP_EWORKSPACE;
  if (n > 0 && !aligned_to(workspace, 16)) return GEAR_HIP_EALIGN;
  hipStream_t st = as_stream(stream);
  char *ws = static_cast<char *>(workspace);
  auto list = [&](size_t at) { return reinterpret_cast<uint32_t *>(ws + at); };
  EmbedArgs e{tokens, tokens_i64 != 0, n, vocab, (int)width, dout, dout_stride, dtable, scale, false};
  const int64_t bytes = vocab * width * element;
  const int bits = 64 - __builtin_clzll((uint64_t)vocab);
  const int64_t fill = std::min<int64_t>(ceil_div64(bytes / 16 + 1, kBlock), 8192);
  char *table = static_cast<char *>(dtable);
  if (n > radix::kRankMax && vocab < kMostBins && ceil_div64(n, kTile) <= kMostTiles) {
    const int tiles = (int)ceil_div64(n, kTile), bins = (int)vocab + 1;
    const CountArgs c{e, tiles, bins, list(p.hist) + kMostBins, list(p.hist), list(p.sorted_keys), list(p.sorted_places)};
    embed_count_kernel<<<dim3((unsigned)(tiles + fill)), dim3(kBlock), 0, st>>>(c, table, bytes);
    embed_prefix_kernel<<<dim3((unsigned)((bins + kWave - 1) / kWave)), dim3(kWave * kStretches), 0, st>>>(c);
    embed_place_kernel<<<dim3((unsigned)tiles), dim3(kBlock), 0, st>>>(c);
    GEARHIP_RETURN_IF_LAUNCH_FAILED();
  } else {
    const bool one = bits > 16 && n > radix::kRankMax && ranges::fits(n) && n <= ranges::worth(bits);
    const bool lists = n > 0 && !one;
    const int64_t blocks = std::max(fill, lists ? std::min<int64_t>(ceil_div64(n, kBlock), 8192) : 0);
    embed_keys_kernel<<<dim3((unsigned)blocks), dim3(kBlock), 0, st>>>(e, lists ? list(p.keys) : nullptr,
                                                                       lists ? list(p.places) : nullptr, table, bytes);
    GEARHIP_RETURN_IF_LAUNCH_FAILED();
    if (n == 0) return 0;
    const int sorted =
        one ? ranges::sort<uint32_t, true>(TokenKeys{e}, n, EmitPlaces{e, list(p.sorted_keys), list(p.sorted_places)}, st)
            : radix::sort_pairs<uint32_t, uint32_t>(list(p.keys), list(p.sorted_keys), list(p.places), list(p.sorted_places),
                                                    list(p.keys_tmp), list(p.places_tmp), n, 0, bits, list(p.hist), st);
    if (sorted != 0) return sorted;
  }
  SumArgs a{e, list(p.sorted_keys), list(p.sorted_places), p.chunks, p.chunk, 0, reinterpret_cast<float *>(ws + p.parts)};
  by_type_and_lanes(dtype, (int)width, [&](auto type, auto lanes) {
    using T = decltype(type);
    constexpr int kLanes = decltype(lanes)::value;
    a.tiles = ((int)width + kPer<T> * kLanes - 1) / (kPer<T> * kLanes);
    const int64_t units = a.chunks * a.tiles;
    hipLaunchKernelGGL((embed_sums_kernel<T, kLanes>), dim3((unsigned)ceil_div64(units, kBlock / kLanes)), dim3(kBlock), 0, st, a);
    const int64_t joins = std::min<int64_t>(ceil_div64(units, kJoinWaves), kMostItems / kJoinBlock);
    hipLaunchKernelGGL((embed_join_kernel<T, kLanes>), dim3((unsigned)joins), dim3(kJoinBlock), 0, st, a);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
