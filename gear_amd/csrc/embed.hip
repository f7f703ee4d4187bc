// Rows of a table by token, scaled, and the gradient of the table (gear_hip_embed and the call beside it).
//
// out[n] = scale * table[token[n]];  dtable[v] = scale * sum over n with token[n] = v of dout[n].  Tokens outside the
// vocabulary give rows of zeros and take part in no sum.
//
// Both are bound by memory.  The gradient has no atomics, so that it is the same on every run: positions are sorted by
// token (stable), and the sorted list is cut into chunks of equal length whatever the tokens are.  A group of lanes, each
// with 16 bytes of columns, goes through a chunk's rows in order and adds up runs of one token in 32 bits.  A run inside
// its chunk goes straight to the table; a run that a border cuts leaves a partial sum on each side of it, and a second
// launch adds those up.  So a token that is half of the batch costs no more than one that is rare.
#include <algorithm>

#include "radix_sort.hpp"
#include "rows.hpp"

namespace gearhip {
namespace {

constexpr int kBlock = 256;
constexpr int kJoinBlock = 1024;
constexpr int kAhead = 8;  // rows in flight

struct EmbedArgs {
  const void *tokens;
  int wide;
  int64_t n, vocab;
  int width;
  const void *rows;  // table, or dout
  int64_t stride;
  void *to;          // out, or dtable: contiguous
  float scale;
};

template <typename T, int kLanes>
__global__ __launch_bounds__(kBlock) void embed_kernel(EmbedArgs a) {
  constexpr int kRows = kBlock / kLanes;
  const int lane = threadIdx.x % kLanes;
  for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes; row < a.n; row += (int64_t)gridDim.x * kRows) {
    const int64_t token = token_at(a.tokens, a.wide, row, a.vocab);
    const T *from = static_cast<const T *>(a.rows) + token * a.stride;
    T *to = static_cast<T *>(a.to) + row * a.width;
    for (int v = lane; v * kPer<T> < a.width; v += kLanes) {
      const Slot<T> s(v, a.width);
      Vals<T> x = {};
      if (token >= 0) x = __builtin_convertvector(load_slot<T>(from, s, a.width < kPer<T>), Vals<T>) * a.scale;
      store_slot(to, s, x);
    }
  }
}

// Keys and positions to sort; tokens that are none come last.  The table begins as zeros, for the rows that nothing is added to.
__global__ __launch_bounds__(kBlock) void embed_keys_kernel(EmbedArgs a, uint32_t *keys, uint32_t *places, char *table,
                                                            int64_t bytes) {
  const int64_t threads = (int64_t)gridDim.x * kBlock, i0 = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  for (int64_t i = i0; i < a.n; i += threads) {
    const int64_t token = token_at(a.tokens, a.wide, i, a.vocab);
    keys[i] = token < 0 ? (uint32_t)a.vocab : (uint32_t)token;
    places[i] = (uint32_t)i;
  }
  // (rows of the table end at any element)
  const int64_t head = (16 - (int64_t)(reinterpret_cast<uintptr_t>(table) & 15)) & 15, whole = bytes > head ? (bytes - head) / 16 : 0;
  for (int64_t i = i0; i < whole; i += threads) reinterpret_cast<u32x4 *>(table + head)[i] = u32x4{0, 0, 0, 0};
  const int64_t edge = bytes - whole * 16;  // bytes before and behind
  for (int64_t i = i0 * 2; i < edge; i += threads * 2)
    *reinterpret_cast<uint16_t *>(table + (i < head ? i : i + whole * 16)) = 0;
}

struct SumArgs {
  EmbedArgs e;
  const uint32_t *keys, *places;  // sorted
  int64_t chunks;
  int chunk, tiles;
  float *parts;  // [chunks][2][tiles * kLanes * kPer]: of the run that a chunk begins in, of the run that it ends in
};

template <typename T, int kLanes>
__global__ __launch_bounds__(kBlock) void embed_sums_kernel(SumArgs a) {
  const int64_t unit = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / kLanes, chunk = unit / a.tiles;
  if (chunk >= a.chunks) return;
  const int v = (int)(unit - chunk * a.tiles) * kLanes + threadIdx.x % kLanes;
  const Slot<T> s(v, a.e.width);
  const int64_t begin = chunk * a.chunk, end = min(begin + a.chunk, a.e.n), pitch = (int64_t)a.tiles * kLanes * kPer<T>;
  const uint32_t none = (uint32_t)a.e.vocab;
  const uint32_t before = begin > 0 ? a.keys[begin - 1] : ~0u, after = end < a.e.n ? a.keys[end] : ~0u;
  uint32_t current = a.keys[begin];
  bool first = true;
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
  for (int64_t at = begin; at < end; at += kAhead) {
    uint32_t key[kAhead];
    Raw<T> row[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      key[i] = at + i < end ? a.keys[at + i] : none;
      row[i] = Raw<T>{};
      if (key[i] != none && s.any())
        row[i] = load_slot<T>(static_cast<const T *>(a.e.rows) + (int64_t)a.places[at + i] * a.e.stride, s, a.e.width < kPer<T>);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (at + i >= end) break;
      if (key[i] != current) {
        flush(false);
        current = key[i], first = false;
        sum = Vals<T>{};
      }
      sum += __builtin_convertvector(row[i], Vals<T>);
    }
  }
  flush(true);
}

// The runs that borders cut: a workgroup for every chunk (and tile of columns) that such a run may begin in.
template <typename T, int kLanes>
__global__ __launch_bounds__(kJoinBlock) void embed_join_kernel(SumArgs a) {
  constexpr int kGroups = kJoinBlock / kLanes;
  __shared__ Vals<T> pile[kJoinBlock];
  for (int64_t unit = blockIdx.x; unit < a.chunks * a.tiles; unit += gridDim.x) {
    const int64_t chunk = unit / a.tiles, begin = chunk * a.chunk, end = begin + a.chunk;
    if (end >= a.e.n) continue;
    const uint32_t key = a.keys[end - 1];
    if (key == (uint32_t)a.e.vocab || a.keys[end] != key) continue;
    if (a.keys[begin] == key && begin > 0 && a.keys[begin - 1] == key) continue;  // it began before
    // the last chunk that begins with it
    int64_t lo = chunk + 1, hi = a.chunks - 1;
    while (lo < hi) {
      const int64_t mid = lo + (hi - lo + 1) / 2;
      if (a.keys[mid * a.chunk] == key)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const int v = (int)(unit - chunk * a.tiles) * kLanes + lane;
    const int64_t pitch = (int64_t)a.tiles * kLanes * kPer<T>;
    Vals<T> sum = {};
    if (group == 0) sum = *reinterpret_cast<const Vals<T> *>(a.parts + (chunk * 2 + 1) * pitch + v * kPer<T>);
#pragma unroll 4
    for (int64_t c = chunk + 1 + group; c <= lo; c += kGroups)
      sum += *reinterpret_cast<const Vals<T> *>(a.parts + c * 2 * pitch + v * kPer<T>);
    __syncthreads();  // (of the run before)
    pile[threadIdx.x] = sum;
    __syncthreads();
    const Slot<T> s(v, a.e.width);
    if (group == 0 && s.any()) {
      for (int g = 1; g < kGroups; ++g) sum += pile[g * kLanes + lane];
      store_slot(static_cast<T *>(a.e.to) + (int64_t)key * a.e.width, s, sum * a.e.scale);
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

constexpr int kTile = 64 * 8;  // most columns of a group of lanes
struct Plan {
  int chunk, pitch;
  int64_t chunks;
  size_t keys, places, keys_tmp, places_tmp, sorted_keys, sorted_places, hist, parts, total;
};
// Chunks of 16 to 256 positions: short ones where there are few (4096 groups of lanes fill the GPU), long ones for fewer borders.
Plan plan_of(int64_t n, int width) {
  Plan p;
  p.chunk = 16;
  while (p.chunk < 256 && ceil_div64(n, p.chunk) > 4096) p.chunk *= 2;
  p.chunks = ceil_div64(n, p.chunk);
  p.pitch = (width + kTile - 1) / kTile * kTile;  // at least what a group of lanes covers, in any type
  const size_t list = align_up((size_t)n * 4, 256);
  p.keys = 0, p.places = list, p.keys_tmp = 2 * list, p.places_tmp = 3 * list, p.sorted_keys = 4 * list, p.sorted_places = 5 * list;
  p.hist = 6 * list;
  p.parts = align_up(p.hist + radix::hist_bytes(n), 256);
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
  const EmbedArgs a{tokens, tokens_i64 != 0, n, vocab, (int)width, table, table_stride, out, scale};
  by_type_and_lanes(dtype, (int)width, [&](auto type, auto lanes) {
    constexpr int kLanes = decltype(lanes)::value;
    const int64_t blocks = ceil_div64(n, kBlock / kLanes), most = kMostItems / kBlock;
    hipLaunchKernelGGL((embed_kernel<decltype(type), kLanes>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(kBlock), 0,
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
  EmbedArgs e{tokens, tokens_i64 != 0, n, vocab, (int)width, dout, dout_stride, dtable, scale};
  const int64_t bytes = vocab * width * element, work = std::max(n, bytes / 16 + 1);
  const unsigned key_blocks = (unsigned)std::min<int64_t>(ceil_div64(work, kBlock), 8192);
  embed_keys_kernel<<<dim3(key_blocks), dim3(kBlock), 0, st>>>(e, n > 0 ? list(p.keys) : nullptr, n > 0 ? list(p.places) : nullptr,
                                                               static_cast<char *>(dtable), bytes);
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  if (n == 0) return 0;
  const int bits = 64 - __builtin_clzll((uint64_t)vocab);
  const int sorted = radix::sort_pairs<uint32_t, uint32_t>(list(p.keys), list(p.sorted_keys), list(p.places), list(p.sorted_places),
                                                           list(p.keys_tmp), list(p.places_tmp), n, 0, bits, list(p.hist), st);
  if (sorted != 0) return sorted;
  SumArgs a{e, list(p.sorted_keys), list(p.sorted_places), p.chunks, p.chunk, 0, reinterpret_cast<float *>(ws + p.parts)};
  by_type_and_lanes(dtype, (int)width, [&](auto type, auto lanes) {
    using T = decltype(type);
    constexpr int kLanes = decltype(lanes)::value;
    a.tiles = ((int)width + kPer<T> * kLanes - 1) / (kPer<T> * kLanes);
    const int64_t units = a.chunks * a.tiles;
    hipLaunchKernelGGL((embed_sums_kernel<T, kLanes>), dim3((unsigned)ceil_div64(units, kBlock / kLanes)), dim3(kBlock), 0, st, a);
    hipLaunchKernelGGL((embed_join_kernel<T, kLanes>), dim3((unsigned)std::min<int64_t>(units, (1 << 22) - 1)), dim3(kJoinBlock), 0, st, a);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
