// Norm of every head's query and key with the rotation of its positions (gear_hip_norm_rotate and the
// calls beside it).
//
// With r = 1 / sqrt(mean(x^2) + eps), n = x r and y = n w, the pair (y[i], y[i + D/2]) is turned by
// angle_i = pos[axis(i)] * freqs[i].  Backwards, g = the gradient turned back, dw = sum of g n over rows,
// h = g w and dx = r (h - n mean(h n)).  Only x is read again: r and n are cheaper to work out than to load.
//
// Bound by memory: 4 bytes a 16-bit element forward, 6 backward.  A lane holds 16 bytes of each half of a row, the same
// elements of both, so that a pair is in one lane; the lanes of a row (rounded up to a power of two) sum by a few
// exchanges in registers.  A workgroup takes
// kTokens tokens with all their heads: a token's sines serve all of them, and are worked out once, into LDS.  The angle is
// reduced in 64 bits -- position times frequency in turns, less the whole turns -- because 32 bits
// leave 6e-5 radians of the fastest pair at position 1000 and nothing at all at 10^7; it costs one
// 64-bit product a pair and token.
// Measured, forward and backward (with the sums of dw): 1024 x 60 tokens, 8 + 8 heads of 32, 32 bits: 58 and 78 us (4.3 and 4.8
// TB/s); 64 x 1470, 16 + 4 of 128, bf16, three axes: 212 and 302 us (4.5 and 4.8 TB/s), where a plain copy of as much reaches 4.8.
#include <type_traits>

#include "half.hpp"

namespace gearhip {
namespace {

constexpr int kBlock = 256;
constexpr int kTurns = 1024;       // sines and cosines of a workgroup's tokens, 8 KB of LDS
constexpr int kTokens = 16;        // its tokens, where there are enough of them
constexpr int kMaxDim = 256;
constexpr int kGradBlocks = 1024;  // workgroups of the backward pass: each leaves one row of weight sums

struct Strides {
  int64_t batch, token, head;
};

struct NormArgs {
  const void *q, *k, *v;
  Strides qs, ks, vs;
  int64_t batch, tokens;
  int q_heads, k_heads, dim;
  const int32_t *pos;
  const double *freqs;
  int axes, upto[4];  // pairs below upto[a] belong to axis a or an earlier one
  const void *q_weight, *k_weight;
  int weight_f32;
  float eps;
  // forward
  int64_t first;  // token of the launch
  void *q_out, *k_out, *v_out;
  const int32_t *slots;  // append: the row of the cache, else null
  int64_t cache_tokens;
  Strides kcs, vcs;
  // backward
  const void *gq, *gk;
  Strides gqs, gks;
  float *sums;  // [blocks][2][dim]
  bool want_weights;
};

template <typename T>
__device__ __forceinline__ const T *row_at(const void *p, const Strides &s, int64_t b, int64_t t, int64_t h) {
  return static_cast<const T *>(p) + b * s.batch + t * s.token + h * s.head;
}

// cos and sin of `count` tokens from `first` on, dim/2 pairs each
__device__ __forceinline__ void turns(const NormArgs &a, int64_t first, int count, float2 *cs) {
  const int half = a.dim / 2, pairs = a.upto[a.axes - 1];
  for (int x = threadIdx.x; x < count * half; x += kBlock) {
    const int token = x / half, i = x - token * half;
    float2 v = make_float2(1.f, 0.f);
    if (i < pairs) {
      const int axis = (a.axes > 1 && i >= a.upto[0]) + (a.axes > 2 && i >= a.upto[1]) + (a.axes > 3 && i >= a.upto[2]);
      double turn = (double)a.pos[(first + token) * a.axes + axis] * (a.freqs[i] * 0.15915494309189533577);
      turn -= rint(turn);
      sincospif((float)(2 * turn), &v.y, &v.x);
    }
    cs[x] = v;
  }
}

// Sum over the LPR lanes of a row, in all of them.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  x = dpp_add<0xB1>(x);                  // lanes 1 apart
  if (LPR > 2) x = dpp_add<0x4E>(x);     // 2 apart
  if (LPR > 4) x = dpp_add<0x141>(x);    // the other half of 8
  if (LPR > 8) x = dpp_add<0x140>(x);    // the other half of 16
  if (LPR > 16) x += __shfl_xor(x, 16);
  return x;
}

__device__ __forceinline__ float sum_of(f32x4 x) { return (x[0] + x[1]) + (x[2] + x[3]); }
__device__ __forceinline__ float sum_of(f32x8 x) {
  return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

// The elements of a half that a lane holds: 16 bytes of them.
template <typename T>
constexpr int kEach = 16 / sizeof(T);
template <typename T>
using Part = float __attribute__((ext_vector_type(16 / sizeof(T))));

template <typename T>
__device__ __forceinline__ Part<T> weights_at(const void *w, int f32, int at) {
  Part<T> x;
#pragma unroll
  for (int e = 0; e < kEach<T>; ++e)
    x[e] = w == nullptr ? 1.f : f32 ? static_cast<const float *>(w)[at + e] : (float)static_cast<const T *>(w)[at + e];
  return x;
}

template <typename T>
struct Halves {
  Part<T> lo, hi;
};

template <typename T>
__device__ __forceinline__ Halves<T> load_halves(const T *row, int at, int half) {
  typedef T raw __attribute__((ext_vector_type(16 / sizeof(T))));
  return Halves<T>{__builtin_convertvector(*reinterpret_cast<const raw *>(row + at), Part<T>),
                   __builtin_convertvector(*reinterpret_cast<const raw *>(row + half + at), Part<T>)};
}
template <typename T>
__device__ __forceinline__ void store_halves(T *row, int at, int half, const Halves<T> &x) {
  typedef T raw __attribute__((ext_vector_type(16 / sizeof(T))));
  *reinterpret_cast<raw *>(row + at) = __builtin_convertvector(x.lo, raw);
  *reinterpret_cast<raw *>(row + half + at) = __builtin_convertvector(x.hi, raw);
}

// (y0, y1) turned by the angle of (c, s), or back
template <typename T>
__device__ __forceinline__ Halves<T> turned(const Halves<T> &y, const float2 *cs, float sign) {
  Halves<T> z;
#pragma unroll
  for (int e = 0; e < kEach<T>; ++e) {
    const float c = cs[e].x, s = sign * cs[e].y;
    z.lo[e] = y.lo[e] * c - y.hi[e] * s;
    z.hi[e] = y.hi[e] * c + y.lo[e] * s;
  }
  return z;
}

template <int LPR, typename T>
__device__ __forceinline__ float inverse_norm(const Halves<T> &x, float over_dim, float eps) {
  return __builtin_amdgcn_rsqf(fmaf(row_sum<LPR>(sum_of(x.lo * x.lo) + sum_of(x.hi * x.hi)), over_dim, eps));
}

// What a workgroup needs of its tokens.
struct Tokens {
  int64_t batch[kTokens], token[kTokens];
};
__device__ __forceinline__ void tokens_of(const NormArgs &a, int64_t first, int count, Tokens &at) {
  if ((int)threadIdx.x < count) {
    const int64_t n = first + threadIdx.x, b = n / a.tokens;
    at.batch[threadIdx.x] = b, at.token[threadIdx.x] = n - b * a.tokens;
  }
}

// The rows (token, head) that a lane's group goes through, kBlock / LPR apart.
struct RowWalk {
  int token, head;
  __device__ __forceinline__ RowWalk(int r, int heads) : token(r / heads), head(r - token * heads) {}
  __device__ __forceinline__ void on(int by, int heads) {
    head += by;
    while (head >= heads) head -= heads, ++token;
  }
};

template <typename T, int LPR>
__global__ __launch_bounds__(kBlock) void norm_rotate_kernel(NormArgs a, int per_block) {
  __shared__ __attribute__((aligned(16))) float2 cs[kTurns];  // [token][dim / 2]
  __shared__ Tokens tokens;
  const int64_t all = a.batch * a.tokens, first = a.first + (int64_t)blockIdx.x * per_block;
  const int count = (int)min((int64_t)per_block, all - first), half = a.dim / 2;
  const int at = (threadIdx.x % LPR) * kEach<T>;
  const bool active = at < half;
  const int heads = a.q_heads + a.k_heads + (a.v_out ? a.k_heads : 0);
  const float over_dim = 1.f / a.dim;
  tokens_of(a, first, count, tokens);
  __syncthreads();
  auto load = [&](const RowWalk &r) __attribute__((always_inline)) {
    Halves<T> x = {};
    if (!active || r.token >= count) return x;
    const int64_t b = tokens.batch[r.token], t = tokens.token[r.token];
    const int kh = r.head - a.q_heads;
    return load_halves(r.head < a.q_heads   ? row_at<T>(a.q, a.qs, b, t, r.head)
                       : kh < a.k_heads     ? row_at<T>(a.k, a.ks, b, t, kh)
                                            : row_at<T>(a.v, a.vs, b, t, kh - a.k_heads),
                       at, half);
  };
  // (the first row is asked for before the sines)
  RowWalk walk(threadIdx.x / LPR, heads), ahead = walk;
  Halves<T> next = load(ahead);
  Part<T> w[2][2] = {};
  if (active) {
    w[0][0] = weights_at<T>(a.q_weight, a.weight_f32, at);
    w[0][1] = weights_at<T>(a.q_weight, a.weight_f32, half + at);
    w[1][0] = weights_at<T>(a.k_weight, a.weight_f32, at);
    w[1][1] = weights_at<T>(a.k_weight, a.weight_f32, half + at);
  }
  turns(a, first, count, cs);
  __syncthreads();
  // (all lanes of a wave go round alike: the sums exchange lanes)
  for (int base = 0; base < count * heads; base += kBlock / LPR, walk = ahead) {
    Halves<T> x = base == 0 ? next : load(walk);
    ahead.on(kBlock / LPR, heads);
    const float r_norm = inverse_norm<LPR>(x, over_dim, a.eps);
    if (!active || walk.token >= count) continue;
    const bool is_q = walk.head < a.q_heads, is_v = walk.head >= a.q_heads + a.k_heads;
    if (!is_v) {
      const Part<T> w0 = is_q ? w[0][0] : w[1][0], w1 = is_q ? w[0][1] : w[1][1];
      x = turned(Halves<T>{x.lo * r_norm * w0, x.hi * r_norm * w1}, cs + walk.token * half + at, 1.f);
    }
    const int64_t n = first + walk.token;
    const int kh = walk.head - a.q_heads - (is_v ? a.k_heads : 0);
    T *to;
    if (is_q) {
      to = static_cast<T *>(a.q_out) + (n * a.q_heads + walk.head) * a.dim;
    } else if (a.slots == nullptr) {
      to = static_cast<T *>(a.k_out) + (n * a.k_heads + kh) * a.dim;
    } else {
      const int64_t slot = a.slots[n], b = tokens.batch[walk.token];
      if (slot < 0 || slot >= a.cache_tokens) continue;
      to = is_v ? static_cast<T *>(a.v_out) + b * a.vcs.batch + slot * a.vcs.token + kh * a.vcs.head
                : static_cast<T *>(a.k_out) + b * a.kcs.batch + slot * a.kcs.token + kh * a.kcs.head;
    }
    store_halves<T>(to, at, half, x);
  }
}

template <typename T, int LPR>
__global__ __launch_bounds__(kBlock) void norm_rotate_grad_kernel(NormArgs a, int per_block) {
  __shared__ __attribute__((aligned(16))) float2 cs[kTurns];  // [token][dim / 2]
  __shared__ Tokens tokens;
  __shared__ __attribute__((aligned(32))) float sums[kBlock / LPR][2 * LPR * kEach<T>];
  const int64_t all = a.batch * a.tokens;
  const int half = a.dim / 2, at = (threadIdx.x % LPR) * kEach<T>;
  const bool active = at < half;
  const float over_dim = 1.f / a.dim;
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {  // queries, then keys: one set of weights and sums at a time
    const void *px = side ? a.k : a.q, *pg = side ? a.gk : a.gq, *pw = side ? a.k_weight : a.q_weight;
    const Strides &sx = side ? a.ks : a.qs, &sg = side ? a.gks : a.gqs;
    const int heads = side ? a.k_heads : a.q_heads;
    T *to = static_cast<T *>(side ? a.k_out : a.q_out);
    Part<T> w0 = {}, w1 = {}, d0 = {}, d1 = {};
    if (active) w0 = weights_at<T>(pw, a.weight_f32, at), w1 = weights_at<T>(pw, a.weight_f32, half + at);
    for (int64_t first = (int64_t)blockIdx.x * per_block; first < all && heads > 0; first += (int64_t)gridDim.x * per_block) {
      const int count = (int)min((int64_t)per_block, all - first);
      __syncthreads();
      tokens_of(a, first, count, tokens);
      turns(a, first, count, cs);
      __syncthreads();
      RowWalk walk(threadIdx.x / LPR, heads);
      for (int base = 0; base < count * heads; base += kBlock / LPR, walk.on(kBlock / LPR, heads)) {
        const bool here = active && walk.token < count;
        Halves<T> x = {}, g = {};
        if (here) {
          const int64_t b = tokens.batch[walk.token], t = tokens.token[walk.token];
          x = load_halves(row_at<T>(px, sx, b, t, walk.head), at, half);
          g = turned(load_halves(row_at<T>(pg, sg, b, t, walk.head), at, half), cs + walk.token * half + at, -1.f);
        }
        const float r_norm = inverse_norm<LPR>(x, over_dim, a.eps);
        x.lo *= r_norm, x.hi *= r_norm;
        d0 += g.lo * x.lo, d1 += g.hi * x.hi;
        g.lo *= w0, g.hi *= w1;
        const float mean = row_sum<LPR>(sum_of(g.lo * x.lo) + sum_of(g.hi * x.hi)) * over_dim;
        if (here)
          store_halves<T>(to + ((first + walk.token) * heads + walk.head) * a.dim, at, half,
                       Halves<T>{r_norm * (g.lo - x.lo * mean), r_norm * (g.hi - x.hi * mean)});
      }
    }
    if (!a.want_weights) continue;
    __syncthreads();
    *reinterpret_cast<Part<T> *>(&sums[threadIdx.x / LPR][at]) = d0;
    *reinterpret_cast<Part<T> *>(&sums[threadIdx.x / LPR][LPR * kEach<T> + at]) = d1;
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += kBlock) {
      const int column = i < half ? i : LPR * kEach<T> + i - half;
      float s = 0;
      for (int r = 0; r < kBlock / LPR; ++r) s += sums[r][column];
      a.sums[((int64_t)blockIdx.x * 2 + side) * a.dim + i] = s;
    }
  }
}

// The sums of all workgroups: 16 of the 2 * dim columns a workgroup, 16 threads a column.
constexpr int kColumns = 16;
template <typename T>
__global__ __launch_bounds__(kBlock) void norm_rotate_weights_kernel(const float *sums, int blocks, int dim, int f32,
                                                                     void *gq, void *gk) {
  __shared__ float part[kBlock / kColumns][kColumns];
  const int c = threadIdx.x % kColumns, group = threadIdx.x / kColumns, column = blockIdx.x * kColumns + c;
  float s = 0;
#pragma unroll 8
  for (int r = group; r < blocks; r += kBlock / kColumns) s += sums[(int64_t)r * 2 * dim + column];
  part[group][c] = s;
  __syncthreads();
  if (group != 0) return;
  for (int x = 1; x < kBlock / kColumns; ++x) s += part[x][c];
  const int side = column >= dim, i = column - side * dim;
  void *to = side ? gk : gq;
  if (to == nullptr) return;
  if (f32)
    static_cast<float *>(to)[i] = s;
  else
    static_cast<T *>(to)[i] = (T)s;
}

bool strides_fit(const void *p, const int64_t *s, int element) {
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (s[i] * element % 16 != 0) return false;
  return true;
}

Strides strides(const int64_t *s) { return Strides{s[0], s[1], s[2]}; }

// 0: go on; 1: nothing to do; else the error
int prepare(const gear_hip_norm_rotate_desc *d, NormArgs &a) {
  if (d == nullptr || d->batch < 0 || d->tokens < 0 || d->q_heads < 0 || d->k_heads < 0) return GEAR_HIP_EINVAL;
  if (d->dtype != GEAR_HIP_F32 && d->dtype != GEAR_HIP_F16 && d->dtype != GEAR_HIP_BF16) return GEAR_HIP_EINVAL;
  if (d->head_dim < 16 || d->head_dim % 16 != 0 || d->axes < 1 || d->axes > 4) return GEAR_HIP_EINVAL;
  if (!(d->eps >= 0)) return GEAR_HIP_EINVAL;
  if (d->head_dim > kMaxDim) return GEAR_HIP_ERANGE;
  int pairs = 0;
  for (int x = 0; x < 4; ++x) {
    if (x < d->axes) {
      if (d->sections[x] < 0 || d->sections[x] > d->head_dim / 2) return GEAR_HIP_EINVAL;
      pairs += d->sections[x];
    }
    a.upto[x] = pairs;
  }
  if (pairs > d->head_dim / 2) return GEAR_HIP_EINVAL;
  constexpr int64_t kMost = (int64_t)1 << 31;
  if (d->batch >= kMost || d->tokens >= kMost || (d->tokens > 0 && d->batch > kMost / d->tokens) ||
      (int64_t)d->q_heads + 2 * (int64_t)d->k_heads > (1 << 24))
    return GEAR_HIP_ERANGE;
  if (d->batch == 0 || d->tokens == 0 || (d->q_heads == 0 && d->k_heads == 0)) return 1;
  if ((d->q_heads > 0 && d->q == nullptr) || (d->k_heads > 0 && d->k == nullptr) || d->pos == nullptr ||
      (pairs > 0 && d->freqs == nullptr))
    return GEAR_HIP_EINVAL;
  const int element = d->dtype == GEAR_HIP_F32 ? 4 : 2;
  if (!strides_fit(d->q, d->q_stride, element) || !strides_fit(d->k, d->k_stride, element)) return GEAR_HIP_EALIGN;
  a.q = d->q, a.k = d->k;
  a.qs = strides(d->q_stride), a.ks = strides(d->k_stride);
  a.batch = d->batch, a.tokens = d->tokens;
  a.q_heads = d->q_heads, a.k_heads = d->k_heads, a.dim = d->head_dim;
  a.pos = d->pos, a.freqs = d->freqs, a.axes = d->axes;
  a.q_weight = d->q_weight, a.k_weight = d->k_weight, a.weight_f32 = d->weight_f32 != 0;
  a.eps = d->eps;
  return 0;
}

// f(T(), lanes of a row)
template <typename F>
void by_type_and_lanes(int dtype, int dim, const F &f) {
  auto lanes = [&](auto type) {
    const int n = dim / 2 / kEach<decltype(type)>;
    if (n <= 2)
      f(type, std::integral_constant<int, 2>());
    else if (n <= 4)
      f(type, std::integral_constant<int, 4>());
    else if (n <= 8)
      f(type, std::integral_constant<int, 8>());
    else if (n <= 16)
      f(type, std::integral_constant<int, 16>());
    else if constexpr (sizeof(type) == 4)
      f(type, std::integral_constant<int, 32>());
  };
  if (dtype == GEAR_HIP_F32)
    lanes(float());
  else if (dtype == GEAR_HIP_F16)
    lanes(f16());
  else
    lanes(bf16());
}

// Tokens a workgroup: the sines of a token serve all its heads, and what is done once a workgroup has to be spread over
// its rows (forward, 94080 tokens of 20 heads of 128: 2 tokens 436 us, 4 296, 8 241, 16 216, 32 224), but few tokens are
// spread over the GPU, two workgroups for each of 256 CUs.  (Few heads of short rows leave most of a workgroup idle, in the
// gradient above all: 61440 tokens, 4 + 1 heads of 32 in bf16, 25 and 41 us where a copy of as much takes 20 for both.)
int tokens_per_block(int64_t tokens, int dim) {
  int n = kTurns / (dim / 2);
  if (n > kTokens) n = kTokens;
  while (n > 1 && ceil_div64(tokens, n) < 512) n /= 2;
  return n;
}

int forward(NormArgs &a, int dtype, void *stream) {
  const int64_t all = a.batch * a.tokens;
  const int n = tokens_per_block(all, a.dim);
  const int64_t most = kMostItems / kBlock;  // workgroups of a launch
  for (a.first = 0; a.first < all; a.first += most * n) {
    const int64_t left = ceil_div64(all - a.first, n), blocks = left < most ? left : most;
    by_type_and_lanes(dtype, a.dim, [&](auto type, auto lanes) {
      hipLaunchKernelGGL((norm_rotate_kernel<decltype(type), decltype(lanes)::value>), dim3((unsigned)blocks), dim3(kBlock), 0,
                         as_stream(stream), a, n);
    });
    GEARHIP_RETURN_IF_LAUNCH_FAILED();
  }
  return 0;
}

}  // namespace
}  // namespace gearhip

using namespace gearhip;

extern "C" int gear_hip_norm_rotate(const gear_hip_norm_rotate_desc *desc, void *q_out, void *k_out, void *stream) {
  NormArgs a = {};
  const int rc = prepare(desc, a);
  if (rc != 0) return rc < 0 ? rc : 0;
  if ((a.q_heads > 0 && q_out == nullptr) || (a.k_heads > 0 && k_out == nullptr)) return GEAR_HIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(q_out) % 16 != 0 || reinterpret_cast<uintptr_t>(k_out) % 16 != 0) return GEAR_HIP_EALIGN;
  a.q_out = q_out, a.k_out = k_out;
  return forward(a, desc->dtype, stream);
}

extern "C" int gear_hip_norm_rotate_append(const gear_hip_norm_rotate_desc *desc, const void *v,
                                           const int64_t *v_stride, void *q_out, const int32_t *slots,
                                           int64_t cache_tokens, void *k_cache, const int64_t *k_cache_stride,
                                           void *v_cache, const int64_t *v_cache_stride, void *stream) {
  NormArgs a = {};
  const int rc = prepare(desc, a);
  if (rc != 0) return rc < 0 ? rc : 0;
  if ((a.q_heads > 0 && q_out == nullptr) || v == nullptr || v_stride == nullptr || slots == nullptr ||
      cache_tokens < 0 || k_cache_stride == nullptr || v_cache_stride == nullptr)
    return GEAR_HIP_EINVAL;
  if (cache_tokens > 0 && (k_cache == nullptr || v_cache == nullptr)) return GEAR_HIP_EINVAL;
  const int element = desc->dtype == GEAR_HIP_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(q_out) % 16 != 0 || !strides_fit(v, v_stride, element) ||
      !strides_fit(k_cache, k_cache_stride, element) || !strides_fit(v_cache, v_cache_stride, element))
    return GEAR_HIP_EALIGN;
  a.v = v, a.vs = strides(v_stride);
  a.q_out = q_out, a.k_out = k_cache, a.v_out = v_cache;
  a.slots = slots, a.cache_tokens = cache_tokens;
  a.kcs = strides(k_cache_stride), a.vcs = strides(v_cache_stride);
  return forward(a, desc->dtype, stream);
}

extern "C" size_t gear_hip_norm_rotate_backward_workspace_bytes(int64_t head_dim) {
  return head_dim > 0 && head_dim <= kMaxDim ? (size_t)kGradBlocks * 2 * head_dim * sizeof(float) : 0;
}

extern "C" int gear_hip_norm_rotate_backward(const gear_hip_norm_rotate_desc *desc, const void *dq_out,
                                             const int64_t *dq_out_stride, const void *dk_out,
                                             const int64_t *dk_out_stride, void *dq, void *dk, void *dq_weight,
                                             void *dk_weight, void *workspace, size_t workspace_bytes, void *stream) {
  NormArgs a = {};
  int rc = prepare(desc, a);
  if (rc < 0) return rc;
  a.want_weights = dq_weight != nullptr || dk_weight != nullptr;
  if (a.want_weights && (workspace == nullptr ||
                         workspace_bytes < gear_hip_norm_rotate_backward_workspace_bytes(desc->head_dim)))
    return GEAR_HIP_EWORKSPACE;
  if (a.want_weights && reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return GEAR_HIP_EALIGN;
  int blocks = 0;  // without rows the weights' gradients are zero
  if (rc == 0) {
    if ((a.q_heads > 0 && (dq_out == nullptr || dq == nullptr)) || (a.k_heads > 0 && (dk_out == nullptr || dk == nullptr)) ||
        dq_out_stride == nullptr || dk_out_stride == nullptr)
      return GEAR_HIP_EINVAL;
    const int element = desc->dtype == GEAR_HIP_F32 ? 4 : 2;
    if (!strides_fit(dq_out, dq_out_stride, element) || !strides_fit(dk_out, dk_out_stride, element) ||
        reinterpret_cast<uintptr_t>(dq) % 16 != 0 || reinterpret_cast<uintptr_t>(dk) % 16 != 0)
      return GEAR_HIP_EALIGN;
    a.gq = dq_out, a.gk = dk_out;
    a.gqs = strides(dq_out_stride), a.gks = strides(dk_out_stride);
    a.q_out = dq, a.k_out = dk;
    a.sums = static_cast<float *>(workspace);
    const int64_t all = a.batch * a.tokens;
    const int n = tokens_per_block(all, a.dim);
    blocks = (int)min(ceil_div64(all, n), (int64_t)kGradBlocks);
    by_type_and_lanes(desc->dtype, a.dim, [&](auto type, auto lanes) {
      hipLaunchKernelGGL((norm_rotate_grad_kernel<decltype(type), decltype(lanes)::value>), dim3(blocks), dim3(kBlock), 0,
                         as_stream(stream), a, n);
    });
    GEARHIP_RETURN_IF_LAUNCH_FAILED();
  }
  if (!a.want_weights) return 0;
  by_type_and_lanes(desc->dtype, 16, [&](auto type, auto) {
    hipLaunchKernelGGL((norm_rotate_weights_kernel<decltype(type)>), dim3(2 * desc->head_dim / kColumns), dim3(kBlock), 0,
                       as_stream(stream), static_cast<const float *>(workspace), blocks, desc->head_dim,
                       desc->weight_f32 != 0, dq_weight, dk_weight);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
