// Norm of every head's query and key with the rotation of its positions (gear_hip_norm_rotate and the
// calls beside it).
//
// With r = 1 / sqrt(mean(x^2) + eps), n = x r and y = n w, the pair (y[i], y[i + D/2]) is turned by
// angle_i = pos[axis(i)] * freqs[i].  Backwards, g = the gradient turned back, dw = sum of g n over rows,
// h = g w and dx = r (h - n mean(h n)).  Only x is read again: r and n are cheaper to work out than to load.
//
// Bound by memory: 4 bytes a 16-bit element forward, 6 backward.  A row takes D/16 lanes (rounded up to a
// power of two), each with the same 8 elements of both halves, so that a pair is in one lane, loads are 16
// bytes and the sums over a row are a few lane exchanges.  A workgroup takes kTokens tokens with all
// their heads: a token's sines serve all of them, and are worked out once, into LDS.  The angle is
// reduced in 64 bits -- position times frequency in turns, less the whole turns -- because 32 bits
// leave 6e-5 radians of the fastest pair at position 1000 and nothing at all at 10^7; it costs one
// 64-bit product a pair and token.
#include <type_traits>

#include "half.hpp"

namespace gearhip {
namespace {

constexpr int kBlock = 256;
constexpr int kTokens = 8;       // a workgroup's tokens, where there are enough of them
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
__device__ __forceinline__ void turns(const NormArgs &a, int64_t first, int count, float2 (*cs)[kMaxDim / 2]) {
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
    cs[token][i] = v;
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int m = 1; m < LPR; m *= 2) x += __shfl_xor(x, m);
  return x;
}

__device__ __forceinline__ float sum8(f32x8 x) {
  return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

template <typename T>
__device__ __forceinline__ f32x8 weights8(const void *w, int f32, int at) {
  f32x8 x = {1, 1, 1, 1, 1, 1, 1, 1};
  if (w == nullptr) return x;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    x[e] = f32 ? static_cast<const float *>(w)[at + e] : (float)static_cast<const T *>(w)[at + e];
  return x;
}

struct Halves {
  f32x8 lo, hi;
};

template <typename T>
__device__ __forceinline__ Halves load_halves(const T *row, int at, int half) {
  Row8<T> a, b;
  a.load(row + at);
  b.load(row + half + at);
  return Halves{a.floats(), b.floats()};
}
template <typename T>
__device__ __forceinline__ void store_halves(T *row, int at, int half, const Halves &x) {
  Row8<T> a, b;
  a.set(x.lo);
  b.set(x.hi);
  a.store(row + at);
  b.store(row + half + at);
}

// (y0, y1) turned by the angle of (c, s), or back
__device__ __forceinline__ Halves turned(const Halves &y, const float2 *cs, float sign) {
  Halves z;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float c = cs[e].x, s = sign * cs[e].y;
    z.lo[e] = y.lo[e] * c - y.hi[e] * s;
    z.hi[e] = y.hi[e] * c + y.lo[e] * s;
  }
  return z;
}

template <int LPR>
__device__ __forceinline__ float inverse_norm(const Halves &x, int dim, float eps) {
  return 1.f / sqrtf(row_sum<LPR>(sum8(x.lo * x.lo) + sum8(x.hi * x.hi)) / dim + eps);
}

template <typename T, int LPR>
__global__ __launch_bounds__(kBlock) void norm_rotate_kernel(NormArgs a, int per_block) {
  __shared__ float2 cs[kTokens][kMaxDim / 2];
  const int64_t all = a.batch * a.tokens, first = (int64_t)blockIdx.x * per_block;
  const int count = (int)min((int64_t)per_block, all - first), half = a.dim / 2;
  turns(a, first, count, cs);
  __syncthreads();
  const int at = (threadIdx.x % LPR) * 8;
  const bool active = at < half;
  const int heads = a.q_heads + a.k_heads + (a.v_out ? a.k_heads : 0);
  f32x8 w[2][2] = {};
  if (active) {
    w[0][0] = weights8<T>(a.q_weight, a.weight_f32, at);
    w[0][1] = weights8<T>(a.q_weight, a.weight_f32, half + at);
    w[1][0] = weights8<T>(a.k_weight, a.weight_f32, at);
    w[1][1] = weights8<T>(a.k_weight, a.weight_f32, half + at);
  }
  // (all lanes of a wave go round alike: the sums exchange lanes)
  for (int base = 0; base < count * heads; base += kBlock / LPR) {
    const int r = base + threadIdx.x / LPR;
    const bool here = active && r < count * heads;
    const int token = here ? r / heads : 0, h = here ? r - token * heads : 0;
    const int64_t n = first + token, b = n / a.tokens, t = n - b * a.tokens;
    const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.k_heads;
    const int64_t kh = is_v ? h - a.q_heads - a.k_heads : h - a.q_heads;
    Halves x = {};
    if (here)
      x = is_q ? load_halves(row_at<T>(a.q, a.qs, b, t, h), at, half)
               : load_halves(is_v ? row_at<T>(a.v, a.vs, b, t, kh) : row_at<T>(a.k, a.ks, b, t, kh), at, half);
    const float r_norm = inverse_norm<LPR>(x, a.dim, a.eps);
    if (!here) continue;
    if (!is_v) {
      const f32x8 w0 = is_q ? w[0][0] : w[1][0], w1 = is_q ? w[0][1] : w[1][1];
      x = turned(Halves{x.lo * r_norm * w0, x.hi * r_norm * w1}, &cs[token][at], 1.f);
    }
    T *to;
    if (is_q) {
      to = static_cast<T *>(a.q_out) + (n * a.q_heads + h) * a.dim;
    } else if (a.slots == nullptr) {
      to = static_cast<T *>(a.k_out) + (n * a.k_heads + kh) * a.dim;
    } else {
      const int64_t slot = a.slots[n];
      if (slot < 0 || slot >= a.cache_tokens) continue;
      to = is_v ? static_cast<T *>(a.v_out) + b * a.vcs.batch + slot * a.vcs.token + kh * a.vcs.head
                : static_cast<T *>(a.k_out) + b * a.kcs.batch + slot * a.kcs.token + kh * a.kcs.head;
    }
    store_halves(to, at, half, x);
  }
}

template <typename T, int LPR>
__global__ __launch_bounds__(kBlock) void norm_rotate_grad_kernel(NormArgs a, int per_block) {
  __shared__ float2 cs[kTokens][kMaxDim / 2];
  __shared__ float sums[kBlock / LPR][LPR * 16];
  const int64_t all = a.batch * a.tokens;
  const int half = a.dim / 2, at = (threadIdx.x % LPR) * 8;
  const bool active = at < half;
  for (int side = 0; side < 2; ++side) {  // queries, then keys: one set of weights and sums at a time
    const void *px = side ? a.k : a.q, *pg = side ? a.gk : a.gq, *pw = side ? a.k_weight : a.q_weight;
    const Strides &sx = side ? a.ks : a.qs, &sg = side ? a.gks : a.gqs;
    const int heads = side ? a.k_heads : a.q_heads;
    T *to = static_cast<T *>(side ? a.k_out : a.q_out);
    f32x8 w0 = {}, w1 = {}, d0 = {}, d1 = {};
    if (active) w0 = weights8<T>(pw, a.weight_f32, at), w1 = weights8<T>(pw, a.weight_f32, half + at);
    for (int64_t first = (int64_t)blockIdx.x * per_block; first < all; first += (int64_t)gridDim.x * per_block) {
      const int count = (int)min((int64_t)per_block, all - first);
      __syncthreads();
      turns(a, first, count, cs);
      __syncthreads();
      for (int base = 0; base < count * heads; base += kBlock / LPR) {
        const int r = base + threadIdx.x / LPR;
        const bool here = active && r < count * heads;
        const int token = here ? r / heads : 0, h = here ? r - token * heads : 0;
        const int64_t n = first + token, b = n / a.tokens, t = n - b * a.tokens;
        Halves x = {}, g = {};
        if (here) {
          x = load_halves(row_at<T>(px, sx, b, t, h), at, half);
          g = turned(load_halves(row_at<T>(pg, sg, b, t, h), at, half), &cs[token][at], -1.f);
        }
        const float r_norm = inverse_norm<LPR>(x, a.dim, a.eps);
        x.lo *= r_norm, x.hi *= r_norm;
        d0 += g.lo * x.lo, d1 += g.hi * x.hi;
        g.lo *= w0, g.hi *= w1;
        const float mean = row_sum<LPR>(sum8(g.lo * x.lo) + sum8(g.hi * x.hi)) / a.dim;
        if (here)
          store_halves(to + (n * heads + h) * a.dim, at, half,
                       Halves{r_norm * (g.lo - x.lo * mean), r_norm * (g.hi - x.hi * mean)});
      }
    }
    if (!a.want_weights) continue;
    __syncthreads();
    *reinterpret_cast<f32x8 *>(&sums[threadIdx.x / LPR][at]) = d0;
    *reinterpret_cast<f32x8 *>(&sums[threadIdx.x / LPR][LPR * 8 + at]) = d1;
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += kBlock) {
      const int column = i < half ? i : LPR * 8 + i - half;
      float s = 0;
      for (int r = 0; r < kBlock / LPR; ++r) s += sums[r][column];
      a.sums[((int64_t)blockIdx.x * 2 + side) * a.dim + i] = s;
    }
  }
}

// The sums of all workgroups, a column a wave.
template <typename T>
__global__ __launch_bounds__(kWave) void norm_rotate_weights_kernel(const float *sums, int blocks, int dim, int f32,
                                                                    void *gq, void *gk) {
  const int side = blockIdx.x >= (unsigned)dim, i = blockIdx.x - side * dim;
  float s = 0;
  for (int r = lane_id(); r < blocks; r += kWave) s += sums[((int64_t)r * 2 + side) * dim + i];
  s = row_sum<kWave>(s);
  void *to = side ? gk : gq;
  if (lane_id() != 0 || to == nullptr) return;
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
    if (dim <= 32)
      f(type, std::integral_constant<int, 2>());
    else if (dim <= 64)
      f(type, std::integral_constant<int, 4>());
    else if (dim <= 128)
      f(type, std::integral_constant<int, 8>());
    else
      f(type, std::integral_constant<int, 16>());
  };
  if (dtype == GEAR_HIP_F32)
    lanes(float());
  else if (dtype == GEAR_HIP_F16)
    lanes(f16());
  else
    lanes(bf16());
}

// Tokens a workgroup: the sines of kTokens serve all their heads, but few tokens are spread over the GPU.
int tokens_per_block(int64_t tokens) {
  int n = kTokens;
  while (n > 1 && ceil_div64(tokens, n) < 512) n /= 2;
  return n;
}

int forward(const NormArgs &a, int dtype, void *stream) {
  const int64_t all = a.batch * a.tokens;
  const int n = tokens_per_block(all);
  by_type_and_lanes(dtype, a.dim, [&](auto type, auto lanes) {
    hipLaunchKernelGGL((norm_rotate_kernel<decltype(type), decltype(lanes)::value>), dim3((unsigned)ceil_div64(all, n)),
                       dim3(kBlock), 0, as_stream(stream), a, n);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
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
    const int n = tokens_per_block(all);
    blocks = (int)min(ceil_div64(all, n), (int64_t)kGradBlocks);
    by_type_and_lanes(desc->dtype, a.dim, [&](auto type, auto lanes) {
      hipLaunchKernelGGL((norm_rotate_grad_kernel<decltype(type), decltype(lanes)::value>), dim3(blocks), dim3(kBlock), 0,
                         as_stream(stream), a, n);
    });
    GEARHIP_RETURN_IF_LAUNCH_FAILED();
  }
  if (!a.want_weights) return 0;
  by_type_and_lanes(desc->dtype, 16, [&](auto type, auto) {
    hipLaunchKernelGGL((norm_rotate_weights_kernel<decltype(type)>), dim3(2 * desc->head_dim), dim3(kWave), 0,
                       as_stream(stream), static_cast<const float *>(workspace), blocks, desc->head_dim,
                       desc->weight_f32 != 0, dq_weight, dk_weight);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
