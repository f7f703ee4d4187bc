// Layer norm of rows, with a second input added before, and its gradients (gear_hip_layer_norm and the call beside it).
//
// u = x + residual as it is stored, c = u - mean u, r = 1 / sqrt(mean c^2 + eps), y = c r w + b.  Backwards, with h = dy w:
// dx = r (h - mean h - c r^2 mean(h c)) + dsum, dw = sum over rows of dy c r, db = sum of dy.  Only u is read again: its
// mean and deviation are cheaper to work out than to store and load.  The squares are of u less its mean, not a
// difference of two sums, which would leave nothing of a small deviation around a large mean; and what the first mean is
// off by (the sum of u less it) is taken off again, so that such a row keeps its digits.
//
// Bound by memory.  kLanes lanes hold a row in registers, two vectors of 16 bytes each (a row of 16384 in 32 bits four), so that
// it is read once; rows of more than 64 lanes exchange sums through LDS.  A workgroup of the gradients goes on to further rows with
// the sums of dw and db in registers, leaves them in the workspace, and a second launch adds those up in a fixed order.
// One vector a lane with twice the lanes is as fast; a row asked for ahead slower (47040 x 2048 bf16: 184 us against 165).
//
// Measured, forward and gradients, us: 47040 x 2048 bf16 with a residual 136 and 145 + 6 (5.7 and 5.3 TB/s), 184320 x 512 of the same 123 and
// 138 + 5 (6.1 and 5.5), 8192 x 8192 92 and 133 + 7; 122880 x 128 in 32 bits 19 and 30 + 5 (6.7 and 6.4, the caches help).
#include "rows.hpp"

namespace gearhip {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxWidth = 16384;
// Workgroups of the backward pass, each of which leaves a row of sums.  47040 x 2048 bf16, 256 / 512 / 768 / 1024 of them: 206 / 152 /
// 146 / 150 us, and the sums of all 5 / 5 / 6 / 7; of 512 threads (8192 x 8192) 128 / 256 / 384 / 512: 217 / 134 / 142 / 130 and 5 / 7 / 9 / 12.
constexpr int kGradBlocks = 768, kGradBlocksWide = 256;
// Results of more than the L2 caches hold are written past them, for what else they hold (122880 x 128 in 32 bits: 21 + 31 -> 19 + 30 us,
// 47040 x 2048 bf16 with a residual 134 + 165 -> 136 + 146).
constexpr int64_t kOnceBytes = 32 << 20;

struct LayerArgs {
  const void *x, *residual, *weight, *bias;
  int64_t xs, rs;  // strides of rows
  int64_t rows;
  int width, weight_f32;
  float eps, over_width;
  bool once;
  void *y, *sum;
  // backward
  const void *dy, *dsum;
  int64_t dys, dss;
  void *dx;
  float *sums;  // [blocks][2][width]
};

template <int kLanes>
constexpr int kThreadsOf = kLanes > kBlock ? kLanes : kBlock;

// Sums over the kLanes threads of a row.  Every thread of the workgroup comes here; `turn` alternates, so that one barrier
// a sum is enough.
template <int kLanes, int kSums>
struct RowSums {
  static constexpr int kWaves = kThreadsOf<kLanes> / kWave;
  static __device__ __forceinline__ void run(float (&x)[kSums], float (*part)[kWaves][4], int &turn) {
#pragma unroll
    for (int i = 0; i < kSums; ++i) x[i] = lanes_sum<(kLanes < kWave ? kLanes : kWave)>(x[i]);
    if constexpr (kLanes > kWave) {
      constexpr int kShare = kLanes / kWave;
      const int wave = threadIdx.x / kWave;
      if (threadIdx.x % kWave == 0)
#pragma unroll
        for (int i = 0; i < kSums; ++i) part[turn][wave][i] = x[i];
      __syncthreads();
      const int first = wave / kShare * kShare;
#pragma unroll
      for (int i = 0; i < kSums; ++i) {
        x[i] = 0;
#pragma unroll
        for (int w = 0; w < kShare; ++w) x[i] += part[turn][first + w][i];
      }
      turn ^= 1;
    }
  }
};

template <typename T, typename P>
__device__ __forceinline__ void store(const LayerArgs &a, T *row, const P &s, const Vals<T> &x) {
  if (a.once && s.whole())
    store_raw<true>(row + s.col, __builtin_convertvector(x, Raw<T>));
  else
    store_slot(row, s, x);
}

template <typename T, typename P>
__device__ __forceinline__ Vals<T> weights_at(const void *w, int f32, const P &s, float none) {
  Vals<T> x;
#pragma unroll
  for (int e = 0; e < kPer<T>; ++e) x[e] = none;
  if (w == nullptr || !s.any()) return x;
  if (s.whole()) {
    if (f32) {
#pragma unroll
      for (int e = 0; e < kPer<T>; ++e) x[e] = static_cast<const float *>(w)[s.col + e];
    } else {
      x = __builtin_convertvector(reinterpret_cast<const AnyRaw<T> *>(static_cast<const T *>(w) + s.col)->v, Vals<T>);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e)
      if (s.own(e)) x[e] = f32 ? static_cast<const float *>(w)[s.col + e] : (float)static_cast<const T *>(w)[s.col + e];
  }
  return x;
}

template <typename T, typename P>
__device__ __forceinline__ Vals<T> own_only(Vals<T> x, const P &s) {
  if (!s.whole()) {
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e)
      if (!s.own(e)) x[e] = 0;
  }
  return x;
}

// 1 / deviation, from the sum of squares around a mean that is `off`
__device__ __forceinline__ float inverse(float squares, float off, const LayerArgs &a) {
  return __builtin_amdgcn_rsqf(fmaxf(fmaf(squares, a.over_width, -off * off), 0.f) + a.eps);
}

template <typename T, int kLanes, int kVecs, bool kWhole, bool kResidual>
__global__ __launch_bounds__(kThreadsOf<kLanes>) void layer_norm_kernel(LayerArgs a) {
  constexpr int kThreads = kThreadsOf<kLanes>, kRows = kThreads / kLanes;
  using At = Place<kWhole, T>;
  __shared__ float part[2][kThreads / kWave][4];
  const int lane = threadIdx.x % kLanes;
  const bool tiny = kLanes == 4 && a.width < kPer<T>;
  int turn = 0;
  Vals<T> w[kVecs], b[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const At s(lane + i * kLanes, a.width);
    w[i] = weights_at<T>(a.weight, a.weight_f32, s, 1.f), b[i] = weights_at<T>(a.bias, a.weight_f32, s, 0.f);
  }
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.rows; base += (int64_t)gridDim.x * kRows) {
    const int64_t row = base + threadIdx.x / kLanes;
    const bool here = row < a.rows;
    Vals<T> u[kVecs];
    float total[1] = {0.f};
    const T *x = static_cast<const T *>(a.x) + row * a.xs, *r = static_cast<const T *>(a.residual) + row * a.rs;
    T *y = static_cast<T *>(a.y) + row * a.width, *sum = static_cast<T *>(a.sum) + row * a.width;
    Raw<T> xs[kVecs], rs[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
      xs[i] = rs[i] = Raw<T>{};
      if (here && s.any()) {
        xs[i] = load_slot<T>(x, s, tiny);
        if constexpr (kResidual) rs[i] = load_slot<T>(r, s, tiny);
      }
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
      u[i] = __builtin_convertvector(xs[i], Vals<T>);
      if constexpr (kResidual) {
        u[i] += __builtin_convertvector(rs[i], Vals<T>);
        if (here && s.any()) store<T>(a, sum, s, u[i]);
        u[i] = __builtin_convertvector(__builtin_convertvector(u[i], Raw<T>), Vals<T>);
      }
      u[i] = own_only<T>(u[i], s);
      total[0] += sum_of(u[i]);
    }
    RowSums<kLanes, 1>::run(total, part, turn);
    const float mean = total[0] / (float)a.width;
    float sums[2] = {0.f, 0.f};  // of c, c^2
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
      u[i] = s.any() ? own_only<T>(u[i] - mean, s) : Vals<T>{};
      sums[0] += sum_of(u[i]), sums[1] += sum_of(u[i] * u[i]);
    }
    RowSums<kLanes, 2>::run(sums, part, turn);
    const float off = sums[0] * a.over_width, inv = inverse(sums[1], off, a);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
      if (here && s.any()) store<T>(a, y, s, (u[i] - off) * inv * w[i] + b[i]);
    }
  }
}

template <typename T, int kLanes, int kVecs, bool kWhole, bool kSum>
__global__ __launch_bounds__(kThreadsOf<kLanes>) void layer_norm_grad_kernel(LayerArgs a) {
  constexpr int kThreads = kThreadsOf<kLanes>, kRows = kThreads / kLanes;
  constexpr bool kHoldWeights = kLanes < 512;
  using At = Place<kWhole, T>;
  __shared__ float part[2][kThreads / kWave][4];
  const int lane = threadIdx.x % kLanes;
  const bool tiny = kLanes == 4 && a.width < kPer<T>;
  int turn = 0;
  Vals<T> w[kVecs], dw[kVecs], db[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    if (kHoldWeights) w[i] = weights_at<T>(a.weight, a.weight_f32, At(lane + i * kLanes, a.width), 1.f);
    dw[i] = db[i] = Vals<T>{};
  }
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.rows; base += (int64_t)gridDim.x * kRows) {
    const int64_t row = base + threadIdx.x / kLanes;
    const bool here = row < a.rows;
    const T *x = static_cast<const T *>(a.x) + row * a.xs, *dy = static_cast<const T *>(a.dy) + row * a.dys,
            *ds = static_cast<const T *>(a.dsum) + row * a.dss;
    T *dx = static_cast<T *>(a.dx) + row * a.width;
    Raw<T> us[kVecs], g[kVecs], plus[kVecs];
    Vals<T> u[kVecs];
    float mean[1] = {0.f};
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
      us[i] = g[i] = plus[i] = Raw<T>{};
      if (here && s.any()) {
        us[i] = load_slot<T>(x, s, tiny), g[i] = load_slot<T>(dy, s, tiny);
        if constexpr (kSum) plus[i] = load_slot<T>(ds, s, tiny);
      }
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
      u[i] = own_only<T>(__builtin_convertvector(us[i], Vals<T>), s);
      mean[0] += sum_of(u[i]);
    }
    RowSums<kLanes, 1>::run(mean, part, turn);
    mean[0] /= (float)a.width;
    float sums[4] = {0.f, 0.f, 0.f, 0.f};  // of c, c^2, h, h c
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
      u[i] = s.any() && here ? own_only<T>(u[i] - mean[0], s) : Vals<T>{};
      if (!kHoldWeights) w[i] = weights_at<T>(a.weight, a.weight_f32, s, 1.f);
      const Vals<T> h = own_only<T>(__builtin_convertvector(g[i], Vals<T>), s) * w[i];
      sums[0] += sum_of(u[i]), sums[1] += sum_of(u[i] * u[i]), sums[2] += sum_of(h), sums[3] += sum_of(h * u[i]);
      as_it_came<T>(g[i]);
    }
    RowSums<kLanes, 4>::run(sums, part, turn);
    const float off = sums[0] * a.over_width, inv = inverse(sums[1], off, a);
    const float mean_h = sums[2] * a.over_width, mean_hn = (sums[3] * a.over_width - off * mean_h) * inv;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
      if (!kHoldWeights) w[i] = weights_at<T>(a.weight, a.weight_f32, s, 1.f);
      if (here && s.any()) {
        const Vals<T> n = (u[i] - off) * inv, gv = own_only<T>(__builtin_convertvector(g[i], Vals<T>), s);
        dw[i] += gv * n, db[i] += gv;
        store<T>(a, dx, s, inv * (gv * w[i] - mean_h - n * mean_hn) + __builtin_convertvector(plus[i], Vals<T>));
      }
    }
  }
  if (a.sums == nullptr) return;
  float *to = a.sums + (int64_t)blockIdx.x * 2 * a.width;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
#pragma unroll
      for (int e = 0; e < kPer<T>; ++e)
        if (s.own(e)) to[s.col + e] = dw[i][e], to[a.width + s.col + e] = db[i][e];
    }
  } else {
    // the rows of the workgroup, one vector and one of both sums at a time
    __shared__ Vals<T> pile[kThreads];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const At s(lane + i * kLanes, a.width);
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        __syncthreads();
        pile[threadIdx.x] = side ? db[i] : dw[i];
        __syncthreads();
        if ((int)threadIdx.x < kLanes) {
          Vals<T> x = pile[threadIdx.x];
          for (int k = 1; k < kRows; ++k) x += pile[k * kLanes + threadIdx.x];
#pragma unroll
          for (int e = 0; e < kPer<T>; ++e)
            if (s.own(e)) to[side * a.width + s.col + e] = x[e];
        }
      }
    }
  }
}

// The sums of all workgroups: 16 of the 2 * width columns a workgroup, 16 threads a column.
constexpr int kColumns = 16;
template <typename T>
__global__ __launch_bounds__(kBlock) void layer_norm_weights_kernel(const float *sums, int blocks, int width, int f32, void *dw,
                                                                    void *db) {
  __shared__ float part[kBlock / kColumns][kColumns];
  const int c = threadIdx.x % kColumns, group = threadIdx.x / kColumns, column = blockIdx.x * kColumns + c;
  float s = 0;
  if (column < 2 * width)
#pragma unroll 8
    for (int r = group; r < blocks; r += kBlock / kColumns) s += sums[(int64_t)r * 2 * width + column];
  part[group][c] = s;
  __syncthreads();
  if (group != 0 || column >= 2 * width) return;
  for (int x = 1; x < kBlock / kColumns; ++x) s += part[x][c];
  const int side = column >= width, i = column - side * width;
  void *to = side ? db : dw;
  if (to == nullptr) return;
  if (f32)
    static_cast<float *>(to)[i] = s;
  else
    static_cast<T *>(to)[i] = (T)s;
}

// f(T(), lanes of a row, vectors of a lane, whether vectors are whole)
template <typename F>
void by_type_and_lanes(int dtype, int width, const F &given) {
  by_type(dtype, [&](auto type) {
    auto f = [&](auto, auto lanes, auto vecs) {
      if (width % kPer<decltype(type)> == 0)
        given(type, lanes, vecs, std::true_type());
      else
        given(type, lanes, vecs, std::false_type());
    };
    const int vecs = (width + kPer<decltype(type)> - 1) / kPer<decltype(type)>;
    using two = std::integral_constant<int, 2>;
    if (vecs <= 8)
      f(type, std::integral_constant<int, 4>(), two());
    else if (vecs <= 16)
      f(type, std::integral_constant<int, 8>(), two());
    else if (vecs <= 32)
      f(type, std::integral_constant<int, 16>(), two());
    else if (vecs <= 64)
      f(type, std::integral_constant<int, 32>(), two());
    else if (vecs <= 128)
      f(type, std::integral_constant<int, 64>(), two());
    else if (vecs <= 256)
      f(type, std::integral_constant<int, 128>(), two());
    else if (vecs <= 512)
      f(type, std::integral_constant<int, 256>(), two());
    else if (vecs <= 1024)
      f(type, std::integral_constant<int, 512>(), two());
    else if (vecs <= 2048)
      f(type, std::integral_constant<int, 1024>(), two());
    else if constexpr (sizeof(type) == 4)
      f(type, std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
  });
}

// 0: go on; 1: nothing to do; else the error
int prepare(const gear_hip_layer_norm_desc *d, LayerArgs &a) {
  if (d == nullptr || d->rows < 0 || d->width < 1 || element_bytes(d->dtype) == 0 || !(d->eps >= 0)) return GEAR_HIP_EINVAL;
  if (d->width > kMaxWidth || d->rows >= (int64_t)1 << 40) return GEAR_HIP_ERANGE;
  if (d->rows == 0) return 1;
  if (d->x == nullptr) return GEAR_HIP_EINVAL;
  const int element = element_bytes(d->dtype), weight = d->weight_f32 ? 4 : element;
  if (!aligned_to(d->x, element) || !aligned_to(d->residual, element) || !aligned_to(d->weight, weight) || !aligned_to(d->bias, weight))
    return GEAR_HIP_EALIGN;
  a.x = d->x, a.xs = d->x_stride, a.residual = d->residual, a.rs = d->residual_stride;
  a.weight = d->weight, a.bias = d->bias, a.weight_f32 = d->weight_f32 != 0;
  a.rows = d->rows, a.width = (int)d->width;
  a.once = d->rows * d->width * element >= kOnceBytes;
  a.eps = d->eps, a.over_width = (float)(1.0 / (double)d->width);
  return 0;
}

// workgroups, where each goes through rows `rows` at a time
int64_t blocks_of(int64_t rows, int each, int64_t most) {
  const int64_t n = ceil_div64(rows, each);
  return n < most ? n : most;
}
int64_t grad_blocks(int threads) { return threads > kBlock ? kGradBlocksWide : kGradBlocks; }

}  // namespace
}  // namespace gearhip

using namespace gearhip;

extern "C" int gear_hip_layer_norm(const gear_hip_layer_norm_desc *desc, void *y, void *sum, void *stream) {
  LayerArgs a = {};
  const int rc = prepare(desc, a);
  if (rc != 0) return rc < 0 ? rc : 0;
  if (y == nullptr || (sum == nullptr) != (a.residual == nullptr)) return GEAR_HIP_EINVAL;
  const int element = element_bytes(desc->dtype);
  if (!aligned_to(y, element) || !aligned_to(sum, element)) return GEAR_HIP_EALIGN;
  a.y = y, a.sum = sum;
  by_type_and_lanes(desc->dtype, a.width, [&](auto type, auto lanes, auto vecs, auto whole) {
    constexpr int kLanes = decltype(lanes)::value, kThreads = kThreadsOf<kLanes>;
    const dim3 grid((unsigned)blocks_of(a.rows, kThreads / kLanes, (1 << 24) / kThreads)), block(kThreads);
    if (a.residual)
      hipLaunchKernelGGL((layer_norm_kernel<decltype(type), kLanes, decltype(vecs)::value, decltype(whole)::value, true>), grid, block, 0,
                         as_stream(stream), a);
    else
      hipLaunchKernelGGL((layer_norm_kernel<decltype(type), kLanes, decltype(vecs)::value, decltype(whole)::value, false>), grid, block, 0,
                         as_stream(stream), a);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}

extern "C" size_t gear_hip_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
  if (rows < 0 || width < 1 || width > kMaxWidth) return 0;
  return (size_t)(rows < kGradBlocks ? rows : kGradBlocks) * 2 * (size_t)width * sizeof(float);
}

extern "C" int gear_hip_layer_norm_backward(const gear_hip_layer_norm_desc *desc, const void *dy, int64_t dy_stride,
                                            const void *dsum, int64_t dsum_stride, void *dx, void *dweight, void *dbias,
                                            void *workspace, size_t workspace_bytes, void *stream) {
  LayerArgs a = {};
  const int rc = prepare(desc, a);
  if (rc < 0) return rc;
  const bool want = dweight != nullptr || dbias != nullptr;
  const int element = element_bytes(desc->dtype), weight = desc->weight_f32 ? 4 : element;
  if (!aligned_to(dweight, weight) || !aligned_to(dbias, weight)) return GEAR_HIP_EALIGN;
  int64_t blocks = 0;  // without rows the weights' gradients are zero
  if (rc == 0) {
    if (want && (workspace == nullptr || workspace_bytes < gear_hip_layer_norm_backward_workspace_bytes(a.rows, a.width)))
      return GEAR_HIP_EWORKSPACE;
    if (dy == nullptr || dx == nullptr) return GEAR_HIP_EINVAL;
    if (!aligned_to(dy, element) || !aligned_to(dsum, element) || !aligned_to(dx, element) || (want && !aligned_to(workspace, 16)))
      return GEAR_HIP_EALIGN;
    a.dy = dy, a.dys = dy_stride, a.dsum = dsum, a.dss = dsum_stride, a.dx = dx;
    a.sums = want ? static_cast<float *>(workspace) : nullptr;
    by_type_and_lanes(desc->dtype, a.width, [&](auto type, auto lanes, auto vecs, auto whole) {
      constexpr int kLanes = decltype(lanes)::value, kThreads = kThreadsOf<kLanes>;
      blocks = blocks_of(a.rows, kThreads / kLanes, grad_blocks(kThreads));
      const dim3 grid((unsigned)blocks), block(kThreads);
      if (dsum)
        hipLaunchKernelGGL((layer_norm_grad_kernel<decltype(type), kLanes, decltype(vecs)::value, decltype(whole)::value, true>), grid, block, 0,
                           as_stream(stream), a);
      else
        hipLaunchKernelGGL((layer_norm_grad_kernel<decltype(type), kLanes, decltype(vecs)::value, decltype(whole)::value, false>), grid, block, 0,
                           as_stream(stream), a);
    });
    GEARHIP_RETURN_IF_LAUNCH_FAILED();
  }
  if (!want) return 0;
  by_type(desc->dtype, [&](auto type) {
    hipLaunchKernelGGL((layer_norm_weights_kernel<decltype(type)>), dim3((unsigned)ceil_div64(2 * desc->width, kColumns)),
                       dim3(kBlock), 0, as_stream(stream), static_cast<const float *>(workspace), (int)blocks, (int)desc->width,
                       desc->weight_f32 != 0, dweight, dbias);
  });
  GEARHIP_RETURN_IF_LAUNCH_FAILED();
  return 0;
}
