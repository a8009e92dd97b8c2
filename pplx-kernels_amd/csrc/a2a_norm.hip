// Root-mean-square norm of rows with the residual's addition, the rows in 8 bits behind it, and the gradients.
//
//   h = x + residual      v = h * r * weight, r = 1 / sqrt(mean(h^2) + eps)
//
// Bound by the rows' bytes: a row stays in registers between the sum of its squares and what is made of it, so that each is
// read once and each result written once.  Sums are fp32.
#include <cfloat>
#include <cmath>

#include "a2a_experts.h"

namespace pplx_amd {
namespace {

struct NormDev {
  const uint8_t *x;
  int64_t x_stride_row;
  const uint8_t *residual;
  int64_t residual_stride_row;
  const uint8_t *weight;
  uint8_t *y;
  int64_t y_stride_row;
  uint8_t *sum;
  int64_t sum_stride_row;
  uint8_t *q;
  int64_t q_stride_row;
  float *scale;
  int64_t scale_stride_row, scale_stride_block;
  float eps, inverse_width;
  uint32_t m, width;
  uint32_t first_group;
};

template <class T> __device__ __forceinline__ PPLX_GLOBAL T *row_at(uint8_t *base, int64_t stride, uint32_t r) {
  return as_global(reinterpret_cast<T *>(base + (int64_t)r * stride));
}
template <class T> __device__ __forceinline__ const PPLX_GLOBAL T *row_at(const uint8_t *base, int64_t stride, uint32_t r) {
  return as_global(reinterpret_cast<const T *>(base + (int64_t)r * stride));
}

// The sum over the LANES threads of a row (64, or all of a workgroup, which all call), the same in each.
template <int LANES> __device__ __forceinline__ float row_sum(float v) {
  v = wave_sum(v);
  if constexpr (LANES > 64) {
    __shared__ float of_wave[LANES / 64];
    __syncthreads();  // (the row before has been read)
    if (lane_id() == 0) of_wave[wave_id()] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) v += of_wave[w];
  }
  return v;
}

// 1 / sqrt(squares / width + eps).
__device__ __forceinline__ float inverse_root(float squares, const float inverse_width, const float eps) {
  return __builtin_amdgcn_rsqf(__builtin_fmaf(squares, inverse_width, eps));
}
// Squares that fp32 does not hold (of 1.8e19 and more) are added up once more of values 2^-70 times as large, beside which eps is
// nothing.  What is an infinity or NaN even then makes the row NaN.
constexpr float kSmall = 0x1p-70f;
__device__ __forceinline__ float inverse_root_of_small(float squares, const float inverse_width) {
  if (!(squares <= FLT_MAX)) return __uint_as_float(0x7fc00000u);
  return __builtin_amdgcn_rsqf(squares * inverse_width) * kSmall;
}
__device__ __forceinline__ float squares_of(f32x8 v, float factor) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = v[i] * factor;
    s = __builtin_fmaf(f, f, s);
  }
  return s;
}

// The largest value of the sixteen lanes around this one, which hold a block of 128 columns.
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
#pragma unroll
  for (int d = 8; d; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, d);
    v = v > o ? v : o;
  }
  return v;
}

// A block's scale and its inverse: a / 448 and 448 / a.  |v| * (448 / a) is at most 448 (1 + 2^-23), which rounds to 448, the
// largest e4m3.
__device__ __forceinline__ RowScale block_scale(uint32_t max_bits) {
  RowScale s;
  if (max_bits >= 0x7f800000u) {
    s.inverse = 0.f;
    s.scale = __uint_as_float(0x7fc00000u);
  } else {
    const float a = __uint_as_float(max_bits > kTinyBits ? max_bits : kTinyBits);
    s.inverse = 448.f / a;
    s.scale = a / 448.f;
  }
  return s;
}
// Eight values as e4m3, rounded to nearest, ties to even (zeros where the inverse is 0).
__device__ __forceinline__ u32x2 e4m3_eight(f32x8 v, float inverse) {
  u32x2 out;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * inverse, v[4 * i + 1] * inverse, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * inverse, v[4 * i + 3] * inverse, w, true);
    out[i] = inverse != 0.f ? (uint32_t)w : 0u;
  }
  return out;
}

// What a thread makes of eight elements of a normed row, whose scale has been found.
template <class T, int FORMAT> __device__ __forceinline__ void store_normed(const NormDev &a, uint32_t r, uint32_t j, f32x8 v, float inverse) {
  if (a.y) store_eight<T>(row_at<T>(a.y, a.y_stride_row, r) + 8ull * j, v);
  if constexpr (FORMAT == PPLX_A2A_ROWS_INT8) *reinterpret_cast<PPLX_GLOBAL u32x2 *>(row_at<uint8_t>(a.q, a.q_stride_row, r) + 8ull * j) = quantize_eight(v, inverse);
  if constexpr (FORMAT == PPLX_A2A_ROWS_E4M3) *reinterpret_cast<PPLX_GLOBAL u32x2 *>(row_at<uint8_t>(a.q, a.q_stride_row, r) + 8ull * j) = e4m3_eight(v, inverse);
}
// The scale of the block of 128 columns around these eight, by sixteen lanes; those behind the row bring zeros.
__device__ __forceinline__ float block_inverse(const NormDev &a, uint32_t r, uint32_t j, bool there, f32x8 v) {
  const RowScale s = block_scale(block_max(magnitude_bits(v)));
  if (there && j % 16 == 0) as_global(a.scale)[(int64_t)r * a.scale_stride_row + (int64_t)(j / 16) * a.scale_stride_block] = s.scale;
  return s.inverse;
}

// Rows of up to 8 LANES PIECES elements, LANES threads to one, which stay in registers; eight elements apart from the next thread's.  All of
// a row's loads, and the weight's, are under way before the first is used.
template <class T, class W, int FORMAT, int LANES, int PIECES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void norm_rows(NormDev a) {
  const uint32_t g = threadIdx.x % LANES, groups = a.width / 8, group = a.first_group + blockIdx.x;
  const uint32_t r = LANES == 64 ? group * 4 + wave_id() : group;
  if (r >= a.m) return;
  const PPLX_GLOBAL W *weight = as_global(reinterpret_cast<const W *>(a.weight));
  typename Eight<W>::raw w[PIECES];
  typename Eight<T>::raw x[PIECES], residual[PIECES];
  // (a thread without elements reads the row's first, which count for nothing)
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const uint32_t j = i * LANES + g, at = j < groups ? j : 0;
    x[i] = load_eight<T>(row_at<T>(a.x, a.x_stride_row, r) + 8ull * at);
    if (a.residual) residual[i] = load_eight<T>(row_at<T>(a.residual, a.residual_stride_row, r) + 8ull * at);
  }
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const uint32_t j = i * LANES + g;
    w[i] = load_eight<W>(weight + 8ull * (j < groups ? j : 0));
  }
  f32x8 v[PIECES];
  float squares = 0.f;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const uint32_t j = i * LANES + g;
    v[i] = Eight<T>::wide(x[i]);
    if (a.residual) {
      // (rounded: what the sum's reader and the gradient see is what the norm is of)
      v[i] = Eight<T>::wide(Eight<T>::narrow(v[i] + Eight<T>::wide(residual[i])));
      if (j < groups) store_eight<T>(row_at<T>(a.sum, a.sum_stride_row, r) + 8ull * j, v[i]);
    }
    if (j >= groups) v[i] = f32x8{};
    squares += squares_of(v[i], 1.f);
  }
  squares = row_sum<LANES>(squares);
  float root;
  if (squares <= FLT_MAX) {
    root = inverse_root(squares, a.inverse_width, a.eps);
  } else {
    float small = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) small += squares_of(v[i], kSmall);
    root = inverse_root_of_small(row_sum<LANES>(small), a.inverse_width);
  }
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    v[i] = v[i] * root * Eight<W>::wide(w[i]);
    if constexpr (FORMAT == PPLX_A2A_ROWS_INT8) {
      const uint32_t b = magnitude_bits(i * LANES + g < groups ? v[i] : f32x8{});
      bits = bits > b ? bits : b;
    }
  }
  float inverse = 0.f;
  if constexpr (FORMAT == PPLX_A2A_ROWS_INT8) {
    const RowScale s = row_scale(row_max<LANES>(bits));
    inverse = s.inverse;
    if (g == 0) as_global(a.scale)[(int64_t)r * a.scale_stride_row] = s.scale;
  }
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const uint32_t j = i * LANES + g;
    if constexpr (FORMAT == PPLX_A2A_ROWS_E4M3) inverse = block_inverse(a, r, j, j < groups, j < groups ? v[i] : f32x8{});
    if (j < groups) store_normed<T, FORMAT>(a, r, j, v[i], inverse);
  }
}

// Longer rows, of which a workgroup reads one twice, or for one scale a row three times.
constexpr int kLongLanes = 512;
template <class T, class W, int FORMAT> __global__ __launch_bounds__(kLongLanes) void norm_long_rows(NormDev a) {
  const uint32_t g = threadIdx.x, groups = a.width / 8, turns = (groups + kLongLanes - 1) / kLongLanes;
  const PPLX_GLOBAL W *weight = as_global(reinterpret_cast<const W *>(a.weight));
  const uint32_t r = a.first_group + blockIdx.x;
  const PPLX_GLOBAL T *x = row_at<T>(a.x, a.x_stride_row, r);
  float squares = 0.f;
  for (uint32_t j = g; j < groups; j += kLongLanes) {
    f32x8 v = Eight<T>::wide(load_eight<T>(x + 8ull * j));
    if (a.residual) {
      v += Eight<T>::wide(load_eight<T>(row_at<T>(a.residual, a.residual_stride_row, r) + 8ull * j));
      v = Eight<T>::wide(Eight<T>::narrow(v));
      store_eight<T>(row_at<T>(a.sum, a.sum_stride_row, r) + 8ull * j, v);
    }
    squares += squares_of(v, 1.f);
  }
  squares = row_sum<kLongLanes>(squares);
  // (a thread reads again what it has written itself)
  const PPLX_GLOBAL T *again = a.residual ? row_at<T>(a.sum, a.sum_stride_row, r) : x;
  float root;
  if (squares <= FLT_MAX) {
    root = inverse_root(squares, a.inverse_width, a.eps);
  } else {
    float small = 0.f;
    for (uint32_t j = g; j < groups; j += kLongLanes) small += squares_of(Eight<T>::wide(load_eight<T>(again + 8ull * j)), kSmall);
    root = inverse_root_of_small(row_sum<kLongLanes>(small), a.inverse_width);
  }
  auto normed = [&](uint32_t j) { return Eight<T>::wide(load_eight<T>(again + 8ull * j)) * root * Eight<W>::wide(load_eight<W>(weight + 8ull * j)); };
  float inverse = 0.f;
  if constexpr (FORMAT == PPLX_A2A_ROWS_INT8) {
    uint32_t bits = 0;
    for (uint32_t j = g; j < groups; j += kLongLanes) {
      const uint32_t b = magnitude_bits(normed(j));
      bits = bits > b ? bits : b;
    }
    const RowScale s = row_scale(row_max<kLongLanes>(bits));
    inverse = s.inverse;
    if (g == 0) as_global(a.scale)[(int64_t)r * a.scale_stride_row] = s.scale;
  }
  for (uint32_t t = 0; t < turns; ++t) {
    const uint32_t j = t * kLongLanes + g;
    const f32x8 v = j < groups ? normed(j) : f32x8{};
    if constexpr (FORMAT == PPLX_A2A_ROWS_E4M3) inverse = block_inverse(a, r, j, j < groups, v);
    if (j < groups) store_normed<T, FORMAT>(a, r, j, v, inverse);
  }
}

// ---------------------------------------------------------------------------
// Gradients
// ---------------------------------------------------------------------------
struct NormBackwardDev {
  const uint8_t *grad_y;
  int64_t grad_y_stride_row;
  const uint8_t *grad_sum;
  int64_t grad_sum_stride_row;
  const uint8_t *h;
  int64_t h_stride_row;
  const uint8_t *weight;
  uint8_t *grad_h;
  int64_t grad_h_stride_row;
  float *partial;  // [gridDim.x, width], or of long rows r of each row
  float eps, inverse_width;
  uint32_t m, width;
};

// Two sums over the threads of a workgroup.  `buffer` alternates from call to call, so that one barrier is enough.
template <int LANES> __device__ __forceinline__ void row_sums(float &a, float &b, uint32_t buffer) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (LANES > 64) {
    __shared__ float of_wave[2][LANES / 64][2];
    if (lane_id() == 0) {
      of_wave[buffer][wave_id()][0] = a;
      of_wave[buffer][wave_id()][1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) {
      a += of_wave[buffer][w][0];
      b += of_wave[buffer][w][1];
    }
  }
}

// Rows of up to 8 LANES PIECES elements, which stay in registers; a workgroup takes one row behind the other, with the loads of the next
// one under way (AHEAD: registers allow it), and holds its share of the weight's gradient.
template <class T, class W, int LANES, int PIECES, bool AHEAD>
__global__ __launch_bounds__(LANES == 64 ? 256 : LANES) void norm_backward_rows(NormBackwardDev a) {
  constexpr uint32_t kAtOnce = LANES == 64 ? 4 : 1;  // rows: a wave to a short one
  const uint32_t g = threadIdx.x % LANES, groups = a.width / 8, step = gridDim.x * kAtOnce;
  const PPLX_GLOBAL W *weight = as_global(reinterpret_cast<const W *>(a.weight));
  struct Rows {
    typename Eight<T>::raw h[PIECES], d[PIECES], s[PIECES];
  };
  // (a thread without elements reads the rows' first, which count for nothing)
  auto load = [&](Rows &to, uint32_t r) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const uint32_t j = i * LANES + g, at = j < groups ? j : 0;
      to.h[i] = load_eight<T>(row_at<T>(a.h, a.h_stride_row, r) + 8ull * at);
      to.d[i] = load_eight<T>(row_at<T>(a.grad_y, a.grad_y_stride_row, r) + 8ull * at);
      if (a.grad_sum && a.grad_h) to.s[i] = load_eight<T>(row_at<T>(a.grad_sum, a.grad_sum_stride_row, r) + 8ull * at);
    }
  };
  typename Eight<W>::raw w[PIECES];
  Rows now, next;
  uint32_t r = blockIdx.x * kAtOnce + (LANES == 64 ? wave_id() : 0);
  bool here = r < a.m;  // (without short rows there are no more workgroups than rows)
  if (AHEAD) load(next, here ? r : 0);
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const uint32_t j = i * LANES + g;
    w[i] = load_eight<W>(weight + 8ull * (j < groups ? j : 0));
  }
  f32x8 of_weight[PIECES] = {};
  for (uint32_t buffer = 0; here; buffer ^= 1) {
    const bool more = a.m - r > step;
    if (AHEAD) {
      now = next;
      if (more) load(next, r + step);
    } else {
      load(now, r);
    }
    float squares = 0.f, along = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if (i * LANES + g >= groups) continue;
      const f32x8 h = Eight<T>::wide(now.h[i]), d = Eight<T>::wide(now.d[i]) * Eight<W>::wide(w[i]);
      squares += squares_of(h, 1.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) along = __builtin_fmaf(d[k], h[k], along);
    }
    row_sums<LANES>(squares, along, buffer);
    float root = inverse_root(squares, a.inverse_width, a.eps);
    if (!(squares <= FLT_MAX)) {
      // (values whose squares fp32 does not hold: both sums of values 2^-70 times as large)
      squares = along = 0.f;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        if (i * LANES + g >= groups) continue;
        const f32x8 h = Eight<T>::wide(now.h[i]) * kSmall, d = Eight<T>::wide(now.d[i]) * Eight<W>::wide(w[i]);
        squares += squares_of(h, 1.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) along = __builtin_fmaf(d[k], h[k], along);
      }
      if (LANES > 64) __syncthreads();  // (the sums have been read)
      row_sums<LANES>(squares, along, buffer);
      if (LANES > 64) __syncthreads();
      root = inverse_root_of_small(squares, a.inverse_width);
      along *= root * (1.f / kSmall);
    } else {
      along *= root;
    }
    along *= a.inverse_width;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const uint32_t j = i * LANES + g;
      if (j >= groups) continue;
      const f32x8 d = Eight<T>::wide(now.d[i]), h = Eight<T>::wide(now.h[i]) * root;
      of_weight[i] += d * h;
      if (!a.grad_h) continue;
      f32x8 out = (d * Eight<W>::wide(w[i]) - h * along) * root;
      if (a.grad_sum) out += Eight<T>::wide(now.s[i]);
      store_eight<T>(row_at<T>(a.grad_h, a.grad_h_stride_row, r) + 8ull * j, out);
    }
    here = more;
    r += step;
  }
  if (!a.partial) return;
  if constexpr (LANES == 64) {
    // The four waves' shares are one.
    __shared__ f32x8 shares[PIECES][256];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) shares[i][threadIdx.x] = of_weight[i];
    __syncthreads();
    if (wave_id()) return;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
#pragma unroll
      for (int w = 1; w < 4; ++w) of_weight[i] += shares[i][w * 64 + g];
    }
  }
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const uint32_t j = i * LANES + g;
    if (j < groups) store_eight<float>(as_global(a.partial) + (uint64_t)blockIdx.x * a.width + 8ull * j, of_weight[i]);
  }
}

// Longer rows, read twice; r of each row is left for the weight's gradient.
template <class T, class W> __global__ __launch_bounds__(kLongLanes) void norm_backward_long(NormBackwardDev a) {
  const uint32_t g = threadIdx.x, groups = a.width / 8;
  const PPLX_GLOBAL W *weight = as_global(reinterpret_cast<const W *>(a.weight));
  for (uint32_t r = blockIdx.x;;) {
    const PPLX_GLOBAL T *grad = row_at<T>(a.grad_y, a.grad_y_stride_row, r), *row = row_at<T>(a.h, a.h_stride_row, r);
    auto squares_times = [&](float factor) {
      float s = 0.f;
      for (uint32_t j = g; j < groups; j += kLongLanes) s += squares_of(Eight<T>::wide(load_eight<T>(row + 8ull * j)), factor);
      return row_sum<kLongLanes>(s);
    };
    const float squares = squares_times(1.f);
    const float root = squares <= FLT_MAX ? inverse_root(squares, a.inverse_width, a.eps)
                                          : inverse_root_of_small(squares_times(kSmall), a.inverse_width);
    if (a.partial && g == 0) as_global(a.partial)[r] = root;
    if (a.grad_h) {
      float along = 0.f;
      for (uint32_t j = g; j < groups; j += kLongLanes) {
        const f32x8 h = Eight<T>::wide(load_eight<T>(row + 8ull * j)) * root;
        const f32x8 d = Eight<T>::wide(load_eight<T>(grad + 8ull * j)) * Eight<W>::wide(load_eight<W>(weight + 8ull * j));
#pragma unroll
        for (int k = 0; k < 8; ++k) along = __builtin_fmaf(d[k], h[k], along);
      }
      along = row_sum<kLongLanes>(along) * a.inverse_width;
      for (uint32_t j = g; j < groups; j += kLongLanes) {
        const f32x8 h = Eight<T>::wide(load_eight<T>(row + 8ull * j)) * root;
        const f32x8 d = Eight<T>::wide(load_eight<T>(grad + 8ull * j)) * Eight<W>::wide(load_eight<W>(weight + 8ull * j));
        f32x8 out = (d - h * along) * root;
        if (a.grad_sum) out += Eight<T>::wide(load_eight<T>(row_at<T>(a.grad_sum, a.grad_sum_stride_row, r) + 8ull * j));
        store_eight<T>(row_at<T>(a.grad_h, a.grad_h_stride_row, r) + 8ull * j, out);
      }
    }
    if (a.m - r <= gridDim.x) break;
    r += gridDim.x;
  }
}

// The weight's gradient out of the workgroups' shares, or of long rows out of the rows: a workgroup to 32 columns, four threads to a
// share or row, whose sums are added in LDS in their order.
constexpr int kSumThreads = 256, kSumSlots = kSumThreads / 4;
template <class W, class Fn> __device__ __forceinline__ void sum_columns(uint32_t count, uint32_t width, W *out, Fn &&of) {
  __shared__ float sums[kSumSlots][33];
  const uint32_t slot = threadIdx.x / 4, j = blockIdx.x * 4 + threadIdx.x % 4;
  f32x8 s = {};
  if (j < width / 8) {
    for (uint32_t i = slot; i < count; i += kSumSlots) s += of(i, j);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) sums[slot][threadIdx.x % 4 * 8 + k] = s[k];
  __syncthreads();
  const uint32_t column = blockIdx.x * 32 + threadIdx.x;
  if (threadIdx.x >= 32 || column >= width) return;
  float sum = 0.f;
#pragma unroll 8
  for (int k = 0; k < kSumSlots; ++k) sum += sums[k][threadIdx.x];
  as_global(out)[column] = (W)sum;
}
template <class W> __global__ __launch_bounds__(kSumThreads) void norm_weight_gradient(const float *partial, uint32_t count, uint32_t width, W *out) {
  sum_columns(count, width, out, [&](uint32_t i, uint32_t j) { return load_eight<float>(as_global(partial) + (uint64_t)i * width + 8ull * j); });
}
template <class T, class W> __global__ __launch_bounds__(kSumThreads) void norm_weight_gradient_long(NormBackwardDev a, W *out) {
  sum_columns(a.m, a.width, out, [&](uint32_t r, uint32_t j) {
    const f32x8 h = Eight<T>::wide(load_eight<T>(row_at<T>(a.h, a.h_stride_row, r) + 8ull * j)) * as_global(a.partial)[r];
    return h * Eight<T>::wide(load_eight<T>(row_at<T>(a.grad_y, a.grad_y_stride_row, r) + 8ull * j));
  });
}

// How many threads a row has, in us of bf16 rows with a residual, out of HBM (16384 x 4096 and longer move at 5.7 TB/s):
//   up to 512         a wave, 8 elements a thread   16384 x 512  13.8 (256 threads 17.4)   262144 x 128  73 (192)
//   up to 2048        256 threads, 8 elements       256 x 2048  3.4 (a wave with 32: 4.4)  8192 x 2048 to e4m3  27.8 (31.8)   16384 x 2048  47.5 (47.5)
//   up to 4096, 8192  512 threads, 8 and 16         512 x 4096  4.8 (256 with 16: 5.7)     8192 x 7168 to e4m3  93 (256 with 32: 98)
//   up to 16384       512 threads, 32               4096 x 16384  94.6 (1024 with 16: 94.9)
// The gradients' workgroups take a row after the other: a wave with 32 elements takes rows of up to 2048 faster than 256 threads do, 16384 x
// 1024  31 (45), since it needs no barrier; longer rows have the same threads as above.
constexpr uint64_t kMostInRegisters = 8 * 4 * 512;

// The gradients' workgroups, each with a share of the weight's gradient to add up: as few as keep memory busy.  One of them has 8192
// elements of each operand under way, or 4096 of rows of up to that, 2048 of short ones.  Both launches, with grad_sum, in a graph over
// tensors and results that no cache holds, us (a step's own results may lie in the caches: 8192 x 4096 then takes 43 + 5):
//   8192 x 7168  256: 89, 512: 97, 1024: 104       8192 x 4096 with weights in fp32  256: 60, 512: 57, 1024: 61     4096 x 2048  256: 17.9, 512: 19.2
//   16384 x 512  256: 19.1, 512: 17.7, 1024: 20.6   262144 x 128  256: 178, 512: 113, 1024: 84
uint32_t backward_groups(uint32_t m, uint64_t width) {
  const uint64_t rows = width <= 2048 ? ((uint64_t)m + 3) / 4 : m;
  const uint64_t most = width <= 128 ? 1024 : width <= 512 || (width > 2048 && width <= 4096) ? 512 : 256;
  return (uint32_t)(rows < most ? rows : most);
}

template <class P> int check_norm_size(const P &p, uint64_t unit) {
  PPLX_REQUIRE(is_dtype(p.dtype), "unsupported dtype of the rows");
  PPLX_REQUIRE(p.weight_dtype == p.dtype || p.weight_dtype == PPLX_A2A_F32, "weight_dtype must be dtype or F32");
  PPLX_REQUIRE(p.hidden_dim > 0 && p.hidden_dim < (1ull << 27) && p.hidden_dim % unit == 0,
               "hidden_dim must be a multiple of %u below 2^27", (unsigned)unit);
  PPLX_REQUIRE(p.eps >= FLT_MIN && p.eps <= FLT_MAX, "eps must be positive, finite and normal");
  if (p.m > kMaxTokens) return refuse(PPLX_A2A_UNSUPPORTED, "2^31 tokens or more");
  return PPLX_A2A_OK;
}

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

extern "C" int pplx_a2a_rms_norm(int device, const pplx_a2a_rms_norm_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_rms_norm_args_t &p = *args;
  PPLX_REQUIRE(p.format >= PPLX_A2A_ROWS_PLAIN && p.format <= PPLX_A2A_ROWS_E4M3, "unknown format of quantised rows");
  const int st = check_norm_size(p, p.format == PPLX_A2A_ROWS_PLAIN ? 8 : 16);
  if (st) return st;
  if (p.m == 0) return PPLX_A2A_OK;
  PPLX_REQUIRE((p.q != nullptr) == (p.format != PPLX_A2A_ROWS_PLAIN), "q goes with a format of quantised rows");
  PPLX_REQUIRE(p.y || p.q, "neither y nor q is asked for");
  PPLX_REQUIRE((p.residual != nullptr) == (p.sum != nullptr), "sum goes with residual");
  PPLX_REQUIRE(!p.q || (p.scale && is_aligned(p.scale, 4)), "scale is NULL or not aligned");
  PPLX_REQUIRE(p.weight && is_aligned(p.weight, 16), "weight is NULL or not 16-byte aligned");
  PPLX_ROWS(p, x);
  if (p.residual) PPLX_ROWS(p, residual);
  if (p.residual) PPLX_ROWS(p, sum);
  if (p.y) PPLX_ROWS(p, y);
  if (p.q) PPLX_ROWS(p, q);
  NormDev a{};
  a.x = static_cast<const uint8_t *>(p.x);
  a.x_stride_row = p.x_stride_row;
  a.residual = static_cast<const uint8_t *>(p.residual);
  a.residual_stride_row = p.residual_stride_row;
  a.weight = static_cast<const uint8_t *>(p.weight);
  a.y = static_cast<uint8_t *>(p.y);
  a.y_stride_row = p.y_stride_row;
  a.sum = static_cast<uint8_t *>(p.sum);
  a.sum_stride_row = p.sum_stride_row;
  a.q = static_cast<uint8_t *>(p.q);
  a.q_stride_row = p.q_stride_row;
  a.scale = p.scale;
  a.scale_stride_row = p.scale_stride_row;
  a.scale_stride_block = p.scale_stride_block;
  a.eps = p.eps;
  a.inverse_width = (float)(1.0 / (double)p.hidden_dim);
  a.m = p.m;
  a.width = (uint32_t)p.hidden_dim;
  return guarded(device, [&] {
    return with_weight_type(p.dtype, p.weight_dtype, [&](auto tag, auto weight_tag) {
      typedef typename decltype(tag)::type T;
      typedef typename decltype(weight_tag)::type W;
      auto launch = [&](auto format) {
        constexpr int F = decltype(format)::value;
        hipStream_t s = (hipStream_t)stream;
        auto rows = [&](auto kernel, uint32_t threads, uint32_t at_once) {
          return launch_groups(kernel, kernel, ((uint64_t)a.m + at_once - 1) / at_once, threads, 0, s, a);
        };
        if (a.width <= 512) PPLX_LAUNCH(rows(norm_rows<T, W, F, 64, 1>, 256, 4));
        else if (a.width <= 2048) PPLX_LAUNCH(rows(norm_rows<T, W, F, 256, 1>, 256, 1));
        else if (a.width <= 4096) PPLX_LAUNCH(rows(norm_rows<T, W, F, 512, 1>, 512, 1));
        else if (a.width <= 8192) PPLX_LAUNCH(rows(norm_rows<T, W, F, 512, 2>, 512, 1));
        else if (a.width <= kMostInRegisters) PPLX_LAUNCH(rows(norm_rows<T, W, F, 512, 4>, 512, 1));
        else PPLX_LAUNCH(rows(norm_long_rows<T, W, F>, kLongLanes, 1));
        return (int)PPLX_A2A_OK;
      };
      switch (p.format) {
        case PPLX_A2A_ROWS_INT8: return launch(std::integral_constant<int, PPLX_A2A_ROWS_INT8>{});
        case PPLX_A2A_ROWS_E4M3: return launch(std::integral_constant<int, PPLX_A2A_ROWS_E4M3>{});
        default: return launch(std::integral_constant<int, PPLX_A2A_ROWS_PLAIN>{});
      }
    });
  });
}

extern "C" int pplx_a2a_rms_norm_workspace(uint32_t m, uint64_t hidden_dim, uint64_t *bytes) {
  PPLX_REQUIRE(bytes, "bytes is NULL");
  PPLX_REQUIRE(hidden_dim > 0 && hidden_dim < (1ull << 27) && hidden_dim % 8 == 0, "hidden_dim must be a multiple of 8 below 2^27");
  if (m > kMaxTokens) return refuse(PPLX_A2A_UNSUPPORTED, "2^31 tokens or more");
  *bytes = 4 * (hidden_dim > kMostInRegisters ? (uint64_t)m : backward_groups(m, hidden_dim) * hidden_dim);
  return PPLX_A2A_OK;
}

extern "C" int pplx_a2a_rms_norm_backward(int device, const pplx_a2a_rms_norm_backward_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_rms_norm_backward_args_t &p = *args;
  const int st = check_norm_size(p, 8);
  if (st) return st;
  PPLX_REQUIRE(p.m > 0, "there are no tokens");
  PPLX_REQUIRE(p.weight && is_aligned(p.weight, 16), "weight is NULL or not 16-byte aligned");
  PPLX_REQUIRE(is_aligned(p.grad_weight, 16), "grad_weight must be 16-byte aligned");
  PPLX_REQUIRE(!p.grad_weight || (p.workspace && is_aligned(p.workspace, 16)), "workspace is NULL or not aligned");
  PPLX_ROWS(p, grad_y);
  if (p.grad_sum) PPLX_ROWS(p, grad_sum);
  PPLX_ROWS(p, h);
  if (p.grad_h) PPLX_ROWS(p, grad_h);
  if (!p.grad_h && !p.grad_weight) return PPLX_A2A_OK;
  NormBackwardDev a{};
  a.grad_y = static_cast<const uint8_t *>(p.grad_y);
  a.grad_y_stride_row = p.grad_y_stride_row;
  a.grad_sum = static_cast<const uint8_t *>(p.grad_sum);
  a.grad_sum_stride_row = p.grad_sum_stride_row;
  a.h = static_cast<const uint8_t *>(p.h);
  a.h_stride_row = p.h_stride_row;
  a.weight = static_cast<const uint8_t *>(p.weight);
  a.grad_h = static_cast<uint8_t *>(p.grad_h);
  a.grad_h_stride_row = p.grad_h_stride_row;
  a.partial = p.grad_weight ? static_cast<float *>(p.workspace) : nullptr;
  a.eps = p.eps;
  a.inverse_width = (float)(1.0 / (double)p.hidden_dim);
  a.m = p.m;
  a.width = (uint32_t)p.hidden_dim;
  return guarded(device, [&] {
    return with_weight_type(p.dtype, p.weight_dtype, [&](auto tag, auto weight_tag) {
      typedef typename decltype(tag)::type T;
      typedef typename decltype(weight_tag)::type W;
      hipStream_t s = (hipStream_t)stream;
      const uint32_t groups = backward_groups(a.m, a.width), columns = (a.width + 31) / 32;
      constexpr bool kAhead = sizeof(T) == 2;  // (32 elements of fp32 in a thread fill its registers once)
      W *out = static_cast<W *>(p.grad_weight);
      if (a.width > kMostInRegisters) {
        // (the weight's gradient reads grad_y once more: grad_h over it comes last, by a launch of its own)
        const bool over = out && a.grad_h && a.grad_h == a.grad_y;
        NormBackwardDev first = a;
        if (over) first.grad_h = nullptr;
        PPLX_LAUNCH(launch_kernel(norm_backward_long<T, W>, dim3(groups), dim3(kLongLanes), 0, s, first));
        if (out) PPLX_LAUNCH(launch_kernel(norm_weight_gradient_long<T, W>, dim3(columns), dim3(kSumThreads), 0, s, a, out));
        a.partial = nullptr;
        if (over) PPLX_LAUNCH(launch_kernel(norm_backward_long<T, W>, dim3(groups), dim3(kLongLanes), 0, s, a));
        return (int)PPLX_A2A_OK;
      }
      if (a.width <= 512) PPLX_LAUNCH(launch_kernel(norm_backward_rows<T, W, 64, 1, true>, dim3(groups), dim3(256), 0, s, a));
      else if (a.width <= 2048) PPLX_LAUNCH(launch_kernel(norm_backward_rows<T, W, 64, 4, kAhead>, dim3(groups), dim3(256), 0, s, a));
      else if (a.width <= 4096) PPLX_LAUNCH(launch_kernel(norm_backward_rows<T, W, 512, 1, true>, dim3(groups), dim3(512), 0, s, a));
      else if (a.width <= 8192) PPLX_LAUNCH(launch_kernel(norm_backward_rows<T, W, 512, 2, true>, dim3(groups), dim3(512), 0, s, a));
      else PPLX_LAUNCH(launch_kernel(norm_backward_rows<T, W, 512, 4, kAhead>, dim3(groups), dim3(512), 0, s, a));
      if (out) {
        const float *partial = a.partial;
        PPLX_LAUNCH(launch_kernel(norm_weight_gradient<W>, dim3(columns), dim3(kSumThreads), 0, s, partial, groups, a.width, out));
      }
      return (int)PPLX_A2A_OK;
    });
  });
}
