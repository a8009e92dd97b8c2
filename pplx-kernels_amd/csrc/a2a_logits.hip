// The router's product and its gradients, on the matrix cores with fp32 sums.
//
//   logits = x weight^T        grad_x = grad_logits weight        grad_weight = grad_logits^T x
//
// All three are sums over k of a[i, k] * b[j, k] of operands whose rows lie along k; for the gradients operands are laid out so
// first.  The matrix cores take 16-bit elements.  What has more bits is a sum of bf16 pieces, each the part of a value
// that the pieces before leave: two hold an fp16 value, three an fp32 one.  Of the products of pieces those below 2^-24 of the
// largest are left out.
#include "a2a_experts.h"

namespace pplx_amd {
namespace {

struct ProductDev {
  const uint8_t *a;
  int64_t a_stride;  // bytes
  const uint8_t *b;
  int64_t b_stride;
  uint8_t *out;
  int64_t out_stride;  // elements
  uint32_t rows, columns, k;
  uint32_t column_blocks;
  uint32_t first_group;
};

template <class T> struct Pieces;
template <> struct Pieces<__bf16> {
  static constexpr int count = 1;
  static __device__ __forceinline__ void of(bf16x8 v, bf16x8 *p) { p[0] = v; }
};
template <> struct Pieces<_Float16> {
  static constexpr int count = 2;
  static __device__ __forceinline__ void of(f16x8 v, bf16x8 *p) {
    const f32x8 w = __builtin_convertvector(v, f32x8);
    p[0] = __builtin_convertvector(w, bf16x8);
    p[1] = __builtin_convertvector(w - __builtin_convertvector(p[0], f32x8), bf16x8);
  }
};
template <> struct Pieces<float> {
  static constexpr int count = 3;
  static __device__ __forceinline__ void of(f32x8 v, bf16x8 *p) {
    p[0] = __builtin_convertvector(v, bf16x8);
    f32x8 left = v - __builtin_convertvector(p[0], f32x8);
    p[1] = __builtin_convertvector(left, bf16x8);
    left -= __builtin_convertvector(p[1], f32x8);
    p[2] = __builtin_convertvector(left, bf16x8);
  }
};

// What a lane holds of an operand, ready for the matrix cores: pieces, or fp16 as it is where both are.
template <class T, class Other> struct Operand {
  static constexpr bool kPlain = std::is_same_v<T, Other> && sizeof(T) == 2;
  static constexpr int count = kPlain ? 1 : Pieces<T>::count;
  typedef std::conditional_t<kPlain, typename Eight<T>::raw, bf16x8> piece;
  piece p[count];
  __device__ __forceinline__ void set(typename Eight<T>::raw v) {
    if constexpr (kPlain) p[0] = v;
    else Pieces<T>::of(v, p);
  }
};
__device__ __forceinline__ f32x4 multiply_16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 multiply_16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
template <class A, class B> __device__ __forceinline__ f32x4 multiply_add(const A &a, const B &b, f32x4 c) {
  // (the smallest first)
#pragma unroll
  for (int order = A::count + B::count - 2 < 2 ? A::count + B::count - 2 : 2; order >= 0; --order) {
#pragma unroll
    for (int i = 0; i < A::count; ++i) {
      if (order - i >= 0 && order - i < B::count) c = multiply_16(a.p[i], b.p[order - i], c);
    }
  }
  return c;
}

// A workgroup to 16 RF rows by 16 CF columns, whose eight waves share out k, 32 elements at a time, and add their sums in
// LDS, in the order of the waves.  Operands go straight to registers.
constexpr int kProductWaves = 8;
template <class TA, class TB, class O, int RF, int CF, int AHEAD>
__global__ __launch_bounds__(kProductWaves * 64) void product_split(ProductDev a) {
  __shared__ float sums[kProductWaves][RF * CF * 4 * 64];
  const uint32_t lane = lane_id(), wave = wave_id(), group = a.first_group + blockIdx.x;
  const uint32_t block = group / a.column_blocks;
  const uint32_t m0 = block * 16 * RF, n0 = (group - block * a.column_blocks) * 16 * CF;
  const PPLX_GLOBAL TA *row[RF];
  const PPLX_GLOBAL TB *column[CF];
#pragma unroll
  for (int i = 0; i < RF; ++i) {
    const uint32_t r = m0 + i * 16 + lane % 16;
    row[i] = as_global(reinterpret_cast<const TA *>(a.a + (int64_t)(r < a.rows ? r : a.rows - 1) * a.a_stride));
  }
#pragma unroll
  for (int i = 0; i < CF; ++i) {
    const uint32_t c = n0 + i * 16 + lane % 16;
    column[i] = as_global(reinterpret_cast<const TB *>(a.b + (int64_t)(c < a.columns ? c : a.columns - 1) * a.b_stride));
  }
  const uint32_t units = (a.k + 31) / 32, own = lane / 16 * 8;
  struct Unit {
    typename Eight<TA>::raw a[RF];
    typename Eight<TB>::raw b[CF];
  };
  Unit u[AHEAD];
  auto load = [&](Unit &to, uint32_t unit) __attribute__((always_inline)) {
    const uint32_t k = unit * 32 + own;
    const uint32_t at = k < a.k ? k : 0;  // (elements behind k are taken for zeros)
#pragma unroll
    for (int i = 0; i < CF; ++i) to.b[i] = load_eight<TB>(column[i] + at);
#pragma unroll
    for (int i = 0; i < RF; ++i) to.a[i] = load_eight<TA>(row[i] + at);
  };
  f32x4 acc[RF][CF] = {};
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    if (wave + i * kProductWaves < units) load(u[i], wave + i * kProductWaves);
  }
  for (uint32_t first = wave; first < units; first += AHEAD * kProductWaves) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const uint32_t unit = first + i * kProductWaves;
      if (unit >= units) break;
      const bool there = unit * 32 + own < a.k;
      Operand<TB, TA> fb[CF];
#pragma unroll
      for (int c = 0; c < CF; ++c) fb[c].set(there ? u[i].b[c] : typename Eight<TB>::raw{});
#pragma unroll
      for (int r = 0; r < RF; ++r) {
        Operand<TA, TB> fa;
        fa.set(there ? u[i].a[r] : typename Eight<TA>::raw{});
#pragma unroll
        for (int c = 0; c < CF; ++c) acc[r][c] = multiply_add(fb[c], fa, acc[r][c]);
      }
      if (unit + AHEAD * kProductWaves < units) load(u[i], unit + AHEAD * kProductWaves);
    }
  }
#pragma unroll
  for (int r = 0; r < RF; ++r) {
#pragma unroll
    for (int c = 0; c < CF; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave][((r * CF + c) * 4 + i) * 64 + lane] = acc[r][c][i];
    }
  }
  __syncthreads();
  // Lane l of fragment (r, c) has columns 16 c + 4 (l / 16) .. + 3 of row 16 r + l % 16.
  if (threadIdx.x >= RF * CF * 64) return;
  const uint32_t fragment = threadIdx.x / 64, r = fragment / CF, c = fragment % CF;
  const uint32_t m = m0 + r * 16 + lane % 16, n = n0 + c * 16 + 4 * (lane / 16);
  if (m >= a.rows) return;
  PPLX_GLOBAL O *out = as_global(reinterpret_cast<O *>(a.out)) + (int64_t)m * a.out_stride;
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kProductWaves; ++w) sum += sums[w][(fragment * 4 + i) * 64 + lane];
    if (n + i < a.columns) out[n + i] = (O)sum;
  }
}

template <class TA, class TB, class O> int launch_product(const ProductDev &from, hipStream_t s) {
  ProductDev a = from;
  a.column_blocks = (a.columns + 31) / 32;
  auto kernel = product_split<TA, TB, O, 2, 2, 2>;
  return launch_groups(kernel, kernel, ((uint64_t)a.rows + 31) / 32 * a.column_blocks, kProductWaves * 64, 0, s, a);
}

// out[c, r] = in[r, c], zeros for r from rows up to the next multiple of eight; a workgroup to 64 by 64.
struct TurnDev {
  const uint8_t *in;
  int64_t in_stride;  // bytes
  uint8_t *out;
  int64_t out_stride;  // bytes
  uint32_t rows, columns;
  uint32_t column_blocks;
  uint32_t first_group;
};
template <class T> __global__ __launch_bounds__(256) void turn(TurnDev a) {
  __shared__ T tile[64][65];
  const uint32_t group = a.first_group + blockIdx.x, block = group / a.column_blocks;
  const uint32_t r0 = block * 64, c0 = (group - block * a.column_blocks) * 64;
  const uint32_t x = threadIdx.x % 64;
  for (uint32_t y = threadIdx.x / 64; y < 64; y += 4) {
    const uint32_t r = r0 + y, c = c0 + x;
    tile[y][x] = r < a.rows && c < a.columns ? as_global(reinterpret_cast<const T *>(a.in + (int64_t)r * a.in_stride))[c] : (T)0;
  }
  __syncthreads();
  const uint32_t most = (a.rows + 7) / 8 * 8;
  for (uint32_t y = threadIdx.x / 64; y < 64; y += 4) {
    const uint32_t r = r0 + x, c = c0 + y;
    if (r < most && c < a.columns) as_global(reinterpret_cast<T *>(a.out + (int64_t)c * a.out_stride))[r] = tile[x][y];
  }
}
template <class T> int launch_turn(const void *in, int64_t in_stride, void *out, int64_t out_stride, uint32_t rows, uint32_t columns, hipStream_t s) {
  TurnDev a{static_cast<const uint8_t *>(in), in_stride, static_cast<uint8_t *>(out), out_stride, rows, columns, (columns + 63) / 64, 0};
  return launch_groups(turn<T>, turn<T>, (uint64_t)((rows + 63) / 64) * a.column_blocks, 256, 0, s, a);
}

// out[r, c] = in[r, c], zeros for c from columns up to the next multiple of eight.
template <class T> __global__ __launch_bounds__(256) void fill_out(TurnDev a) {
  const uint64_t width = (a.columns + 7) / 8 * 8, i = (uint64_t)(a.first_group + blockIdx.x) * 256 + threadIdx.x;
  const uint32_t r = (uint32_t)(i / width), c = (uint32_t)(i - r * width);
  if (r >= a.rows) return;
  as_global(reinterpret_cast<T *>(a.out + (int64_t)r * a.out_stride))[c] =
      c < a.columns ? as_global(reinterpret_cast<const T *>(a.in + (int64_t)r * a.in_stride))[c] : (T)0;
}

uint64_t in_eights(uint64_t n) { return (n + 7) / 8 * 8; }

// The workspace of the gradients: grad_logits with rows of whole eights, the same turned, and the weight and x turned.
struct BackwardSpace {
  uint64_t grad, grad_turned, weight_turned, x_turned, bytes;
};
BackwardSpace backward_space(uint64_t m, uint64_t experts, uint64_t hidden, int64_t size, int64_t weight_size) {
  BackwardSpace s{};
  s.grad = 0;
  s.grad_turned = s.grad + 4 * m * in_eights(experts);
  s.weight_turned = s.grad_turned + 4 * experts * in_eights(m);
  s.x_turned = s.weight_turned + (hidden * in_eights(experts) * weight_size + 15) / 16 * 16;
  s.bytes = s.x_turned + hidden * in_eights(m) * size;
  return s;
}

template <class Fn> int with_weight_type(int32_t dtype, int32_t weight_dtype, Fn &&fn) {
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    return weight_dtype == dtype ? fn(tag, TypeTag<T>{}) : fn(tag, TypeTag<float>{});
  });
}

int check_router_size(uint32_t experts, uint64_t hidden, int32_t dtype, int32_t weight_dtype) {
  PPLX_REQUIRE(is_dtype(dtype), "unsupported dtype of the rows");
  PPLX_REQUIRE(weight_dtype == dtype || weight_dtype == PPLX_A2A_F32, "weight_dtype must be dtype or F32");
  PPLX_REQUIRE(experts >= 1 && experts <= kMaxExperts, "num_experts must be in [1, %u]", kMaxExperts);
  PPLX_REQUIRE(hidden > 0 && hidden < (1ull << 27) && hidden % 8 == 0, "hidden_dim must be a multiple of 8 below 2^27");
  return PPLX_A2A_OK;
}
int check_rows_of(const void *p, int64_t stride, const char *name) {
  PPLX_REQUIRE(p, "%s is NULL", name);
  PPLX_REQUIRE(is_aligned(p, 16) && stride % 16 == 0, "%s must be 16-byte aligned with 16-byte strides", name);
  return PPLX_A2A_OK;
}
#define PPLX_ROWS(p, name)                                               \
  do {                                                                   \
    const int st_ = check_rows_of(p.name, p.name##_stride_row, #name);   \
    if (st_) return st_;                                                 \
  } while (0)

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

extern "C" int pplx_a2a_router_workspace(uint32_t m, uint32_t num_experts, uint64_t hidden_dim, int32_t dtype,
                                         int32_t weight_dtype, int32_t backward, uint64_t *bytes) {
  PPLX_REQUIRE(bytes, "bytes is NULL");
  const int st = check_router_size(num_experts, hidden_dim, dtype, weight_dtype);
  if (st) return st;
  *bytes = backward ? backward_space(m, num_experts, hidden_dim, dtype_bytes(dtype), dtype_bytes(weight_dtype)).bytes : 0;
  return PPLX_A2A_OK;
}

extern "C" int pplx_a2a_router_logits(int device, const pplx_a2a_router_logits_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_router_logits_args_t &p = *args;
  const int st = check_router_size(p.num_experts, p.hidden_dim, p.dtype, p.weight_dtype);
  if (st) return st;
  if (p.m == 0) return PPLX_A2A_OK;
  PPLX_ROWS(p, x);
  PPLX_ROWS(p, weight);
  PPLX_REQUIRE(p.logits && is_aligned(p.logits, 4), "logits is NULL or not aligned");
  ProductDev a{};
  a.a = static_cast<const uint8_t *>(p.x);
  a.a_stride = p.x_stride_row;
  a.b = static_cast<const uint8_t *>(p.weight);
  a.b_stride = p.weight_stride_row;
  a.out = reinterpret_cast<uint8_t *>(p.logits);
  a.out_stride = p.logits_stride_row;
  a.rows = p.m;
  a.columns = p.num_experts;
  a.k = (uint32_t)p.hidden_dim;
  return guarded(device, [&] {
    return with_weight_type(p.dtype, p.weight_dtype, [&](auto tag, auto weight_tag) {
      typedef typename decltype(tag)::type T;
      typedef typename decltype(weight_tag)::type W;
      PPLX_LAUNCH((launch_product<T, W, float>(a, (hipStream_t)stream)));
      return (int)PPLX_A2A_OK;
    });
  });
}

extern "C" int pplx_a2a_router_logits_backward(int device, const pplx_a2a_router_logits_backward_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_router_logits_backward_args_t &p = *args;
  const int st = check_router_size(p.num_experts, p.hidden_dim, p.dtype, p.weight_dtype);
  if (st) return st;
  PPLX_REQUIRE(p.m > 0, "there are no tokens");
  PPLX_REQUIRE(p.grad_logits && is_aligned(p.grad_logits, 4), "grad_logits is NULL or not aligned");
  if (p.grad_x) {
    PPLX_ROWS(p, grad_x);
    PPLX_ROWS(p, weight);
  }
  if (p.grad_weight) {
    PPLX_ROWS(p, grad_weight);
    PPLX_ROWS(p, x);
  }
  if (!p.grad_x && !p.grad_weight) return PPLX_A2A_OK;
  PPLX_REQUIRE(p.workspace && is_aligned(p.workspace, 16), "workspace is NULL or not aligned");
  const uint32_t m = p.m, experts = p.num_experts, hidden = (uint32_t)p.hidden_dim;
  const BackwardSpace space = backward_space(m, experts, hidden, dtype_bytes(p.dtype), dtype_bytes(p.weight_dtype));
  uint8_t *work = static_cast<uint8_t *>(p.workspace);
  const int64_t by_experts = (int64_t)in_eights(experts), by_tokens = (int64_t)in_eights(m);
  return guarded(device, [&] {
    return with_weight_type(p.dtype, p.weight_dtype, [&](auto tag, auto weight_tag) {
      typedef typename decltype(tag)::type T;
      typedef typename decltype(weight_tag)::type W;
      hipStream_t s = (hipStream_t)stream;
      if (p.grad_x) {
        const TurnDev fill{reinterpret_cast<const uint8_t *>(p.grad_logits), 4 * p.grad_logits_stride_row, work + space.grad,
                           4 * by_experts, m, experts, 0, 0};
        PPLX_LAUNCH(launch_groups(fill_out<float>, fill_out<float>, ((uint64_t)m * by_experts + 255) / 256, 256, 0, s, fill));
        PPLX_LAUNCH(launch_turn<W>(p.weight, p.weight_stride_row, work + space.weight_turned, by_experts * (int64_t)sizeof(W),
                                   experts, hidden, s));
        ProductDev a{};
        a.a = work + space.grad;
        a.a_stride = 4 * by_experts;
        a.b = work + space.weight_turned;
        a.b_stride = by_experts * (int64_t)sizeof(W);
        a.out = static_cast<uint8_t *>(p.grad_x);
        a.out_stride = p.grad_x_stride_row / (int64_t)sizeof(T);
        a.rows = m;
        a.columns = hidden;
        a.k = (uint32_t)by_experts;
        PPLX_LAUNCH((launch_product<float, W, T>(a, s)));
      }
      if (p.grad_weight) {
        PPLX_LAUNCH(launch_turn<float>(p.grad_logits, 4 * p.grad_logits_stride_row, work + space.grad_turned, 4 * by_tokens, m,
                                       experts, s));
        PPLX_LAUNCH(launch_turn<T>(p.x, p.x_stride_row, work + space.x_turned, by_tokens * (int64_t)sizeof(T), m, hidden, s));
        ProductDev a{};
        a.a = work + space.grad_turned;
        a.a_stride = 4 * by_tokens;
        a.b = work + space.x_turned;
        a.b_stride = by_tokens * (int64_t)sizeof(T);
        a.out = static_cast<uint8_t *>(p.grad_weight);
        a.out_stride = p.grad_weight_stride_row / (int64_t)sizeof(W);
        a.rows = experts;
        a.columns = hidden;
        a.k = (uint32_t)by_tokens;
        PPLX_LAUNCH((launch_product<float, T, W>(a, s)));
      }
      return (int)PPLX_A2A_OK;
    });
  });
}
