// Rows to 8 bits with one scale each, with the gated activation in front: the input of the experts' products.
#include "a2a_experts.h"

namespace pplx_amd {
namespace {

constexpr uint64_t kStreamBytes = 192ull << 20;

struct QuantizeDev {
  RowsDev rows;
  uint8_t *out;
  int64_t out_stride_row, out_stride_expert;
  float *scale;
  int64_t scale_stride_row, scale_stride_expert;
  const uint8_t *x;
  int64_t x_stride_row, x_stride_expert;
  uint32_t width;
  uint32_t first_group;
};

// What one thread holds of a row: PIECES times eight elements, eight elements apart from the next thread's.
template <class T, bool SWIGLU, int LANES, int PIECES, bool NT> struct Piece {
  const PPLX_GLOBAL T *row;
  uint32_t width, groups, g, first_of_wave;
  f32x8 v[PIECES];

  // (the same for all lanes of a wave: pieces that no lane has cost nothing)
  __device__ __forceinline__ bool any(uint32_t base, int i) const { return base + i * LANES + first_of_wave < groups; }

  __device__ __forceinline__ void load(uint32_t base) {
    typename Eight<T>::raw gate[PIECES], up[SWIGLU ? PIECES : 1];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if (!any(base, i)) continue;
      uint32_t j = base + i * LANES + g;
      j = j < groups ? j : groups - 1;
      gate[i] = load_eight<T, NT>(row + 8ull * j);
      if constexpr (SWIGLU) up[i] = load_eight<T, NT>(row + width + 8ull * j);
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if (!any(base, i)) continue;
      v[i] = Eight<T>::wide(gate[i]);
      if constexpr (SWIGLU) {
        const f32x8 u = Eight<T>::wide(up[i]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          // (A reciprocal of one ulp: a quotient to the last bit is ten instructions more, which the rows' bytes do not hide.  Of
          // a sixteenth: that of 2^126 and more is subnormal, and comes as zero.)
          v[i][k] = 0.0625f * v[i][k] * __builtin_amdgcn_rcpf(__builtin_fmaf(__expf(-v[i][k]), 0.0625f, 0.0625f)) * u[k];
        }
      }
    }
  }
};

// LANES threads to a row; up to 8 * PIECES * LANES elements stay in registers between the search for the largest value and the
// conversion, longer rows are read twice.
template <class T, bool SWIGLU, int LANES, int PIECES, bool NT>
__device__ __forceinline__ void quantize_one(const QuantizeDev &a, uint32_t e, uint32_t r, uint32_t g) {
  constexpr uint32_t kStep = LANES * PIECES;
  Piece<T, SWIGLU, LANES, PIECES, NT> p;
  p.row = as_global(reinterpret_cast<const T *>(a.x + (int64_t)e * a.x_stride_expert + (int64_t)r * a.x_stride_row));
  p.width = a.width;
  p.groups = a.width / 8;
  p.g = g;
  p.first_of_wave = LANES == 64 ? 0 : wave_id() * 64;
  uint32_t bits = 0;
  for (uint32_t base = 0; base < p.groups; base += kStep) {
    p.load(base);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if (!p.any(base, i)) continue;
      const uint32_t b = magnitude_bits(p.v[i]);
      bits = bits > b ? bits : b;
    }
  }
  const RowScale s = row_scale(row_max<LANES>(bits));
  if (g == 0) as_global(a.scale)[(int64_t)e * a.scale_stride_expert + (int64_t)r * a.scale_stride_row] = s.scale;
  PPLX_GLOBAL u32x2 *out =
      as_global(reinterpret_cast<u32x2 *>(a.out + (int64_t)e * a.out_stride_expert + (int64_t)r * a.out_stride_row));
  for (uint32_t base = 0; base < p.groups; base += kStep) {
    if (p.groups > kStep) p.load(base);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if (!p.any(base, i)) continue;
      const uint32_t j = base + i * LANES + g;
      if (j < p.groups) out[j] = quantize_eight(p.v[i], s.inverse);
    }
  }
}

// Rows of one buffer: as many as are there, 256 / LANES to a workgroup.
template <class T, bool SWIGLU, int LANES, int PIECES, bool NT>
__global__ __launch_bounds__(256) void quantize_flat(QuantizeDev a) {
  uint32_t there = a.rows.rows;
  if (a.rows.layout == PPLX_A2A_ROWS_SORTED) {
    const int32_t last = as_global(a.rows.starts_or_counts)[a.rows.experts];
    there = last < 0 ? 0 : (uint32_t)last < there ? (uint32_t)last : there;
  }
  const uint32_t group = a.first_group + blockIdx.x;
  const uint32_t r = LANES == 64 ? group * 4 + wave_id() : group;
  if (r < there) quantize_one<T, SWIGLU, LANES, PIECES, NT>(a, 0, r, threadIdx.x % LANES);
}

// Rows of the experts' buffers: workgroups share out the rows that are there, whose experts they find in the sums of the
// counts.
template <class T, bool SWIGLU, int LANES, int PIECES>
__global__ __launch_bounds__(256) void quantize_padded(QuantizeDev a) {
  extern __shared__ uint32_t upto[];  // rows of the experts up to and with each
  __shared__ uint32_t of_wave[4];
  const uint32_t E = a.rows.experts;
  const uint32_t per = (E + 255) / 256, first = threadIdx.x * per;
  uint32_t own = 0;
  for (uint32_t i = 0; i < per; ++i) own += first + i < E ? span_of(a.rows, first + i).count : 0u;
  uint32_t sum = wave_scan(own, lane_id());
  if (lane_id() == 63) of_wave[wave_id()] = sum;
  __syncthreads();
  sum -= own;
#pragma unroll
  for (int w = 0; w < 4; ++w) sum += (uint32_t)w < wave_id() ? of_wave[w] : 0u;
  for (uint32_t i = 0; i < per; ++i) {
    if (first + i < E) upto[first + i] = sum += span_of(a.rows, first + i).count;
  }
  __syncthreads();
  const uint32_t there = upto[E - 1];
  constexpr uint32_t kAtOnce = 256 / LANES;
  for (uint32_t i = blockIdx.x * kAtOnce; i < there; i += gridDim.x * kAtOnce) {
    const uint32_t r = i + (LANES == 64 ? wave_id() : 0);
    if (r >= there) break;  // (with 256 lanes to a row r is i)
    uint32_t lo = 0, hi = E - 1;
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (upto[mid] > r) hi = mid;
      else lo = mid + 1;
    }
    const uint32_t e = __builtin_amdgcn_readfirstlane(lo);
    quantize_one<T, SWIGLU, LANES, PIECES, false>(a, e, r - (e ? upto[e - 1] : 0u), threadIdx.x % LANES);
  }
}

template <class T, bool SWIGLU, int LANES, int PIECES> int launch_quantize(const QuantizeDev &a, hipStream_t s) {
  constexpr uint32_t kAtOnce = 256 / LANES;
  if (a.rows.layout == PPLX_A2A_ROWS_PADDED) {
    const uint64_t groups = ((uint64_t)a.rows.rows * a.rows.experts + kAtOnce - 1) / kAtOnce;
    const uint32_t grid = groups < 2048 ? (uint32_t)groups : 2048;  // eight workgroups to a compute unit
    PPLX_LAUNCH(launch_kernel(quantize_padded<T, SWIGLU, LANES, PIECES>, dim3(grid), dim3(256), 4 * a.rows.experts, s, a));
  } else {
    // Bound by its bytes: 49152 activated rows of 1408 (277 MB read, 69 MB written) take 62.6 us, 5.5 TB/s, 8192 of 14336 102.6, 5.7
    // TB/s, and 32768 plain ones of 7168 120, 5.9 TB/s.  (Pieces of sixteen elements instead of eight leave lanes idle, and
    // arithmetic then binds the activated ones: 74.7 us, 4.6 TB/s.)
    // Rows that would fill the last-level cache are read past it, unless they are read twice, so that the result is in it for
    // whoever reads it next.  us with a read of the result behind it, plain / so: 49152 rows of 1408 231.9 / 226.2; 16384 of 2048
    // (134 MB) with their product 95.4 / 97.7.  Storing the result past the cache is faster alone and slower with its reader
    // (253.5).
    const bool large = (uint64_t)a.rows.rows * a.width * sizeof(T) * (SWIGLU ? 2 : 1) > kStreamBytes && a.width <= 8 * PIECES * LANES;
    auto kernel = large ? quantize_flat<T, SWIGLU, LANES, PIECES, true> : quantize_flat<T, SWIGLU, LANES, PIECES, false>;
    PPLX_LAUNCH(launch_groups(kernel, kernel, (a.rows.rows + kAtOnce - 1) / kAtOnce, 256, 0, s, a));
  }
  return PPLX_A2A_OK;
}

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

extern "C" int pplx_a2a_quantize_rows(int device, const pplx_a2a_quantize_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_quantize_args_t &p = *args;
  QuantizeDev a{};
  const int st = check_rows(p.rows, &a.rows);
  if (st) return st;
  PPLX_REQUIRE(is_dtype(p.dtype), "unsupported dtype of x");
  PPLX_REQUIRE(p.width > 0 && p.width < (1ull << 27) && p.width % 16 == 0, "width must be a multiple of 16 below 2^27");
  if (p.rows.rows == 0) return PPLX_A2A_OK;
  PPLX_REQUIRE(p.out && p.out_scale && p.x, "out / out_scale / x is NULL");
  PPLX_REQUIRE(is_aligned(p.out, 16) && p.out_stride_row % 16 == 0 && p.out_stride_expert % 16 == 0,
               "out must be 16-byte aligned with 16-byte strides");
  PPLX_REQUIRE(is_aligned(p.x, 16) && p.x_stride_row % 16 == 0 && p.x_stride_expert % 16 == 0,
               "x must be 16-byte aligned with 16-byte strides");
  PPLX_REQUIRE(is_aligned(p.out_scale, 4), "out_scale must be aligned to its elements");
  a.out = static_cast<uint8_t *>(p.out);
  a.out_stride_row = p.out_stride_row;
  a.out_stride_expert = p.out_stride_expert;
  a.scale = p.out_scale;
  a.scale_stride_row = p.out_scale_stride_row;
  a.scale_stride_expert = p.out_scale_stride_expert;
  a.x = static_cast<const uint8_t *>(p.x);
  a.x_stride_row = p.x_stride_row;
  a.x_stride_expert = p.x_stride_expert;
  a.width = (uint32_t)p.width;
  return guarded(device, [&] {
    return with_type(p.dtype, [&](auto tag) {
      typedef typename decltype(tag)::type T;
      hipStream_t s = (hipStream_t)stream;
      // A wave to a row, whose largest value needs no barrier, where four pieces a thread hold the row; us, 64 threads / 256:
      // 32768 plain rows of 512 11.2 / 29.3, of 2048 37.2 / 44.0, activated 54.4 / 63.1; with eight pieces in one wave rows of 4096
      // 115 / 111, 2000 of them 11.7 / 9.2.  Eight pieces a thread hold rows of up to 16384.
      if (a.width <= 2048) return p.swiglu ? launch_quantize<T, true, 64, 4>(a, s) : launch_quantize<T, false, 64, 4>(a, s);
      if (a.width <= 8192) return p.swiglu ? launch_quantize<T, true, 256, 4>(a, s) : launch_quantize<T, false, 256, 4>(a, s);
      return p.swiglu ? launch_quantize<T, true, 256, 8>(a, s) : launch_quantize<T, false, 256, 8>(a, s);
    });
  });
}
