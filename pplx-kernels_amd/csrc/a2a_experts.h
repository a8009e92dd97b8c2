// What the kernels between dispatch and combine share: element types, reductions over the lanes of a row, quantisation,
// and where the rows of the experts lie.  Included only by the .hip sources.
#pragma once
#include <cstdarg>
#include <cstdio>
#include <new>

#include "a2a_common.h"
#include "a2a_device_scope.h"
#include "a2a_host.h"
#include "pplx_a2a.h"

namespace pplx_amd {
namespace {

// ---------------------------------------------------------------------------
// Host side: failures of the C entry points
// ---------------------------------------------------------------------------
inline int refuse(int status, const char *fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return report_failure(status, buf);
}
#define PPLX_REQUIRE(cond, ...)                                                     \
  do {                                                                              \
    if (!(cond)) return refuse(PPLX_A2A_INVALID_ARGUMENT, __VA_ARGS__);             \
  } while (0)
#define PPLX_LAUNCH(expr)                                                           \
  do {                                                                              \
    const int err_ = (expr);                                                        \
    if (err_ != 0)                                                                  \
      return refuse(PPLX_A2A_HIP_ERROR, "%s failed: %s", __func__, hipGetErrorString((hipError_t)err_)); \
  } while (0)

inline bool is_aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool is_dtype(int32_t t) { return t == PPLX_A2A_F32 || t == PPLX_A2A_BF16 || t == PPLX_A2A_F16; }
inline int64_t dtype_bytes(int32_t t) { return t == PPLX_A2A_F32 ? 4 : 2; }
constexpr uint32_t kMaxExperts = 5461;  // as in a world: three tables of an expert's words fit 64 KiB of LDS

template <class T> struct TypeTag { typedef T type; };
// Calls fn with the tag of the element type; dtype has been checked.
template <class Fn> int with_type(int32_t dtype, Fn &&fn) {
  switch (dtype) {
    case PPLX_A2A_BF16: return fn(TypeTag<__bf16>{});
    case PPLX_A2A_F16: return fn(TypeTag<_Float16>{});
    default: return fn(TypeTag<float>{});
  }
}

// A grid of any number of workgroups: a launch takes fewer than 2^32 threads along a dimension, so that more go out in several,
// whose first argument's first_group is the number of the first one.  Those behind the first launch may be of another
// kernel.
template <typename A, typename... P, typename... R>
int launch_groups(void (*kernel)(A, P...), void (*later)(A, P...), uint64_t groups, uint32_t threads, uint32_t lds, hipStream_t s,
                  A a, const R &...rest) {
  const uint64_t most = 0xffffffffu / threads;
  for (uint64_t first = 0; first < groups; first += most) {
    a.first_group = (uint32_t)first;
    const uint64_t left = groups - first;
    const int err =
        launch_kernel(first ? later : kernel, dim3((uint32_t)(left < most ? left : most)), dim3(threads), lds, s, a, rest...);
    if (err) return err;
  }
  return 0;
}

// ---------------------------------------------------------------------------
// Eight consecutive elements as fp32 and back (rounded to nearest, ties to even)
// ---------------------------------------------------------------------------
template <class T> struct Eight;
template <> struct Eight<__bf16> {
  typedef bf16x8 raw;
  static __device__ __forceinline__ f32x8 wide(raw v) { return __builtin_convertvector(v, f32x8); }
  static __device__ __forceinline__ raw narrow(f32x8 v) { return __builtin_convertvector(v, bf16x8); }
};
template <> struct Eight<_Float16> {
  typedef f16x8 raw;
  static __device__ __forceinline__ f32x8 wide(raw v) { return __builtin_convertvector(v, f32x8); }
  static __device__ __forceinline__ raw narrow(f32x8 v) { return __builtin_convertvector(v, f16x8); }
};
template <> struct Eight<float> {
  typedef f32x8 raw;
  static __device__ __forceinline__ f32x8 wide(raw v) { return v; }
  static __device__ __forceinline__ raw narrow(f32x8 v) { return v; }
};
// NT: past the caches.
template <bool NT, class V> __device__ __forceinline__ V load_vector(const PPLX_GLOBAL V *p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}
template <class T, bool NT = false> __device__ __forceinline__ typename Eight<T>::raw load_eight(const PPLX_GLOBAL T *p) {
  if constexpr (sizeof(T) == 4) {
    // (two 16-byte loads: rows are 16-byte aligned, not 32)
    const PPLX_GLOBAL f32x4 *q = reinterpret_cast<const PPLX_GLOBAL f32x4 *>(p);
    const f32x4 a = load_vector<NT>(q), b = load_vector<NT>(q + 1);
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  } else {
    return load_vector<NT>(reinterpret_cast<const PPLX_GLOBAL typename Eight<T>::raw *>(p));
  }
}
template <class T> __device__ __forceinline__ void store_eight(PPLX_GLOBAL T *p, f32x8 v) {
  if constexpr (sizeof(T) == 4) {
    PPLX_GLOBAL f32x4 *q = reinterpret_cast<PPLX_GLOBAL f32x4 *>(p);
    q[0] = f32x4{v[0], v[1], v[2], v[3]};
    q[1] = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    *reinterpret_cast<PPLX_GLOBAL typename Eight<T>::raw *>(p) = Eight<T>::narrow(v);
  }
}

// The same past the caches.
template <class T> __device__ __forceinline__ void stream_eight(PPLX_GLOBAL T *p, f32x8 v) {
  if constexpr (sizeof(T) == 4) {
    PPLX_GLOBAL f32x4 *q = reinterpret_cast<PPLX_GLOBAL f32x4 *>(p);
    __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, q);
    __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, q + 1);
  } else {
    __builtin_nontemporal_store(Eight<T>::narrow(v), reinterpret_cast<PPLX_GLOBAL typename Eight<T>::raw *>(p));
  }
}

// ---------------------------------------------------------------------------
// Lanes
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, d);
    v = v > o ? v : o;
  }
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)v, d);
    v += lane >= (uint32_t)d ? o : 0u;
  }
  return v;
}

// ---------------------------------------------------------------------------
// Quantisation of a row: q = rint(x * (127 / a)), scale = a / 127, a = max(max |x|, 2^-100).  The largest value is found
// on the bits of the magnitudes, where an infinity and a NaN come out on top: such a row becomes zeros with a scale of
// NaN, so that everything made from it is NaN.  2^-100 keeps 127 / a finite; the only rows that it changes are those whose
// values are all below 1e-30.  |q| <= 127: a * (127 / a) is at most 127 (1 + 2^-23), which rounds to 127.
// ---------------------------------------------------------------------------
constexpr uint32_t kTinyBits = (127u - 100u) << 23;  // 2^-100
struct RowScale {
  float inverse, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t max_bits) {
  RowScale s;
  if (max_bits >= 0x7f800000u) {
    s.inverse = 0.f;
    s.scale = __uint_as_float(0x7fc00000u);
  } else {
    const float a = __uint_as_float(max_bits > kTinyBits ? max_bits : kTinyBits);
    s.inverse = 127.f / a;
    s.scale = a / 127.f;
  }
  return s;
}
__device__ __forceinline__ uint32_t magnitude_bits(f32x8 v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    m = m > b ? m : b;
  }
  return m;
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Eight values as bytes.  1.5 * 2^23 + p is p rounded to an integer, ties to even, whose low byte is the low byte of the sum's
// bits: |p| <= 127.  (A row with an infinity or a NaN has inverse 0 and becomes zeros, whatever its products are.)
__device__ __forceinline__ u32x2 quantize_eight(f32x8 v, float inverse) {
#pragma clang fp contract(off)
  uint32_t bits[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float p = v[i] * inverse;  // (rounded, as the oracle's product is)
    bits[i] = __float_as_uint(p + 12582912.f);
  }
  const uint32_t keep = inverse != 0.f ? 0xffffffffu : 0u;
  uint32_t q[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t *b = bits + 4 * i;
    // (a selector's bytes 0-3 are of the second operand, 4-7 of the first)
    const uint32_t low = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), high = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0c);
    q[i] = (low | high) & keep;
  }
  return u32x2{q[0], q[1]};
}
__device__ __forceinline__ u32x4 quantize_sixteen(f32x8 a, f32x8 b, float inverse) {
  const u32x2 lo = quantize_eight(a, inverse), hi = quantize_eight(b, inverse);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// The largest of the magnitudes that the LANES threads of a row found (64, or the 256 of a workgroup, which all call).
template <int LANES> __device__ __forceinline__ uint32_t row_max(uint32_t bits) {
  bits = wave_max(bits);
  if constexpr (LANES > 64) {
    __shared__ uint32_t of_wave[LANES / 64];
    __syncthreads();  // (the row before has been read)
    if (lane_id() == 0) of_wave[wave_id()] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) bits = bits > of_wave[w] ? bits : of_wave[w];
  }
  return bits;
}

// ---------------------------------------------------------------------------
// Where the experts' rows lie
// ---------------------------------------------------------------------------
struct RowsDev {
  const int32_t *starts_or_counts;
  uint32_t rows;
  uint32_t experts;
  int32_t layout;
};
// Rows [begin, begin + count) of expert e, from its buffer's first (PADDED) or from the first of all.
struct Span {
  uint32_t begin, count;
};
__device__ __forceinline__ Span span_of(const RowsDev &r, uint32_t e) {
  if (r.layout == PPLX_A2A_ROWS_DENSE) return Span{0, r.rows};
  const PPLX_GLOBAL int32_t *p = as_global(r.starts_or_counts);
  auto clamped = [&](int32_t v) { return v < 0 ? 0u : (uint32_t)v < r.rows ? (uint32_t)v : r.rows; };
  if (r.layout == PPLX_A2A_ROWS_PADDED) return Span{0, clamped(p[e])};
  const uint32_t a = clamped(p[e]), b = clamped(p[e + 1]);
  return Span{a, b > a ? b - a : 0};
}

inline int check_row_numbers(const pplx_a2a_rows_t &r, RowsDev *out) {
  PPLX_REQUIRE(r.layout == PPLX_A2A_ROWS_DENSE || r.layout == PPLX_A2A_ROWS_SORTED || r.layout == PPLX_A2A_ROWS_PADDED,
               "unknown layout of rows");
  PPLX_REQUIRE(r.num_experts >= 1 && r.num_experts <= kMaxExperts, "num_experts must be in [1, %u]", kMaxExperts);
  PPLX_REQUIRE(r.layout != PPLX_A2A_ROWS_DENSE || r.num_experts == 1, "rows without offsets or counts have one expert");
  const uint64_t per = r.layout == PPLX_A2A_ROWS_PADDED ? r.num_experts : 1;
  if (r.rows >= (1ull << 31) / per) return refuse(PPLX_A2A_UNSUPPORTED, "2^31 rows or more");
  out->rows = (uint32_t)r.rows;
  out->experts = r.num_experts;
  out->layout = r.layout;
  return PPLX_A2A_OK;
}
inline int check_rows(const pplx_a2a_rows_t &r, RowsDev *out) {
  const int st = check_row_numbers(r, out);
  if (st) return st;
  PPLX_REQUIRE(r.layout == PPLX_A2A_ROWS_DENSE || (r.starts_or_counts && is_aligned(r.starts_or_counts, 4)),
               "starts_or_counts is NULL or not aligned");
  out->starts_or_counts = r.starts_or_counts;
  return PPLX_A2A_OK;
}

// C++ exceptions end at the C entry points (the launches allocate nothing; the runtime might).
template <class Fn> int guarded(int device, Fn &&fn) {
  try {
    DeviceScope scope(device);
    if (!scope.ok()) {
      (void)hipGetLastError();
      return refuse(PPLX_A2A_HIP_ERROR, "cannot select HIP device %d", device);
    }
    return fn();
  } catch (const std::exception &e) {
    return refuse(PPLX_A2A_HIP_ERROR, "%s", e.what());
  } catch (...) {
    return refuse(PPLX_A2A_HIP_ERROR, "unknown failure");
  }
}

}  // namespace
}  // namespace pplx_amd
