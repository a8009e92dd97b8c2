// Sorted rows back to tokens, weighted, and the gradients of that.  The gradient of the sort itself is the gather without
// weights.  Both go by token: a token's picks are gathered (or written) by the lanes that hold its row, so nothing is
// added by atomics and every sum has one order.
#include "a2a_experts.h"

namespace pplx_amd {
namespace {

constexpr uint64_t kStreamRowsBytes = 96ull << 20, kStreamGradientBytes = 56ull << 20;

struct UnsortDev {
  void *out;
  int64_t out_stride;  // bytes
  const uint8_t *y;
  int64_t y_stride;    // bytes
  uint32_t y_rows;
  const int32_t *slots;
  const float *weights;
  uint32_t m, K, width;
  uint32_t first_group;
};

// Where the eight elements of a lane lie in a piece of 512: together where they are 16 bytes, in two halves of the piece where
// they are 32, so that each load of the wave takes whole lines.
template <class Y> __device__ __forceinline__ void lane_columns(uint32_t lane, uint32_t *at) {
  at[0] = sizeof(Y) == 4 ? lane * 4 : lane * 8;
  at[1] = sizeof(Y) == 4 ? 256 + lane * 4 : lane * 8 + 4;
}
template <class Y, bool NT>
__device__ __forceinline__ typename Eight<Y>::raw load_columns(const PPLX_GLOBAL Y *row, const uint32_t *at) {
  if constexpr (sizeof(Y) == 4) {
    const f32x4 a = load_vector<NT>(reinterpret_cast<const PPLX_GLOBAL f32x4 *>(row + at[0]));
    const f32x4 b = load_vector<NT>(reinterpret_cast<const PPLX_GLOBAL f32x4 *>(row + at[1]));
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  } else {
    return load_vector<NT>(reinterpret_cast<const PPLX_GLOBAL typename Eight<Y>::raw *>(row + at[0]));
  }
}

// Adds N rows of the token to acc, in the order of `left`'s bits, which it takes away.
template <class Y, int N, bool NT>
__device__ __forceinline__ void gather_some(const UnsortDev &a, int32_t slot, float w, uint64_t &left, const uint32_t *from,
                                            f32x8 &acc) {
  typename Eight<Y>::raw raw[N];
  float weight[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = __builtin_ctzll(left);
    left &= left - 1;
    const uint32_t s = (uint32_t)__builtin_amdgcn_readlane(slot, k);
    weight[i] = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(w), k));
    raw[i] = load_columns<Y, NT>(as_global(reinterpret_cast<const Y *>(a.y + (int64_t)s * a.y_stride)), from);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const f32x8 v = Eight<Y>::wide(raw[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = __builtin_fmaf(weight[i], v[j], acc[j]);
  }
}

// One wave to 512 elements of a token's row, eight to a lane, and up to eight rows in flight.
template <class Y, class O, bool NT>
__global__ __launch_bounds__(256) void unsort_gather(UnsortDev a, uint32_t pieces, FastDiv by_pieces) {
  const uint32_t lane = lane_id();
  const uint32_t wave = __builtin_amdgcn_readfirstlane((a.first_group + blockIdx.x) * 4 + threadIdx.x / kWave);
  const uint32_t t = fast_div(wave, by_pieces);
  if (t >= a.m) return;
  const uint32_t piece = (wave - t * pieces) * 512;
  uint32_t at[2], from[2];
  lane_columns<Y>(lane, at);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    at[h] += piece;
    from[h] = at[h] < a.width ? at[h] : a.width - 8 + 4 * h;  // (loads stay unconditional)
  }
  int32_t slot = -1;
  float w = 1.f;
  if (lane < a.K) {
    slot = as_global(a.slots)[(size_t)t * a.K + lane];
    if (a.weights) w = as_global(a.weights)[(size_t)t * a.K + lane];
  }
  uint64_t left = __ballot((uint32_t)slot < a.y_rows);
  f32x8 acc = {0, 0, 0, 0, 0, 0, 0, 0};
  uint32_t n = __builtin_popcountll(left);
  for (; n >= 8; n -= 8) gather_some<Y, 8, NT>(a, slot, w, left, from, acc);
  if (n & 4) gather_some<Y, 4, NT>(a, slot, w, left, from, acc);
  if (n & 2) gather_some<Y, 2, NT>(a, slot, w, left, from, acc);
  if (n & 1) gather_some<Y, 1, NT>(a, slot, w, left, from, acc);
  PPLX_GLOBAL O *out = as_global(reinterpret_cast<O *>(static_cast<uint8_t *>(a.out) + (int64_t)t * a.out_stride));
  if constexpr (sizeof(Y) == 4) {
    typedef O four __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 v = {acc[4 * h], acc[4 * h + 1], acc[4 * h + 2], acc[4 * h + 3]};
      if (at[h] < a.width) {
        PPLX_GLOBAL four *p = reinterpret_cast<PPLX_GLOBAL four *>(out + at[h]);
        __builtin_nontemporal_store(__builtin_convertvector(v, four), p);
      }
    }
  } else if (at[0] < a.width) {
    stream_eight<O>(out + at[0], acc);
  }
}

struct UnsortBackwardDev {
  uint8_t *grad_y;
  int64_t grad_y_stride;
  float *grad_weights;
  const uint8_t *grad_out;
  int64_t grad_out_stride;
  const uint8_t *y;
  int64_t y_stride;
  uint32_t y_rows;
  const int32_t *slots;
  const int32_t *num_rows;
  const float *weights;
  uint32_t m, K, width;
  uint32_t first_group;
  uint32_t sweeps, sweep_rows;  // workgroups in front of the tokens', rows of grad_y that one looks at
};

// Rows of grad_y that no slot names are zeros.  Those from *num_rows on are shared out over the tokens.  In front of it every
// row is named by the slots of a whole sort, but not by those of some of its tokens, or with picks taken out: workgroups in
// front of the tokens' count the slots that name a row, and where these are fewer than the rows go through them once more, for
// sweep_rows rows each, mark in LDS what is named and clear the rest.  They write what nobody else writes, so they run beside
// the others.
constexpr uint32_t kMaxSweepRows = 16384;
template <uint32_t AT_ONCE, class Fn> __device__ __forceinline__ void for_slots(const UnsortBackwardDev &a, Fn &&fn) {
  typedef uint32_t four __attribute__((ext_vector_type(4), aligned(4)));
  const PPLX_GLOBAL four *slots = as_global(reinterpret_cast<const four *>(a.slots));
  const uint32_t picks = a.m * a.K, fours = picks / 4;
  uint32_t base = threadIdx.x;
  for (; base + 256 * (AT_ONCE - 1) < fours; base += 256 * AT_ONCE) {
    four s[AT_ONCE];
#pragma unroll
    for (uint32_t u = 0; u < AT_ONCE; ++u) s[u] = slots[base + u * 256];
#pragma unroll
    for (uint32_t u = 0; u < AT_ONCE; ++u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) fn(s[u][i]);
    }
  }
  for (; base < fours; base += 256) {
    const four s = slots[base];
#pragma unroll
    for (int i = 0; i < 4; ++i) fn(s[i]);
  }
  if (threadIdx.x < picks % 4) fn((uint32_t)as_global(a.slots)[4 * fours + threadIdx.x]);
}

template <class T> __device__ void clear_unnamed(const UnsortBackwardDev &a, uint32_t total, uint32_t *named) {
  const uint32_t rows = total < a.y_rows ? total : a.y_rows;
  const uint32_t first = (a.first_group + blockIdx.x) * a.sweep_rows;
  if (first >= rows) return;
  const uint32_t count = rows - first < a.sweep_rows ? rows - first : a.sweep_rows;
  uint32_t own = 0;
  for_slots<16>(a, [&](uint32_t slot) { own += slot < rows ? 1u : 0u; });
#pragma unroll
  for (int d = 32; d; d >>= 1) own += (uint32_t)__shfl_xor((int)own, d);
  if (lane_id() == 0) named[wave_id()] = own;
  __syncthreads();
  if (named[0] + named[1] + named[2] + named[3] >= rows) return;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < (count + 31) / 32; i += 256) named[i] = 0;
  __syncthreads();
  for_slots<8>(a, [&](uint32_t slot) {
    const uint32_t r = slot - first;
    if (r < count) atomicOr(&named[r / 32], 1u << (r % 32));
  });
  __syncthreads();
  for (uint32_t r = wave_id(); r < count; r += 4) {
    if ((named[r / 32] >> (r % 32)) & 1) continue;
    PPLX_GLOBAL T *row = as_global(reinterpret_cast<T *>(a.grad_y + (int64_t)(first + r) * a.grad_y_stride));
    for (uint32_t col = lane_id() * 8; col < a.width; col += 64 * 8) store_eight<T>(row + col, f32x8{0, 0, 0, 0, 0, 0, 0, 0});
  }
}

// All rows of grad_y, in front of the gradient.
template <class T> __global__ __launch_bounds__(256) void clear_rows(UnsortBackwardDev a) {
  const uint32_t pieces = a.width / 8;
  const uint64_t all = (uint64_t)a.y_rows * pieces, step = (uint64_t)gridDim.x * 256;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
    const uint64_t r = i / pieces;
    PPLX_GLOBAL T *row = as_global(reinterpret_cast<T *>(a.grad_y + (int64_t)r * a.grad_y_stride));
    store_eight<T>(row + (i - r * pieces) * 8, f32x8{0, 0, 0, 0, 0, 0, 0, 0});
  }
}

// LANES threads to a token (a wave, or the workgroup).  Eight picks at a time: their rows of y are read, their rows of
// grad_y written, and the eight products summed over the row at the end.
template <class T, class G, int LANES, bool NT>
__global__ __launch_bounds__(256) void unsort_backward(UnsortBackwardDev a) {
  constexpr int kPicks = 8;
  const uint32_t lane = lane_id(), wave = wave_id(), g = threadIdx.x % LANES;
  __shared__ uint32_t named[kMaxSweepRows / 32];
  if (a.first_group + blockIdx.x < a.sweeps) {
    const int32_t live_rows = *as_global(a.num_rows);
    clear_unnamed<T>(a, live_rows > 0 ? (uint32_t)live_rows : 0u, named);
    return;
  }
  const uint32_t group = a.first_group + blockIdx.x - a.sweeps;
  const uint32_t t = LANES == 64 ? group * 4 + wave : group;
  if (t >= a.m) return;  // (with 256 lanes to a token the grid has one workgroup a token)
  int32_t slot = -1;
  float w = 1.f;
  if (lane < a.K) {
    slot = as_global(a.slots)[(size_t)t * a.K + lane];
    if (a.weights) w = as_global(a.weights)[(size_t)t * a.K + lane];
  }
  const uint64_t live = __ballot((uint32_t)slot < a.y_rows);
  const PPLX_GLOBAL G *go_row = as_global(reinterpret_cast<const G *>(a.grad_out + (int64_t)t * a.grad_out_stride));
  const bool want_y = a.grad_y != nullptr, want_w = a.grad_weights != nullptr;
  __shared__ float partial[LANES / 64][kPicks];
  for (uint32_t first = 0; first < a.K; first += kPicks) {
    float acc[kPicks] = {};
    for (uint32_t col = g * 8; col < a.width; col += LANES * 8) {
      typename Eight<T>::raw raw[kPicks];
      if (want_w) {
#pragma unroll
        for (int i = 0; i < kPicks; ++i) {
          const uint32_t k = first + i;
          if (k < a.K && (live >> k) & 1) {
            const uint32_t s = (uint32_t)__builtin_amdgcn_readlane(slot, k);
            raw[i] = load_eight<T, NT>(as_global(reinterpret_cast<const T *>(a.y + (int64_t)s * a.y_stride)) + col);
          }
        }
      }
      const f32x8 go = Eight<G>::wide(load_eight<G>(go_row + col));
#pragma unroll
      for (int i = 0; i < kPicks; ++i) {
        const uint32_t k = first + i;
        if (!(k < a.K && (live >> k) & 1)) continue;
        if (want_w) {
          const f32x8 v = Eight<T>::wide(raw[i]);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[i] = __builtin_fmaf(go[j], v[j], acc[i]);
        }
        if (want_y) {
          const float weight = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(w), k));
          const uint32_t s = (uint32_t)__builtin_amdgcn_readlane(slot, k);
          stream_eight<T>(as_global(reinterpret_cast<T *>(a.grad_y + (int64_t)s * a.grad_y_stride)) + col, go * weight);
        }
      }
    }
    if (want_w) {
#pragma unroll
      for (int i = 0; i < kPicks; ++i) acc[i] = wave_sum(acc[i]);
      if constexpr (LANES > 64) {
        __syncthreads();  // (the picks before have been read)
#pragma unroll
        for (int i = 0; i < kPicks; ++i) {
          if (lane == 0) partial[wave][i] = acc[i];
        }
        __syncthreads();
        if (threadIdx.x < kPicks && first + threadIdx.x < a.K) {
          float sum = 0.f;
#pragma unroll
          for (int v = 0; v < LANES / 64; ++v) sum += partial[v][threadIdx.x];
          const uint32_t k = first + threadIdx.x;
          as_global(a.grad_weights)[(size_t)t * a.K + k] = (live >> k) & 1 ? sum : 0.f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPicks; ++i) {
          if (lane == (uint32_t)i && first + i < a.K) {
            as_global(a.grad_weights)[(size_t)t * a.K + first + i] = (live >> (first + i)) & 1 ? acc[i] : 0.f;
          }
        }
      }
    }
  }
  if (!want_y) return;
  // The rows behind the last live one.
  const int32_t there = *as_global(a.num_rows);
  const uint32_t total = there > 0 ? (uint32_t)there : 0u;
  const uint64_t stride = (uint64_t)a.m * a.K;
  for (uint32_t k = 0; k < a.K; ++k) {
    for (uint64_t r = (uint64_t)t * a.K + k; r < a.y_rows; r += stride) {
      if (r < total) continue;
      PPLX_GLOBAL T *row = as_global(reinterpret_cast<T *>(a.grad_y + (int64_t)r * a.grad_y_stride));
      for (uint32_t col = g * 8; col < a.width; col += LANES * 8) store_eight<T>(row + col, f32x8{0, 0, 0, 0, 0, 0, 0, 0});
    }
  }
}

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

namespace {
int check_unsort_size(uint64_t m, uint64_t K, uint64_t hidden_dim, int64_t y_rows) {
  PPLX_REQUIRE(K >= 1 && K <= 64, "experts_per_token must be in [1, 64]");
  PPLX_REQUIRE(hidden_dim > 0 && hidden_dim < (1ull << 28) && hidden_dim % 8 == 0,
               "hidden_dim must be a multiple of 8 below 2^28");
  PPLX_REQUIRE(y_rows >= 0 && y_rows < (1ll << 31), "y must have fewer than 2^31 rows");
  if (m * K >= (1ull << 31) || m * ((hidden_dim + 511) / 512) >= (1ull << 31))
    return refuse(PPLX_A2A_UNSUPPORTED, "too many picks or elements");
  return PPLX_A2A_OK;
}

// Rows of grad_y to each of the workgroups that look for rows without a name, 0 for all rows cleared in front.  128 of them
// or more each go through all slots, which grows with the square of the picks.  us, as if all rows had names / so / cleared:
// 4096 x 8 rows of 64 bytes 9.2 / 8.9 / 11.9, 8192 x 8 of 128 13.3 / 13.9 / 16.7, of 4096 101 / 102 / 141; 131072 x 8 of 128
// 146 / 163 / 166, of 512 202 / 223 / 293, of 4096 1785 / 1755 / 2709; 1000000 x 8 of 256 1202 / 1733 / 1614.
uint32_t rows_to_sweep(uint32_t y_rows, uint64_t picks, uint64_t row_bytes) {
  uint32_t rows = (y_rows + 127) / 128;
  rows = rows < 256 ? 256 : rows > kMaxSweepRows ? kMaxSweepRows : rows;
  const uint64_t sweeps = (y_rows + rows - 1) / rows;
  return picks <= 1 << 18 || sweeps <= 2 * row_bytes ? rows : 0;
}
}  // namespace

extern "C" int pplx_a2a_unsort_tokens(int device, const pplx_a2a_unsort_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_unsort_args_t &p = *args;
  const int st = check_unsort_size(p.m, p.experts_per_token, p.hidden_dim, p.y_rows);
  if (st) return st;
  PPLX_REQUIRE(is_dtype(p.y_dtype) && is_dtype(p.out_dtype), "unsupported dtype of y or out");
  if (p.m == 0) return PPLX_A2A_OK;
  PPLX_REQUIRE(p.out && p.slots && (p.y || p.y_rows == 0), "out / slots / y is NULL");
  PPLX_REQUIRE(is_aligned(p.out, 16) && p.out_stride_row % 16 == 0, "out must be 16-byte aligned with a 16-byte row stride");
  PPLX_REQUIRE(is_aligned(p.y, 16) && p.y_stride_row % 16 == 0, "y must be 16-byte aligned with a 16-byte row stride");
  PPLX_REQUIRE(is_aligned(p.slots, 4) && is_aligned(p.weights, 4), "slots and weights must be aligned to their elements");
  UnsortDev a{};
  a.out = p.out;
  a.out_stride = p.out_stride_row;
  a.y = static_cast<const uint8_t *>(p.y);
  a.y_stride = p.y_stride_row;
  a.y_rows = (uint32_t)p.y_rows;
  a.slots = p.slots;
  a.weights = p.weights;
  a.m = p.m;
  a.K = p.experts_per_token;
  a.width = (uint32_t)p.hidden_dim;
  const uint32_t pieces = (a.width + 511) / 512;
  const uint64_t groups = ((uint64_t)a.m * pieces + 3) / 4;
  return guarded(device, [&] {
    return with_type(p.y_dtype, [&](auto y) {
      return with_type(p.out_dtype, [&](auto out) {
        typedef typename decltype(y)::type Y;
        typedef typename decltype(out)::type O;
        // Results go past the caches, and rows that are more than the last-level cache's share come past them.  us, plain /
        // stores / loads and stores non-temporal: 8192 x 2 rows of 4096 bf16 (134 MB) 39.4 / 36.6 / 33.0, 8192 x 8 of 7168
        // 204 / 189 / 176, 3001 x 5 of 2880 fp32 (173 MB) 38.9 / 35.4 / 31.5; 4096 x 3 of 2880 (71 MB) 17.9 / 15.4 / 16.6,
        // 8192 of 4096 (67 MB) 26.7 / 20.6 / 23.0, 1024 x 2 of 7168 8.6 / 8.2 / 8.9.  Large ones run at 6.0 TB/s.
        const uint64_t bytes = (uint64_t)a.m * a.K * a.width * sizeof(Y);
        auto kernel = bytes > kStreamRowsBytes ? unsort_gather<Y, O, true> : unsort_gather<Y, O, false>;
        PPLX_LAUNCH(launch_groups(kernel, kernel, groups, 256, 0, (hipStream_t)stream, a, pieces, make_fast_div(pieces)));
        return (int)PPLX_A2A_OK;
      });
    });
  });
}

extern "C" int pplx_a2a_unsort_tokens_backward(int device, const pplx_a2a_unsort_backward_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_unsort_backward_args_t &p = *args;
  const int st = check_unsort_size(p.m, p.experts_per_token, p.hidden_dim, p.y_rows);
  if (st) return st;
  PPLX_REQUIRE(is_dtype(p.dtype) && is_dtype(p.grad_dtype), "unsupported dtype of y or grad_out");
  if (!p.grad_y && !p.grad_weights) return PPLX_A2A_OK;
  PPLX_REQUIRE(p.m > 0 || !p.grad_y || p.y_rows == 0, "without tokens there is no gradient of rows");
  if (p.m == 0) return PPLX_A2A_OK;
  PPLX_REQUIRE(p.grad_out && p.slots, "grad_out / slots is NULL");
  PPLX_REQUIRE(!p.grad_y || (p.num_rows && is_aligned(p.num_rows, 4)), "num_rows is NULL or not aligned");
  PPLX_REQUIRE(!p.grad_weights || p.y || p.y_rows == 0, "y is NULL, which grad_weights needs");
  PPLX_REQUIRE(is_aligned(p.grad_out, 16) && p.grad_out_stride_row % 16 == 0 && is_aligned(p.grad_y, 16) &&
                   p.grad_y_stride_row % 16 == 0 && is_aligned(p.y, 16) && p.y_stride_row % 16 == 0,
               "grad_out, grad_y and y must be 16-byte aligned with 16-byte row strides");
  PPLX_REQUIRE(is_aligned(p.slots, 4) && is_aligned(p.weights, 4) && is_aligned(p.grad_weights, 4),
               "slots, weights and grad_weights must be aligned to their elements");
  UnsortBackwardDev a{};
  a.grad_y = static_cast<uint8_t *>(p.grad_y);
  a.grad_y_stride = p.grad_y_stride_row;
  a.grad_weights = p.grad_weights;
  a.grad_out = static_cast<const uint8_t *>(p.grad_out);
  a.grad_out_stride = p.grad_out_stride_row;
  a.y = static_cast<const uint8_t *>(p.y);
  a.y_stride = p.y_stride_row;
  a.y_rows = (uint32_t)p.y_rows;
  a.slots = p.slots;
  a.num_rows = p.num_rows;
  a.weights = p.weights;
  a.m = p.m;
  a.K = p.experts_per_token;
  a.width = (uint32_t)p.hidden_dim;
  return guarded(device, [&] {
    return with_type(p.dtype, [&](auto y) {
      return with_type(p.grad_dtype, [&](auto grad) {
        typedef typename decltype(y)::type Y;
        typedef typename decltype(grad)::type G;
        // us, plain / stores / loads and stores non-temporal: 8192 x 2 rows of 4096 bf16 (134 MB) 71.7 / 68.3 / 56.5, 8192 x 8 of
        // 2048 (268 MB) 112 / 109 / 100, 16384 x 2 of 1024 (67 MB) 36.3 / 31.4 / 30.2; 2048 x 6 of 2048 (50 MB) 24.6 / 19.6 /
        // 23.0, 1024 x 2 of 7168 (29 MB) 13.8 / 13.9 / 15.1.
        const bool large = (uint64_t)a.m * a.K * a.width * sizeof(Y) > kStreamGradientBytes;
        if (a.grad_y && a.y_rows > 0) {
          if (const uint32_t rows = rows_to_sweep(a.y_rows, (uint64_t)a.m * a.K, a.width * sizeof(Y))) {
            a.sweep_rows = rows;
            a.sweeps = (a.y_rows + rows - 1) / rows;
          } else {
            const uint64_t groups = ((uint64_t)a.y_rows * (a.width / 8) + 255) / 256;
            PPLX_LAUNCH(launch_kernel(clear_rows<Y>, dim3(groups < 4096 ? (uint32_t)groups : 4096), dim3(256), 0, (hipStream_t)stream, a));
          }
        }
        auto launch = [&](auto lanes) {
          constexpr int L = decltype(lanes)::value;
          auto kernel = large ? unsort_backward<Y, G, L, true> : unsort_backward<Y, G, L, false>;
          const uint64_t groups = (uint64_t)a.sweeps + (L == 64 ? (a.m + 3) / 4 : a.m);
          PPLX_LAUNCH(launch_groups(kernel, kernel, groups, 256, 0, (hipStream_t)stream, a));
          return (int)PPLX_A2A_OK;
        };
        return a.width <= 1024 ? launch(std::integral_constant<int, 64>{}) : launch(std::integral_constant<int, 256>{});
      });
    });
  });
}
