// Rows times their experts' weights in 8-bit integers.
//
//   out[r, n] = x_scale[r] * weight_scale[e, n] * sum over k of x[r, k] * weight[e, n, k]
//
// on the matrix cores (v_mfma_i32_*_i8), whose int32 sums are exact for every k that the entry point admits.  The weights
// are the first operand, so that the accumulators of a lane are consecutive columns of one row of the result.
//
// Tiles of BM rows by BN columns go through LDS, 128 bytes of k at a time, which loads write there directly.  A row of a
// tile is a line of eight 16-byte chunks; chunk c of row r lies at place c ^ (r & 7) of its line, so that the lanes of a
// fragment, which read one chunk each of consecutive rows, read all banks.  How many rows each expert has is known on the
// device only: every workgroup sums the experts' blocks of rows and takes tiles from the list that follows from them.
#include "a2a_experts.h"

namespace pplx_amd {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct MatmulDev {
  RowsDev rows;
  uint8_t *out;
  int64_t out_stride_row, out_stride_expert;  // elements
  const int8_t *x;
  int64_t x_stride_row, x_stride_expert;
  const float *x_scale;
  int64_t x_scale_stride_row, x_scale_stride_expert;
  const int8_t *weight;
  const float *weight_scale;
  uint32_t n, k;
  uint32_t n_blocks;
  uint32_t vector_stores;  // out rows are aligned to four elements
};

constexpr uint32_t kStepBytes = 128;

// Waits until at most `left` of the wave's loads and stores are under way.
template <int LEFT> __device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((LEFT & 15) | ((LEFT >> 4) << 14) | (7 << 4) | (15 << 8));
  asm volatile("" ::: "memory");
}

// Sixteen bytes a lane from global memory to LDS, lane i's at `lds` + 16 i.
__device__ __forceinline__ void load_to_lds(const PPLX_GLOBAL int8_t *p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}

__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}

// Four consecutive columns of a row of the result, of which `n` exist.
template <class O>
__device__ __forceinline__ void store_four(PPLX_GLOBAL O *p, f32x4 v, uint32_t n, bool whole) {
  if (whole && n >= 4) {
    typedef O four __attribute__((ext_vector_type(4)));
    *reinterpret_cast<PPLX_GLOBAL four *>(p) = __builtin_convertvector(v, four);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      if (i < n) p[i] = (O)v[i];
    }
  }
}

// Inclusive sums of the experts' blocks of BM rows in `upto`, by all THREADS threads of the workgroup.
template <int THREADS, int BM> __device__ __forceinline__ void sum_blocks(const RowsDev &rows, uint32_t *upto, uint32_t *of_wave) {
  const uint32_t E = rows.experts, per = (E + THREADS - 1) / THREADS, first = threadIdx.x * per;
  uint32_t own = 0;
  for (uint32_t i = 0; i < per; ++i) own += first + i < E ? (span_of(rows, first + i).count + BM - 1) / BM : 0u;
  uint32_t sum = wave_scan(own, lane_id());
  if (lane_id() == 63) of_wave[wave_id()] = sum;
  __syncthreads();
  sum -= own;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) sum += (uint32_t)w < wave_id() ? of_wave[w] : 0u;
  for (uint32_t i = 0; i < per; ++i) {
    if (first + i < E) upto[first + i] = sum += (span_of(rows, first + i).count + BM - 1) / BM;
  }
  __syncthreads();
}

struct Tile {
  uint32_t e, m0, n0, begin, count;
};
// Tile number `id` of the list: by expert, then by groups of kGroup blocks of rows, in a group by columns.  Workgroups
// that run at the same time on one XCD take consecutive ones, about kGroup by eight of them, whose operands its L2 serves.
constexpr uint32_t kGroup = 4;
template <int BM, int BN> __device__ __forceinline__ Tile tile_of(const MatmulDev &a, const uint32_t *upto, uint32_t id) {
  uint32_t lo = 0, hi = a.rows.experts - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (upto[mid] * a.n_blocks > id) hi = mid;
    else lo = mid + 1;
  }
  Tile t;
  t.e = __builtin_amdgcn_readfirstlane(lo);
  const uint32_t before = t.e ? upto[t.e - 1] : 0u;
  const uint32_t blocks = upto[t.e] - before;
  const uint32_t local = id - before * a.n_blocks;
  const uint32_t group = local / (kGroup * a.n_blocks);
  const uint32_t in_group = local - group * kGroup * a.n_blocks;
  const uint32_t size = blocks - group * kGroup < kGroup ? blocks - group * kGroup : kGroup;
  const uint32_t nb = in_group / size;
  const Span s = span_of(a.rows, t.e);
  t.m0 = __builtin_amdgcn_readfirstlane((group * kGroup + in_group - nb * size) * BM);
  t.n0 = __builtin_amdgcn_readfirstlane(nb * BN);
  t.begin = __builtin_amdgcn_readfirstlane(s.begin);
  t.count = __builtin_amdgcn_readfirstlane(s.count);
  return t;
}

// The fragments of one matrix instruction: 32 rows and 32 bytes of k, or 16 rows and 64 bytes of k, 16 bytes to a lane.
template <int F> struct Mfma;
template <> struct Mfma<32> {
  typedef i32x16 acc;
  static constexpr int kChunks = 2;
  static __device__ __forceinline__ acc run(i32x4 a, i32x4 b, acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
  }
};
template <> struct Mfma<16> {
  typedef i32x4 acc;
  static constexpr int kChunks = 4;
  static __device__ __forceinline__ acc run(i32x4 a, i32x4 b, acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};

// WM by WN waves, each BM / WM rows by BN / WN columns in fragments of F; STAGES steps of k in LDS.
template <int BM, int BN, int WM, int WN, int F, int STAGES, class O>
__global__ __launch_bounds__(WM *WN * 64) void matmul_tiles(MatmulDev a) {
  constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
  constexpr int MF = BM / WM / F, NF = BN / WN / F;  // fragments of a wave
  constexpr int kLoads = (BM + BN) / 8 / kWaves;     // of a wave in a step, eight rows each
  static_assert((BM + BN) % (8 * kWaves) == 0 && BM % (WM * F) == 0 && BN % (WN * F) == 0, "tile");
  constexpr int kStage = (BM + BN) * (int)kStepBytes;
  extern __shared__ __align__(128) uint8_t lds[];  // [STAGES][BM rows of x, BN of the weight][128], then the sums
  uint32_t *upto = reinterpret_cast<uint32_t *>(lds + STAGES * kStage);
  __shared__ uint32_t of_wave[kWaves];
  sum_blocks<kThreads, BM>(a.rows, upto, of_wave);
  const uint32_t tiles = __builtin_amdgcn_readfirstlane(upto[a.rows.experts - 1] * a.n_blocks);
  const uint32_t lane = lane_id(), wave = wave_id();
  const uint32_t wm = wave % WM, wn = wave / WM;
  const uint32_t lds0 = lds_address(lds);
  const uint32_t steps = (a.k + kStepBytes - 1) / kStepBytes;
  const uint32_t chunk = ((lane & 7) ^ (lane >> 3)) * 16;  // of its line that this lane fetches
  // Places of the fragments' chunks in their lines (rows of a fragment differ by 8 or more in what the lanes share).
  const uint32_t frag_row = (lane % F) * kStepBytes, frag_chunk = lane / F;

  // (blockIdx goes round the eight XCDs)
  const uint32_t block = (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
  for (uint32_t id = block; id < tiles; id += gridDim.x) {
    const Tile t = tile_of<BM, BN>(a, upto, id);
    if (t.m0 >= t.count) continue;  // (offsets that descend make a list that is too long)
    const int8_t *x = a.x + (int64_t)t.e * a.x_stride_expert + (int64_t)t.begin * a.x_stride_row;
    const int8_t *weight = a.weight + (uint64_t)t.e * a.n * a.k;
    const PPLX_GLOBAL int8_t *from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t row = (i * kWaves + wave) * 8 + (lane >> 3);  // of the stage
      if ((i * kWaves + wave) * 8 < BM) {
        const uint32_t r = t.m0 + row;
        from[i] = as_global(x + (int64_t)(r < t.count ? r : t.count - 1) * a.x_stride_row);
      } else {
        const uint32_t r = t.n0 + row - BM;
        from[i] = as_global(weight + (uint64_t)(r < a.n ? r : a.n - 1) * a.k);
      }
    }
    auto fetch = [&](uint32_t step, uint32_t stage) __attribute__((always_inline)) {
      const uint32_t k = step * kStepBytes + chunk;
      const uint32_t at = k < a.k ? k : 0;  // (bytes behind k are taken for zeros when they are used)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        load_to_lds(from[i] + at, __builtin_amdgcn_readfirstlane(lds0 + stage * kStage + (i * kWaves + wave) * 1024));
      }
    };

    typename Mfma<F>::acc acc[NF][MF] = {};
    // The tile before has been read; its stores are done, so that what is counted below are loads.
    wait_loads<0>();
    __syncthreads();
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      if ((uint32_t)s < steps) fetch(s, s);
    }
    uint32_t stage = 0;
    for (uint32_t step = 0; step < steps; ++step) {
      if (step + STAGES - 1 <= steps) wait_loads<(STAGES - 2) * kLoads>();
      else wait_loads<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (step + STAGES - 1 < steps) fetch(step + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
      const uint8_t *rows_x = lds + stage * kStage + wm * (BM / WM) * kStepBytes + frag_row;
      const uint8_t *rows_w = lds + stage * kStage + (BM + wn * (BN / WN)) * kStepBytes + frag_row;
      const uint32_t left = a.k - step * kStepBytes;
      constexpr int kChunks = Mfma<F>::kChunks;
#pragma unroll
      for (int kk = 0; kk < 8 / kChunks; ++kk) {
        const uint32_t c = kk * kChunks + frag_chunk;
        const uint32_t place = (c ^ (lane & 7)) * 16;
        i32x4 fx[MF], fw[NF];
#pragma unroll
        for (int i = 0; i < MF; ++i) fx[i] = *reinterpret_cast<const i32x4 *>(rows_x + i * F * kStepBytes + place);
#pragma unroll
        for (int i = 0; i < NF; ++i) fw[i] = *reinterpret_cast<const i32x4 *>(rows_w + i * F * kStepBytes + place);
        if (left < kStepBytes) {
          const bool there = c * 16 < left;
#pragma unroll
          for (int i = 0; i < MF; ++i) fx[i] = there ? fx[i] : i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < NF; ++j) {
#pragma unroll
          for (int i = 0; i < MF; ++i) acc[j][i] = Mfma<F>::run(fw[j], fx[i], acc[j][i]);
        }
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }

    // Lane l holds row l % F of each fragment and, in its accumulators, columns 4 (l / F) .. + 3 of every 256 / F.
    constexpr uint32_t kSpan = 256 / F;
    const float *ws = a.weight_scale + (uint64_t)t.e * a.n;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const uint32_t r = t.m0 + wm * (BM / WM) + i * F + lane % F;
      if (r >= t.count) continue;
      const float xs = as_global(a.x_scale)[(int64_t)t.e * a.x_scale_stride_expert + (int64_t)(t.begin + r) * a.x_scale_stride_row];
      PPLX_GLOBAL O *out = as_global(reinterpret_cast<O *>(a.out)) + (int64_t)t.e * a.out_stride_expert +
                           (int64_t)(t.begin + r) * a.out_stride_row;
#pragma unroll
      for (int j = 0; j < NF; ++j) {
#pragma unroll
        for (int q = 0; q < F * F / 256; ++q) {
          const uint32_t n = t.n0 + wn * (BN / WN) + j * F + q * kSpan + 4 * (lane / F);
          if (n >= a.n) continue;
          const uint32_t exist = a.n - n;
          f32x4 v;
#pragma unroll
          for (uint32_t u = 0; u < 4; ++u) {
            v[u] = (float)acc[j][i][4 * q + u] * (xs * as_global(ws)[n + (u < exist ? u : 0)]);
          }
          store_four<O>(out + n, v, exist, a.vector_stores);
        }
      }
    }
  }
}

constexpr uint32_t kComputeUnits = 256;

template <int BM, int BN, int WM, int WN, int F, int STAGES, class O>
int launch_tiles(const MatmulDev &from, uint64_t most_blocks, hipStream_t s) {
  MatmulDev a = from;
  constexpr uint32_t kTileLds = STAGES * (BM + BN) * kStepBytes;
  const uint32_t lds = kTileLds + 4 * a.rows.experts;
  constexpr uint32_t kPerUnit = kTileLds <= 64 * 1024 ? 2 : 1;
  a.n_blocks = (a.n + BN - 1) / BN;
  const uint64_t tiles = most_blocks * a.n_blocks;
  if (tiles >= (1ull << 31)) return refuse(PPLX_A2A_UNSUPPORTED, "too many tiles");
  uint64_t grid = kPerUnit * kComputeUnits;
  grid = tiles < grid ? (tiles + 7) / 8 * 8 : grid;  // (whole rounds of the XCDs)
  auto kernel = matmul_tiles<BM, BN, WM, WN, F, STAGES, O>;
  if (lds > 64 * 1024) {
    const hipError_t err =
        hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (err != hipSuccess) (void)hipGetLastError();  // (the launch says so if it matters)
  }
  PPLX_LAUNCH(launch_kernel(kernel, dim3((uint32_t)grid), dim3(WM * WN * 64), lds, s, a));
  return PPLX_A2A_OK;
}

template <class O> int launch_matmul(const MatmulDev &a, hipStream_t s) {
  const uint64_t E = a.rows.experts;
  const uint64_t all = a.rows.layout == PPLX_A2A_ROWS_PADDED ? E * a.rows.rows : a.rows.rows;
  auto most_blocks = [&](uint64_t bm) {  // that the rows of all experts can make
    if (a.rows.layout == PPLX_A2A_ROWS_PADDED) return E * ((a.rows.rows + bm - 1) / bm);
    return (all + bm - 1) / bm + (E < all ? E : all) - 1;
  };
  const uint64_t even = all / E;
  if (even <= 24) return launch_tiles<32, 128, 1, 4, 32, 3, O>(a, most_blocks(32), s);
  if (even <= 128) return launch_tiles<64, 128, 1, 4, 32, 3, O>(a, most_blocks(64), s);
  return launch_tiles<256, 256, 2, 4, 32, 2, O>(a, most_blocks(256), s);
}

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

extern "C" int pplx_a2a_int8_matmul(int device, const pplx_a2a_int8_matmul_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_int8_matmul_args_t &p = *args;
  MatmulDev a{};
  const int st = check_rows(p.rows, &a.rows);
  if (st) return st;
  PPLX_REQUIRE(is_dtype(p.out_dtype), "unsupported dtype of out");
  PPLX_REQUIRE(p.n < (1ull << 31), "n must be below 2^31");
  PPLX_REQUIRE(p.k > 0 && p.k % 16 == 0 && p.k <= 131056, "k must be a multiple of 16 in [16, 131056]");
  if (p.rows.rows == 0 || p.n == 0) return PPLX_A2A_OK;
  PPLX_REQUIRE(p.out && p.x && p.x_scale && p.weight && p.weight_scale, "out / x / x_scale / weight / weight_scale is NULL");
  PPLX_REQUIRE(is_aligned(p.x, 16) && p.x_stride_row % 16 == 0 && p.x_stride_expert % 16 == 0,
               "x must be 16-byte aligned with 16-byte strides");
  PPLX_REQUIRE(is_aligned(p.weight, 16), "weight must be 16-byte aligned");
  PPLX_REQUIRE(is_aligned(p.out, dtype_bytes(p.out_dtype)) && is_aligned(p.x_scale, 4) && is_aligned(p.weight_scale, 4),
               "out, x_scale and weight_scale must be aligned to their elements");
  a.out = static_cast<uint8_t *>(p.out);
  a.out_stride_row = p.out_stride_row;
  a.out_stride_expert = p.out_stride_expert;
  a.x = p.x;
  a.x_stride_row = p.x_stride_row;
  a.x_stride_expert = p.x_stride_expert;
  a.x_scale = p.x_scale;
  a.x_scale_stride_row = p.x_scale_stride_row;
  a.x_scale_stride_expert = p.x_scale_stride_expert;
  a.weight = p.weight;
  a.weight_scale = p.weight_scale;
  a.n = (uint32_t)p.n;
  a.k = (uint32_t)p.k;
  a.vector_stores = is_aligned(p.out, 4 * dtype_bytes(p.out_dtype)) && p.out_stride_row % 4 == 0 && p.out_stride_expert % 4 == 0;
  return guarded(device, [&] {
    return with_type(p.out_dtype, [&](auto tag) { return launch_matmul<typename decltype(tag)::type>(a, (hipStream_t)stream); });
  });
}
