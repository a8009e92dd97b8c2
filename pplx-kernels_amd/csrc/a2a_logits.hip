// The router's product and its gradients, on the matrix cores with fp32 sums.
//
//   logits = x weight^T        grad_x = grad_logits weight        grad_weight = grad_logits^T x
//
// All three are sums over k of a[i, k] * b[j, k] of operands whose rows lie along k; for the gradients operands are laid out so
// first.  The matrix cores take 16-bit elements.  What has more bits is a sum of bf16 pieces, each the part of a value
// that the pieces before leave: two hold an fp16 value, three an fp32 one.  Of the products of pieces those below 2^-24 of the
// largest are left out.
#include <cmath>

#include "a2a_experts.h"
#include "a2a_tiles.h"

namespace pplx_amd {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

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

// N pieces of eight values, each rounded to nearest; two fp32 words to a pair of bf16 and back take one instruction each way.
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <int N> __device__ __forceinline__ void cut(f32x8 v, bf16x8 *p) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int n = 0; n < N; ++n) {
    words w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, bf16x2));
      if (n + 1 == N) continue;
      v[2 * i] -= __uint_as_float(w[i] << 16);
      v[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
    }
    p[n] = __builtin_bit_cast(bf16x8, w);
  }
}
// Pieces that hold a value in full.
template <class T> struct Pieces {
  static constexpr int count = std::is_same_v<T, __bf16> ? 1 : std::is_same_v<T, _Float16> ? 2 : 3;
  static __device__ __forceinline__ void of(typename Eight<T>::raw v, bf16x8 *p) {
    if constexpr (std::is_same_v<T, __bf16>) p[0] = v;
    else cut<count>(Eight<T>::wide(v), p);
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

// A workgroup to 16 rows by 16 columns, whose eight waves share out k, 32 elements at a time, and add their sums in LDS, in the order of
// the waves.  Operands go straight to registers.
constexpr int kProductWaves = 8;
template <class TA, class TB> __global__ __launch_bounds__(kProductWaves * 64) void product_split(ProductDev a) {
  constexpr int kAhead = 2;
  __shared__ float sums[kProductWaves][4 * 64];
  const uint32_t lane = lane_id(), wave = wave_id(), group = a.first_group + blockIdx.x;
  const uint32_t block = group / a.column_blocks, m = block * 16 + lane % 16, n0 = (group - block * a.column_blocks) * 16;
  const uint32_t r = m < a.rows ? m : a.rows - 1, c = n0 + lane % 16 < a.columns ? n0 + lane % 16 : a.columns - 1;
  const PPLX_GLOBAL TA *row = as_global(reinterpret_cast<const TA *>(a.a + (int64_t)r * a.a_stride));
  const PPLX_GLOBAL TB *column = as_global(reinterpret_cast<const TB *>(a.b + (int64_t)c * a.b_stride));
  const uint32_t units = (a.k + 31) / 32, own = lane / 16 * 8;
  struct Unit {
    typename Eight<TA>::raw a;
    typename Eight<TB>::raw b;
  };
  Unit u[kAhead];
  // (units behind the last are loads of the first elements, which are taken for zeros: a branch would wait for all loads)
  auto load = [&](Unit &to, uint32_t unit) __attribute__((always_inline)) {
    const uint32_t k = unit * 32 + own, at = k < a.k ? k : 0;
    to.b = load_eight<TB>(column + at);
    to.a = load_eight<TA>(row + at);
  };
  f32x4 acc = {};
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(u[i], wave + i * kProductWaves);
  for (uint32_t first = wave; first < units; first += kAhead * kProductWaves) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const uint32_t unit = first + i * kProductWaves;
      const bool there = unit * 32 + own < a.k;
      Operand<TA, TB> fa;
      Operand<TB, TA> fb;
      fa.set(there ? u[i].a : typename Eight<TA>::raw{});
      fb.set(there ? u[i].b : typename Eight<TB>::raw{});
      acc = multiply_add(fb, fa, acc);
      load(u[i], unit + kAhead * kProductWaves);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sums[wave][i * 64 + lane] = acc[i];
  __syncthreads();
  // Lane l has columns 4 (l / 16) .. + 3 of row l % 16.
  if (wave || m >= a.rows) return;
  PPLX_GLOBAL float *out = as_global(reinterpret_cast<float *>(a.out)) + (int64_t)m * a.out_stride;
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kProductWaves; ++w) sum += sums[w][i * 64 + lane];
    const uint32_t n = n0 + 4 * (lane / 16) + i;
    if (n < a.columns) out[n] = sum;
  }
}

// ---------------------------------------------------------------------------
// Tiles of BM rows by BN columns through LDS, which loads write directly
// ---------------------------------------------------------------------------
struct TilesDev {
  const int8_t *a, *b;
  int64_t a_stride, b_stride;  // bytes
  float *out;
  int64_t out_stride;  // elements
  uint64_t out_split;  // elements from one split's sums to the next's
  uint32_t rows, columns, k;
  uint32_t row_blocks, column_blocks, splits, steps_per_split;
};

__device__ __forceinline__ f32x16 multiply_32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 multiply_32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Lines of 64 elements of a row: of 128 bytes, or 256.  Chunk c of line r lies at c ^ exchange(r): sixteen consecutive lines hold a
// chunk at sixteen places of 256 bytes, which is what LDS reads at a time.
template <class T> struct Lines {
  static constexpr uint32_t kBytes = 64 * sizeof(T), kChunks = kBytes / 16, kPerLoad = 64 / kChunks;
  static __device__ __forceinline__ uint32_t exchange(uint32_t line) { return kChunks == 8 ? (line >> 1) & 7 : line & 15; }
};

// WM by WN waves, each BM / WM rows by BN / WN columns in fragments of 32 by 32; STAGES steps of 64 elements of k in LDS.  A wave
// reads the fragments of the next sixteen k before it multiplies those at hand, over the border between two steps too: there it
// waits for the next step's loads, and behind the barrier this step's place takes those of a step to come.  What is cut into pieces
// is cut between LDS and the matrix cores.  TAIL: k is no multiple of 64.
template <class TA, class TB, int BM, int BN, int WM, int WN, int STAGES, bool TAIL>
__global__ __launch_bounds__(WM *WN * 64) void logits_tiles(TilesDev a) {
  typedef Lines<TA> LA;
  typedef Lines<TB> LB;
  constexpr int kWaves = WM * WN;
  constexpr int kRows = BM / WM, kColumns = BN / WN, MF = kRows / 32, NF = kColumns / 32;
  constexpr int kLoadsA = BM / (int)LA::kPerLoad / kWaves, kLoadsB = BN / (int)LB::kPerLoad / kWaves, kLoads = kLoadsA + kLoadsB;
  static_assert(kLoadsA * LA::kPerLoad * kWaves == BM && kLoadsB * LB::kPerLoad * kWaves == BN, "whole loads");
  static_assert(MF >= 1 && NF >= 1 && kRows % 32 == 0 && kColumns % 32 == 0, "whole fragments");
  static_assert((STAGES - 1) * kLoads < 63, "loads that can be counted");
  constexpr uint32_t kPlaceB = BM * LA::kBytes, kStage = kPlaceB + BN * LB::kBytes;
  static_assert(STAGES * kStage <= kLdsBytes, "loads to LDS stay in front of kLdsBytes");
  extern __shared__ __align__(128) uint8_t lds[];  // [STAGES][BM lines of the rows, BN of the columns]
  const uint32_t lane = lane_id(), wave = wave_id();
  const uint32_t wm = wave % WM, wn = wave / WM;
  // (blockIdx goes round the eight XCDs: one of them takes tiles of one split, whose part of the columns' operand its L2 holds, and all
  // tiles of a block of rows)
  const uint32_t id = (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
  const uint32_t block = id / a.column_blocks, split = block / a.row_blocks;
  if (split >= a.splits) return;
  const uint32_t m0 = __builtin_amdgcn_readfirstlane((block - split * a.row_blocks) * BM);
  const uint32_t n0 = __builtin_amdgcn_readfirstlane((id - block * a.column_blocks) * BN);
  const uint32_t all_steps = (a.k + 63) / 64;
  const uint32_t begin = __builtin_amdgcn_readfirstlane(split * a.steps_per_split);
  const uint32_t end = begin + a.steps_per_split < all_steps ? begin + a.steps_per_split : all_steps;
  const uint32_t lds0 = lds_address(lds);

  const int8_t *first_a = a.a + (int64_t)m0 * a.a_stride, *first_b = a.b + (int64_t)n0 * a.b_stride;
  const uint32_t rows_left = a.rows - m0, columns_left = a.columns - n0;
  uint32_t offset[kLoads], chunk[kLoads];  // (the chunks are the same for all loads of an operand, or alternate)
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const bool of_a = i < kLoadsA;
    const uint32_t chunks = of_a ? LA::kChunks : LB::kChunks, per_load = 64 / chunks;
    const uint32_t line = ((of_a ? i : i - kLoadsA) * kWaves + wave) * per_load + lane / chunks;
    chunk[i] = (lane % chunks) ^ (of_a ? LA::exchange(line) : LB::exchange(line));
    offset[i] = chunk[i] * 16 + (of_a ? (line < rows_left ? line : rows_left - 1) * (uint32_t)a.a_stride
                                      : (line < columns_left ? line : columns_left - 1) * (uint32_t)a.b_stride);
  }
  // Load number i of a step.  Behind k a lane fetches the first chunk of its line; what it brings is taken for zeros.  Loads of
  // steps that do not exist bring nothing, and count.
  auto fetch = [&](auto last, int i, uint32_t step, uint32_t stage) __attribute__((always_inline)) {
    const bool of_a = i < kLoadsA;
    const uint32_t bytes = of_a ? LA::kBytes : LB::kBytes, size = of_a ? sizeof(TA) : sizeof(TB);
    const int8_t *base = (of_a ? first_a : first_b) + (uint64_t)step * bytes;
    const bool behind = decltype(last)::value && step * 64 + chunk[i] * (16 / size) >= a.k;
    const uint32_t place = of_a ? i * kWaves + wave : (i - kLoadsA) * kWaves + wave;
    load_to_lds(base, behind ? offset[i] - chunk[i] * 16 : offset[i], lds0 + stage * kStage + (of_a ? 0 : kPlaceB) + place * 1024,
                step < end ? ~0u : 0u);
  };
  typename Eight<TA>::raw ra[2][MF];
  typename Eight<TB>::raw rb[2][NF];
  constexpr int kReads = MF + NF;
  auto read_line = [&](auto last, auto &to, auto lines, const uint8_t *line, int kk, uint32_t step) __attribute__((always_inline)) {
    typedef decltype(lines) L;
    u32x4 v[L::kChunks / 8];
#pragma unroll
    for (uint32_t h = 0; h < L::kChunks / 8; ++h) {
      const uint32_t c = (2 * kk + lane / 32) * (L::kChunks / 8) + h;
      v[h] = *reinterpret_cast<const u32x4 *>(line + (c ^ L::exchange(lane % 32)) * 16);
      if constexpr (decltype(last)::value) v[h] &= step * 64 + kk * 16 + lane / 32 * 8 < a.k ? ~0u : 0u;
    }
    __builtin_memcpy(&to, v, sizeof(v));
  };
  auto read = [&](auto last, int i, int to, int kk, uint32_t step, uint32_t stage) __attribute__((always_inline)) {
    const uint8_t *lines = lds + stage * kStage;
    if (i < MF) read_line(last, ra[to][i], LA{}, lines + (wm * kRows + i * 32 + lane % 32) * LA::kBytes, kk, step);
    else read_line(last, rb[to][i - MF], LB{}, lines + kPlaceB + (wn * kColumns + (i - MF) * 32 + lane % 32) * LB::kBytes, kk, step);
  };
  typedef std::bool_constant<TAIL> Tail;
  f32x16 acc[NF][MF] = {};
#pragma unroll
  for (int s = 0; s < STAGES; ++s) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) fetch(Tail{}, i, begin + s, s);
  }
  wait_loads<(STAGES - 1) * kLoads>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < kReads; ++i) read(Tail{}, i, 0, 0, begin, 0);
  typedef Operand<TA, TB> OA;
  typedef Operand<TB, TA> OB;
  constexpr int kMost = OA::count + OB::count - 2 < 2 ? OA::count + OB::count - 2 : 2;
  constexpr int kPairs = OA::count + OB::count < 4 || OA::count == 1 || OB::count == 1 ? OA::count * OB::count
                         : OA::count + OB::count == 6                                  ? 6
                                                                                       : 5;
  constexpr int kProducts = MF * NF * kPairs;
  // The products of sixteen k, between which the reads of the next sixteen and the loads of a step go out: a wave issues in order, and
  // one that hands over all its reads or loads at once waits for them to be taken.
  auto multiply = [&](int from, auto read_next, auto fetch_next) __attribute__((always_inline)) {
    OA fa[MF];
    OB fb[NF];
#pragma unroll
    for (int i = 0; i < MF; ++i) fa[i].set(ra[from][i]);
#pragma unroll
    for (int j = 0; j < NF; ++j) fb[j].set(rb[from][j]);
    int q = 0;
#pragma unroll
    for (int order = kMost; order >= 0; --order) {
#pragma unroll
      for (int pa = 0; pa < OA::count; ++pa) {
        const int pb = order - pa;
        if (pb < 0 || pb >= OB::count) continue;
#pragma unroll
        for (int j = 0; j < NF; ++j) {
#pragma unroll
          for (int i = 0; i < MF; ++i) {
            acc[j][i] = multiply_32(fb[j].p[pb], fa[i].p[pa], acc[j][i]);
#pragma unroll
            for (int r = q * kReads / kProducts; r < (q + 1) * kReads / kProducts; ++r) read_next(r);
#pragma unroll
            for (int l = q * kLoads / kProducts; l < (q + 1) * kLoads / kProducts; ++l) fetch_next(l);
            __builtin_amdgcn_sched_barrier(0);
            ++q;
          }
        }
      }
    }
  };
  uint32_t stage = 0, step = begin;
  auto take = [&](auto last_read, auto last_fetched) __attribute__((always_inline)) {
    const uint32_t next = stage + 1 == STAGES ? 0 : stage + 1;
#pragma unroll
    for (int kk = 0; kk < 3; ++kk) {
      multiply(kk % 2, [&](int r) { read(last_read, r, (kk + 1) % 2, kk + 1, step, stage); }, [](int) {});
    }
    // Loads under way are those of steps step + 1 .. step + STAGES - 1; this step's place is free behind the barrier.
    wait_loads<(STAGES - 2) * kLoads, true>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    multiply(1, [&](int r) { read(last_read, r, 0, 0, step + 1, next); }, [&](int l) { fetch(last_fetched, l, step + STAGES, stage); });
    stage = next;
    ++step;
  };
  // (what lies behind k is looked for in the last steps only)
  const uint32_t last = all_steps - 1;
  while (step < end && (!TAIL || step + STAGES < last)) take(std::false_type{}, std::false_type{});
  if constexpr (TAIL) {
    while (step < end && step + 1 < last) take(std::false_type{}, std::true_type{});
    while (step < end) take(std::true_type{}, std::true_type{});
  }
  wait_loads<0, true>();
  // Lane l holds row l % 32 of each fragment and columns 4 (l / 32) .. + 3 of every eight.
  typedef float four __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const uint32_t row = m0 + wm * kRows + i * 32 + lane % 32;
    if (row >= a.rows) continue;
    PPLX_GLOBAL float *out = as_global(a.out) + split * a.out_split + (int64_t)row * a.out_stride;
#pragma unroll
    for (int j = 0; j < NF; ++j) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t n = n0 + wn * kColumns + j * 32 + q * 8 + 4 * (lane / 32);
        if (n + 4 <= a.columns) {
          *reinterpret_cast<PPLX_GLOBAL four *>(out + n) = four{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
        } else {
#pragma unroll
          for (uint32_t u = 0; u < 3; ++u) {
            if (n + u < a.columns) out[n + u] = acc[j][i][4 * q + u];
          }
        }
      }
    }
  }
}

// The sums of the splits as results: eight threads to four columns, each with every eighth split, whose sums are added in order.
// Rows of the sums are `columns` long, a multiple of four, of which `width` are there.
struct SumDev {
  const float *sums;
  uint64_t split;  // elements
  uint8_t *out;
  int64_t out_stride;  // elements
  uint32_t rows, columns, width, splits;
  uint32_t first_group;
};
template <class O, int SHARES> __global__ __launch_bounds__(256) void sum_splits(SumDev a) {
  __shared__ f32x4 shares[SHARES > 1 ? 256 : 1];
  constexpr uint32_t kPer = 256 / SHARES;  // results of a workgroup
  const uint32_t per_row = a.columns / 4, share = threadIdx.x / kPer;
  const uint64_t i = (uint64_t)(a.first_group + blockIdx.x) * kPer + threadIdx.x % kPer;
  const uint32_t r = i >> 32 ? (uint32_t)(i / per_row) : (uint32_t)i / per_row, c = (uint32_t)(i - (uint64_t)r * per_row) * 4;
  f32x4 s = {};
  if (r < a.rows) {
    const PPLX_GLOBAL float *p = as_global(a.sums) + (uint64_t)r * a.columns + c;
#pragma unroll 4
    for (uint32_t k = share; k < a.splits; k += SHARES) s += *reinterpret_cast<const PPLX_GLOBAL f32x4 *>(p + k * a.split);
  }
  if constexpr (SHARES > 1) {
    shares[threadIdx.x] = s;
    __syncthreads();
    if (share) return;
#pragma unroll
    for (int k = 1; k < SHARES; ++k) s += shares[k * kPer + threadIdx.x];
  }
  if (r >= a.rows) return;
  PPLX_GLOBAL O *out = as_global(reinterpret_cast<O *>(a.out)) + (int64_t)r * a.out_stride + c;
  typedef O four __attribute__((ext_vector_type(4), aligned(sizeof(O))));
  if (c + 4 <= a.width) {
    *reinterpret_cast<PPLX_GLOBAL four *>(out) = four{(O)s[0], (O)s[1], (O)s[2], (O)s[3]};
  } else {
#pragma unroll
    for (uint32_t u = 0; u < 3; ++u) {
      if (c + u < a.width) out[u] = (O)s[u];
    }
  }
}
template <class O> int launch_sum(const SumDev &a, hipStream_t s) {
  const uint64_t results = (uint64_t)a.rows * (a.columns / 4);
  if (a.splits <= 8) return launch_groups(sum_splits<O, 1>, sum_splits<O, 1>, (results + 255) / 256, 256, 0, s, a);
  return launch_groups(sum_splits<O, 8>, sum_splits<O, 8>, (results + 31) / 32, 256, 0, s, a);
}

// ---------------------------------------------------------------------------
// Gradients: sums over k of a[i, k] * b[k, n], where the rows of b lie along n
// ---------------------------------------------------------------------------
// The matrix cores want eight consecutive k of a column in a lane.  A lane fetches NV consecutive columns of eight rows of b, and the
// vectors are turned in its registers: fragment f has the columns f, NV + f, 2 NV + f .. of a block of 32 NV, and the sums of a lane,
// one for each fragment, are consecutive columns again.  Fragments go to LDS, from where all waves of a workgroup take them.
// The other operand, grad_logits, is cut into pieces once, by split_gradient, and lies in the order in which lanes take them.  It has
// all three pieces whatever the results' type: two leave out up to 2^-17 of a value (and the products of second pieces 2^-16), which shows
// in a result of 16 bits where products cancel.  What the third one costs, us with all launches, two pieces and three:
//   both bf16       3001 x 7168 of 256  grad_x 34 / 44, grad_weight 38 / 48     8192 x 7168 of 256  78 / 103, 81 / 107
//                   8192 x 4096 of 8  17 / 18, 20 / 21
//   both fp16       3001 x 7168 of 256  45 / 61, 50 / 63     16384 x 4096 of 64  44 / 58, 59 / 75
//   bf16, fp32      3001 x 7168 of 256  44 / 76 (two pieces of the weight too, without the product of second pieces)
struct GradientDev {
  const uint8_t *a;  // [blocks of 32 rows][sixteens of k][pieces][64 lanes] of 16 bytes
  const uint8_t *b;
  int64_t b_stride;  // bytes
  uint8_t *out;
  int64_t out_stride;  // elements
  uint64_t out_split;  // elements
  uint32_t rows, columns, k;
  uint32_t column_blocks, parts;  // (parts: of the rows, or of k)
  uint32_t first_group;
};

template <class TB, int NV> struct Turned {
  typedef Pieces<TB> Cut;
  static constexpr int kPieces = Cut::count;
  static constexpr int kBytes = kPieces * NV * 1024;  // of sixteen k in LDS
  typedef TB vec __attribute__((ext_vector_type(NV)));
  vec row[8];

  // Columns `column` .. + NV of rows k .. k + 7.  What lies behind the last k is zeros.
  __device__ __forceinline__ void load(const GradientDev &a, uint32_t column, uint32_t k) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const uint32_t at = k + r < a.k ? k + r : a.k - 1;
      row[r] = *reinterpret_cast<const PPLX_GLOBAL vec *>(as_global(reinterpret_cast<const TB *>(a.b + (int64_t)at * a.b_stride)) + column);
    }
  }
  __device__ __forceinline__ void store(uint8_t *to, uint32_t left, uint32_t lane) const {  // (left: k that are there)
#pragma unroll
    for (int f = 0; f < NV; ++f) {
      typename Eight<TB>::raw v;
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = (uint32_t)r < left ? row[r][f] : (TB)0;
      bf16x8 p[kPieces];
      Cut::of(v, p);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) *reinterpret_cast<bf16x8 *>(to + ((i * NV + f) * 64 + lane) * 16) = p[i];
    }
  }
};

typedef const PPLX_GLOBAL bf16x8 *FragmentPtr;
constexpr int kPiecesOfGradient = 3;
struct Fragments {  // of 32 rows and sixteen k
  bf16x8 p[kPiecesOfGradient];
  // Number i of those at `from`, the first where there are not so many.
  __device__ __forceinline__ void load(FragmentPtr from, uint32_t i, uint32_t all) {
    from += (uint64_t)(i < all ? i : 0) * (64 * kPiecesOfGradient);
#pragma unroll
    for (int n = 0; n < kPiecesOfGradient; ++n) p[n] = from[n * 64];
  }
};
// Their products with the columns' fragments at `from`.
template <int PIECES, int NV>
__device__ __forceinline__ void multiply_turned(const Fragments &fa, const uint8_t *from, uint32_t lane, f32x16 *acc) {
#pragma unroll
  for (int pb = PIECES - 1; pb >= 0; --pb) {
    bf16x8 fb[NV];
#pragma unroll
    for (int f = 0; f < NV; ++f) fb[f] = *reinterpret_cast<const bf16x8 *>(from + ((pb * NV + f) * 64 + lane) * 16);
#pragma unroll
    for (int pa = kPiecesOfGradient - 1 - pb; pa >= 0; --pa) {
#pragma unroll
      for (int f = 0; f < NV; ++f) acc[f] = multiply_32(fa.p[pa], fb[f], acc[f]);
    }
  }
}

// Pieces of grad_logits [rows, columns] as fragments of its rows, and of its columns (either may be left out).
struct PiecesDev {
  const float *in;
  int64_t in_stride;  // elements
  uint32_t rows, columns;
  uint8_t *by_rows, *by_columns;
  uint32_t first_group;
};
// A workgroup to 32 rows by 32 columns, of which a wave each takes half a block of rows, and of columns.
__global__ __launch_bounds__(128) void split_gradient(PiecesDev a) {
  __shared__ float tile[32][33];
  const uint32_t lane = lane_id(), wave = wave_id();
  const uint32_t column_blocks = (a.columns + 31) / 32, group = a.first_group + blockIdx.x;
  const uint32_t block = group / column_blocks, column_block = group - block * column_blocks;
  const uint32_t r0 = block * 32, c0 = column_block * 32;
  const uint32_t y = threadIdx.x / 32, x = threadIdx.x % 32, c = c0 + x < a.columns ? c0 + x : a.columns - 1;
  float in[8];
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) {
    const uint32_t r = r0 + i * 4 + y;
    in[i] = as_global(a.in)[(int64_t)(r < a.rows ? r : a.rows - 1) * a.in_stride + c];
  }
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) tile[i * 4 + y][x] = r0 + i * 4 + y < a.rows && c0 + x < a.columns ? in[i] : 0.f;
  __syncthreads();
  auto write = [&](uint8_t *to, uint64_t fragment, auto at) {
    f32x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = at(lane % 32, wave * 16 + lane / 32 * 8 + i);
    bf16x8 p[kPiecesOfGradient];
    cut<kPiecesOfGradient>(v, p);
    PPLX_GLOBAL bf16x8 *out = as_global(reinterpret_cast<bf16x8 *>(to)) + fragment * (64 * kPiecesOfGradient) + lane;
#pragma unroll
    for (int i = 0; i < kPiecesOfGradient; ++i) out[i * 64] = p[i];
  };
  const uint32_t row_sixteens = (a.rows + 15) / 16, column_sixteens = (a.columns + 15) / 16;
  if (a.by_rows && column_block * 2 + wave < column_sixteens) {
    write(a.by_rows, (uint64_t)block * column_sixteens + column_block * 2 + wave,
          [&](uint32_t r, uint32_t k) { return tile[r][k]; });
  }
  if (a.by_columns && block * 2 + wave < row_sixteens) {
    write(a.by_columns, (uint64_t)column_block * row_sixteens + block * 2 + wave,
          [&](uint32_t c, uint32_t k) { return tile[k][c]; });
  }
}
uint64_t fragment_bytes(uint64_t rows, uint64_t k) { return (rows + 31) / 32 * ((k + 15) / 16) * (1024 * kPiecesOfGradient); }
int launch_split(const PiecesDev &a, hipStream_t s) {
  return launch_groups(split_gradient, split_gradient, ((uint64_t)a.rows + 31) / 32 * ((a.columns + 31) / 32), 128, 0, s, a);
}

// Lane l holds NV columns of rows 8 i + 4 (l / 32) .. + 3.
template <class O, int NV>
__device__ __forceinline__ void store_turned(const GradientDev &a, uint64_t first, uint32_t m0, uint32_t column, uint32_t lane, const f32x16 *acc) {
  typedef O vec __attribute__((ext_vector_type(NV)));
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const uint32_t r = m0 + q / 4 * 8 + 4 * (lane / 32) + q % 4;
    if (r >= a.rows) continue;
    vec v;
#pragma unroll
    for (int f = 0; f < NV; ++f) v[f] = (O)acc[f][q];
    *reinterpret_cast<PPLX_GLOBAL vec *>(as_global(reinterpret_cast<O *>(a.out)) + first + (int64_t)r * a.out_stride + column) = v;
  }
}

// Of x: a workgroup keeps the fragments of 32 NV columns of the weight in LDS, CHUNK k of them at a time, and its waves take 32 rows
// of grad_logits each, a round after the other.  3001 x 7168 of 256 in bf16: 38 us, 860 TFLOP/s with the three pieces of grad_logits.  With
// two of them 28, of which the products alone took 18, the stores 6 and the loads 2 to 4 (what another order of loads and stores,
// priorities of waves or fewer rows to a workgroup do not hide).
constexpr int kGradientWaves = 8;
template <class TB, class O, int NV>
__global__ __launch_bounds__(kGradientWaves * 64) void gradient_of_rows(GradientDev a, uint32_t chunk) {
  typedef Turned<TB, NV> B;
  extern __shared__ __align__(16) uint8_t lds[];  // [chunk / 16][pieces][NV][64 lanes]
  const uint32_t lane = lane_id(), wave = wave_id(), half = lane / 32 * 8;
  const uint32_t group = a.first_group + blockIdx.x;
  const uint32_t part = group / a.column_blocks, n0 = (group - part * a.column_blocks) * 32 * NV;
  const uint32_t column = n0 + lane % 32 * NV;
  const bool there = column < a.columns;
  const uint32_t rounds = (a.rows + 32 * kGradientWaves - 1) / (32 * kGradientWaves);
  const uint32_t chunks = (a.k + chunk - 1) / chunk;
  auto fill = [&](uint32_t first) {
    const uint32_t sixteens = ((a.k - first < chunk ? a.k - first : chunk) + 15) / 16;
    for (uint32_t i = wave; i < sixteens; i += kGradientWaves) {
      const uint32_t k = first + i * 16 + half;
      B b;
      b.load(a, there ? column : 0, k);
      b.store(lds + i * B::kBytes, k < a.k ? a.k - k : 0, lane);
    }
  };
  if (chunks == 1) {
    fill(0);
    __syncthreads();
  }
  const uint32_t all = (a.k + 15) / 16;
  for (uint32_t round = part; round < rounds; round += a.parts) {
    const uint32_t block = round * kGradientWaves + wave, m0 = block * 32;
    const FragmentPtr from = as_global(reinterpret_cast<const bf16x8 *>(a.a)) + (uint64_t)(m0 < a.rows ? block : 0) * all * (64 * kPiecesOfGradient) + lane;
    constexpr int kAhead = 4;  // fragments under way
    Fragments fa[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fa[i].load(from, i, all);
    f32x16 acc[NV] = {};
    for (uint32_t c = 0; c < chunks; ++c) {
      const uint32_t first = c * chunk / 16, count = all - first < chunk / 16 ? all - first : chunk / 16;
      if (chunks > 1) {
        __syncthreads();  // (the chunk before has been read)
        fill(c * chunk);
        __syncthreads();
      }
      if (m0 >= a.rows) continue;
      for (uint32_t i = 0; i < count; i += kAhead) {  // (a chunk that is not the last is a multiple of 16 kAhead)
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (i + u >= count) break;
          multiply_turned<B::kPieces, NV>(fa[u], lds + (i + u) * B::kBytes, lane, acc);
          fa[u].load(from, first + i + u + kAhead, all);
        }
      }
    }
    if (there) store_turned<O, NV>(a, 0, m0, column, lane, acc);
  }
}

// Of the weight: waves take 32 experts each, a workgroup all of a block of them, and go through the tokens sixteen for each wave at a
// time: every wave turns sixteen of x, and all multiply with what the others turned.  Parts of the tokens add up in sum_splits.
// 256 x 7168 of 3001 in bf16: 38 us, 860 TFLOP/s with the three pieces, and 6 for the sum of the parts.  Memory answers a wave in order: the
// fragments of a step are all under way before the rows of x that come after it (with two pieces four of eight 30.5 us, all 26.5).
template <class TB, class O, int NV, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void gradient_of_weight(GradientDev a, uint32_t tokens_per_part, uint32_t row_blocks) {
  typedef Turned<TB, NV> B;
  extern __shared__ __align__(16) uint8_t lds[];  // [2][waves][pieces][NV][64 lanes]
  const uint32_t lane = lane_id(), wave = wave_id(), half = lane / 32 * 8;
  const uint32_t group = a.first_group + blockIdx.x;
  const uint32_t block = group / a.column_blocks, n0 = (group - block * a.column_blocks) * 32 * NV;
  const uint32_t part = block / row_blocks, m0 = ((block - part * row_blocks) * WAVES + wave) * 32;
  const uint32_t column = n0 + lane % 32 * NV;
  const bool there = column < a.columns;
  const uint32_t begin = part * tokens_per_part, end = a.k - begin < tokens_per_part ? a.k : begin + tokens_per_part;
  constexpr uint32_t step = 16 * WAVES, size = WAVES * B::kBytes;
  const uint32_t all = (a.k + 15) / 16, first = begin / 16;
  const FragmentPtr from = as_global(reinterpret_cast<const bf16x8 *>(a.a)) + (uint64_t)(m0 < a.rows ? m0 / 32 : 0) * all * (64 * kPiecesOfGradient) + lane;
  auto left_at = [&](uint32_t k) { return k < end ? end - k : 0u; };
  B b;
  f32x16 acc[NV] = {};
  b.load(a, there ? column : 0, begin + wave * 16 + half);
  Fragments fa[WAVES];
#pragma unroll
  for (uint32_t i = 0; i < WAVES; ++i) fa[i].load(from, first + i, all);
  uint32_t buffer = 0, at = begin;
  auto take = [&](auto last, auto idle) __attribute__((always_inline)) {
    constexpr bool kLast = decltype(last)::value, kIdle = decltype(idle)::value;
    b.store(lds + buffer * size + wave * B::kBytes, left_at(at + wave * 16 + half), lane);
    __syncthreads();
    if constexpr (!kLast) b.load(a, there ? column : 0, at + step + wave * 16 + half);
#pragma unroll
    for (uint32_t u = 0; u < (kIdle ? 0 : WAVES); ++u) {
      const uint32_t now = at / 16 + u;
      if (!kLast || now < all) multiply_turned<B::kPieces, NV>(fa[u], lds + buffer * size + u * B::kBytes, lane, acc);
      if constexpr (!kLast) fa[u].load(from, now + WAVES, all);
    }
    buffer ^= 1;
    at += step;
  };
  // (waves without experts turn rows for the others, and leave the matrix cores to them)
  if (m0 < a.rows) {
    while (at + step < end) take(std::false_type{}, std::false_type{});
    take(std::true_type{}, std::false_type{});
  } else {
    while (at + step < end) take(std::false_type{}, std::true_type{});
    take(std::true_type{}, std::true_type{});
  }
  if (there && m0 < a.rows) store_turned<O, NV>(a, part * a.out_split, m0, column, lane, acc);
}

uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Kernels that take more than 64 KiB of LDS say so.
template <class K> void allow_lds(K *kernel, uint32_t bytes) {
  if (bytes <= 64 * 1024) return;
  const hipError_t err =
      hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (err != hipSuccess) (void)hipGetLastError();  // (the launch says so if it matters)
}

// ---------------------------------------------------------------------------
// Which form a product takes, and in how many splits of k
// ---------------------------------------------------------------------------
// What a product costs in microseconds: a start, `per_step` for every 64 k of a tile and every round of the compute units, and where k is
// split the sums' launch and bytes.  Measured with rows that come from HBM, forms 64 x 64 / 128 x 128 with their best splits, us:
//   both bf16       8192 x 256 x 7168  65 (1) / 47.8 (2)     3001 x 256 x 7168  32.9 (4) / 27.2 (4)   1024 x 256 x 7168  15.0 (4) / 17.2 (12)
//                   16384 x 64 x 4096  32.0 (1) / 37.5 (4)   256 x 256 x 7168  9.4 (16) / 11.9 (16)   64 x 256 x 7168   7.6 (28) / 9.0 (28)
//   bf16, fp32      8192 x 256 x 7168  199 (2) / 97.7 (2)    256 x 256 x 7168  14.1 (16) / 16.1 (28)   64 x 256 x 7168   9.9 (56) / 11.1 (56)
//   both fp32       4096 x 256 x 7168  144 (4) / 101 (4)     256 x 256 x 7168  17.2 (16) / 21.3 (38)   64 x 256 x 7168  10.9 (56) / 14.5 (56)
// and 128 x 192, for 16-bit operands, beside 128 x 128:
//   both bf16       16384 x 384 x 7168  91 (1) / 143 (1)     8192 x 384 x 7168  57.6 (2) / 72.2 (1)   4096 x 384 x 7168  36.2 (4) / 42.2 (2)   1024 x 384 x 7168  21.4 (14) / 19.7 (8)
//                   3001 x 384 x 7168  32.2 (4) / 32.8 (3)
// and 64 x 128, for 16-bit operands of few steps, beside 64 x 64 and 128 x 128:
//   both bf16       16384 x 128 x 2048  20.4 / 25.1 / 25.4   8192 x 256 x 2048  17.7 / 21.3 / 23.0   4096 x 300 x 2048  15.1 / 17.9 / 18.9
//                   16384 x 256 x 2048  35.8 / 41.8 / 28.2   2048 x 128 x 4096  14.0 / 12.0 / 16.4
// and 128 x 32, where operands are cut into pieces (what a wave cuts of the rows is not cut by a second one), beside 64 x 64:
//   bf16, fp32      16384 x 8 x 4096  38.4 (4) / 60.4 (1)    4096 x 32 x 2048  12.8 (8) / 13.6 (4)   64 x 8 x 4096  7.9 (32) / 8.7 (16)
//   both fp32       16384 x 8 x 4096  63.5 (2) / 89.0 (2)    4096 x 32 x 2048  14.4 (8) / 17.8 (4)   both bf16, 16384 x 8 x 4096  30.4 (4) / 29.1 (4)
// What bounds a tile of 128 x 128 is what a compute unit fetches into its LDS, 31 bytes a cycle: 0.43 us a step with rows in L2, and
// 0.63 with rows out of HBM.  (Not for their latency: with a wave of its own that reads them into L2 one to eight steps ahead,
// 16384 x 512 x 7168 takes 147 to 151 and not 145.)  Larger tiles fetch less and hold fewer steps: 128 x 256 and
// 256 x 128 take 1.1 us a step, 256 x 256 1.4.  Tiles of 64 x 192, 64 x 256, 32 x 64 and 32 x 128 were within 5 % of the best of
// these, or slower, in all of thirty products.
// product_split, which is one launch: 4 x 64 x 2048 4.3 (tiles 5.8), 1 x 256 x 7168 9.5 (6.5), 64 x 256 x 7168 14.2, with fp32
// weights 20.9: its loads take a cycle for each row of 64 bytes, whatever else is under way.
struct LogitsForm {
  uint32_t bm, bn;
  double start[4], per_step[4];  // 16-bit operands; bf16 and fp32; fp16 and fp32; fp32
};
constexpr double kNever = 1e9;
constexpr LogitsForm kForms[] = {{64, 64, {3.0, 4.7, 5.0, 5.4}, {0.25, 0.8, 1.0, 1.08}},
                                 {128, 128, {3.0, 6.0, 6.5, 7.0}, {0.66, 1.5, 2.4, 3.0}},
                                 {128, 192, {4.5, kNever, kNever, kNever}, {0.85, kNever, kNever, kNever}},
                                 {128, 32, {kNever, 5.0, 5.4, 5.0}, {kNever, 0.95, 1.1, 1.75}},
                                 {64, 128, {3.0, kNever, kNever, kNever}, {0.48, kNever, kNever, kNever}}};
struct LogitsPlan {
  int form = -1;  // -1: product_split
  uint32_t splits = 1, steps_per_split = 0;
  uint64_t bytes = 0;  // of workspace
};
uint64_t sums_width(uint64_t columns) { return (columns + 3) / 4 * 4; }
LogitsPlan plan_logits(uint64_t m, uint64_t experts, uint64_t hidden, int32_t dtype, int32_t weight_dtype, bool far_apart) {
  LogitsPlan best;
  if (far_apart) return best;
  const int kind = dtype == PPLX_A2A_F32 ? 3 : weight_dtype != PPLX_A2A_F32 ? 0 : dtype == PPLX_A2A_BF16 ? 1 : 2;
  const uint32_t steps = (uint32_t)((hidden + 63) / 64), of_rows = (m < 16 ? (uint32_t)m : 16) * (dtype == PPLX_A2A_F32 ? 8 : 4),
                 of_columns = weight_dtype == PPLX_A2A_F32 ? 128 : 64;
  auto rounds = [](uint64_t groups) { return (double)((groups + kComputeUnits - 1) / kComputeUnits); };
  double least = 2.2 + rounds(((m + 15) / 16) * ((experts + 15) / 16)) * (double)(steps * 2 * (of_rows + of_columns)) / 2400;
  for (int f = 0; f < (int)(sizeof(kForms) / sizeof(kForms[0])); ++f) {
    const LogitsForm &form = kForms[f];
    const uint64_t tiles = ((m + form.bm - 1) / form.bm) * ((experts + form.bn - 1) / form.bn);
    const double per_step = form.per_step[kind], start = form.start[kind];
    if (tiles >= (1ull << 28) || start + per_step * rounds(tiles) >= least) continue;  // (no split of k is faster than one step)
    // As many splits as go into one, two or three rounds of the compute units, fewer where their sums cost more than they gain, and some
    // that make the last of a few rounds a short one: 1 % of products have a plan that costs 3 % more than the best of all splits.
    auto consider = [&](uint32_t wanted) {
      if (wanted < 1) return;
      const uint32_t most = wanted < 64 ? wanted : 64, per = (steps + most - 1) / most, splits = (steps + per - 1) / per;
      const uint64_t bytes = splits > 1 ? 4 * splits * m * sums_width(experts) : 0;
      if (bytes > (512ull << 20)) return;
      const double cost = start + rounds(tiles * splits) * (double)per * per_step +
                          (splits > 1 ? 2.2 + 0.02 * (double)splits + (double)bytes / 5.5e6 : 0.0);
      if (cost < least) {
        least = cost;
        best.form = f;
        best.splits = splits;
        best.steps_per_split = per;
        best.bytes = bytes;
      }
    };
    const uint32_t a_round = tiles < kComputeUnits ? kComputeUnits / (uint32_t)tiles : 0;
    consider(1);
    for (uint32_t n : {a_round, a_round * 3 / 4, a_round / 2, a_round / 4}) consider(n);
    if (tiles < 3 * kComputeUnits) {
      consider((uint32_t)(2 * kComputeUnits / tiles));
      consider((uint32_t)(3 * kComputeUnits / tiles));
    }
    if (tiles > kComputeUnits && tiles < 8 * kComputeUnits) {
      for (uint32_t n : {4, 8, 16}) consider(n);
    }
  }
  return best;
}

template <class T, class W, int BM, int BN, int WM, int WN, int STAGES> int launch_tiles(const TilesDev &from, hipStream_t s) {
  TilesDev a = from;
  a.row_blocks = (uint32_t)ceil_div(a.rows, BM);
  a.column_blocks = (uint32_t)ceil_div(a.columns, BN);
  constexpr uint32_t lds = STAGES * 64 * (BM * sizeof(T) + BN * sizeof(W));
  auto kernel = a.k % 64 ? logits_tiles<T, W, BM, BN, WM, WN, STAGES, true> : logits_tiles<T, W, BM, BN, WM, WN, STAGES, false>;
  allow_lds(kernel, lds);
  // (a launch takes fewer than 2^32 threads: more rows go out in several, which steps of few rows, the only ones that are split, never
  // come to)
  const uint32_t most = (1u << 22) / a.column_blocks;
  const int8_t *first = a.a;
  float *out = a.out;
  for (uint64_t block = 0, blocks = a.row_blocks; block < blocks; block += most) {
    a.a = first + (int64_t)block * BM * a.a_stride;
    a.out = out + (int64_t)block * BM * a.out_stride;
    a.rows = from.rows - (uint32_t)(block * BM);
    a.row_blocks = (uint32_t)(blocks - block);
    if (blocks - block > most) {
      a.row_blocks = most;
      a.rows = most * BM;
    }
    const uint64_t grid = ceil_div((uint64_t)a.row_blocks * a.column_blocks * a.splits, 8) * 8;
    const int err = launch_kernel(kernel, dim3((uint32_t)grid), dim3(WM * WN * 64), lds, s, a);
    if (err) return err;
  }
  return 0;
}
template <class T, class W> int launch_form(int form, const TilesDev &a, hipStream_t s) {
  if (form == 0) return launch_tiles<T, W, 64, 64, 2, 2, 4>(a, s);
  if constexpr (sizeof(W) == 2) {
    if (form == 2) return launch_tiles<T, W, 128, 192, 2, 2, 3>(a, s);
    if (form == 4) return launch_tiles<T, W, 64, 128, 2, 2, 4>(a, s);
  } else {
    if (form == 3) return launch_tiles<T, W, 128, 32, 4, 1, sizeof(T) == 2 ? 5 : 3>(a, s);
  }
  return launch_tiles<T, W, 128, 128, 2, 4, sizeof(W) == 2 ? 4 : 2>(a, s);
}

// ---------------------------------------------------------------------------
// The gradients' shares
// ---------------------------------------------------------------------------
// Columns of a lane: four where their pieces fit LDS.
template <class TB> constexpr int kColumnsOfLane = Pieces<TB>::count <= 2 ? 4 : 2;

struct WeightShares {
  uint32_t waves, row_blocks, parts, tokens_per_part;
};
// Into how many parts the tokens go, by cost in us: a start, a step of 16 tokens for each wave, and the parts' sums.  Up to 64 experts
// leave two of four waves without work for the matrix cores, and a second workgroup costs a compute unit half a step.  With all launches:
// 8192 x 4096 of 8 in 8 parts 30.4 and in 16 (two to a unit) 22.0; 16384 x 4096 of 64 in fp16 in 8, 16 and 32 parts 83.5, 68.4 and 71.7; but
// 8192 x 2048 of 128 in 16 parts 28.8 and in 32 34.0, and 3001 x 7168 of 256 in 4 parts 47.1 and in 8 58.8 (the best of all parts in each of
// eleven such sizes, or within 2 %).  Workgroups of two waves, each in its best parts, with two pieces of grad_logits: 8192 x 4096 of 8 17.4
// and not 16.9, 4452 x 1960 of 47 in fp32 18.2 and not 18.3, 2000 x 2048 of 60 12.7 and not 8.0.
WeightShares weight_shares(uint64_t m, uint64_t experts, uint64_t hidden, uint32_t columns) {
  WeightShares w{};
  w.waves = experts > 128 ? 8 : 4;
  w.row_blocks = (uint32_t)ceil_div(experts, 32 * w.waves);
  const uint64_t step = 16 * w.waves, steps = ceil_div(m, step), blocks = ceil_div(hidden, columns) * w.row_blocks;
  double least = 0;
  for (uint64_t most = steps; most >= 1; most = most > 8 ? most * 7 / 8 : most - 1) {
    const uint64_t parts = ceil_div(steps, most), per = ceil_div(steps, parts);
    if (parts > 32) break;
    const double at_once = (double)ceil_div(blocks * parts, kComputeUnits), shared = at_once > 1 && experts <= 64 ? at_once - 0.5 : at_once;
    const double cost = shared * (double)per * (w.waves == 8 ? 3.2 : 1.2) + 2.0 * at_once +
                        (parts > 1 ? 2.0 + (double)(parts * experts * hidden) * 8 / 6e6 : 0.0);
    if (w.parts == 0 || cost < least) {
      least = cost;
      w.parts = (uint32_t)parts;
      w.tokens_per_part = (uint32_t)(per * step);
    }
  }
  return w;
}

struct BackwardSpace {
  WeightShares shares;
  uint64_t by_columns, sums, bytes;  // (fragments of the rows come first)
};
template <class T> BackwardSpace backward_space(uint64_t m, uint64_t experts, uint64_t hidden) {
  BackwardSpace s{};
  s.shares = weight_shares(m, experts, hidden, 32 * kColumnsOfLane<T>);
  s.by_columns = fragment_bytes(m, experts);
  s.sums = s.by_columns + fragment_bytes(experts, m);
  s.bytes = s.sums + (s.shares.parts > 1 ? 4 * s.shares.parts * experts * hidden : 0);
  return s;
}

template <class T, class W> int launch_gradient_of_rows(GradientDev a, hipStream_t s) {
  constexpr int kNV = kColumnsOfLane<W>;
  typedef Turned<W, kNV> B;
  constexpr uint32_t kMost = kLdsBytes / B::kBytes / 4 * 64;  // k of a chunk
  const uint32_t whole = (a.k + 15) / 16 * 16, chunk = whole < kMost ? whole : kMost;
  a.column_blocks = (uint32_t)ceil_div(a.columns, 32 * kNV);
  // Workgroups keep the weight's columns for as many rounds of rows as leaves no compute unit idle for long.
  const uint64_t rounds = ceil_div(a.rows, 32 * kGradientWaves);
  uint64_t least = 0;
  for (uint64_t most = rounds; most >= 1; most = most > 8 ? most * 7 / 8 : most - 1) {
    const uint64_t parts = ceil_div(rounds, most), per = ceil_div(rounds, parts), cost = ceil_div(a.column_blocks * parts, kComputeUnits) * (per + 1);
    if (a.parts == 0 || cost < least) {
      least = cost;
      a.parts = (uint32_t)parts;
    }
  }
  auto kernel = gradient_of_rows<W, T, kNV>;
  const uint32_t lds = chunk / 16 * B::kBytes;
  allow_lds(kernel, lds);
  return launch_groups(kernel, kernel, (uint64_t)a.column_blocks * a.parts, kGradientWaves * 64, lds, s, a, chunk);
}

template <class T, class W> int launch_gradient_of_weight(GradientDev a, const WeightShares &w, float *sums, hipStream_t s) {
  constexpr int kNV = kColumnsOfLane<T>;
  a.column_blocks = (uint32_t)ceil_div(a.columns, 32 * kNV);
  a.parts = w.parts;
  const uint64_t groups = (uint64_t)a.column_blocks * w.row_blocks * w.parts;
  const uint32_t lds = 2 * w.waves * Turned<T, kNV>::kBytes;
  auto launch = [&](auto kernel) {
    allow_lds(kernel, lds);
    return launch_groups(kernel, kernel, groups, w.waves * 64, lds, s, a, w.tokens_per_part, w.row_blocks);
  };
  if (w.parts == 1) return w.waves == 8 ? launch(gradient_of_weight<T, W, kNV, 8>) : launch(gradient_of_weight<T, W, kNV, 4>);
  const SumDev sum{sums, (uint64_t)a.rows * a.columns, a.out, a.out_stride, a.rows, a.columns, a.columns, w.parts, 0};
  a.out = reinterpret_cast<uint8_t *>(sums);
  a.out_stride = a.columns;
  a.out_split = sum.split;
  const int err = w.waves == 8 ? launch(gradient_of_weight<T, float, kNV, 8>) : launch(gradient_of_weight<T, float, kNV, 4>);
  return err ? err : launch_sum<W>(sum, s);
}

int check_router_size(uint64_t m, uint32_t experts, uint64_t hidden, int32_t dtype, int32_t weight_dtype) {
  PPLX_REQUIRE(is_dtype(dtype), "unsupported dtype of the rows");
  PPLX_REQUIRE(weight_dtype == dtype || weight_dtype == PPLX_A2A_F32, "weight_dtype must be dtype or F32");
  PPLX_REQUIRE(experts >= 1 && experts <= kMaxExperts, "num_experts must be in [1, %u]", kMaxExperts);
  PPLX_REQUIRE(hidden > 0 && hidden < (1ull << 27) && hidden % 8 == 0, "hidden_dim must be a multiple of 8 below 2^27");
  if (m > kMaxTokens) return refuse(PPLX_A2A_UNSUPPORTED, "2^31 tokens or more");
  return PPLX_A2A_OK;
}
// A tile's rows are reached by 32-bit offsets.
bool is_far(int64_t stride) { return stride < 0 || stride >= (1 << 23); }

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

extern "C" int pplx_a2a_router_workspace(uint32_t m, uint32_t num_experts, uint64_t hidden_dim, int32_t dtype,
                                         int32_t weight_dtype, int32_t backward, uint64_t *bytes) {
  PPLX_REQUIRE(bytes, "bytes is NULL");
  const int st = check_router_size(m, num_experts, hidden_dim, dtype, weight_dtype);
  if (st) return st;
  if (!backward) {
    *bytes = plan_logits(m, num_experts, hidden_dim, dtype, weight_dtype, false).bytes;
    return PPLX_A2A_OK;
  }
  return with_type(dtype, [&](auto tag) {
    *bytes = backward_space<typename decltype(tag)::type>(m, num_experts, hidden_dim).bytes;
    return (int)PPLX_A2A_OK;
  });
}

extern "C" int pplx_a2a_router_logits(int device, const pplx_a2a_router_logits_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_router_logits_args_t &p = *args;
  const int st = check_router_size(p.m, p.num_experts, p.hidden_dim, p.dtype, p.weight_dtype);
  if (st) return st;
  if (p.m == 0) return PPLX_A2A_OK;
  PPLX_ROWS(p, x);
  PPLX_ROWS(p, weight);
  PPLX_REQUIRE(p.logits && is_aligned(p.logits, 4), "logits is NULL or not aligned");
  const LogitsPlan plan =
      plan_logits(p.m, p.num_experts, p.hidden_dim, p.dtype, p.weight_dtype, is_far(p.x_stride_row) || is_far(p.weight_stride_row));
  PPLX_REQUIRE(plan.bytes == 0 || (p.workspace && is_aligned(p.workspace, 16)), "workspace is NULL or not aligned");
  return guarded(device, [&] {
    return with_weight_type(p.dtype, p.weight_dtype, [&](auto tag, auto weight_tag) {
      typedef typename decltype(tag)::type T;
      typedef typename decltype(weight_tag)::type W;
      hipStream_t s = (hipStream_t)stream;
      if (plan.form < 0) {
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
        a.column_blocks = (uint32_t)ceil_div(a.columns, 16);
        auto kernel = product_split<T, W>;
        PPLX_LAUNCH(launch_groups(kernel, kernel, ceil_div(a.rows, 16) * a.column_blocks, kProductWaves * 64, 0, s, a));
        return (int)PPLX_A2A_OK;
      }
      const uint64_t width = sums_width(p.num_experts);
      TilesDev a{};
      a.a = static_cast<const int8_t *>(p.x);
      a.a_stride = p.x_stride_row;
      a.b = static_cast<const int8_t *>(p.weight);
      a.b_stride = p.weight_stride_row;
      a.rows = p.m;
      a.columns = p.num_experts;
      a.k = (uint32_t)p.hidden_dim;
      a.splits = plan.splits;
      a.steps_per_split = plan.steps_per_split;
      a.out = plan.splits > 1 ? static_cast<float *>(p.workspace) : p.logits;
      a.out_stride = plan.splits > 1 ? (int64_t)width : p.logits_stride_row;
      a.out_split = (uint64_t)p.m * width;
      PPLX_LAUNCH((launch_form<T, W>(plan.form, a, s)));
      if (plan.splits > 1) {
        const SumDev sum{a.out, a.out_split, reinterpret_cast<uint8_t *>(p.logits), p.logits_stride_row, p.m, (uint32_t)width, p.num_experts, plan.splits, 0};
        PPLX_LAUNCH(launch_sum<float>(sum, s));
      }
      return (int)PPLX_A2A_OK;
    });
  });
}

extern "C" int pplx_a2a_router_logits_backward(int device, const pplx_a2a_router_logits_backward_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_router_logits_backward_args_t &p = *args;
  const int st = check_router_size(p.m, p.num_experts, p.hidden_dim, p.dtype, p.weight_dtype);
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
  return guarded(device, [&] {
    return with_weight_type(p.dtype, p.weight_dtype, [&](auto tag, auto weight_tag) {
      typedef typename decltype(tag)::type T;
      typedef typename decltype(weight_tag)::type W;
      hipStream_t s = (hipStream_t)stream;
      const BackwardSpace space = backward_space<T>(p.m, p.num_experts, p.hidden_dim);
      uint8_t *work = static_cast<uint8_t *>(p.workspace);
      PiecesDev pieces{};
      pieces.in = p.grad_logits;
      pieces.in_stride = p.grad_logits_stride_row;
      pieces.rows = p.m;
      pieces.columns = p.num_experts;
      pieces.by_rows = p.grad_x ? work : nullptr;
      pieces.by_columns = p.grad_weight ? work + space.by_columns : nullptr;
      PPLX_LAUNCH(launch_split(pieces, s));
      if (p.grad_x) {
        GradientDev a{};
        a.a = pieces.by_rows;
        a.b = static_cast<const uint8_t *>(p.weight);
        a.b_stride = p.weight_stride_row;
        a.out = static_cast<uint8_t *>(p.grad_x);
        a.out_stride = p.grad_x_stride_row / (int64_t)sizeof(T);
        a.rows = p.m;
        a.columns = (uint32_t)p.hidden_dim;
        a.k = p.num_experts;
        PPLX_LAUNCH((launch_gradient_of_rows<T, W>(a, s)));
      }
      if (p.grad_weight) {
        GradientDev a{};
        a.a = pieces.by_columns;
        a.b = static_cast<const uint8_t *>(p.x);
        a.b_stride = p.x_stride_row;
        a.out = static_cast<uint8_t *>(p.grad_weight);
        a.out_stride = p.grad_weight_stride_row / (int64_t)sizeof(W);
        a.rows = p.num_experts;
        a.columns = (uint32_t)p.hidden_dim;
        a.k = p.m;
        PPLX_LAUNCH((launch_gradient_of_weight<T, W>(a, space.shares, reinterpret_cast<float *>(work + space.sums), s)));
      }
      return (int)PPLX_A2A_OK;
    });
  });
}
