// Rows times their experts' weights in 8-bit integers.
//
//   out[r, n] = x_scale[r] * weight_scale[e, n] * sum over k of x[r, k] * weight[e, n, k]
//
// on the matrix cores (v_mfma_i32_*_i8), whose int32 sums are exact for every k that the entry point admits.  The weights
// are the first operand, so that the accumulators of a lane are consecutive columns of one row of the result.
//
// Tiles of BM rows by BN columns go through LDS, BK bytes of k at a time, which loads write there directly.  A row of a
// tile is a line of 16-byte chunks, whose places are exchanged from row to row so that the lanes of a fragment, which read one
// chunk each of consecutive rows, read all banks.  How many rows each expert has is known on the
// device only: every workgroup sums the experts' blocks of rows and takes tiles from the list that follows from them.
#include <cmath>

#include "a2a_experts.h"
#include "a2a_tiles.h"

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
  uint32_t first_group;    // of the split forms
  uint32_t large_weights;  // more than the last-level cache is likely to hold until they are read again
};

// A store of the lanes in `lanes` that counts whether there are any or not.  (All lanes are active where it stands.  Its data
// registers may be written again two wait states later.)
__device__ __forceinline__ void store_counted(PPLX_GLOBAL void *p, u32x4 v, uint64_t lanes) {
  asm volatile(
      "s_mov_b64 exec, %2\n\t"
      "global_store_dwordx4 %0, %1, off\n\t"
      "s_mov_b64 exec, -1\n\t"
      "s_nop 1"
      ::"v"(p), "v"(v), "s"(lanes)
      : "memory");
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
template <int BM, int BN>
__device__ __forceinline__ Tile tile_of(const RowsDev &rows, uint32_t n_blocks, const uint32_t *upto, uint32_t id) {
  uint32_t lo = 0, hi = rows.experts - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (upto[mid] * n_blocks > id) hi = mid;
    else lo = mid + 1;
  }
  Tile t;
  t.e = __builtin_amdgcn_readfirstlane(lo);
  const uint32_t before = t.e ? upto[t.e - 1] : 0u;
  const uint32_t blocks = upto[t.e] - before;
  const uint32_t local = id - before * n_blocks;
  const uint32_t group = local / (kGroup * n_blocks);
  const uint32_t in_group = local - group * kGroup * n_blocks;
  const uint32_t size = blocks - group * kGroup < kGroup ? blocks - group * kGroup : kGroup;
  const uint32_t nb = in_group / size;
  const Span s = span_of(rows, t.e);
  t.m0 = __builtin_amdgcn_readfirstlane((group * kGroup + in_group - nb * size) * BM);
  t.n0 = __builtin_amdgcn_readfirstlane(nb * BN);
  t.begin = __builtin_amdgcn_readfirstlane(s.begin);
  t.count = __builtin_amdgcn_readfirstlane(s.count);
  return t;
}

// Four results at any address that one may have.
template <class O> struct FourOf;
template <> struct FourOf<float> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct FourOf<__bf16> {
  typedef __bf16 type __attribute__((ext_vector_type(4), aligned(2)));
};
template <> struct FourOf<_Float16> {
  typedef _Float16 type __attribute__((ext_vector_type(4), aligned(2)));
};

// Four columns of a row, 4 bytes or 2 each, as words.
template <class O> __device__ __forceinline__ void pack_four(f32x4 v, uint32_t *words) {
  if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) words[i] = __float_as_uint(v[i]);
  } else {
    typedef O four __attribute__((ext_vector_type(4)));
    typedef uint32_t two __attribute__((ext_vector_type(2)));
    const two w = __builtin_bit_cast(two, __builtin_convertvector(v, four));
    words[0] = w[0];
    words[1] = w[1];
  }
}

// WM by WN waves, each BM / WM rows by BN / WN columns in fragments of 32 by 32; STAGES steps of BK bytes of k in LDS.  A wave
// reads the fragments of the next 32 bytes of k before it multiplies those at hand, over the border between two steps too:
// there it waits for the next step's loads, and behind the barrier this step's place takes those of a step to come.  The
// loads of the next tile's first steps go out before this tile's results are stored.
// TAIL: k is no multiple of BK.
template <int BM, int BN, int WM, int WN, int BK, int STAGES, bool TAIL, class O>
__global__ __launch_bounds__(WM *WN * 64) void matmul_tiles(MatmulDev) {
  constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
  constexpr int kRows = BM / WM, kColumns = BN / WN, MF = kRows / 32, NF = kColumns / 32;
  constexpr int kChunks = BK / 16, kRowsPerLoad = 64 / kChunks;
  constexpr int kLoads = (BM + BN) / kRowsPerLoad / kWaves;  // of a wave in a step
  constexpr int kSteps = BK / 32;                            // matrix instructions along k in a step
  static_assert(BK == 64 || BK == 128, "a line is four or eight chunks");
  static_assert((BM + BN) % (kRowsPerLoad * kWaves) == 0 && BM % kRowsPerLoad == 0, "whole loads");
  static_assert(kRows % 32 == 0 && kColumns % 32 == 0, "whole fragments");
  static_assert((STAGES - 1) * kLoads < 63, "loads that can be counted");
  constexpr int kScales = (BM + BN + kThreads - 1) / kThreads;  // of a thread
  static_assert(kSteps % 2 == 0, "a step begins with the first fragments");
  // A wave of few products reads a step's fragments all at once: read for the next product only, each waits for LDS.
  constexpr bool kWhole = MF * NF <= 2;
  constexpr int kSets = kWhole ? kSteps : 2;            // of fragments in registers
  // Weights that one tile reads, and no other, go past the caches: 32 rows or fewer of each of 32 experts, 4096 x 7168, take
  // 138 us instead of 159 (6.8 TB/s).  Not in pieces of 64 bytes, half of what a read brings: the other half, read a step later,
  // is gone by then (64 rows each 254 us instead of 193), and not weights that the last-level cache may hold from one call to
  // the next (32 rows of 16384 x 4096 20.8 instead of 15.2).
  constexpr bool kLines = BK == 128;
  constexpr int kAhead = kWhole ? STAGES - 1 : STAGES;  // steps loaded in front of a tile's first
  constexpr int kStage = (BM + BN) * BK;
  // [STAGES][BM rows of x, BN of the weight][BK], scales, sums of blocks, sums of waves.  All of a workgroup's share is in here,
  // so that the stages, which loads write directly, begin at its first byte.
  extern __shared__ __align__(128) uint8_t lds[];
  static_assert(STAGES * kStage <= kLdsBytes, "loads to LDS stay in front of kLdsBytes");
  float *scales = reinterpret_cast<float *>(lds + STAGES * kStage);  // of BM rows and BN columns
  uint32_t *upto = reinterpret_cast<uint32_t *>(scales + BM + BN);
  // The arguments are read where they are used, once a tile: kept in scalar registers they are more than there are.
  auto arguments = []() __attribute__((always_inline)) {
    auto *p = (const PPLX_CONSTANT MatmulDev *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
  };
  uint32_t tiles;
  {
    const auto *a = arguments();
    const RowsDev rows{a->rows.starts_or_counts, a->rows.rows, a->rows.experts, a->rows.layout};
    sum_blocks<kThreads, BM>(rows, upto, upto + rows.experts);
    // (offsets that do not ascend give a list of any length, of which only tiles that exist are taken)
    const uint32_t listed = upto[rows.experts - 1] * a->n_blocks;
    tiles = __builtin_amdgcn_readfirstlane(listed < 1u << 31 ? listed : 1u << 31);
  }
  const uint32_t lane = lane_id(), wave = wave_id();
  const uint32_t wm = wave % WM, wn = wave / WM;
  const uint32_t lds0 = lds_address(lds);
  const uint32_t depth = arguments()->k;
  const uint32_t steps = (depth + BK - 1) / BK;
  // Chunk c of row r lies at c ^ swizzle(r): sixteen consecutive rows hold a chunk at sixteen places of 256 bytes, which is
  // what LDS reads at a time.  (With exchanges for 128 bytes reads took 8.8 cycles instead of 4.9.)
  auto swizzle = [](uint32_t row) { return kChunks == 8 ? (row >> 1) & 7 : (row >> 2) & 3; };
  static_assert(kWaves * kRowsPerLoad % 16 == 0 && BM % 16 == 0, "a lane's rows have one exchange");
  const uint32_t load_row = lane / kChunks;
  const uint32_t load_chunk = (lane % kChunks) ^ swizzle(wave * kRowsPerLoad + load_row);
  const uint32_t frag_base = (lane % 32) * BK;
  uint32_t frag_place[kSteps];
#pragma unroll
  for (int kk = 0; kk < kSteps; ++kk) frag_place[kk] = ((2 * kk + lane / 32) ^ swizzle(lane % 32)) * 16;

  // The tile whose steps are loaded: where its operands begin, and what the lane's loads add to that.
  const int8_t *x = nullptr, *weight = nullptr;
  uint32_t once = 0;  // no other tile reads this one's part of the weight
  uint32_t offset[kLoads];
  float scale[kScales];  // of row threadIdx.x, threadIdx.x + kThreads .. of the tile, its columns behind its rows
  // Load number i of a step.  Behind k a lane fetches the first chunk of its line; what it brings is taken for zeros.  Loads of
  // steps that do not exist bring nothing, and count: the loop has one path.
  auto fetch = [&](int i, uint32_t step, uint32_t stage) __attribute__((always_inline)) {
    const uint32_t first = (i * kWaves + wave) * kRowsPerLoad;
    const int8_t *base = (first < BM ? x : weight) + step * BK;
    const bool behind = TAIL && step * BK + load_chunk * 16 >= depth;
    const uint32_t at = behind ? offset[i] - load_chunk * 16 : offset[i], place = lds0 + stage * kStage + first * BK;
    const uint32_t lanes = step < steps ? ~0u : 0u;
    if (kLines && i * kWaves * kRowsPerLoad >= BM) load_past_to_lds(base, at, place, lanes, once);
    else load_to_lds(base, at, place, lanes);
  };
  auto begin = [&](const Tile &t) __attribute__((always_inline)) {
    const auto *a = arguments();
    x = a->x + (int64_t)t.e * a->x_stride_expert + (int64_t)(t.begin + t.m0) * a->x_stride_row;
    weight = a->weight + ((uint64_t)t.e * a->n + t.n0) * depth;
    const uint32_t rows_left = t.count - t.m0, columns_left = a->n - t.n0;
    once = a->large_weights && t.count <= BM;
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      const uint32_t p = threadIdx.x + i * kThreads;
      if (p < BM) {
        const uint32_t r = p < rows_left ? p : rows_left - 1;
        scale[i] = as_global(a->x_scale)[(int64_t)t.e * a->x_scale_stride_expert + (int64_t)(t.begin + t.m0 + r) * a->x_scale_stride_row];
      } else if (p < BM + BN) {
        const uint32_t c = p - BM < columns_left ? p - BM : columns_left - 1;
        scale[i] = as_global(a->weight_scale)[(uint64_t)t.e * a->n + t.n0 + c];
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t first = (i * kWaves + wave) * kRowsPerLoad;  // row of the stage
      const uint32_t r = first + load_row - (first < BM ? 0 : BM);
      offset[i] = load_chunk * 16 + (first < BM ? (r < rows_left ? r : rows_left - 1) * (uint32_t)a->x_stride_row
                                                : (r < columns_left ? r : columns_left - 1) * depth);
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) fetch(i, s, s);
    }
  };
  i32x4 fx[kSets][MF], fw[kSets][NF];
  // Fragment number i (of the rows, then of the columns) for matrix instructions kk of a step.
  auto read = [&](int i, int to, int kk, uint32_t step, uint32_t stage) __attribute__((always_inline)) {
    const uint8_t *lines = lds + stage * kStage + frag_base + frag_place[kk];
    if (i < MF) {
      fx[to][i] = *reinterpret_cast<const i32x4 *>(lines + (wm * kRows + i * 32) * BK);
      if constexpr (TAIL) fx[to][i] &= step * BK + kk * 32 + (lane / 32) * 16 < depth ? -1 : 0;
    } else {
      fw[to][i - MF] = *reinterpret_cast<const i32x4 *>(lines + (BM + wn * kColumns + (i - MF) * 32) * BK);
    }
  };

  // (blockIdx goes round the eight XCDs)
  uint32_t id = (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
  Tile t{};
  auto find = [&]() __attribute__((always_inline)) {
    const auto *a = arguments();
    const RowsDev rows{a->rows.starts_or_counts, a->rows.rows, a->rows.experts, a->rows.layout};
    const uint32_t n_blocks = a->n_blocks;
    for (; id < tiles; id += gridDim.x) {
      t = tile_of<BM, BN>(rows, n_blocks, upto, id);
      if (t.m0 < t.count && t.n0 < a->n) break;
    }
    return id < tiles;
  };
  // Stores of a tile's results by a wave that are counted.
  constexpr int kStores = MF * NF * (sizeof(O) == 4 ? 4 : 2);
  constexpr int kBehind = (STAGES - 1) * kLoads + kStores <= 63 ? kStores : 0;  // as far as the counter goes
  bool stored = false;  // the stores of the tile before stand behind the loads of the first steps
  bool more = find();
  if (more) begin(t);
  while (more) {
    const Tile at = t;
    i32x16 acc[NF][MF] = {};
    if constexpr (kWhole) {
      uint32_t stage = 0;
      for (uint32_t step = 0; step < steps; ++step) {
        const uint32_t before = stage == 0 ? STAGES - 1 : stage - 1;
        // Loads under way are those of steps step .. step + STAGES - 2; the place of the step before is free behind the barrier.
        if (stored && step < STAGES - 1) wait_loads<(STAGES - 2) * kLoads + kBehind>();
        else wait_loads<(STAGES - 2) * kLoads>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
#pragma unroll
          for (int i = 0; i < MF + NF; ++i) read(i, kk, kk, step, stage);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) fetch(i, step + STAGES - 1, before);
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
#pragma unroll
          for (int j = 0; j < NF; ++j) {
#pragma unroll
            for (int i = 0; i < MF; ++i) {
              acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[kk][j], fx[kk][i], acc[j][i], 0, 0, 0);
            }
          }
        }
        stage = stage + 1 == STAGES ? 0 : stage + 1;
      }
    } else {
      if (stored) wait_loads<(STAGES - 1) * kLoads + kBehind>();
      else wait_loads<(STAGES - 1) * kLoads>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < MF + NF; ++i) read(i, 0, 0, 0, 0);
      // The matrix instructions of 32 bytes of k, between which the reads of the next 32 and the loads of a step go out: a wave
      // issues in order, and one that hands over all its reads or loads at once waits for them to be taken.
      constexpr int kProducts = MF * NF;
      auto multiply = [&](int from, auto read_next, auto fetch_next) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < kProducts; ++q) {
          const int j = q / MF, i = q % MF;
          acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[from][j], fx[from][i], acc[j][i], 0, 0, 0);
#pragma unroll
          for (int r = q * (MF + NF) / kProducts; r < (q + 1) * (MF + NF) / kProducts; ++r) read_next(r);
#pragma unroll
          for (int l = q * kLoads / kProducts; l < (q + 1) * kLoads / kProducts; ++l) fetch_next(l);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      uint32_t stage = 0;
      for (uint32_t step = 0; step < steps; ++step) {
        const uint32_t next = stage + 1 == STAGES ? 0 : stage + 1;
#pragma unroll
        for (int kk = 0; kk + 1 < kSteps; ++kk) {
          multiply(kk % 2, [&](int r) { read(r, (kk + 1) % 2, kk + 1, step, stage); }, [](int) {});
        }
        // Loads under way are those of steps step + 1 .. step + STAGES - 1; this step's place is free behind the barrier.
        if (stored && step < STAGES - 1) wait_loads<(STAGES - 2) * kLoads + kBehind, true>();
        else wait_loads<(STAGES - 2) * kLoads, true>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        multiply((kSteps - 1) % 2, [&](int r) { read(r, kSteps % 2, 0, step + 1, next); },
                 [&](int l) { fetch(l, step + STAGES, stage); });
        stage = next;
      }
    }

    wait_loads<0, true>();
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      if (threadIdx.x + i * kThreads < BM + BN) scales[threadIdx.x + i * kThreads] = scale[i];
    }
    __syncthreads();  // (the stages have been read, the scales are there)
    id += gridDim.x;
    more = find();
    if (more) begin(t);
    stored = true;

    // Lane l holds row l % 32 of each fragment and, in its accumulators, columns 4 (l / 32) .. + 3 of every eight.  Of 2-byte
    // results two such groups change places between the halves of the wave, so that every lane has 16 bytes of its row; then two
    // such stores change places between the quarters, so that each takes 64 bytes of sixteen rows instead of 32 of 32: 16384 x
    // 14336 of 1024 304 to 298 us, of 14340, whose rows do not begin at lines, 344 to 323.
    const auto *a = arguments();
    const uint32_t columns = a->n;
    const int64_t out_stride = a->out_stride_row;
    PPLX_GLOBAL O *out_first = as_global(reinterpret_cast<O *>(a->out)) + (int64_t)at.e * a->out_stride_expert +
                               (int64_t)(at.begin + at.m0) * out_stride;
    const uint32_t half = lane / 32;
    constexpr uint32_t kVec = 16 / sizeof(O);        // results of a lane in a store
    constexpr int kGroups = sizeof(O) == 4 ? 1 : 2;  // of eight columns in a store
    const uint32_t lane_column = kVec * (half + lane / 16 % 2 * 2);
    // Rows of 2-byte results that begin between two words are stored one result earlier, by words, where a lane has the result
    // before its own from the lane that holds it; the strip's first lanes, which do not, store as they are.  (Stores that split words
    // are slow: 14335 columns 428 us, so 339.)
    const bool odd = sizeof(O) == 2 && (((uintptr_t)out_first | (uintptr_t)(out_stride * 2)) & 2);
    const uint32_t before = 4 * (half ? lane - 32 : lane < 16 ? lane + 48 : lane + 16);
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      uint32_t carry[2] = {0, 0};  // the last words of the columns before, for the first lanes
      const float xs = scales[wm * kRows + i * 32 + lane % 32];
#pragma unroll
      for (int j = 0; j < NF; ++j) {
#pragma unroll
        for (int q = 0; q < 4; q += 2 * kGroups) {
          uint32_t words[2][4];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
              const int group = q + p * kGroups + g;
              const f32x4 ws = *reinterpret_cast<const f32x4 *>(scales + BM + wn * kColumns + j * 32 + group * 8 + 4 * half);
              f32x4 v;
#pragma unroll
              for (int u = 0; u < 4; ++u) v[u] = (float)acc[j][i][4 * group + u] * (xs * ws[u]);
              pack_four<O>(v, words[p] + 2 * g);
            }
            if constexpr (kGroups == 2) {
              const auto first = __builtin_amdgcn_permlane32_swap(words[p][0], words[p][2], false, false);
              const auto second = __builtin_amdgcn_permlane32_swap(words[p][1], words[p][3], false, false);
              words[p][0] = first[0];
              words[p][1] = second[0];
              words[p][2] = first[1];
              words[p][3] = second[1];
            }
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const auto both = __builtin_amdgcn_permlane16_swap(words[0][w], words[1][w], false, false);
            words[0][w] = both[0];
            words[1][w] = both[1];
          }
          uint32_t n = at.n0 + wn * kColumns + j * 32 + q * 8 + lane_column;
          asm volatile("" : "+v"(n));  // (the masks of a column for all rows at once are more scalar registers than there are)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint32_t row = wm * kRows + i * 32 + p * 16 + lane % 16;
            const bool there = at.m0 + row < at.count;
            PPLX_GLOBAL O *out = out_first + (int64_t)row * out_stride;
            // Rows that begin anywhere take whole vectors all the same; what is left of a row goes one by one (behind stores that
            // count, where more of them make the waits longer and not shorter).
            u32x4 v = {words[p][0], words[p][1], words[p][2], words[p][3]};
            const uint64_t whole = __ballot(there && n + kVec <= columns);
            if (odd) {
              const uint32_t last = (uint32_t)__builtin_amdgcn_ds_bpermute((int)before, (int)v[3]);
              const bool shift = ((uintptr_t)out & 2) && !(j == 0 && q == 0 && lane < 16);
              const uint32_t own[5] = {lane < 16 ? carry[p] : last, v[0], v[1], v[2], v[3]};
              carry[p] = last;
#pragma unroll
              for (int w = 0; w < 4; ++w) v[w] = shift ? __builtin_amdgcn_alignbit(own[w + 1], own[w], 16) : own[w + 1];
              store_counted(out + n - (shift ? 1 : 0), v, whole);
              // (nobody behind it stores its last result)
              if (shift && there && n + kVec <= columns && (n + 2 * kVec > columns || (j == NF - 1 && lane >= 48))) {
                reinterpret_cast<PPLX_GLOBAL uint16_t *>(out)[n + kVec - 1] = (uint16_t)(own[4] >> 16);
              }
            } else {
              store_counted(out + n, v, whole);
            }
            if (there && n < columns && n + kVec > columns) {
              typedef O vec __attribute__((ext_vector_type(kVec)));
              const vec one = __builtin_bit_cast(vec, u32x4{words[p][0], words[p][1], words[p][2], words[p][3]});
#pragma unroll
              for (uint32_t u = 0; u + 1 < kVec; ++u) {
                if (u < columns - n) out[n + u] = one[u];
              }
            }
          }
        }
      }
    }
  }
}

// Launches take a plan to fill instead, or NULL.
template <int BM, int BN, int WM, int WN, int BK, int STAGES, class O>
int launch_tiles(const MatmulDev &from, uint64_t most_blocks, hipStream_t s, pplx_a2a_int8_matmul_plan_t *plan) {
  MatmulDev a = from;
  constexpr uint32_t kTileLds = STAGES * (BM + BN) * BK;
  const uint32_t lds = kTileLds + 4 * (BM + BN) + 4 * a.rows.experts + 4 * WM * WN;
  constexpr uint32_t per_unit = kLdsBytes / kTileLds;
  static_assert(per_unit >= 1, "a tile's steps fit");
  a.n_blocks = (a.n + BN - 1) / BN;
  const uint64_t tiles = most_blocks * a.n_blocks;
  if (tiles >= (1ull << 31)) return refuse(PPLX_A2A_UNSUPPORTED, "too many tiles");
  uint64_t grid = per_unit * kComputeUnits;
  grid = tiles < grid ? (tiles + 7) / 8 * 8 : grid;  // (whole rounds of the XCDs)
  if (plan) {
    *plan = {BM, BN, 0, (uint32_t)grid, tiles};
    return PPLX_A2A_OK;
  }
  auto kernel = a.k % BK ? matmul_tiles<BM, BN, WM, WN, BK, STAGES, true, O> : matmul_tiles<BM, BN, WM, WN, BK, STAGES, false, O>;
  if (lds > 64 * 1024) {
    const hipError_t err =
        hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (err != hipSuccess) (void)hipGetLastError();  // (the launch says so if it matters)
  }
  PPLX_LAUNCH(launch_kernel(kernel, dim3((uint32_t)grid), dim3(WM * WN * 64), lds, s, a));
  return PPLX_A2A_OK;
}

// Products of few tiles: one workgroup to 16 RF rows by 32 columns, whose eight waves share out k, 128 bytes at a time, and
// add their sums in LDS (whole numbers: in any order the same).  Operands go straight to registers, in fragments of 16 rows by
// 64 bytes: the lanes of an instruction take 64 bytes in one piece of each row (32 by 32 bytes, which takes 16, was 1.2
// to 1.6 times as long).  AHEAD units of a wave are in flight.
constexpr int kSplitWaves = 8;
template <int RF, int CF, int AHEAD, class O> __global__ __launch_bounds__(kSplitWaves * 64) void matmul_split(MatmulDev a) {
  constexpr int kRows = 16 * RF, kColumns = 16 * CF;
  extern __shared__ uint32_t upto[];
  __shared__ uint32_t of_wave[kSplitWaves];
  __shared__ int32_t sums[kSplitWaves][RF * CF * 4 * 64];
  const uint32_t lane = lane_id(), wave = wave_id(), group = a.first_group + blockIdx.x;
  Tile t;
  if (a.rows.layout == PPLX_A2A_ROWS_DENSE) {
    t.e = t.begin = 0;
    t.count = a.rows.rows;
    const uint32_t block = group / a.n_blocks;
    t.m0 = block * kRows;
    t.n0 = (group - block * a.n_blocks) * kColumns;
  } else {
    sum_blocks<kSplitWaves * 64, kRows>(a.rows, upto, of_wave);
    if (group >= upto[a.rows.experts - 1] * a.n_blocks) return;
    t = tile_of<kRows, kColumns>(a.rows, a.n_blocks, upto, group);
    if (t.m0 >= t.count || t.n0 >= a.n) return;  // (offsets that do not ascend)
  }
  const int8_t *x_first = a.x + (int64_t)t.e * a.x_stride_expert + (int64_t)(t.begin + t.m0) * a.x_stride_row;
  const int8_t *w_first = a.weight + ((uint64_t)t.e * a.n + t.n0) * a.k;
  const uint32_t rows_left = t.count - t.m0, columns_left = a.n - t.n0;
  const PPLX_GLOBAL int8_t *x[RF], *weight[CF];
#pragma unroll
  for (int i = 0; i < RF; ++i) {
    const uint32_t r = i * 16 + lane % 16;
    x[i] = as_global(x_first + (int64_t)(r < rows_left ? r : rows_left - 1) * a.x_stride_row);
  }
#pragma unroll
  for (int i = 0; i < CF; ++i) {
    const uint32_t c = i * 16 + lane % 16;
    weight[i] = as_global(w_first + (uint64_t)(c < columns_left ? c : columns_left - 1) * a.k);
  }
  const uint32_t units = (a.k + 127) / 128, own = lane / 16 * 16;
  struct Unit {
    i32x4 x[2][RF], w[2][CF];
  };
  Unit u[AHEAD];
  auto load = [&](Unit &to, uint32_t unit) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t k = unit * 128 + h * 64 + own;
      const uint32_t at = k < a.k ? k : 0;
#pragma unroll
      for (int i = 0; i < CF; ++i) to.w[h][i] = *reinterpret_cast<const PPLX_GLOBAL i32x4 *>(weight[i] + at);
#pragma unroll
      for (int i = 0; i < RF; ++i) to.x[h][i] = *reinterpret_cast<const PPLX_GLOBAL i32x4 *>(x[i] + at);
    }
  };
  i32x4 acc[CF][RF] = {};
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    if (wave + i * kSplitWaves < units) load(u[i], wave + i * kSplitWaves);
  }
  for (uint32_t first = wave; first < units; first += AHEAD * kSplitWaves) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const uint32_t unit = first + i * kSplitWaves;
      if (unit >= units) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int there = unit * 128 + h * 64 + own < a.k ? -1 : 0;  // (bytes behind k are taken for zeros)
#pragma unroll
        for (int r = 0; r < RF; ++r) {
          const i32x4 fx = u[i].x[h][r] & there;
#pragma unroll
          for (int c = 0; c < CF; ++c) acc[c][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(u[i].w[h][c], fx, acc[c][r], 0, 0, 0);
        }
      }
      if (unit + AHEAD * kSplitWaves < units) load(u[i], unit + AHEAD * kSplitWaves);
    }
  }
#pragma unroll
  for (int c = 0; c < CF; ++c) {
#pragma unroll
    for (int r = 0; r < RF; ++r) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave][((c * RF + r) * 4 + i) * 64 + lane] = acc[c][r][i];
    }
  }
  __syncthreads();
  // Lane l of fragment (c, r) has columns 16 c + 4 (l / 16) .. + 3 of row 16 r + l % 16.
  if (threadIdx.x >= RF * CF * 64) return;
  const uint32_t fragment = threadIdx.x / 64, c = fragment / RF, r = fragment % RF;
  const uint32_t row = t.m0 + r * 16 + lane % 16, n = t.n0 + c * 16 + 4 * (lane / 16);
  if (row >= t.count || n >= a.n) return;
  const float xs = as_global(a.x_scale)[(int64_t)t.e * a.x_scale_stride_expert + (int64_t)(t.begin + row) * a.x_scale_stride_row];
  const PPLX_GLOBAL float *ws = as_global(a.weight_scale) + (uint64_t)t.e * a.n;
  PPLX_GLOBAL O *out = as_global(reinterpret_cast<O *>(a.out)) + (int64_t)t.e * a.out_stride_expert +
                       (int64_t)(t.begin + row) * a.out_stride_row;
  float sum[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    int32_t whole = 0;
#pragma unroll
    for (int w = 0; w < kSplitWaves; ++w) whole += sums[w][(fragment * 4 + i) * 64 + lane];
    sum[i] = (float)whole * (xs * ws[n + i < a.n ? n + i : n]);
  }
  if (a.n - n >= 4) {
    typedef typename FourOf<O>::type four;
    four v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (O)sum[i];
    *reinterpret_cast<PPLX_GLOBAL four *>(out + n) = v;
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i) {
      if (i < a.n - n) out[n + i] = (O)sum[i];
    }
  }
}

template <int RF, int CF, int AHEAD, class O>
int launch_split(const MatmulDev &from, uint64_t most_blocks, hipStream_t s, pplx_a2a_int8_matmul_plan_t *plan) {
  MatmulDev a = from;
  a.n_blocks = (a.n + 16 * CF - 1) / (16 * CF);
  const uint64_t tiles = most_blocks * a.n_blocks;
  if (tiles >= (1ull << 31)) return refuse(PPLX_A2A_UNSUPPORTED, "too many tiles");
  if (plan) {
    *plan = {16 * RF, 16 * CF, 1, (uint32_t)tiles, tiles};
    return PPLX_A2A_OK;
  }
  auto kernel = matmul_split<RF, CF, AHEAD, O>;
  PPLX_LAUNCH(launch_groups(kernel, kernel, tiles, kSplitWaves * 64, 4 * a.rows.experts, s, a));
  return PPLX_A2A_OK;
}

// What a form costs, in microseconds, from the number of workgroups that its blocks make: `start` once, and for every round
// of the compute units `per_line` for each 128 bytes of k and `per_tile`, or what the weights take at `rate` megabytes a
// microsecond.  (The loads of a workgroup's steps go to LDS at some 32 bytes a cycle, which is what the lines of the tiles
// cost.)  Fitted to 3670 products of 1 to 32768 rows with 1 to 64
// experts, even and skewed, k of 256 to 16384 and n of 100 to 16384, each run in every form.  The form with the least estimate is
// on average 2 % slower than the fastest with one weight, 4 % with sorted rows, and 11 % in buffers of the experts: how their
// rows spread is known on the device only.  Without any one of the forms the fastest is 1 to 4 % slower, at worst 1.3 to 1.6 times.
// Measured, us, with the tiles of 32 x 128 / 64 x 128 / 64 x 256 / 128 x 128 / 128 x 256 / 256 x 256:
//   2816 x 2048, 64 experts   2048 rows 84 / 76 / 72 / 86 / 84 / 107      16384 278 / 250 / 204 / 184 / 175 / 170
//   4096 x 7168, 32 experts   512 rows 142 / 148 / 144 / 185 / 176 / 205  1500  214 / 165 / 153 / 199 / 187 / 211
//                             3000 309 / 262 / 218 / 215 / 200 / 227      6000  510 / 409 / 331 / 342 / 318 / 252
//   131072 x 4096, one weight 32 rows 112 / 116 / 122 / 120 / 132 / 139   128   209 / 164 / 151 / 139 / 141 / 149
// and, for few rows, split 16 x 16 / split 16 x 32 / split 32 x 32 / tiles of 32 x 128:
//   4096 x 4096   1 row 5.6 / 7.0 / 7.5 / 13.0     16 rows 7.0 / 8.5 / 9.1 / 13.2     64 rows 18.3 / 13.8 / 10.6 / 13.0
//   16384 x 4096  8 rows 16.6 / 14.4 / 15.9 / 13.5     2048 x 7168  8 rows 8.2 / 11.1 / 11.7 / 20.0
struct MatmulForm {
  uint32_t bm, bn;
  double start, per_line, per_tile, rate;
};
constexpr int kSplitForms = 3;
constexpr MatmulForm kForms[] = {
    {16, 16, 1.3, 0.10, 1.25, 5.0},  {16, 32, 1.1, 0.14, 1.77, 6.2},  {32, 32, 0.9, 0.16, 2.30, 4.5},  // split
    {32, 128, 4.4, 0.29, 0.78, 6.5}, {64, 128, 1.5, 0.34, 4.16, 6.0}, {128, 128, 5.2, 0.70, 1.07, 4.2},
    {128, 256, 0.1, 0.95, 7.01, 3.0}, {256, 256, 0.7, 1.38, 9.15, 2.8}, {64, 256, 5.7, 0.56, 3.35, 5.3},
};

int matmul_form(const MatmulDev &a) {
  const double E = a.rows.experts;
  // Of the experts' buffers an eighth is taken to be there.
  double rows = a.rows.rows;
  if (a.rows.layout == PPLX_A2A_ROWS_PADDED) rows = rows * E < 8 ? 1 : rows * E / 8;
  const double with_rows = rows < E ? rows : E, lines = (a.k + 127) / 128;
  int best = 0;
  double least = 0;
  for (int f = 0; f < (int)(sizeof(kForms) / sizeof(kForms[0])); ++f) {
    const MatmulForm &form = kForms[f];
    // (between experts of even sizes, and sizes that spread as an exponential does)
    const double blocks = a.rows.layout == PPLX_A2A_ROWS_DENSE ? (double)((a.rows.rows + form.bm - 1) / form.bm)
                                                               : with_rows / -std::expm1(-0.75 * form.bm * with_rows / rows);
    double rounds = blocks * ((a.n + form.bn - 1) / form.bn) / kComputeUnits;
    if (rounds < 1) rounds = 1;
    // (small workgroups share the units; the last round of tiles is a whole one, of which a guess at their number makes a quarter)
    if (f >= kSplitForms) rounds += (std::ceil(rounds) - rounds) * (a.rows.layout == PPLX_A2A_ROWS_DENSE ? 1.0 : 0.25);
    const double work = rounds * (lines * form.per_line + form.per_tile);
    const double weights = with_rows * a.n * a.k / (1e6 * form.rate);
    const double cost = form.start + (work < weights ? weights : work);
    if (f == 0 || cost < least) {
      best = f;
      least = cost;
    }
  }
  return best;
}

template <class O> int launch_matmul(const MatmulDev &a, hipStream_t s, pplx_a2a_int8_matmul_plan_t *plan = nullptr) {
  const uint64_t E = a.rows.experts;
  auto most_blocks = [&](uint64_t bm) -> uint64_t {  // that the rows of all experts can make
    const uint64_t rows = a.rows.rows;
    if (a.rows.layout == PPLX_A2A_ROWS_PADDED) return E * ((rows + bm - 1) / bm);
    return (rows + bm - 1) / bm + (E < rows ? E : rows) - 1;
  };
  switch (matmul_form(a)) {
    case 0: return launch_split<1, 1, 4, O>(a, most_blocks(16), s, plan);
    case 1: return launch_split<1, 2, 4, O>(a, most_blocks(16), s, plan);
    case 2: return launch_split<2, 2, 2, O>(a, most_blocks(32), s, plan);
    case 3: return launch_tiles<32, 128, 1, 4, 128, 3, O>(a, most_blocks(32), s, plan);
    case 4: return launch_tiles<64, 128, 1, 4, 128, 3, O>(a, most_blocks(64), s, plan);
    case 5: return launch_tiles<128, 128, 2, 2, 64, 4, O>(a, most_blocks(128), s, plan);
    case 6: return launch_tiles<128, 256, 2, 4, 64, 4, O>(a, most_blocks(128), s, plan);
    case 7: return launch_tiles<256, 256, 2, 4, 64, 4, O>(a, most_blocks(256), s, plan);
    default: return launch_tiles<64, 256, 1, 4, 128, 3, O>(a, most_blocks(64), s, plan);
  }
}

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

namespace {
int check_matmul_size(uint64_t n, uint64_t k) {
  PPLX_REQUIRE(n < (1ull << 31), "n must be below 2^31");
  PPLX_REQUIRE(k > 0 && k % 16 == 0 && k <= 131056, "k must be a multiple of 16 in [16, 131056]");
  return PPLX_A2A_OK;
}
}  // namespace

extern "C" int pplx_a2a_int8_matmul_plan(const pplx_a2a_rows_t *rows, uint64_t n, uint64_t k, pplx_a2a_int8_matmul_plan_t *out) {
  PPLX_REQUIRE(rows && out, "rows or out is NULL");
  MatmulDev a{};
  int st = check_row_numbers(*rows, &a.rows);
  if (!st) st = check_matmul_size(n, k);
  if (st) return st;
  a.n = (uint32_t)n;
  a.k = (uint32_t)k;
  *out = {};
  return a.rows.rows == 0 || n == 0 ? (int)PPLX_A2A_OK : launch_matmul<float>(a, nullptr, out);
}

extern "C" int pplx_a2a_int8_matmul(int device, const pplx_a2a_int8_matmul_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_int8_matmul_args_t &p = *args;
  MatmulDev a{};
  int st = check_rows(p.rows, &a.rows);
  if (st) return st;
  PPLX_REQUIRE(is_dtype(p.out_dtype), "unsupported dtype of out");
  st = check_matmul_size(p.n, p.k);
  if (st) return st;
  if (p.rows.rows == 0 || p.n == 0) return PPLX_A2A_OK;
  PPLX_REQUIRE(p.out && p.x && p.x_scale && p.weight && p.weight_scale, "out / x / x_scale / weight / weight_scale is NULL");
  PPLX_REQUIRE(is_aligned(p.x, 16) && p.x_stride_row % 16 == 0 && p.x_stride_expert % 16 == 0,
               "x must be 16-byte aligned with 16-byte strides");
  if (p.x_stride_row < 0 || p.x_stride_row >= (1 << 23))  // (a tile's rows are reached by 32-bit offsets)
    return refuse(PPLX_A2A_UNSUPPORTED, "rows of x must be less than 8 MiB apart");
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
  a.large_weights = (uint64_t)a.rows.experts * p.n * p.k > (96ull << 20);
  return guarded(device, [&] {
    return with_type(p.out_dtype, [&](auto tag) { return launch_matmul<typename decltype(tag)::type>(a, (hipStream_t)stream); });
  });
}
