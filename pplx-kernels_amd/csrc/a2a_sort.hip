// Tokens sorted by expert: a stable counting sort of the picks by (expert, token, pick) and the copies of the tokens' rows,
// quantised on the way if asked for.  Everything is placed by counting, no atomic's order decides where a row goes.
//
// Few picks: one launch.  Every workgroup counts all picks by expert in LDS (and, of those, the picks in front of its own
// tokens), which costs it one read of indices that the L2 holds, and then copies its tokens.
// Many picks: three launches.  Tiles of picks are counted into the workspace, then every tile sums the counts of all
// tiles (at most 64 of them) and gives its picks their slots, and then the rows are copied.
#include "a2a_experts.h"

namespace pplx_amd {
namespace {

struct SortDev {
  const uint8_t *x;
  int64_t x_stride_row;
  const uint32_t *indices;
  const uint32_t *bound_m;
  uint8_t *rows;
  int64_t rows_stride;
  float *scale;
  int32_t *slots;
  int32_t *offsets;
  uint32_t *tile_counts;  // [tiles][E]
  uint32_t m, K, E, width;  // width: elements of a row
  uint32_t row_vecs;        // 16-byte vectors of a row of x
  uint32_t tile, tiles;     // picks of a tile, tiles
  uint32_t first_group;
};

__device__ __forceinline__ uint32_t tokens_there(const SortDev &a) {
  if (!a.bound_m) return a.m;
  const uint32_t n = *as_global(a.bound_m);
  return n < a.m ? n : a.m;
}

// The lanes of the wave whose value of `id` is this lane's, among those of `live`.
__device__ __forceinline__ uint64_t same_id(uint32_t id, uint64_t live, uint32_t bits) {
  uint64_t mask = live;
  for (uint32_t b = 0; b < bits; ++b) {
    const bool set = (id >> b) & 1u;
    const uint64_t with = __ballot(set);
    mask &= set ? with : ~with;
  }
  return mask;
}
__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Exclusive sums of counts[0..E) over the experts, written to out[0..E) (which may be counts), by all threads of the
// workgroup; returns the sum of all.  `of_wave` holds a word for each wave.
template <int THREADS>
__device__ __forceinline__ uint32_t scan_experts(const uint32_t *counts, uint32_t *out, uint32_t E, uint32_t *of_wave) {
  const uint32_t per = (E + THREADS - 1) / THREADS, first = threadIdx.x * per;
  const uint32_t lane = lane_id(), wave = wave_id();
  uint32_t own = 0;
  for (uint32_t i = 0; i < per; ++i) own += first + i < E ? counts[first + i] : 0u;
  const uint32_t upto = wave_scan(own, lane);
  if (lane == 63) of_wave[wave] = upto;
  __syncthreads();
  uint32_t before = upto - own, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const uint32_t n = of_wave[w];
    before += (uint32_t)w < wave ? n : 0u;
    total += n;
  }
  for (uint32_t i = 0; i < per; ++i) {
    if (first + i < E) {
      const uint32_t n = counts[first + i];
      out[first + i] = before;
      before += n;
    }
  }
  __syncthreads();
  return total;
}

// Rows are stored through to memory at agent scope and stay in the last-level cache as far as it goes.  8192 tokens x 8
// rows of 14 KiB, us: so 214, non-temporal 225, non-temporal through 220, plain 218; whole rows in a wave's registers
// 220-227, four to sixteen waves to a compute unit 213-227.  5.2 TB/s, of which eight parts in nine are writes to rows
// all over the buffer, is what the memory takes of these.
//
// The copies of one token's row, by LANES threads of which `g` is this one's number.  Lane k of every wave holds the
// slot of pick k; rows t * K + k from `total` on are the ones that nobody else fills.
template <int LANES>
__device__ __forceinline__ void copy_row(const SortDev &a, uint32_t t, int32_t slot, uint32_t total, uint32_t g) {
  const uint32_t lane = lane_id();
  const uint32_t spare = t * a.K + lane;
  uint64_t live = __ballot(lane < a.K && slot >= 0);
  uint64_t empty = __ballot(lane < a.K && spare >= total);
  constexpr int NV = 4;
  const PPLX_GLOBAL u32x4 *row = as_global(reinterpret_cast<const u32x4 *>(a.x + (int64_t)t * a.x_stride_row));
  for (uint32_t base = 0; base < a.row_vecs; base += LANES * NV) {
    if (live) {
      u32x4 v[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const uint32_t j = base + i * LANES + g;
        v[i] = row[j < a.row_vecs ? j : a.row_vecs - 1];
      }
      SettleAll<NV>::of(v);
      for (uint64_t left = live; left; left &= left - 1) {
        const uint32_t s = (uint32_t)__builtin_amdgcn_readlane(slot, __builtin_ctzll(left));
        PPLX_GLOBAL u32x4 *out = as_global(reinterpret_cast<u32x4 *>(a.rows + (int64_t)s * a.rows_stride));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const uint32_t j = base + i * LANES + g;
          if (j < a.row_vecs) row_store<RowStore::kKeep>(v[i], out + j);
        }
      }
    }
    for (uint64_t left = empty; left; left &= left - 1) {
      const uint32_t r = t * a.K + (uint32_t)__builtin_ctzll(left);
      PPLX_GLOBAL u32x4 *out = as_global(reinterpret_cast<u32x4 *>(a.rows + (int64_t)r * a.rows_stride));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const uint32_t j = base + i * LANES + g;
        if (j < a.row_vecs) row_store<RowStore::kKeep>(u32x4{0, 0, 0, 0}, out + j);
      }
    }
  }
}

// The same with quantised copies.  Up to 32 * LANES elements of the row stay in registers between the search for its
// largest value and its conversion, longer rows are read twice.
template <int LANES, class T>
__device__ __forceinline__ void quantize_row(const SortDev &a, uint32_t t, int32_t slot, uint32_t total, uint32_t g) {
  const uint32_t lane = lane_id();
  const uint32_t spare = t * a.K + lane;
  const uint64_t live = __ballot(lane < a.K && slot >= 0);
  const uint64_t empty = __ballot(lane < a.K && spare >= total);
  constexpr int NS = 2;
  const PPLX_GLOBAL T *row = as_global(reinterpret_cast<const T *>(a.x + (int64_t)t * a.x_stride_row));
  const uint32_t groups = a.width / 16;
  const bool held = groups <= LANES * NS;
  f32x8 v[2 * NS];
  uint32_t bits = 0;
  if (live) {
    for (uint32_t base = 0; base < groups; base += LANES * NS) {
      typename Eight<T>::raw raw[2 * NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        uint32_t j = base + i * LANES + g;
        j = j < groups ? j : groups - 1;
        raw[2 * i] = load_eight<T>(row + 16ull * j);
        raw[2 * i + 1] = load_eight<T>(row + 16ull * j + 8);
      }
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        v[i] = Eight<T>::wide(raw[i]);
        const uint32_t b = magnitude_bits(v[i]);
        bits = bits > b ? bits : b;
      }
    }
  }
  const RowScale s = row_scale(row_max<LANES>(bits));
  // lane k writes the scale of pick k (the first wave of the row, once)
  if (g < 64 && lane < a.K) {
    PPLX_GLOBAL float *scale = as_global(a.scale);
    if (slot >= 0) scale[slot] = s.scale;
    if (spare >= total) scale[spare] = 0.f;
  }
  for (uint32_t base = 0; base < groups; base += LANES * NS) {
    u32x4 q[NS];
    if (live) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        if (!held) {
          uint32_t j = base + i * LANES + g;
          j = j < groups ? j : groups - 1;
          v[2 * i] = Eight<T>::wide(load_eight<T>(row + 16ull * j));
          v[2 * i + 1] = Eight<T>::wide(load_eight<T>(row + 16ull * j + 8));
        }
        q[i] = quantize_sixteen(v[2 * i], v[2 * i + 1], s.inverse);
      }
      for (uint64_t left = live; left; left &= left - 1) {
        const uint32_t r = (uint32_t)__builtin_amdgcn_readlane(slot, __builtin_ctzll(left));
        PPLX_GLOBAL u32x4 *out = as_global(reinterpret_cast<u32x4 *>(a.rows + (int64_t)r * a.rows_stride));
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const uint32_t j = base + i * LANES + g;
          if (j < groups) row_store<RowStore::kKeep>(q[i], out + j);
        }
      }
    }
    for (uint64_t left = empty; left; left &= left - 1) {
      const uint32_t r = t * a.K + (uint32_t)__builtin_ctzll(left);
      PPLX_GLOBAL u32x4 *out = as_global(reinterpret_cast<u32x4 *>(a.rows + (int64_t)r * a.rows_stride));
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const uint32_t j = base + i * LANES + g;
        if (j < groups) row_store<RowStore::kKeep>(u32x4{0, 0, 0, 0}, out + j);
      }
    }
  }
}

// T: the element type of quantised rows, void for copies.
template <int LANES, class T>
__device__ __forceinline__ void place_row(const SortDev &a, uint32_t t, int32_t slot, uint32_t total, uint32_t g) {
  if constexpr (std::is_void_v<T>) copy_row<LANES>(a, t, slot, total, g);
  else quantize_row<LANES, T>(a, t, slot, total, g);
}

// One launch: `per` tokens to a workgroup of 256 threads, 256 / LANES of them at a time.
constexpr uint32_t kMaxPer = 16;
template <int LANES, class T>
__global__ __launch_bounds__(256) void sort_one_launch(SortDev a, uint32_t per, uint32_t id_bits) {
  extern __shared__ uint32_t tables[];  // [E] picks from this workgroup's on, then first rows; [E] picks in front of them
  __shared__ uint32_t of_wave[4];
  __shared__ int32_t own_slots[kMaxPer * 64];
  uint32_t *all = tables, *before = tables + a.E;
  const uint32_t lane = lane_id(), wave = wave_id();
  const uint32_t t0 = blockIdx.x * per;
  const uint32_t n = tokens_there(a);
  const uint32_t picks = n * a.K, first = t0 * a.K;
  for (uint32_t e = threadIdx.x; e < 2 * a.E; e += 256) tables[e] = 0;
  __syncthreads();
  const PPLX_GLOBAL uint32_t *idx = as_global(a.indices);
  constexpr uint32_t kAtOnce = 8;  // loads in flight
  for (uint32_t base = 0; base < picks; base += 256 * kAtOnce) {
    uint32_t e[kAtOnce];
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) {
      const uint32_t p = base + u * 256 + threadIdx.x;
      e[u] = p < picks ? idx[p] : a.E;
    }
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) {
      if (e[u] < a.E) atomicAdd(base + u * 256 + threadIdx.x < first ? &before[e[u]] : &all[e[u]], 1u);
    }
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < a.E; e += 256) all[e] += before[e];
  __syncthreads();
  const uint32_t total = scan_experts<256>(all, all, a.E, of_wave);
  if (blockIdx.x == 0) {
    for (uint32_t e = threadIdx.x; e < a.E; e += 256) as_global(a.offsets)[e] = (int32_t)all[e];
    if (threadIdx.x == 0) as_global(a.offsets)[a.E] = (int32_t)total;
  }
  const uint32_t tokens = a.m - t0 < per ? a.m - t0 : per;  // (the grid has no workgroup behind the last token)
  if (wave == 0) {
    const uint32_t own = tokens * a.K;
    for (uint32_t base = 0; base < own; base += 64) {
      const uint32_t p = first + base + lane;
      const bool there = base + lane < own && p < picks;
      const uint32_t e = there ? idx[p] : a.E;
      const bool live = e < a.E;
      const uint64_t same = same_id(e, __ballot(live), id_bits);
      int32_t slot = -1;
      if (live) {
        const uint32_t leader = (uint32_t)__builtin_ctzll(same);
        slot = (int32_t)(all[e] + before[e] + lanes_below(same));
        __builtin_amdgcn_wave_barrier();
        if (lane == leader) atomicAdd(&before[e], (uint32_t)__builtin_popcountll(same));
        __builtin_amdgcn_wave_barrier();
      }
      if (base + lane < own) {
        own_slots[base + lane] = slot;
        as_global(a.slots)[p] = slot;
      }
    }
  }
  __syncthreads();
  constexpr uint32_t kRowsAtOnce = 256 / LANES;
  const uint32_t g = threadIdx.x % LANES;
  for (uint32_t i = 0; i < per; i += kRowsAtOnce) {
    const uint32_t mine = i + (LANES == 64 ? wave : 0);
    if (mine >= tokens) break;  // (with 256 lanes to a row the whole workgroup leaves)
    const int32_t slot = lane < a.K ? own_slots[mine * a.K + lane] : -1;
    place_row<LANES, T>(a, t0 + mine, slot, total, g);
  }
}

// Many picks, first launch: the picks of each tile by expert.
__global__ __launch_bounds__(1024) void sort_count(SortDev a) {
  extern __shared__ uint32_t counts[];
  const uint32_t picks = tokens_there(a) * a.K;
  const uint32_t first = blockIdx.x * a.tile;
  const uint32_t end = first + a.tile < picks ? first + a.tile : picks;
  for (uint32_t e = threadIdx.x; e < a.E; e += 1024) counts[e] = 0;
  __syncthreads();
  for (uint32_t p = first + threadIdx.x; p < end; p += 1024) {
    const uint32_t e = as_global(a.indices)[p];
    if (e < a.E) atomicAdd(&counts[e], 1u);
  }
  __syncthreads();
  PPLX_GLOBAL uint32_t *out = as_global(a.tile_counts) + (size_t)blockIdx.x * a.E;
  for (uint32_t e = threadIdx.x; e < a.E; e += 1024) out[e] = counts[e];
}

// Second launch: the slots of each tile's picks.  Each of the WAVES waves takes a part of the tile's picks that are
// consecutive, counts them first, and then goes through them 64 at a time.
template <int WAVES>
__global__ __launch_bounds__(WAVES * 64) void sort_slots(SortDev a, uint32_t id_bits) {
  extern __shared__ uint32_t tables[];  // [E] first rows of the experts, then for each wave [E] its next rows behind those
  __shared__ uint32_t of_wave[WAVES];
  uint32_t *start = tables, *next = tables + a.E;
  const uint32_t lane = lane_id(), wave = wave_id();
  const uint32_t picks = tokens_there(a) * a.K, all_picks = a.m * a.K;
  const uint32_t part = a.tile / WAVES;  // (a multiple of 64)
  const uint32_t first = blockIdx.x * a.tile + wave * part;
  const PPLX_GLOBAL uint32_t *idx = as_global(a.indices);
  for (uint32_t e = threadIdx.x; e < WAVES * a.E; e += WAVES * 64) next[e] = 0;
  __syncthreads();
  uint32_t *own = next + (size_t)wave * a.E;
  for (uint32_t i = lane; i < part; i += 64) {
    const uint32_t p = first + i;
    const uint32_t e = p < picks ? idx[p] : a.E;
    if (e < a.E) atomicAdd(&own[e], 1u);
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < a.E; e += WAVES * 64) {
    // (sixteen tiles' counts in flight: one behind the other they are 64 trips to the L2)
    uint32_t all = 0, row = 0;
    constexpr uint32_t kAtOnce = 16;
    for (uint32_t i = 0; i < a.tiles; i += kAtOnce) {
      uint32_t n[kAtOnce];
#pragma unroll
      for (uint32_t u = 0; u < kAtOnce; ++u) {
        n[u] = as_global(a.tile_counts)[(size_t)(i + u < a.tiles ? i + u : 0) * a.E + e];
      }
#pragma unroll
      for (uint32_t u = 0; u < kAtOnce; ++u) {
        all += i + u < a.tiles ? n[u] : 0;
        row += i + u < blockIdx.x ? n[u] : 0;
      }
    }
    start[e] = all;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const uint32_t n = next[(size_t)w * a.E + e];
      next[(size_t)w * a.E + e] = row;
      row += n;
    }
  }
  __syncthreads();
  const uint32_t total = scan_experts<WAVES * 64>(start, start, a.E, of_wave);
  if (blockIdx.x == 0) {
    for (uint32_t e = threadIdx.x; e < a.E; e += WAVES * 64) as_global(a.offsets)[e] = (int32_t)start[e];
    if (threadIdx.x == 0) as_global(a.offsets)[a.E] = (int32_t)total;
  }
  for (uint32_t i = lane; i < part; i += 64) {
    const uint32_t p = first + i;
    if (p - lane >= all_picks) break;
    const uint32_t e = p < picks ? idx[p] : a.E;
    const bool live = e < a.E;
    const uint64_t same = same_id(e, __ballot(live), id_bits);
    int32_t slot = -1;
    if (live) {
      const uint32_t leader = (uint32_t)__builtin_ctzll(same);
      slot = (int32_t)(start[e] + own[e] + lanes_below(same));
      __builtin_amdgcn_wave_barrier();
      if (lane == leader) atomicAdd(&own[e], (uint32_t)__builtin_popcountll(same));
      __builtin_amdgcn_wave_barrier();
    }
    if (p < all_picks) as_global(a.slots)[p] = slot;
  }
}

// Third launch: the rows.  LATER: workgroups behind those of one launch.  (Two scalar instructions that add first_group, a
// zero, to the number of the workgroup cost 8192 tokens x 8 rows of 14 KiB 6 of 195 us, in whatever way they are written.)
template <int LANES, class T, bool LATER>
__global__ __launch_bounds__(256) void sort_rows(SortDev a) {
  const uint32_t lane = lane_id();
  const uint32_t group = LATER ? a.first_group + blockIdx.x : blockIdx.x;
  const uint32_t t = LANES == 64 ? group * 4 + wave_id() : group;
  if (t >= a.m) return;  // (with 256 lanes to a row the grid has one workgroup a token)
  const uint32_t total = (uint32_t)as_global(a.offsets)[a.E];
  const int32_t slot = lane < a.K ? as_global(a.slots)[(size_t)t * a.K + lane] : -1;
  place_row<LANES, T>(a, t, slot, total, threadIdx.x % LANES);
}

// us a call, one launch / three: 1024 x 8 picks of rows of 4 KiB 10.2 / 14.9, 2048 x 4 of 8 KiB 17.8 / 19.7; beyond, 2048 x 6 of
// quantised 8 KiB 20.3 / 19.1, 8192 x 2 of 8 KiB (with the gradients) 185.6 / 181.3.
constexpr uint32_t kOneLaunchPicks = 8192;
constexpr uint32_t kMaxTiles = 64;

uint32_t sort_waves(uint32_t E) {
  return E <= 963 ? 16 : E <= 1820 ? 8 : 2;  // (waves + 1) * E words in 64 KiB
}
void sort_tiling(uint32_t picks, uint32_t E, uint32_t *tile, uint32_t *tiles) {
  *tile = *tiles = 0;
  if (picks <= kOneLaunchPicks) return;
  const uint32_t unit = sort_waves(E) * 64;
  uint32_t per = (picks + kMaxTiles - 1) / kMaxTiles;
  per = (per + unit - 1) / unit * unit;
  *tile = per;
  *tiles = (picks + per - 1) / per;
}

template <int LANES, class T> int launch_sort(const SortDev &a, hipStream_t s) {
  uint32_t bits = 0;
  while ((1u << bits) < a.E) ++bits;
  if (a.tiles == 0) {
    // a token to a workgroup until there are two workgroups to a compute unit
    uint32_t per = (a.m + 511) / 512;
    const uint32_t at_once = 256 / LANES;
    per = per < at_once ? at_once : per > kMaxPer ? kMaxPer : per;
    const uint32_t groups = a.m ? (a.m + per - 1) / per : 1;  // (without tokens the offsets are still written)
    PPLX_LAUNCH(launch_kernel(sort_one_launch<LANES, T>, dim3(groups), dim3(256), 8 * a.E, s, a, per, bits));
    return PPLX_A2A_OK;
  }
  PPLX_LAUNCH(launch_kernel(sort_count, dim3(a.tiles), dim3(1024), 4 * a.E, s, a));
  const uint32_t waves = sort_waves(a.E), lds = 4 * (waves + 1) * a.E;
  const dim3 grid(a.tiles), block(waves * 64);
  if (waves == 16) PPLX_LAUNCH(launch_kernel(sort_slots<16>, grid, block, lds, s, a, bits));
  else if (waves == 8) PPLX_LAUNCH(launch_kernel(sort_slots<8>, grid, block, lds, s, a, bits));
  else PPLX_LAUNCH(launch_kernel(sort_slots<2>, grid, block, lds, s, a, bits));
  PPLX_LAUNCH(launch_groups(sort_rows<LANES, T, false>, sort_rows<LANES, T, true>, LANES == 64 ? (a.m + 3) / 4 : a.m, 256, 0, s, a));
  return PPLX_A2A_OK;
}

template <class T> int launch_sort_form(const SortDev &a, hipStream_t s) {
  const bool wave_rows = std::is_void_v<T> ? a.row_vecs <= 256 : a.width <= 2048;  // what its registers hold
  return wave_rows ? launch_sort<64, T>(a, s) : launch_sort<256, T>(a, s);
}

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

namespace {
int check_sort_size(uint64_t m, uint64_t K, uint64_t E) {
  PPLX_REQUIRE(K >= 1 && K <= 64, "experts_per_token must be in [1, 64]");
  PPLX_REQUIRE(E >= 1 && E <= kMaxExperts, "num_experts must be in [1, %u]", kMaxExperts);
  if (m * K >= (1ull << 31)) return refuse(PPLX_A2A_UNSUPPORTED, "2^31 picks or more");
  return PPLX_A2A_OK;
}
}  // namespace

extern "C" int pplx_a2a_sort_workspace(uint32_t m, uint32_t experts_per_token, uint32_t num_experts, uint64_t *bytes) {
  PPLX_REQUIRE(bytes, "bytes is NULL");
  const int st = check_sort_size(m, experts_per_token, num_experts);
  if (st) return st;
  uint32_t tile, tiles;
  sort_tiling(m * experts_per_token, num_experts, &tile, &tiles);
  *bytes = 4ull * tiles * num_experts;
  return PPLX_A2A_OK;
}

extern "C" int pplx_a2a_sort_tokens(int device, const pplx_a2a_sort_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_sort_args_t &p = *args;
  int st = check_sort_size(p.m, p.experts_per_token, p.num_experts);
  if (st) return st;
  PPLX_REQUIRE(is_dtype(p.dtype), "unsupported dtype of x");
  PPLX_REQUIRE(p.offsets && is_aligned(p.offsets, 4), "offsets is NULL or not aligned");
  const uint64_t x_bytes = p.hidden_dim * (uint64_t)dtype_bytes(p.dtype);
  const uint64_t out_bytes = p.out_scale ? p.hidden_dim : x_bytes;
  PPLX_REQUIRE(p.hidden_dim > 0 && p.hidden_dim < (1ull << 28) && x_bytes % 16 == 0 && out_bytes % 16 == 0,
               "rows must be multiples of 16 bytes, shorter than 2^28 elements");
  if (p.m > 0) {
    PPLX_REQUIRE(p.x && p.indices && p.out_rows && p.slots, "x / indices / out_rows / slots is NULL with m > 0");
    PPLX_REQUIRE(is_aligned(p.x, 16) && p.x_stride_row % 16 == 0, "x must be 16-byte aligned with a 16-byte row stride");
    PPLX_REQUIRE(is_aligned(p.out_rows, 16) && p.out_stride_row % 16 == 0,
                 "out_rows must be 16-byte aligned with a 16-byte row stride");
    PPLX_REQUIRE(is_aligned(p.indices, 4) && is_aligned(p.bound_m, 4) && is_aligned(p.slots, 4) && is_aligned(p.out_scale, 4),
                 "indices, bound_m, slots and out_scale must be aligned to their elements");
  }
  SortDev a{};
  a.x = static_cast<const uint8_t *>(p.x);
  a.x_stride_row = p.x_stride_row;
  a.indices = p.indices;
  a.bound_m = p.bound_m;
  a.rows = static_cast<uint8_t *>(p.out_rows);
  a.rows_stride = p.out_stride_row;
  a.scale = p.out_scale;
  a.slots = p.slots;
  a.offsets = p.offsets;
  a.m = p.m;
  a.K = p.experts_per_token;
  a.E = p.num_experts;
  a.width = (uint32_t)p.hidden_dim;
  a.row_vecs = (uint32_t)(x_bytes / 16);
  sort_tiling(a.m * a.K, a.E, &a.tile, &a.tiles);
  PPLX_REQUIRE(a.tiles == 0 || (p.workspace && is_aligned(p.workspace, 4)), "workspace is NULL or not aligned");
  a.tile_counts = static_cast<uint32_t *>(p.workspace);
  return guarded(device, [&] {
    hipStream_t s = (hipStream_t)stream;
    if (!p.out_scale || a.m == 0) return launch_sort_form<void>(a, s);
    return with_type(p.dtype, [&](auto tag) { return launch_sort_form<typename decltype(tag)::type>(a, s); });
  });
}
