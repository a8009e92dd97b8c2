// Tiles that loads write to LDS directly: what the kernels of the products share.  Included only by the .hip sources.
#pragma once
#include "a2a_common.h"

namespace pplx_amd {
namespace {

constexpr uint32_t kComputeUnits = 256;

#define PPLX_CONSTANT __attribute__((address_space(4)))

// Waits until at most LEFT of the wave's loads are under way, and for its LDS reads where asked to.
template <int LEFT, bool LDS = false> __device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((LEFT & 15) | ((LEFT >> 4) << 14) | (7 << 4) | ((LDS ? 0 : 15) << 8));
  asm volatile("" ::: "memory");
}

// Sixteen bytes a lane from `base` + `offset` to LDS, lane i's at `lds` + 16 i; `lanes` is ~0, or 0 for a load that only
// counts.  (asm: behind the builtin the compiler waits for the loads of the steps to come before it reads the step at
// hand out of LDS.  Nothing is returned to registers, and the kernel waits by itself.  All lanes are active where it
// stands.  The load wants one wait state behind the write of m0, and five behind a vector instruction that wrote the
// registers of `base`, of which the compiler keeps count for its own loads only.)
__device__ __forceinline__ void load_to_lds(const int8_t *base, uint32_t offset, uint32_t lds, uint32_t lanes) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_mov_b32 exec_lo, %3\n\t"
      "s_mov_b32 exec_hi, %3\n\t"
      "s_nop 1\n\t"
      "global_load_lds_dwordx4 %0, %1\n\t"
      "s_mov_b64 exec, -1"
      ::"v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds)), "s"(__builtin_amdgcn_readfirstlane(lanes))
      : "memory");
}

// The same, past the caches if `past`.  (The branch stands in the asm: one of the compiler's, between the matrix instructions,
// costs registers.)
__device__ __forceinline__ void load_past_to_lds(const int8_t *base, uint32_t offset, uint32_t lds, uint32_t lanes, uint32_t past) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_cmp_eq_u32 %4, 0\n\t"
      "s_mov_b32 exec_lo, %3\n\t"
      "s_mov_b32 exec_hi, %3\n\t"
      "s_cbranch_scc1 .Lkept%=\n\t"
      "s_nop 1\n\t"
      "global_load_lds_dwordx4 %0, %1 nt\n\t"
      "s_branch .Lloaded%=\n"
      ".Lkept%=:\n\t"
      "s_nop 1\n\t"
      "global_load_lds_dwordx4 %0, %1\n"
      ".Lloaded%=:\n\t"
      "s_mov_b64 exec, -1"
      ::"v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds)), "s"(__builtin_amdgcn_readfirstlane(lanes)),
        "s"(__builtin_amdgcn_readfirstlane(past))
      : "memory", "scc");
}

__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}

// The steps in flight take 128 KiB of a compute unit's LDS; what else a workgroup has there lies behind them.
constexpr uint32_t kLdsBytes = 128 * 1024;

}  // namespace
}  // namespace pplx_amd
