/*
 * pplx_a2a.h -- C ABI of the MI355X (gfx950) MoE dispatch / combine library.
 *
 * This is the boundary a host-language binding attaches to.  Every entry point
 * takes plain pointers, sizes and strides; no torch / C++ types cross it.  The
 * library replaces the host classes and kernels of ppl-ai/pplx-kernels'
 * intranode all-to-all for a single-GPU loopback: all `world_size` simulated
 * expert-parallel (EP) ranks live in one process and one GPU's HBM.
 *
 * Reference interfaces replaced (paths relative to the reference tree):
 *   csrc/all_to_all/all_to_all.h:9-13    SplitMode                -> pplx_a2a_split_mode
 *   csrc/all_to_all/all_to_all.h:29-39   AllToAll ctor arguments  -> pplx_a2a_config_t
 *   csrc/all_to_all/intranode.h:23-63    AllToAllIntraNode        -> pplx_a2a_t + dispatch/combine
 *   csrc/core/buffer.h:116-161           Strided1D/2D/3D views    -> pointer + stride fields
 *   csrc/bindings/all_to_all_ops.cpp:54-108,122-196,238-311  create/destroy/dispatch/combine ops
 *
 * Conventions
 *   - Every function returns a pplx_a2a_status; 0 is success.  The library never
 *     exits or traps; pplx_a2a_last_error() returns the message of the calling
 *     thread's last failure.
 *   - Device pointers are HBM addresses on the world's device.  `stream` is a
 *     hipStream_t passed as void* (NULL = the legacy default stream).
 *   - Only *_create, *_destroy and pplx_a2a_world_reserve_split allocate, free
 *     or synchronise (pplx_a2a_world_faults synchronises the stream it reads
 *     behind); dispatch / combine only enqueue kernels, so they may be captured
 *     in a hipGraph and replayed.
 *   - Outputs of a send+recv step made of per-rank calls are valid once the
 *     LAST rank's call has returned, in stream order of any stream a rank of
 *     the step called on.
 */
#ifndef PPLX_A2A_H_
#define PPLX_A2A_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum pplx_a2a_status {
  PPLX_A2A_OK = 0,
  PPLX_A2A_INVALID_ARGUMENT = 1, /* a precondition on the arguments does not hold */
  PPLX_A2A_INVALID_STATE = 2,    /* call order violated (e.g. RECV before every SEND) */
  PPLX_A2A_HIP_ERROR = 3,        /* a HIP runtime call failed */
  PPLX_A2A_UNSUPPORTED = 4       /* valid request that this build cannot serve */
} pplx_a2a_status;

/* csrc/all_to_all/all_to_all.h:9-13 */
typedef enum pplx_a2a_split_mode {
  PPLX_A2A_SPLIT_NONE = 0, /* send and receive in one call */
  PPLX_A2A_SPLIT_SEND = 1,
  PPLX_A2A_SPLIT_RECV = 2
} pplx_a2a_split_mode;

/* element types of combine: csrc/bindings/all_to_all_ops.cpp:265-310 */
typedef enum pplx_a2a_dtype {
  PPLX_A2A_F32 = 0,
  PPLX_A2A_BF16 = 1,
  PPLX_A2A_F16 = 2
} pplx_a2a_dtype;

/* The AllToAll constructor arguments, csrc/all_to_all/all_to_all.h:29-39.
 * Invariants checked at world creation (csrc/all_to_all/all_to_all.cpp:32-39):
 * hidden_dim_bytes % 16 == 0, hidden_dim_scale_bytes % 16 == 0,
 * hidden_dim_scale_bytes <= hidden_dim_bytes, num_experts % world_size == 0,
 * world_size % dp_size == 0.  Unlike the reference a single DP group
 * (world_size == dp_size) is accepted. */
typedef struct pplx_a2a_config {
  uint64_t max_num_tokens;         /* M: max tokens per DP group per step */
  uint64_t num_experts;            /* E: global expert count */
  uint64_t experts_per_token;      /* K: top-k */
  uint32_t world_size;             /* R: number of simulated EP ranks */
  uint32_t dp_size;                /* ranks per DP group (hold identical tokens) */
  uint64_t hidden_dim;             /* H: elements per token row */
  uint64_t hidden_dim_bytes;       /* bytes of one dispatched activation row */
  uint64_t hidden_dim_scale_bytes; /* bytes of one row of fp32 block scales, 0 if none */
} pplx_a2a_config_t;

/* Owner of the state shared by all simulated ranks (routing tables, slot map,
 * staging for split mode).  Takes the place of the IPC-mapped peer buffers set
 * up in csrc/all_to_all/intranode.cpp:11-137. */
typedef struct pplx_a2a_world pplx_a2a_world_t;
/* One simulated EP rank; takes the place of an AllToAllIntraNode object. */
typedef struct pplx_a2a pplx_a2a_t;
/* An instantiated hipGraph. */
typedef struct pplx_a2a_graph pplx_a2a_graph_t;
typedef struct pplx_a2a_bound pplx_a2a_bound_t;

/* Arguments of one rank's dispatch: the views built in
 * csrc/bindings/all_to_all_ops.cpp:165-195 for AllToAllIntraNode::dispatch
 * (csrc/all_to_all/intranode.h:39-50). */
typedef struct pplx_a2a_dispatch_args {
  int32_t *out_expert_num_tokens;        /* [L] */
  int64_t out_expert_num_tokens_stride;  /* elements */
  void *out_expert_x;                    /* [L, rows, hidden_dim_bytes] */
  int64_t out_expert_x_stride_row;       /* bytes between rows */
  int64_t out_expert_x_stride_expert;    /* bytes between local experts */
  int64_t out_expert_x_rows;             /* size(1): row capacity per expert; 0 = M * num_dp_groups */
  float *out_expert_x_scale;             /* [L, rows, S] or NULL */
  int64_t out_expert_x_scale_stride_elem;   /* floats */
  int64_t out_expert_x_scale_stride_row;    /* floats */
  int64_t out_expert_x_scale_stride_expert; /* floats */
  const void *dp_x;                      /* [m, hidden_dim_bytes] */
  int64_t dp_x_stride_row;               /* bytes */
  const float *dp_x_scale;               /* [m, S] or NULL */
  int64_t dp_x_scale_stride_elem;        /* floats */
  int64_t dp_x_scale_stride_row;         /* floats */
  const uint32_t *indices;               /* [m, K] contiguous */
  uint32_t m;                            /* rows of dp_x / indices */
  const uint32_t *bound_m;               /* device scalar: tokens actually present, or NULL (= m) */
} pplx_a2a_dispatch_args_t;

/* Arguments of one rank's combine: the views built in
 * csrc/bindings/all_to_all_ops.cpp:222-235 for AllToAllIntraNode::combine<T,U>
 * (csrc/all_to_all/intranode.h:53-63).  Strides are in elements. */
typedef struct pplx_a2a_combine_args {
  void *out_tokens;                 /* [>= m, H] of out_dtype */
  int64_t out_tokens_stride_row;
  int32_t out_dtype;                /* pplx_a2a_dtype: BF16 or F16 */
  const uint32_t *indices;          /* [m, K] contiguous */
  const float *weights;             /* [m, K] */
  int64_t weights_stride_row;
  const void *expert_y;             /* [L, rows, H] of in_dtype */
  int64_t expert_y_stride_row;
  int64_t expert_y_stride_expert;
  int64_t expert_y_rows;            /* size(1); 0 = M * num_dp_groups */
  int32_t in_dtype;                 /* pplx_a2a_dtype: F32, BF16 or F16 */
  uint32_t m;
  const uint32_t *bound_m;          /* device scalar or NULL (= m) */
} pplx_a2a_combine_args_t;

/* ---- lifecycle ------------------------------------------------------- */

/* Allocates the world's device state on `device` (a HIP device ordinal): with
 * T = world_size / dp_size * max_num_tokens, a slot map of T * experts_per_token * 4
 * bytes and routing tables of about T * num_experts / 8 bytes (the 8192-token
 * DSv3 shape: 2 MiB + 2.3 MiB), plus rank tables for worlds of more than 64 ranks.
 * Replaces the buffer set-up of csrc/all_to_all/intranode.cpp:11-137. */
int pplx_a2a_world_create(const pplx_a2a_config_t *cfg, int device, pplx_a2a_world_t **out);
/* Frees the world.  Fails with INVALID_STATE while rank handles are attached. */
int pplx_a2a_world_destroy(pplx_a2a_world_t *world);

/* Attaches simulated rank `rank`; replaces create_intranode,
 * csrc/bindings/all_to_all_ops.cpp:79-106. */
int pplx_a2a_create(pplx_a2a_world_t *world, uint32_t rank, pplx_a2a_t **out);
/* Replaces destroy, csrc/bindings/all_to_all_ops.cpp:108. */
int pplx_a2a_destroy(pplx_a2a_t *handle);
/* AllToAll::getNumExpertsPerToken, csrc/all_to_all/all_to_all.h:44. */
uint64_t pplx_a2a_num_experts_per_token(const pplx_a2a_t *handle);
uint32_t pplx_a2a_rank(const pplx_a2a_t *handle);

/* ---- per-rank calls (the reference API) ------------------------------ */

/* AllToAllIntraNode::dispatch, csrc/all_to_all/intranode_dispatch.cu:288-390.
 * The call is collective over the world, like the reference's: with
 * PPLX_A2A_SPLIT_NONE the kernels are enqueued when the last of the world_size
 * ranks has made its call for the step, on that call's `stream`, and every
 * rank's outputs are complete once they finish.  Ranks may call on different
 * streams (csrc/bindings/all_to_all_ops.cpp:163,194 runs each rank on its own
 * current stream): the launching stream first waits for the work the other
 * streams held when the last call came in, and those streams then wait for the
 * kernels; work a rank enqueues BETWEEN its own call and the last rank's call
 * is not ordered against the step.  The ranks of a captured step must share
 * one stream (PPLX_A2A_INVALID_STATE otherwise).
 * SEND and RECV are collective in the same way, phase by phase: the last
 * rank's SEND enqueues the sends of all ranks (inputs may be reused once it has
 * returned, in stream order; no output is touched), the last rank's RECV the
 * receives (outputs are those named by the RECV calls).  A SEND takes over
 * everything its call's inputs hold: dispatch SEND copies every present token
 * (row, scales, picks) and the groups' token counts into the staging area and
 * RECV routes and places them; combine SEND reads expert_y, indices, weights
 * and bound_m and leaves the combined rows in the staging area, and RECV copies
 * them to out_tokens (the reference reads indices and weights in its RECV,
 * csrc/all_to_all/intranode_combine.cu:127-169: pass the same ones to both
 * calls, as its callers do).  Every rank's SEND must
 * come before the first RECV, and staging must have been reserved with
 * pplx_a2a_world_reserve_split (PPLX_A2A_INVALID_STATE otherwise).
 * Without bound_m, m may not exceed max_num_tokens
 * (csrc/all_to_all/intranode_dispatch.cu:65); the members of a DP group must
 * pass the same m. */
int pplx_a2a_dispatch(pplx_a2a_t *handle, const pplx_a2a_dispatch_args_t *args,
                      int split_mode, void *stream);
/* AllToAllIntraNode::combine<T,U>, csrc/all_to_all/intranode_combine.cu:190-266. */
int pplx_a2a_combine(pplx_a2a_t *handle, const pplx_a2a_combine_args_t *args,
                     int split_mode, void *stream);

/* ---- all ranks in one call ------------------------------------------- */

/* One step for all ranks: `per_rank` is a host array of world_size entries,
 * entry r holding rank r's arguments.  Equivalent to world_size calls of
 * pplx_a2a_dispatch(..., PPLX_A2A_SPLIT_NONE, stream). */
int pplx_a2a_world_dispatch(pplx_a2a_world_t *world, const pplx_a2a_dispatch_args_t *per_rank,
                            void *stream);
int pplx_a2a_world_combine(pplx_a2a_world_t *world, const pplx_a2a_combine_args_t *per_rank,
                           void *stream);

/* One step (dispatch, combine, or dispatch then combine) for all ranks without a
 * world and without any allocation.  It has no counterpart in the reference; it
 * is for callers that cannot allocate device memory around the call: code under
 * hipGraph capture that has no world yet, tight serving loops, harnesses that
 * forbid hipMalloc.  `dispatch_per_rank` / `combine_per_rank` are host arrays
 * of world_size entries as for pplx_a2a_world_dispatch / _combine (either may be
 * NULL to skip that half); the kernels and the results are the same.  The state
 * a world would own (slot map, routing tables) lives in a 10 MiB array that
 * is part of the library's code object on every GPU; a geometry that needs more
 * (world_size / dp_size * max_num_tokens * experts_per_token * 4 bytes of slot
 * map plus about world_size / dp_size * max_num_tokens * num_experts * 5 / 32 bytes of
 * routing tables), or more than 64 ranks, is refused with
 * PPLX_A2A_INVALID_ARGUMENT / PPLX_A2A_UNSUPPORTED.  The slot map written by a
 * dispatch stays there for the combine of a later call.  All calls on one GPU
 * share the array: calls that overlap in time on one GPU (different streams or
 * threads) race, and a step of a different geometry overwrites the slot map.
 * `fault_bits`: optional device word that the kernels OR the fault bits of
 * pplx_a2a_world_faults into (the caller clears and reads it); NULL discards them.
 * Calls no hipMalloc / hipFree and never synchronises.  The first call on a device looks the
 * array's address up (pplx_a2a_world_create on that device does the same): it cannot be made
 * under stream capture and returns PPLX_A2A_INVALID_STATE there. */
int pplx_a2a_static_step(const pplx_a2a_config_t *cfg, int device,
                         const pplx_a2a_dispatch_args_t *dispatch_per_rank,
                         const pplx_a2a_combine_args_t *combine_per_rank, uint32_t *fault_bits,
                         void *stream);

/* Which kernels a step of a geometry runs as; for tests and tools.  Needs no GPU (it answers for one
 * with 160 KiB of LDS per compute unit). */
typedef enum pplx_a2a_dispatch_form {
  PPLX_A2A_DISPATCH_ONE_LAUNCH = 0,     /* routing and scatter in one */
  PPLX_A2A_DISPATCH_SLOT_MAP = 1,       /* the routing launches write the slots */
  PPLX_A2A_DISPATCH_TABLES = 2,         /* the scatter works the slots out of the routing tables */
  PPLX_A2A_DISPATCH_SCANNED_TABLES = 3  /* the same behind a scan of the tiles' counts */
} pplx_a2a_dispatch_form;
typedef struct pplx_a2a_plan {
  int32_t dispatch_form;          /* pplx_a2a_dispatch_form */
  uint32_t routing_tiles;
  uint32_t scatter_waves_per_cu;  /* 0 = as many as fit, or no scatter launch */
  int32_t scatter_in_turn;   /* 1: its waves fetch row, slots and buffers one behind the other */
  int32_t combine_per_group;      /* 1: combine gathers once for the ranks of a DP group */
} pplx_a2a_plan_t;
/* in_dtype: pplx_a2a_dtype of expert_y */
int pplx_a2a_plan(const pplx_a2a_config_t *cfg, int in_dtype, pplx_a2a_plan_t *out);
/* The same for a GPU with `lds_per_cu` bytes of LDS per compute unit (0: it does not say).
 * `rows_in_lds` (optional) receives 1 when dispatch takes its rows through LDS, not registers. */
int pplx_a2a_plan_on(const pplx_a2a_config_t *cfg, int in_dtype, uint32_t lds_per_cu, pplx_a2a_plan_t *out,
                     int32_t *rows_in_lds);

/* How combine takes a step: `picks` rows of a token at a time, `pieces` times 512 elements of each (1 KiB of
 * a 16-bit row, 2 KiB of an fp32 one), once for all ranks of a DP group when per_group is 1. */
typedef struct pplx_a2a_combine_plan {
  uint32_t picks;
  uint32_t pieces;
  int32_t per_group;
} pplx_a2a_combine_plan_t;
int pplx_a2a_combine_plan(const pplx_a2a_config_t *cfg, int in_dtype, pplx_a2a_combine_plan_t *out);
/* Whether combine stores the rows of a step plainly (1) or past the caches (0). */
int pplx_a2a_combine_stores(const pplx_a2a_config_t *cfg, int32_t *plain);

/* Parts of a step for pplx_a2a_world_abandon_step. */
#define PPLX_A2A_ABANDON_DISPATCH 1u
#define PPLX_A2A_ABANDON_COMBINE 2u

/* Drops the calls recorded so far for the dispatch and / or combine step (or split phase)
 * that is being assembled and returns that half of the world to idle, so that every rank can
 * call again.  For the caller whose rank r fails its argument checks after other ranks of the
 * step have called: nothing of a step reaches the GPU before its last rank has called, so the
 * recorded calls are forgotten and no kernel runs.  A split step between its SEND and RECV
 * phases is given up as a whole (what SEND staged is overwritten by the next SEND).
 * `dropped_calls` (optional) receives the number of recorded calls that were dropped.  The
 * reference has no such exit because it has no such state: a failed check there ends the
 * process (csrc/core/cuda_utils.h:7-14, csrc/core/utils.h:16-24).  Only host state changes:
 * no allocation, no synchronisation. */
int pplx_a2a_world_abandon_step(pplx_a2a_world_t *world, uint32_t which, uint32_t *dropped_calls);
/* A step whose buffers stay where they are: pplx_a2a_bound_create checks the arguments of
 * pplx_a2a_world_dispatch and pplx_a2a_world_combine once and enqueues the writing of their rank
 * tables into `device_memory` (pplx_a2a_bound_bytes, 16-byte aligned, the caller's), on `stream`;
 * pplx_a2a_bound_launch then runs dispatch (op 0) or combine (op 1).  On that stream the kernels
 * read the tables from there; on another one, on hipStreamPerThread, or while the stream is captured, they
 * go with the launch as always (a graph never refers to device_memory).  device_memory is to stay untouched
 * until the last launch on that stream is done with it; the bound step is to be destroyed before
 * its world.  The capture of `stream` refuses pplx_a2a_bound_create. */
int pplx_a2a_bound_bytes(const pplx_a2a_world_t *world, uint64_t *out);
int pplx_a2a_bound_create(pplx_a2a_world_t *world, const pplx_a2a_dispatch_args_t *dispatch_per_rank,
                          const pplx_a2a_combine_args_t *combine_per_rank, void *device_memory, void *stream,
                          pplx_a2a_bound_t **out);
int pplx_a2a_bound_launch(pplx_a2a_world_t *world, const pplx_a2a_bound_t *bound, int op, void *stream);
int pplx_a2a_bound_destroy(pplx_a2a_bound_t *bound);
/* Number of per-rank calls of `op` (0 = dispatch, 1 = combine) in `split_mode` that the world
 * has recorded and not launched yet; 0 once the last rank's call has enqueued the phase.  A
 * binding that keeps the callers' buffers alive for the ranks that called early reads this to
 * know when to let them go. */
int pplx_a2a_world_recorded_calls(pplx_a2a_world_t *world, int op, int split_mode, uint32_t *out);
/* The world a rank handle is attached to. */
pplx_a2a_world_t *pplx_a2a_world_of(const pplx_a2a_t *handle);

/* Allocates the staging that split send / recv calls go through (the reference
 * allocates its inboxes in the constructor, csrc/all_to_all/intranode.cpp:37-136;
 * here a world that never splits does not pay for them).  With G = world_size /
 * dp_size DP groups and M = max_num_tokens: G*M * (hidden_dim_bytes +
 * hidden_dim_scale_bytes + 4 * experts_per_token) bytes for dispatch (one copy
 * of every token, its scales and its picks) and, when expert_y_elem_bytes is not
 * 0, world_size*M * hidden_dim * 2 bytes for combine (one combined row per rank
 * and token, in the 2-byte dtype of out_tokens whatever expert_y holds; 2 and 4
 * ask for the same).  May be called again: what has been allocated stays where
 * it is until the world is destroyed, so graphs that recorded split calls remain
 * valid.  The first call (and the first that asks for combine staging)
 * allocates and clears memory, which synchronises the device. */
int pplx_a2a_world_reserve_split(pplx_a2a_world_t *world, uint32_t expert_y_elem_bytes);

/* Reads and clears the world's device-side fault word (synchronises `stream`):
 * bit 0 = a routed row did not fit out_expert_x_rows and was dropped,
 * bit 1 = an expert index >= num_experts was ignored,
 * bit 2 = combine met a slot beyond expert_y_rows,
 * bit 3 = an expert id repeated inside one token: the repeat took no row, was
 *         not counted and adds nothing in combine (the reference gives every
 *         pick a slot, csrc/all_to_all/intranode_dispatch.cu:139-144; top-k
 *         routing never repeats an expert),
 * bit 4 = a bound_m beyond max_num_tokens (or beyond m) was clamped
 *         (csrc/all_to_all/intranode_dispatch.cu:65 asserts). */
int pplx_a2a_world_faults(pplx_a2a_world_t *world, void *stream, uint32_t *out_bits);

/* ---- hipGraph plumbing ------------------------------------------------ */

/* Thin wrappers over stream capture so that a binding without HIP access can
 * record a dispatch+combine step once and replay it
 * (the reference's "CUDA graph support", README.md:5). */
int pplx_a2a_graph_begin_capture(void *stream);
int pplx_a2a_graph_end_capture(void *stream, pplx_a2a_graph_t **out);
int pplx_a2a_graph_launch(pplx_a2a_graph_t *graph, void *stream);
int pplx_a2a_graph_destroy(pplx_a2a_graph_t *graph);

/* ---- between dispatch and combine ------------------------------------------ */

/* Operators on plain device buffers: no world, no handle, nothing kept between calls.  They only
 * enqueue kernels on `stream` of `device` (a HIP device ordinal), so they may be captured; every
 * buffer, the workspace among them, is the caller's and stays valid until the kernels are done.
 * Two calls that may overlap in time need workspaces of their own.  They have no counterpart in the
 * reference, which leaves the experts to its caller. */

/* Tokens sorted by expert.  Pick (t, k) is live when t < min(m, *bound_m) and indices[t, k] <
 * num_experts; its row is slots[t, k], its rank among the live picks ordered by (expert, t, k), and
 * -1 when it is not live.  Rows offsets[e] .. offsets[e + 1] - 1 are expert e's; out_rows[slot] is a copy of
 * x[t], or its quantised form, and the rows of out_rows[0 .. m * experts_per_token) behind the last
 * live one are zeros (their scales too).  Unlike dispatch every pick has a row, one that repeats an expert of
 * its token too.  Quantised rows (out_scale not NULL): a = max(max |x[t, :]|, 2^-100),
 * out_rows = rint(x * (127 / a)) as int8 and out_scale = a / 127; a row that holds an infinity or a NaN
 * becomes zeros with a scale of NaN. */
typedef struct pplx_a2a_sort_args {
  const void *x;               /* [m, hidden_dim] of dtype, 16-byte aligned */
  int64_t x_stride_row;        /* bytes, a multiple of 16 */
  int32_t dtype;               /* pplx_a2a_dtype */
  uint32_t m;
  uint32_t experts_per_token;  /* 1..64; m * experts_per_token < 2^31 */
  uint32_t num_experts;        /* 1..5461 */
  uint64_t hidden_dim;         /* rows, and quantised rows, are multiples of 16 bytes */
  const uint32_t *indices;     /* [m, K] contiguous */
  const uint32_t *bound_m;     /* device scalar or NULL (= m) */
  void *out_rows;              /* [m * K, hidden_dim] of dtype, or int8 */
  int64_t out_stride_row;      /* bytes, a multiple of 16 */
  float *out_scale;            /* [m * K] or NULL */
  int32_t *slots;              /* [m, K] contiguous */
  int32_t *offsets;            /* [num_experts + 1] */
  void *workspace;             /* pplx_a2a_sort_workspace bytes, 4-byte aligned; may be NULL when that is 0 */
} pplx_a2a_sort_args_t;
int pplx_a2a_sort_workspace(uint32_t m, uint32_t experts_per_token, uint32_t num_experts, uint64_t *bytes);
int pplx_a2a_sort_tokens(int device, const pplx_a2a_sort_args_t *args, void *stream);

/* Sorted rows back to tokens: out[t] = sum over k of weights[t, k] * y[slots[t, k]], accumulated in
 * fp32 in the order of k and rounded once; picks with a slot outside [0, y_rows) add nothing, whatever their
 * weight, and a token without others becomes zeros.  Without weights the sum of the rows, which is the gradient of
 * sort_tokens. */
typedef struct pplx_a2a_unsort_args {
  void *out;                 /* [m, hidden_dim] of out_dtype, 16-byte aligned */
  int64_t out_stride_row;    /* bytes, a multiple of 16 */
  int32_t out_dtype;         /* pplx_a2a_dtype */
  int32_t y_dtype;           /* pplx_a2a_dtype */
  const void *y;             /* [y_rows, hidden_dim] of y_dtype, 16-byte aligned */
  int64_t y_stride_row;      /* bytes, a multiple of 16 */
  int64_t y_rows;
  const int32_t *slots;      /* [m, K] contiguous */
  const float *weights;      /* [m, K] contiguous or NULL */
  uint32_t m;                /* m * experts_per_token and m * ceil(hidden_dim / 512) are below 2^31 */
  uint32_t experts_per_token; /* 1..64 */
  uint64_t hidden_dim;       /* a multiple of 8 */
} pplx_a2a_unsort_args_t;
int pplx_a2a_unsort_tokens(int device, const pplx_a2a_unsort_args_t *args, void *stream);

/* Gradients of unsort_tokens: grad_y[slots[t, k]] = weights[t, k] * grad_out[t] and grad_weights[t, k] =
 * <grad_out[t], y[slots[t, k]]>, summed in fp32; rows of grad_y that no slot names and weights of picks without a
 * row get zeros.  The slots are those of a sort, of all its tokens or of some, with any of them taken out (-1): no two
 * name one row, and none names a row from *num_rows on.  Either gradient may be left out (NULL). */
typedef struct pplx_a2a_unsort_backward_args {
  void *grad_y;               /* [y_rows, hidden_dim] of dtype, 16-byte aligned, or NULL */
  int64_t grad_y_stride_row;  /* bytes, a multiple of 16 */
  float *grad_weights;        /* [m, K] contiguous or NULL */
  const void *grad_out;       /* [m, hidden_dim] of grad_dtype, 16-byte aligned */
  int64_t grad_out_stride_row; /* bytes, a multiple of 16 */
  int32_t grad_dtype;         /* pplx_a2a_dtype of grad_out */
  int32_t dtype;              /* pplx_a2a_dtype of y and grad_y */
  const void *y;              /* read for grad_weights only */
  int64_t y_stride_row;       /* bytes, a multiple of 16 */
  int64_t y_rows;             /* of y and grad_y */
  const int32_t *slots;       /* [m, K] contiguous */
  const int32_t *num_rows;    /* device scalar: live rows, which is offsets + num_experts */
  const float *weights;       /* [m, K] contiguous or NULL (ones) */
  uint32_t m;                 /* as above */
  uint32_t experts_per_token; /* 1..64 */
  uint64_t hidden_dim;        /* a multiple of 8 */
} pplx_a2a_unsort_backward_args_t;
int pplx_a2a_unsort_tokens_backward(int device, const pplx_a2a_unsort_backward_args_t *args, void *stream);

/* Where the rows of the experts lie.  PADDED: [num_experts, rows], of which expert e's first starts_or_counts[e] (clamped
 * to 0 .. rows) are there, as dispatch leaves them; SORTED: [rows], of which starts_or_counts[e] ..
 * starts_or_counts[e + 1] - 1 are expert e's (num_experts + 1 entries that do not descend from 0 on, clamped to rows);
 * DENSE: [rows], all of them there (one expert, starts_or_counts NULL). */
typedef enum pplx_a2a_row_layout {
  PPLX_A2A_ROWS_DENSE = 0,
  PPLX_A2A_ROWS_SORTED = 1,
  PPLX_A2A_ROWS_PADDED = 2
} pplx_a2a_row_layout;
typedef struct pplx_a2a_rows {
  int32_t layout;                   /* pplx_a2a_row_layout */
  uint32_t num_experts;             /* 1..5461 */
  uint64_t rows;                    /* of the buffer, PADDED: of each expert's; all of them < 2^31 */
  const int32_t *starts_or_counts;
} pplx_a2a_rows_t;

/* Rows to 8 bits with one scale each, as sort_tokens does it: of x [.., width], or with swiglu of
 * silu(x[.., :width]) * x[.., width:2 * width] in fp32, silu(g) = g / (1 + exp(-g)), which is -0 where exp(-g) is
 * more than fp32 holds (g < -88.7).  Rows that are not there are neither read nor written. */
typedef struct pplx_a2a_quantize_args {
  pplx_a2a_rows_t rows;
  void *out;                       /* int8 [.., width], 16-byte aligned */
  int64_t out_stride_row;          /* bytes, a multiple of 16, as is the next */
  int64_t out_stride_expert;       /* (PADDED) */
  float *out_scale;
  int64_t out_scale_stride_row;    /* floats */
  int64_t out_scale_stride_expert;
  const void *x;                   /* of dtype, 16-byte aligned */
  int64_t x_stride_row;            /* bytes, a multiple of 16, as is the next */
  int64_t x_stride_expert;
  int32_t dtype;                   /* pplx_a2a_dtype */
  int32_t swiglu;
  uint64_t width;                  /* a multiple of 16 */
} pplx_a2a_quantize_args_t;
int pplx_a2a_quantize_rows(int device, const pplx_a2a_quantize_args_t *args, void *stream);

/* Rows times their experts' weights in 8-bit integers: out[r, n] = x_scale[r] * weight_scale[e, n] *
 * sum over k of x[r, k] * weight[e, n, k].  The sums are exact (int32); the sum, the product of the scales and the product
 * of both are rounded to fp32, and the result to out_dtype.
 * Rows that are not there are neither read nor written. */
typedef struct pplx_a2a_int8_matmul_args {
  pplx_a2a_rows_t rows;
  void *out;                     /* [.., n] of out_dtype, aligned to its elements */
  int64_t out_stride_row;        /* elements */
  int64_t out_stride_expert;
  int32_t out_dtype;             /* pplx_a2a_dtype */
  const int8_t *x;               /* [.., k], 16-byte aligned */
  int64_t x_stride_row;          /* bytes, a multiple of 16, as is the next */
  int64_t x_stride_expert;
  const float *x_scale;
  int64_t x_scale_stride_row;    /* floats */
  int64_t x_scale_stride_expert;
  const int8_t *weight;          /* [num_experts, n, k] contiguous, 16-byte aligned */
  const float *weight_scale;     /* [num_experts, n] contiguous */
  uint64_t n;                    /* < 2^31 */
  uint64_t k;                    /* a multiple of 16, at most 131056: 128 * 128 * k < 2^31 */
} pplx_a2a_int8_matmul_args_t;
int pplx_a2a_int8_matmul(int device, const pplx_a2a_int8_matmul_args_t *args, void *stream);

/* Which form a product takes (rows->starts_or_counts is not looked at; no GPU needed). */
typedef struct pplx_a2a_int8_matmul_plan {
  uint32_t tile_rows, tile_columns; /* of the result, to a workgroup at a time; 0 where there is nothing to do */
  int32_t split;                    /* the waves of a workgroup share out k, and it takes one tile */
  uint32_t workgroups;
  uint64_t tiles;                   /* at most: as the rows of the experts spread */
} pplx_a2a_int8_matmul_plan_t;
int pplx_a2a_int8_matmul_plan(const pplx_a2a_rows_t *rows, uint64_t n, uint64_t k, pplx_a2a_int8_matmul_plan_t *out);

/* ---- before dispatch ------------------------------------------------------- */

/* Operators on plain device buffers as above: what makes the rows that dispatch sends, and its picks and weights.  Fewer than 2^31
 * tokens. */

/* Root-mean-square norm of rows, with the addition of a residual in front and the rows in 8 bits behind it:
 *   h = x + residual, rounded to dtype (h = x without residual)            -> sum
 *   v = h * weight / sqrt(mean(h^2) + eps), in fp32, rounded to dtype      -> y
 *   the quantised v, of which y is not a part                              -> q, scale
 * PPLX_A2A_ROWS_INT8: one scale a row, as pplx_a2a_quantize_rows.  PPLX_A2A_ROWS_E4M3: one scale for each 128 columns, which
 * is how dispatch carries fp8 rows: a = max(max |v|, 2^-100), scale = a / 448, q = v * (448 / a) rounded to e4m3.  (A v that lies in the
 * middle between two codes but for the roundings of fp32 has either of them; the same inputs have the same.)  A row that holds an
 * infinity or a NaN becomes NaN: y and the scales are NaN, q is zeros.  y and sum may be x or residual themselves (same address and
 * stride). */
typedef enum pplx_a2a_row_format { PPLX_A2A_ROWS_PLAIN = 0, PPLX_A2A_ROWS_INT8 = 1, PPLX_A2A_ROWS_E4M3 = 2 } pplx_a2a_row_format;
typedef struct pplx_a2a_rms_norm_args {
  const void *x;               /* [m, hidden_dim] of dtype; all rows 16-byte aligned, strides in bytes, multiples of 16 */
  int64_t x_stride_row;
  const void *residual;        /* the same, or NULL */
  int64_t residual_stride_row;
  const void *weight;          /* [hidden_dim] of weight_dtype, 16-byte aligned */
  int32_t dtype;               /* pplx_a2a_dtype */
  int32_t weight_dtype;        /* dtype or F32 */
  float eps;                   /* positive, a normal number */
  uint32_t m;
  uint64_t hidden_dim;         /* a multiple of 8, with q of 16; below 2^27 */
  void *y;                     /* [m, hidden_dim] of dtype, or NULL */
  int64_t y_stride_row;
  void *sum;                   /* the same: with residual and only with it */
  int64_t sum_stride_row;
  void *q;                     /* [m, hidden_dim] bytes, or NULL */
  int64_t q_stride_row;
  float *scale;                /* [m], or [m, ceil(hidden_dim / 128)], with q */
  int64_t scale_stride_row;    /* floats */
  int64_t scale_stride_block;  /* floats (E4M3) */
  int32_t format;              /* pplx_a2a_row_format */
} pplx_a2a_rms_norm_args_t;
int pplx_a2a_rms_norm(int device, const pplx_a2a_rms_norm_args_t *args, void *stream);

/* Gradients of y = rms_norm(h) and of h itself, with r = 1 / sqrt(mean(h^2) + eps) and g = grad_y * weight:
 *   grad_h = r * (g - h * r^2 * mean(g * h)) + grad_sum, rounded once: that of x and of residual
 *   grad_weight = sum over rows of grad_y * h * r, in fp32, in an order that the sizes alone decide
 * Either may be left out (NULL).  grad_h may be grad_y or grad_sum itself. */
typedef struct pplx_a2a_rms_norm_backward_args {
  const void *grad_y;          /* [m, hidden_dim] of dtype, as above */
  int64_t grad_y_stride_row;
  const void *grad_sum;        /* the same, or NULL (zeros) */
  int64_t grad_sum_stride_row;
  const void *h;               /* the same: x, or sum where there was a residual */
  int64_t h_stride_row;
  const void *weight;          /* [hidden_dim] of weight_dtype, 16-byte aligned */
  int32_t dtype;               /* pplx_a2a_dtype */
  int32_t weight_dtype;        /* dtype or F32 */
  float eps;
  uint32_t m;
  uint64_t hidden_dim;         /* a multiple of 8 below 2^27 */
  void *grad_h;                /* [m, hidden_dim] of dtype, or NULL */
  int64_t grad_h_stride_row;
  void *grad_weight;           /* [hidden_dim] of weight_dtype, 16-byte aligned, or NULL */
  void *workspace;             /* pplx_a2a_rms_norm_workspace bytes, 16-byte aligned: with grad_weight */
} pplx_a2a_rms_norm_backward_args_t;
int pplx_a2a_rms_norm_workspace(uint32_t m, uint64_t hidden_dim, uint64_t *bytes);
int pplx_a2a_rms_norm_backward(int device, const pplx_a2a_rms_norm_backward_args_t *args, void *stream);

/* The router's product: logits[t, e] = sum over k of x[t, k] * weight[e, k], added up in fp32.  Products of 16-bit elements are
 * exact; fp32 elements count to 24 bits.  (With weights of fp32 an infinity in a row or a weight, or a value above 3.38e38, may make a NaN.) */
typedef struct pplx_a2a_router_logits_args {
  const void *x;               /* [m, hidden_dim] of dtype; rows 16-byte aligned, strides in bytes, multiples of 16 */
  int64_t x_stride_row;
  const void *weight;          /* [num_experts, hidden_dim] of weight_dtype, the same */
  int64_t weight_stride_row;
  int32_t dtype;               /* pplx_a2a_dtype */
  int32_t weight_dtype;        /* dtype or F32 */
  uint32_t m;
  uint32_t num_experts;        /* 1..5461 */
  uint64_t hidden_dim;         /* a multiple of 8 below 2^27 */
  float *logits;               /* [m, num_experts], 4-byte aligned */
  int64_t logits_stride_row;   /* floats */
  void *workspace;             /* pplx_a2a_router_workspace bytes, 16-byte aligned; may be NULL when that is 0 */
} pplx_a2a_router_logits_args_t;
/* backward: of pplx_a2a_router_logits_backward. */
int pplx_a2a_router_workspace(uint32_t m, uint32_t num_experts, uint64_t hidden_dim, int32_t dtype, int32_t weight_dtype,
                              int32_t backward, uint64_t *bytes);
int pplx_a2a_router_logits(int device, const pplx_a2a_router_logits_args_t *args, void *stream);

/* Its gradients: grad_x = grad_logits * weight and grad_weight = grad_logits^T * x, added up in fp32 and rounded once.  Operands count to 24
 * bits whatever the results' type; an infinity, or a value above 3.38e38, may make a NaN of what it has a part in.  Either may be left out
 * (NULL). */
typedef struct pplx_a2a_router_logits_backward_args {
  const float *grad_logits;    /* [m, num_experts], 4-byte aligned */
  int64_t grad_logits_stride_row; /* floats */
  const void *x;               /* [m, hidden_dim] of dtype, as above: read for grad_weight */
  int64_t x_stride_row;
  const void *weight;          /* [num_experts, hidden_dim] of weight_dtype, as above: read for grad_x */
  int64_t weight_stride_row;
  int32_t dtype;
  int32_t weight_dtype;
  uint32_t m;
  uint32_t num_experts;
  uint64_t hidden_dim;
  void *grad_x;                /* [m, hidden_dim] of dtype, as x, or NULL */
  int64_t grad_x_stride_row;
  void *grad_weight;           /* [num_experts, hidden_dim] of weight_dtype, as weight, or NULL */
  int64_t grad_weight_stride_row;
  void *workspace;             /* pplx_a2a_router_workspace bytes, 16-byte aligned */
} pplx_a2a_router_logits_backward_args_t;
int pplx_a2a_router_logits_backward(int device, const pplx_a2a_router_logits_backward_args_t *args, void *stream);

/* Each token's experts and their weights.  With s the softmax of a token's logits, or the sigmoid of each:
 *   key[e] = s[e] + bias[e], in an order as if computed in 64 bits; without a bias the logits' order
 *   the experts are num_groups groups of consecutive ones, of which the top_groups take part whose group_top best keys
 *   (s + bias) have the largest sums
 *   indices = the experts_per_token experts of the largest keys, largest first; equal ones, and equal groups, by number
 *   weights = weight_scale * s[indices], divided by the sum of the s[indices] with renormalize
 * An expert whose logit or key is -inf is not there.  Picks that no expert is left for, and those of tokens from *bound_m on,
 * have index num_experts and weight 0.  A token with a logit or key that is NaN or +inf gets the first experts and weights of
 * NaN. */
typedef enum pplx_a2a_scores { PPLX_A2A_SOFTMAX = 0, PPLX_A2A_SIGMOID = 1 } pplx_a2a_scores;
typedef struct pplx_a2a_route_args {
  const void *logits;          /* [m, num_experts] of dtype, aligned to its elements */
  int64_t logits_stride_row;   /* elements */
  int32_t dtype;               /* pplx_a2a_dtype */
  uint32_t m;
  uint32_t num_experts;        /* 1..5461 */
  uint32_t experts_per_token;  /* 1..64, at most top_groups * num_experts / num_groups */
  const float *bias;           /* [num_experts] or NULL */
  const uint32_t *bound_m;     /* device scalar or NULL (= m) */
  uint32_t num_groups;         /* divides num_experts; 1: no groups */
  uint32_t top_groups;         /* 1..num_groups */
  uint32_t group_top;          /* 1 or 2, at most num_experts / num_groups (where top_groups < num_groups) */
  int32_t scores;              /* pplx_a2a_scores */
  int32_t renormalize;
  float weight_scale;          /* finite */
  uint32_t *indices;           /* [m, experts_per_token] contiguous */
  float *weights;              /* [m, experts_per_token] contiguous */
} pplx_a2a_route_args_t;
int pplx_a2a_route_tokens(int device, const pplx_a2a_route_args_t *args, void *stream);

/* The gradient of the weights with respect to the logits, for the picks (distinct in each token) that route_tokens made;
 * picks with an index of num_experts or more have none.  Every logit's gradient is written: NaN for all of a token's that has picks
 * and a logit that is NaN or +inf.  (The bias is not read: a token whose weights are NaN by the bias alone has a gradient all the same.) */
typedef struct pplx_a2a_route_backward_args {
  const float *grad_weights;   /* [m, experts_per_token] contiguous */
  const void *logits;          /* [m, num_experts] of dtype, as above */
  int64_t logits_stride_row;
  const uint32_t *indices;     /* [m, experts_per_token] contiguous */
  int32_t dtype;
  uint32_t m;
  uint32_t num_experts;
  uint32_t experts_per_token;
  int32_t scores;
  int32_t renormalize;
  float weight_scale;
  void *grad_logits;           /* [m, num_experts] of dtype, aligned to its elements */
  int64_t grad_logits_stride_row; /* elements */
} pplx_a2a_route_backward_args_t;
int pplx_a2a_route_tokens_backward(int device, const pplx_a2a_route_backward_args_t *args, void *stream);

/* ---- misc -------------------------------------------------------------- */

const char *pplx_a2a_last_error(void);
/* "major.minor.patch" of this library. */
const char *pplx_a2a_version(void);
/* Hash of the sources the library was built from (a binding can tell a stale build). */
const char *pplx_a2a_build_id(void);

#ifdef __cplusplus
}
#endif
#endif /* PPLX_A2A_H_ */
