// Each token's experts and their weights out of the router's logits, and the gradient of the weights.
//
// Experts are put in order as if everything were computed in 64 bits: two whose scores with bias are closer than fp32 tells
// apart come out in the same order everywhere.
#include <cfloat>
#include <cmath>

#include "a2a_experts.h"

namespace pplx_amd {
namespace {

struct PicksDev {
  const uint8_t *logits;
  int64_t logits_stride_row;  // elements
  const float *bias;
  const uint32_t *bound_m;
  uint32_t *indices;
  float *weights;
  uint32_t m, experts, picks;
  uint32_t groups, top_groups, group_top;
  int32_t scores, renormalize;
  float weight_scale;
  uint32_t first_group;
};

constexpr double kNone = -HUGE_VAL;

template <class Op> __device__ __forceinline__ double wave_all(double v, Op &&op) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = op(v, __shfl_xor(v, d));
  return v;
}
__device__ __forceinline__ double wave_max_of(double v) {
  return wave_all(v, [](double a, double b) { return a > b ? a : b; });
}
__device__ __forceinline__ double wave_sum_of(double v) {
  return wave_all(v, [](double a, double b) { return a + b; });
}

// The number of the largest key of `keys`, the first of several (count where all are -inf).  Called by a wave.
__device__ __forceinline__ uint32_t first_of_largest(const double *keys, uint32_t count) {
  double best = kNone;
  uint32_t at = count;
  for (uint32_t e = lane_id(); e < count; e += 64) {
    if (keys[e] > best) {
      best = keys[e];
      at = e;
    }
  }
  const double most = wave_max_of(best);
  at = best == most && most > kNone ? at : count;
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)at, d);
    at = at < o ? at : o;
  }
  return at;
}

// A wave to a token, whose keys are in LDS.
template <class T> __global__ __launch_bounds__(64) void pick_experts(PicksDev a) {
  extern __shared__ double keys[];  // of the experts, then the sums of the groups
  const uint32_t t = a.first_group + blockIdx.x, lane = lane_id(), E = a.experts;
  uint32_t there = a.m;
  if (a.bound_m) there = *as_global(a.bound_m) < there ? *as_global(a.bound_m) : there;
  PPLX_GLOBAL uint32_t *indices = as_global(a.indices) + (uint64_t)t * a.picks;
  PPLX_GLOBAL float *weights = as_global(a.weights) + (uint64_t)t * a.picks;
  if (t >= there) {
    if (lane < a.picks) {
      indices[lane] = E;
      weights[lane] = 0.f;
    }
    return;
  }
  const PPLX_GLOBAL T *logits = as_global(reinterpret_cast<const T *>(a.logits)) + (int64_t)t * a.logits_stride_row;
  const PPLX_GLOBAL float *bias = as_global(a.bias);
  bool bad = false;
  double most = kNone, total = 0;
  for (uint32_t e = lane; e < E; e += 64) {
    const double l = (float)logits[e];
    bad |= !(l < HUGE_VAL);
    most = l > most ? l : most;
  }
  most = wave_max_of(most);
  const bool softmax = a.scores == PPLX_A2A_SOFTMAX, grouped = a.top_groups < a.groups;
  if (softmax && (a.bias || grouped || !a.renormalize)) {
    for (uint32_t e = lane; e < E; e += 64) total += exp((double)(float)logits[e] - most);
    total = wave_sum_of(total);
  }
  auto score = [&](double l) { return softmax ? exp(l - most) / total : 1.0 / (1.0 + exp(-l)); };
  // An expert's chance beside the others' of its group; -inf where it is not there.
  auto chance = [&](uint32_t e) {
    const double l = (float)logits[e];
    return l > kNone ? score(l) + (a.bias ? (double)bias[e] : 0.0) : kNone;
  };
  for (uint32_t e = lane; e < E; e += 64) {
    const double key = a.bias ? chance(e) : (double)(float)logits[e];
    keys[e] = key;
    bad |= !(key < HUGE_VAL);
  }
  if (__ballot(bad)) {
    if (lane < a.picks) {
      indices[lane] = lane;
      weights[lane] = __uint_as_float(0x7fc00000u);
    }
    return;
  }
  __syncthreads();
  if (grouped) {
    double *sums = keys + E;
    const uint32_t size = E / a.groups;
    for (uint32_t g = lane; g < a.groups; g += 64) {
      double first = kNone, second = kNone;
      for (uint32_t e = g * size; e < (g + 1) * size; ++e) {
        const double c = a.bias ? keys[e] : chance(e);
        second = c > first ? first : c > second ? c : second;
        first = c > first ? c : first;
      }
      sums[g] = a.group_top == 1 ? first : first + second;
    }
    __syncthreads();
    // (groups that are taken have a sum of NaN; one whose sum is -inf comes after all others, by number)
    for (uint32_t i = 0; i < a.top_groups; ++i) {
      uint32_t g = first_of_largest(sums, a.groups);
      if (g == a.groups) {
        for (uint32_t j = lane; j < a.groups; j += 64) g = j < g && sums[j] == kNone ? j : g;
#pragma unroll
        for (int d = 32; d; d >>= 1) {
          const uint32_t o = (uint32_t)__shfl_xor((int)g, d);
          g = g < o ? g : o;
        }
      }
      __syncthreads();
      if (lane == 0) sums[g] = __longlong_as_double(0x7ff8000000000000ll);
      __syncthreads();
    }
    for (uint32_t e = lane; e < E; e += 64) keys[e] = sums[e / size] != sums[e / size] ? keys[e] : kNone;
    __syncthreads();
  }
  uint32_t own = E;  // lane k: pick k
  for (uint32_t k = 0; k < a.picks; ++k) {
    const uint32_t e = first_of_largest(keys, E);
    if (e == E) break;
    own = lane == k ? e : own;
    __syncthreads();
    if (lane == 0) keys[e] = kNone;
    __syncthreads();
  }
  const bool picked = own < E;
  const double l = picked ? (double)(float)logits[own] : kNone;
  double w;
  if (a.renormalize) {
    // The scores over the largest of them: none of them is 0 because 64 bits do not hold it.
    const double top = wave_max_of(l), up = top < 0 ? -top : 0;
    w = !picked ? 0 : softmax ? exp(l - top) : 1.0 / (exp(-up) + exp(-l - up));
    w /= wave_sum_of(w);
  } else {
    w = score(l);
  }
  if (lane < a.picks) {
    indices[lane] = own;
    weights[lane] = picked ? (float)(w * (double)a.weight_scale) : 0.f;
  }
}

struct PicksBackwardDev {
  const float *grad_weights;
  const uint8_t *logits;
  int64_t logits_stride_row;
  const uint32_t *indices;
  uint8_t *grad_logits;
  int64_t grad_logits_stride_row;
  uint32_t m, experts, picks;
  int32_t scores, renormalize;
  float weight_scale;
  uint32_t first_group;
};

// A wave to a token.  Without renormalisation the gradient of a softmax has a part for every expert, p_e times the sum of
// g_k w_k; everything else is that of the picks alone.
template <class T> __global__ __launch_bounds__(64) void pick_gradient(PicksBackwardDev a) {
  extern __shared__ float of_picks[];  // an expert's own part
  const uint32_t t = a.first_group + blockIdx.x, lane = lane_id(), E = a.experts;
  const PPLX_GLOBAL T *logits = as_global(reinterpret_cast<const T *>(a.logits)) + (int64_t)t * a.logits_stride_row;
  PPLX_GLOBAL T *out = as_global(reinterpret_cast<T *>(a.grad_logits)) + (int64_t)t * a.grad_logits_stride_row;
  const bool softmax = a.scores == PPLX_A2A_SOFTMAX;
  const uint32_t own = lane < a.picks ? as_global(a.indices)[(uint64_t)t * a.picks + lane] : E;
  const bool picked = own < E;
  const double g = picked ? (double)as_global(a.grad_weights)[(uint64_t)t * a.picks + lane] : 0.0;
  const double l = picked ? (double)(float)logits[own] : kNone;
  for (uint32_t e = lane; e < E; e += 64) of_picks[e] = 0.f;
  double most = kNone, total = 0, inner = 0, part = 0;
  const bool dense = softmax && !a.renormalize;
  if (dense) {
    for (uint32_t e = lane; e < E; e += 64) {
      const double x = (float)logits[e];
      most = x > most ? x : most;
    }
    most = wave_max_of(most);
    for (uint32_t e = lane; e < E; e += 64) total += exp((double)(float)logits[e] - most);
    total = wave_sum_of(total);
    const double w = picked ? exp(l - most) / total * a.weight_scale : 0.0;
    inner = wave_sum_of(g * w);
    part = g * w;
  } else {
    const double s = picked ? 1.0 / (1.0 + exp(-l)) : 0.0;
    double w = s;
    if (a.renormalize) {
      const double top = wave_max_of(l), up = top < 0 ? -top : 0;
      w = !picked ? 0 : softmax ? exp(l - top) : 1.0 / (exp(-up) + exp(-l - up));
      w /= wave_sum_of(w);
      part = w * a.weight_scale * (g - wave_sum_of(g * w));
    } else {
      part = g * w * a.weight_scale;
    }
    if (!softmax) part *= 1.0 - s;
  }
  __syncthreads();
  if (picked) of_picks[own] = (float)part;
  __syncthreads();
  for (uint32_t e = lane; e < E; e += 64) {
    double d = of_picks[e];
    if (dense && inner != 0) d -= exp((double)(float)logits[e] - most) / total * inner;
    out[e] = (T)(float)d;
  }
}

int check_picks(int32_t dtype, uint32_t experts, uint32_t picks, int32_t scores, float scale) {
  PPLX_REQUIRE(is_dtype(dtype), "unsupported dtype of the logits");
  PPLX_REQUIRE(experts >= 1 && experts <= kMaxExperts, "num_experts must be in [1, %u]", kMaxExperts);
  PPLX_REQUIRE(picks >= 1 && picks <= 64 && picks <= experts, "experts_per_token must be in [1, 64] and at most num_experts");
  PPLX_REQUIRE(scores == PPLX_A2A_SOFTMAX || scores == PPLX_A2A_SIGMOID, "unknown scores");
  PPLX_REQUIRE(std::isfinite(scale), "weight_scale must be finite");
  return PPLX_A2A_OK;
}

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

extern "C" int pplx_a2a_route_tokens(int device, const pplx_a2a_route_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_route_args_t &p = *args;
  const int st = check_picks(p.dtype, p.num_experts, p.experts_per_token, p.scores, p.weight_scale);
  if (st) return st;
  PPLX_REQUIRE(p.num_groups >= 1 && p.num_experts % p.num_groups == 0, "num_groups must divide num_experts");
  PPLX_REQUIRE(p.top_groups >= 1 && p.top_groups <= p.num_groups, "top_groups must be in [1, num_groups]");
  const uint32_t size = p.num_experts / p.num_groups;
  PPLX_REQUIRE(p.top_groups == p.num_groups || p.group_top == 1 || (p.group_top == 2 && size >= 2),
               "group_top must be 1 or 2 and at most the experts of a group");
  PPLX_REQUIRE(p.experts_per_token <= p.top_groups * size, "the groups that take part have fewer than experts_per_token experts");
  if (p.m == 0) return PPLX_A2A_OK;
  PPLX_REQUIRE(p.logits && p.indices && p.weights, "logits / indices / weights is NULL");
  PPLX_REQUIRE(is_aligned(p.logits, dtype_bytes(p.dtype)) && is_aligned(p.bias, 4) && is_aligned(p.bound_m, 4) &&
                   is_aligned(p.indices, 4) && is_aligned(p.weights, 4),
               "logits, bias, bound_m, indices and weights must be aligned to their elements");
  PicksDev a{};
  a.logits = static_cast<const uint8_t *>(p.logits);
  a.logits_stride_row = p.logits_stride_row;
  a.bias = p.bias;
  a.bound_m = p.bound_m;
  a.indices = p.indices;
  a.weights = p.weights;
  a.m = p.m;
  a.experts = p.num_experts;
  a.picks = p.experts_per_token;
  a.groups = p.num_groups;
  a.top_groups = p.top_groups;
  a.group_top = p.group_top;
  a.scores = p.scores;
  a.renormalize = p.renormalize;
  a.weight_scale = p.weight_scale;
  return guarded(device, [&] {
    return with_type(p.dtype, [&](auto tag) {
      auto kernel = pick_experts<typename decltype(tag)::type>;
      // (5461 experts in as many groups take 85 KiB)
      const uint32_t lds = 8 * (a.experts + (a.top_groups < a.groups ? a.groups : 0));
      if (lds > 64 * 1024) {
        const hipError_t err =
            hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (err != hipSuccess) (void)hipGetLastError();  // (the launch says so if it matters)
      }
      PPLX_LAUNCH(launch_groups(kernel, kernel, a.m, 64, lds, (hipStream_t)stream, a));
      return (int)PPLX_A2A_OK;
    });
  });
}

extern "C" int pplx_a2a_route_tokens_backward(int device, const pplx_a2a_route_backward_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_route_backward_args_t &p = *args;
  const int st = check_picks(p.dtype, p.num_experts, p.experts_per_token, p.scores, p.weight_scale);
  if (st) return st;
  if (p.m == 0) return PPLX_A2A_OK;
  PPLX_REQUIRE(p.grad_weights && p.logits && p.indices && p.grad_logits, "grad_weights / logits / indices / grad_logits is NULL");
  const int64_t size = dtype_bytes(p.dtype);
  PPLX_REQUIRE(is_aligned(p.logits, size) && is_aligned(p.grad_logits, size) && is_aligned(p.grad_weights, 4) && is_aligned(p.indices, 4),
               "logits, grad_logits, grad_weights and indices must be aligned to their elements");
  PicksBackwardDev a{};
  a.grad_weights = p.grad_weights;
  a.logits = static_cast<const uint8_t *>(p.logits);
  a.logits_stride_row = p.logits_stride_row;
  a.indices = p.indices;
  a.grad_logits = static_cast<uint8_t *>(p.grad_logits);
  a.grad_logits_stride_row = p.grad_logits_stride_row;
  a.m = p.m;
  a.experts = p.num_experts;
  a.picks = p.experts_per_token;
  a.scores = p.scores;
  a.renormalize = p.renormalize;
  a.weight_scale = p.weight_scale;
  return guarded(device, [&] {
    return with_type(p.dtype, [&](auto tag) {
      auto kernel = pick_gradient<typename decltype(tag)::type>;
      PPLX_LAUNCH(launch_groups(kernel, kernel, a.m, 64, 4 * a.experts, (hipStream_t)stream, a));
      return (int)PPLX_A2A_OK;
    });
  });
}
