// Each token's experts and their weights out of the router's logits, and the gradient of the weights.
//
// Experts are put in order as if everything were computed in 64 bits: two whose scores with bias are closer than fp32 tells
// apart come out in the same order everywhere.  Without a bias the logits themselves have that order.  Otherwise fp32 makes the
// choice and watches how near its keys come: a token with two of them closer than their errors is chosen for once more in 64 bits, out of
// the registers that hold its logits.
// A wave takes a token, whose logits it reads once.  What bounds it is the instructions of the choice, six dependent steps over the wave for
// each pick, 0.16 us of a wave: 256 experts in fp32, a pick and eight, us in a graph: 64 tokens 2.4 and 3.5, with scores and biases
// 3.0 and 4.3, with groups too 3.8 and 5.0; 8192 tokens 3.7 and 6.9 (1.2 TB/s of logits), with scores and biases 5.6 and 11.6, with
// groups too 7.8 and 15.1, of which some tokens' second choice is 2 to 4.
#include <cfloat>
#include <climits>
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
  uint32_t group_lanes, lanes_shift;  // lanes that hold a group's experts, a power of two
  uint32_t first_group;
};

constexpr double kNone = -HUGE_VAL;
constexpr float kNoLogit = -HUGE_VALF;

// What a wave's lanes wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <class F, class Op> __device__ __forceinline__ F wave_all(F v, Op &&op) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = op(v, __shfl_xor(v, d));
  return v;
}
template <class F> __device__ __forceinline__ F wave_max_of(F v) {
  return wave_all(v, [](F a, F b) { return a > b ? a : b; });
}
template <class F> __device__ __forceinline__ F wave_sum_of(F v) {
  return wave_all(v, [](F a, F b) { return a + b; });
}
__device__ __forceinline__ uint32_t wave_min_of(uint32_t v) {
  return wave_all(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// Reductions without LDS, whose results are in scalar registers: lanes pass theirs on inside rows of sixteen, to the lane 1, 2, 4 and 8
// above, then the last lane of a row to the next row, and that of the second to the last two.
template <int CONTROL, int ROWS> __device__ __forceinline__ int from_lane(int otherwise, int v) {
  return __builtin_amdgcn_update_dpp(otherwise, v, CONTROL, ROWS, 0xf, false);
}
template <class Fn> __device__ __forceinline__ int over_lanes(int v, Fn &&step) {
  v = step(v, std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});
  v = step(v, std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  v = step(v, std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  v = step(v, std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  v = step(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  v = step(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ int wave_largest(int v) {
  return over_lanes(v, [](int x, auto control, auto rows) {
    const int o = from_lane<decltype(control)::value, decltype(rows)::value>(INT_MIN, x);
    return o > x ? o : x;
  });
}
__device__ __forceinline__ float wave_total(float v) {
  return __int_as_float(over_lanes(__float_as_int(v), [](int x, auto control, auto rows) {
    return __float_as_int(__int_as_float(x) + __int_as_float(from_lane<decltype(control)::value, decltype(rows)::value>(0, x)));
  }));
}
__device__ __forceinline__ int of_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float of_lane(float v, int lane) { return __int_as_float(of_lane(__float_as_int(v), lane)); }
__device__ __forceinline__ double of_lane(double v, int lane) {
  return __hiloint2double(of_lane(__double2hiint(v), lane), of_lane(__double2loint(v), lane));
}
// The upper halves' largest, then of the lower halves that come with it.
__device__ __forceinline__ int64_t wave_largest(int64_t v) {
  const int high = (int)(v >> 32), most = wave_largest(high);
  const int low = wave_largest(high == most ? (int)((uint32_t)v ^ 0x80000000u) : INT_MIN);
  return (int64_t)((uint64_t)(uint32_t)most << 32 | ((uint32_t)low ^ 0x80000000u));
}
// What the lanes of a group of `lanes` (1, 2, 4, ... 64) hold, joined by `join`, in all of them; where the lanes next to each other hold the
// same already, a mirrored row is as good as an exchange.
__device__ __forceinline__ float of_partner(float v, int control) {
  const int x = __float_as_int(v);
  switch (control) {
    case 1: return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0xb1, 0xf, 0xf, true));
    case 2: return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0x4e, 0xf, 0xf, true));
    case 4: return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0x141, 0xf, 0xf, true));
    case 8: return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0x140, 0xf, 0xf, true));
    default: return __shfl_xor(v, control);
  }
}
__device__ __forceinline__ double of_partner(double v, int control) {
  return __hiloint2double(__float_as_int(of_partner(__int_as_float(__double2hiint(v)), control)),
                          __float_as_int(of_partner(__int_as_float(__double2loint(v)), control)));
}
template <class Join> __device__ __forceinline__ void over_group(uint32_t lanes, Join &&join) {
  if (lanes > 1) join(std::integral_constant<int, 1>{});
  if (lanes > 2) join(std::integral_constant<int, 2>{});
  if (lanes > 4) join(std::integral_constant<int, 4>{});
  if (lanes > 8) join(std::integral_constant<int, 8>{});
  if (lanes > 16) join(std::integral_constant<int, 16>{});
  if (lanes > 32) join(std::integral_constant<int, 32>{});
}
// Numbers, none of them NaN, as integers of the same order, and back; 0 and -0 are one.
__device__ __forceinline__ int order_of(float v) {
  const int b = __float_as_int(v + 0.f);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ int64_t order_of(double v) {
  const int64_t b = __double_as_longlong(v + 0.0);
  return b ^ ((b >> 63) & 0x7fffffffffffffffll);
}
__device__ __forceinline__ float number_of(int order) { return __int_as_float(order ^ ((order >> 31) & 0x7fffffff)); }
__device__ __forceinline__ double number_of(int64_t order) {
  return __longlong_as_double(order ^ ((order >> 63) & 0x7fffffffffffffffll));
}
__device__ __forceinline__ float wave_max_of_lanes(float v) { return number_of(wave_largest(order_of(v))); }
__device__ __forceinline__ double wave_max_of_lanes(double v) { return number_of(wave_largest(order_of(v))); }
__device__ __forceinline__ double wave_total(double v) { return wave_sum_of(v); }

// exp(x) to two ulps, of x <= 88 (of more, exp(88); of NaN, NaN): 2^p for the rounded product p = x log2(e), times 1 + what the rounding
// left, in two steps where the result is subnormal (the instruction has none).
__device__ __forceinline__ float exp_of(float x) {
  x = x > 88.f ? 88.f : x;
  constexpr float kLog2e = 1.44269504088896340736f, kRest = 1.925963033500865e-8f;  // (their sum is log2(e))
  const float p = x * kLog2e;
  const float left = __builtin_fmaf(x, kLog2e, -p) + x * kRest;
  const float shift = p < -100.f ? 64.f : 0.f;
  float v = __builtin_amdgcn_exp2f(p + shift);
  v = __builtin_fmaf(v, left * 0.69314718055994530942f, v);
  return p < -1000.f ? 0.f : p < -100.f ? v * 0x1p-64f : v;  // (-inf brings a NaN from `left`)
}
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
template <class F> __device__ __forceinline__ F sigmoid_of(F l) { return (F)1 / ((F)1 + exp_of(-l)); }
// The same for keys, where an absolute error counts: in a few instructions and without branches.  exp(x) of x <= 0 to 2^-22 of it, or 2^-100.
__device__ __forceinline__ float key_exp(float x) {
  constexpr float kLog2e = 1.44269504088896340736f, kRest = 1.925963033500865e-8f;
  x = __builtin_fmaxf(x, -100.f);
  const float p = x * kLog2e, left = __builtin_fmaf(x, kLog2e, -p) + x * kRest, v = __builtin_amdgcn_exp2f(p);
  return __builtin_fmaf(v, left * 0.69314718055994530942f, v);
}
__device__ __forceinline__ double key_exp(double x) { return exp(x); }
// Off by 2^-22 at most.  The product rounds: |x| s (1 - s) <= 0.23 times 1.5 * 2^-24; the exponential: 2^-23 s (1 - s); the sum: 2^-24; the
// reciprocal: 2^-23.
__device__ __forceinline__ float key_sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f));
}
__device__ __forceinline__ double key_sigmoid(double x) { return sigmoid_of(x); }

// The weights of a wave's picks, lane k's of pick k with logit l: their scores, or their shares of the sum.
template <class F> __device__ __forceinline__ F weight_of_pick(bool picked, F l, bool softmax, bool renormalize, F most, F total) {
  if (renormalize) {
    // (scores over the largest of them: none of them is 0 because its type does not hold it)
    const F top = wave_max_of_lanes(picked ? l : (F)kNone), up = top < 0 ? -top : (F)0;
    F w = !picked ? (F)0 : softmax ? exp_of(l - top) : (F)1 / (exp_of(-up) + exp_of(-l - up));
    const F sum = wave_total(w);
    return picked ? w / sum : (F)0;
  }
  return !picked ? (F)0 : softmax ? exp_of(l - most) / total : sigmoid_of(l);
}
// Whether fp32 holds what weight_of_pick comes to: the distances from the largest logit, and from 0.
__device__ __forceinline__ bool picks_are_near(bool picked, float l, float most) {
  return __ballot(picked && !(l - most > -80.f && l > -80.f && l < 80.f)) == 0;
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
  return wave_min_of(best == most && most > kNone ? at : count);
}

__device__ __forceinline__ void store_pick(const PicksDev &a, uint32_t t, uint32_t lane, uint32_t expert, float weight) {
  if (lane >= a.picks) return;
  as_global(a.indices)[(uint64_t)t * a.picks + lane] = expert;
  as_global(a.weights)[(uint64_t)t * a.picks + lane] = weight;
}
// A token with a logit or key that is no number, or +inf.
__device__ __forceinline__ void store_bad(const PicksDev &a, uint32_t t, uint32_t lane) {
  store_pick(a, t, lane, lane, __uint_as_float(0x7fc00000u));
}

// A token's choice in 64 bits by a wave, with keys in LDS: of the experts, then the sums of the groups.
template <class T> __device__ __forceinline__ void pick_exactly(const PicksDev &a, uint32_t t, double *keys) {
  const uint32_t lane = lane_id(), E = a.experts;
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
  // An expert's chance beside the others' of its group; -inf where it is not there.
  auto chance = [&](uint32_t e) {
    const double l = (float)logits[e];
    const double s = softmax ? exp(l - most) / total : sigmoid_of(l);
    return l > kNone ? s + (a.bias ? (double)bias[e] : 0.0) : kNone;
  };
  for (uint32_t e = lane; e < E; e += 64) {
    const double key = a.bias ? chance(e) : (double)(float)logits[e];
    keys[e] = key;
    bad |= !(key < HUGE_VAL);
  }
  if (__ballot(bad)) return store_bad(a, t, lane);
  wave_sync();
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
    wave_sync();
    // (groups that are taken have a sum of NaN; those whose sum is -inf come after all others, by number)
    for (uint32_t i = 0; i < a.top_groups; ++i) {
      uint32_t g = first_of_largest(sums, a.groups);
      if (g == a.groups) {
        for (uint32_t j = lane; j < a.groups; j += 64) g = j < g && sums[j] == kNone ? j : g;
        g = wave_min_of(g);
      }
      wave_sync();
      if (lane == 0) sums[g] = __longlong_as_double(0x7ff8000000000000ll);
      wave_sync();
    }
    for (uint32_t e = lane; e < E; e += 64) keys[e] = sums[e / size] != sums[e / size] ? keys[e] : kNone;
    wave_sync();
  }
  uint32_t own = E;  // lane k: pick k
  for (uint32_t k = 0; k < a.picks; ++k) {
    const uint32_t e = first_of_largest(keys, E);
    if (e == E) break;
    own = lane == k ? e : own;
    wave_sync();
    if (lane == 0) keys[e] = kNone;
    wave_sync();
  }
  const bool picked = own < E;
  const double l = picked ? (double)(float)logits[own] : kNone;
  const double w = weight_of_pick(picked, l, softmax, a.renormalize, most, total);
  store_pick(a, t, lane, own, (float)(w * (double)a.weight_scale));
}

constexpr uint32_t kTokensAtOnce = 4;  // of a workgroup, a wave to each (no wave waits for another)
// Whether a token is there; those from bound_m on are done here.
__device__ __forceinline__ bool is_there(const PicksDev &a, uint32_t t, uint32_t lane) {
  if (!a.bound_m || t < *as_global(a.bound_m)) return true;
  store_pick(a, t, lane, a.experts, 0.f);
  return false;
}

template <class T> __global__ __launch_bounds__(64) void pick_experts_exactly(PicksDev a) {
  extern __shared__ double keys[];
  const uint32_t t = a.first_group + blockIdx.x;
  if (is_there(a, t, lane_id())) pick_exactly<T>(a, t, keys);
}

// PER consecutive elements from `base` on, of which those from `end` on are `otherwise`.
template <class T, int PER>
__device__ __forceinline__ void load_some(const PPLX_GLOBAL T *row, uint32_t base, uint32_t end, float otherwise, float *l) {
  typedef T vec __attribute__((ext_vector_type(PER), aligned(sizeof(T))));
  if (base + PER <= end) {
    if constexpr (PER == 1) {
      l[0] = (float)row[base];
    } else {
      const vec v = *reinterpret_cast<const PPLX_GLOBAL vec *>(row + base);
#pragma unroll
      for (int j = 0; j < PER; ++j) l[j] = (float)v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) l[j] = base + j < end ? (float)row[base + j] : otherwise;
  }
}

constexpr int kMostExperts = 16;  // of a lane
// A token's choice in F, with its logits and biases in registers: of experts `base` on in this lane, which are of `group`.  False,
// with nothing stored, if fp32 doesn't tell.  SCORED: keys (with a bias) or the groups' sums are scores, not logits.
template <class F, int PER, bool SCORED>
__device__ __forceinline__ bool choose(const PicksDev &a, uint32_t t, uint32_t lane, uint32_t group, uint32_t base, const float *l,
                                       const float *bias, float most) {
  constexpr bool kWatched = SCORED && sizeof(F) == 4;
  typedef decltype(order_of(F())) Order;
  const bool softmax = a.scores == PPLX_A2A_SOFTMAX, grouped = (SCORED || PER < kMostExperts) && a.top_groups < a.groups;
  const Order none = order_of((F)kNone);
  F score[PER], total = 0;
  if (softmax && (SCORED || !a.renormalize)) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      score[j] = key_exp((F)l[j] - (F)most);
      score[j] = l[j] > kNoLogit ? score[j] : (F)0;
      total += score[j];
    }
    total = wave_total(total);
    const F share = (F)1 / total;
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] *= share;
  } else if (SCORED) {
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] = key_sigmoid((F)l[j]);
  }
  Order key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    F k = l[j];
    if (SCORED) k = l[j] > kNoLogit ? score[j] + (F)bias[j] : (F)kNone;
    key[j] = order_of(k);
  }
  // How far keys may be from their values in 64 bits: a sigmoid by 2^-22.  A softmax by 2^-22 for its exponential, and it is divided by a
  // sum of as much and PER + 6 roundings: 2^-19 of a score that is 1 / total at most.  Two keys are off by twice as much, the sums
  // of two groups by four times; the sums with the bias and of two scores round by 2^-24 of what they come to.
  const float off = !kWatched ? 0.f : softmax ? 0x1p-18f / (float)total : 0x1p-21f;
  auto are_near = [](float larger, float smaller, float off) {
    // (so that what is no number, the difference of sums that fp32 does not hold, is near)
    return !(larger - smaller > __builtin_fmaf(0x1p-22f, __builtin_fabsf(larger) + __builtin_fabsf(smaller), off));
  };
  bool near = false;
  if (grouped) {
    auto larger_of = [](F x, F y) { return x > y ? x : y; };
    auto smaller_of = [](F x, F y) { return x > y ? y : x; };
    F first = kNone, second = kNone;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const F c = number_of(key[j]);
      second = larger_of(second, smaller_of(first, c));
      first = larger_of(first, c);
    }
    over_group(a.group_lanes, [&](auto distance) {
      const F c = of_partner(first, distance), d = of_partner(second, distance);
      second = larger_of(larger_of(second, d), smaller_of(first, c));
      first = larger_of(first, c);
    });
    const F sum = a.group_top == 1 ? first : first + second;
    uint32_t before = 0;  // groups in front of this one
    for (uint32_t g = 0; g < a.groups; ++g) {
      const F other = of_lane(sum, (int)(g * a.group_lanes));
      before += other > sum || (other == sum && g < group) ? 1 : 0;
    }
    const bool taken = before < a.top_groups;
    if (kWatched) {
      // Of the groups that are taken the least that the last may come to, and the most of the others.  Keys round by their own size, which
      // the sum of two of different signs does not show.  (A sum that fp32 does not hold is not told; one of a single expert is -inf.)
      const bool whole = a.group_top == 1 ? first > (F)kNone : second > (F)kNone;
      const float size = a.group_top == 1 ? __builtin_fabsf((float)first) : __builtin_fabsf((float)first) + __builtin_fabsf((float)second);
      const float error = __builtin_fmaf(0x1p-22f, size, off);
      near |= whole && !(size <= FLT_MAX);
      const float last = -wave_max_of_lanes(!taken ? kNoLogit : whole ? error - (float)sum : HUGE_VALF);
      const float next = wave_max_of_lanes(taken || !whole ? kNoLogit : (float)sum + error);
      near |= next > kNoLogit && !(last > next);
    } else if (!SCORED) {
      // Groups by their largest logit: the order of the scores, but where two of these are one in 64 bits.  They are not for logits 2^-20
      // apart, of which the less is not beyond 12 (a sigmoid's slope is 2^-18 there) and the larger one's exponential is a normal number.
      const float last = -wave_max_of_lanes(taken ? -(float)sum : kNoLogit), mine = (float)sum;
      const float more = mine > last ? mine : last, less = mine > last ? last : mine;
      const bool apart = more - less > 0x1p-20f && (softmax ? more - most > -700.f : less < 12.f && more > -700.f);
      near |= group < a.groups && mine != last && less > kNoLogit && !apart;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (!a.bias) key[j] = order_of((F)l[j]);  // (equal scores may be of logits that are not)
      key[j] = taken ? key[j] : none;
    }
  }
  // The largest key of each lane; the largest of all is taken, and its lane looks for its next one.
  Order head;
  float head_logit;
  uint32_t head_at;
  auto find_head = [&]() __attribute__((always_inline)) {
    head = key[0];
    head_logit = l[0];
    head_at = 0;
#pragma unroll
    for (int j = 1; j < PER; ++j) {
      const bool more = key[j] > head;
      head = more ? key[j] : head;
      head_logit = more ? l[j] : head_logit;
      head_at = more ? j : head_at;
    }
  };
  find_head();
  uint32_t own = a.experts;  // lane k: pick k, its key and logit
  float own_key = kNoLogit, own_logit = kNoLogit;
  for (uint32_t k = 0; k < a.picks; ++k) {
    const Order order = wave_largest(head);
    if (order == none) break;
    const int winner = __builtin_ctzll(__ballot(head == order));
    const uint32_t expert = (uint32_t)of_lane((int)(base + head_at), winner);
    const float number = (float)number_of(order), logit = SCORED ? of_lane(head_logit, winner) : number;
    if (lane == k) {
      own = expert;
      own_key = number;
      own_logit = logit;
    }
    if ((int)lane == winner) {
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] = (uint32_t)j == head_at ? none : key[j];
      find_head();
    }
  }
  const bool picked = own < a.experts;
  if (kWatched && a.bias) {
    // Each pick beside the next, the last one beside all that are left.  Equal logits with equal biases are equal in any arithmetic.
    const PPLX_GLOBAL float *biases = as_global(a.bias);
    const float next_key = __shfl(own_key, (int)(lane + 1));
    const bool close = lane + 1 < a.picks && next_key > kNoLogit && are_near(own_key, next_key, off);
    if (__ballot(close)) {
      const float next_logit = __shfl(own_logit, (int)(lane + 1));
      const uint32_t next = __shfl(own, (int)(lane + 1));
      if (close) near |= !(own_logit == next_logit && biases[own] == biases[next]);
    }
    const Order order = wave_largest(head);
    const float last_key = of_lane(own_key, (int)a.picks - 1), last_logit = of_lane(own_logit, (int)a.picks - 1);
    const int last = of_lane((int)own, (int)a.picks - 1);
    if (order != none && are_near(last_key, number_of(order), off)) {
      const float last_bias = biases[last];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        near |= key[j] != none && are_near(last_key, number_of(key[j]), off) && !(l[j] == last_logit && bias[j] == last_bias);
      }
    }
  }
  if (sizeof(F) == 4 && __ballot(near)) return false;
  float w;
  if (sizeof(F) == 4 && picks_are_near(picked, own_logit, most)) {
    w = (float)weight_of_pick<F>(picked, own_logit, softmax, a.renormalize, most, total) * a.weight_scale;
  } else {
    w = (float)(weight_of_pick<double>(picked, own_logit, softmax, a.renormalize, most, total) * (double)a.weight_scale);
  }
  store_pick(a, t, lane, own, w);
  return true;
}

// Up to 64 PER experts, PER consecutive ones in a lane, so that the first of equal keys is that of the first lane; where groups are
// chosen, no lane has experts of two.
template <class T, int PER, bool SCORED> __global__ __launch_bounds__(64 * kTokensAtOnce) void pick_experts(PicksDev a) {
  const uint32_t lane = lane_id(), wave = wave_id(), E = a.experts;
  const uint32_t t = (a.first_group + blockIdx.x) * kTokensAtOnce + wave;
  if (t >= a.m) return;
  const PPLX_GLOBAL T *logits = as_global(reinterpret_cast<const T *>(a.logits)) + (int64_t)t * a.logits_stride_row;
  uint32_t group = 0, base = lane * PER, end = E;
  if (a.top_groups < a.groups) {
    const uint32_t size = E / a.groups;
    group = lane >> a.lanes_shift;
    base = group * size + (lane - group * a.group_lanes) * PER;
    end = group < a.groups ? (group + 1) * size : 0;
  }
  float l[PER], bias[PER];
  load_some<T, PER>(logits, base, end, kNoLogit, l);
#pragma unroll
  for (int j = 0; j < PER; ++j) bias[j] = 0.f;
  if (SCORED && a.bias) load_some<float, PER>(as_global(a.bias), base, end, 0.f, bias);
  if (!is_there(a, t, lane)) return;
  bool bad = false;
  float most = kNoLogit;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    bad |= !(l[j] < HUGE_VALF);
    if (SCORED) bad |= l[j] > kNoLogit && !(bias[j] < HUGE_VALF);
    most = l[j] > most ? l[j] : most;
  }
  if (__ballot(bad)) return store_bad(a, t, lane);
  most = wave_max_of_lanes(most);
  if (choose<float, PER, SCORED>(a, t, lane, group, base, l, bias, most)) return;
  if constexpr (SCORED || PER < kMostExperts) choose<double, PER, true>(a, t, lane, group, base, l, bias, most);
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

// The parts of a token's gradient that are its picks' own, lane k's of pick k, and what all experts' scores are multiplied with: without
// renormalisation the gradient of a softmax has a part for every expert, p_e times the sum of g_k w_k.
template <class F>
__device__ __forceinline__ F gradient_of_pick(const PicksBackwardDev &a, bool picked, F g, F l, F most, F total, F *inner) {
  const bool softmax = a.scores == PPLX_A2A_SOFTMAX;
  const F w = weight_of_pick(picked, l, softmax, a.renormalize, most, total);
  const F sum = wave_total(picked ? g * w : (F)0);
  F part = picked ? w * g : (F)0;
  if (a.renormalize) part = picked ? w * (g - sum) : (F)0;
  if (!softmax) part *= sigmoid_of(-l);  // 1 - s
  *inner = softmax && !a.renormalize ? sum * (F)a.weight_scale : (F)0;
  return picked ? part * (F)a.weight_scale : (F)0;
}

// A wave to a token, PER consecutive experts in a lane and 64 PER at a time; rows of up to that are read once, whole in every form: a
// token with a logit that is NaN or +inf has weights of NaN, and so has its gradient.  An expert's own part goes through LDS to the lane
// that writes it.  16384 tokens of 256 experts, us in a graph: softmax without renormalisation 13.5 (2.5 TB/s), the other forms 10.4 (8.4
// if they read the picks' logits alone).
template <class T, int PER> __global__ __launch_bounds__(64 * kTokensAtOnce) void pick_gradient(PicksBackwardDev a) {
  extern __shared__ float of_picks[];  // [waves][experts]: an expert's own part
  const uint32_t lane = lane_id(), wave = wave_id(), E = a.experts;
  const uint32_t t = (a.first_group + blockIdx.x) * kTokensAtOnce + wave;
  if (t >= a.m) return;
  float *own_parts = of_picks + wave * E;
  const PPLX_GLOBAL T *logits = as_global(reinterpret_cast<const T *>(a.logits)) + (int64_t)t * a.logits_stride_row;
  PPLX_GLOBAL T *out = as_global(reinterpret_cast<T *>(a.grad_logits)) + (int64_t)t * a.grad_logits_stride_row;
  const uint32_t own = lane < a.picks ? as_global(a.indices)[(uint64_t)t * a.picks + lane] : E;
  const bool picked = own < E;
  const float g = picked ? as_global(a.grad_weights)[(uint64_t)t * a.picks + lane] : 0.f;
  const bool dense = a.scores == PPLX_A2A_SOFTMAX && !a.renormalize, once = E <= 64 * PER;
  float l[PER];
  float most = kNoLogit, total = 0.f;
  bool bad = false;
  for (uint32_t first = 0; first < E; first += 64 * PER) {
    load_some<T, PER>(logits, first + lane * PER, E, kNoLogit, l);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      bad |= !(l[j] < HUGE_VALF);
      most = l[j] > most ? l[j] : most;
    }
  }
  bad = __ballot(bad) && __ballot(picked);  // (without picks it has no part in anything)
  if (dense) {
    most = wave_max_of_lanes(most);
    for (uint32_t first = 0; first < E; first += 64 * PER) {
      if (!once) load_some<T, PER>(logits, first + lane * PER, E, kNoLogit, l);
#pragma unroll
      for (int j = 0; j < PER; ++j) total += l[j] == kNoLogit ? 0.f : exp_of(l[j] - most);
    }
    total = wave_total(total);
  }
  for (uint32_t e = lane; e < E; e += 64) own_parts[e] = 0.f;
  const float own_logit = picked ? (float)logits[own] : kNoLogit;
  float inner, part;
  if (picks_are_near(picked, own_logit, dense ? most : own_logit)) {
    part = gradient_of_pick<float>(a, picked, g, own_logit, most, total, &inner);
  } else {
    double sum;
    part = (float)gradient_of_pick<double>(a, picked, g, own_logit, most, total, &sum);
    inner = (float)sum;
  }
  wave_sync();
  if (picked) own_parts[own] = part;
  wave_sync();
  const float share = inner / total;
  for (uint32_t first = 0; first < E; first += 64 * PER) {
    const uint32_t base = first + lane * PER;
    if (dense && !once) load_some<T, PER>(logits, base, E, kNoLogit, l);
    float d[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      d[j] = base + j < E ? own_parts[base + j] : 0.f;
      if (dense && inner != 0.f) d[j] -= l[j] == kNoLogit ? 0.f : exp_of(l[j] - most) * share;
      if (bad) d[j] = __uint_as_float(0x7fc00000u);
    }
    if constexpr (PER > 1) {
      typedef T vec __attribute__((ext_vector_type(PER), aligned(sizeof(T))));
      if (base + PER <= E) {
        vec v;
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = (T)d[j];
        *reinterpret_cast<PPLX_GLOBAL vec *>(out + base) = v;
        continue;
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (base + j < E) out[base + j] = (T)d[j];
    }
  }
}

int check_picks(int32_t dtype, uint32_t m, uint32_t experts, uint32_t picks, int32_t scores, float scale) {
  PPLX_REQUIRE(is_dtype(dtype), "unsupported dtype of the logits");
  PPLX_REQUIRE(experts >= 1 && experts <= kMaxExperts, "num_experts must be in [1, %u]", kMaxExperts);
  PPLX_REQUIRE(picks >= 1 && picks <= 64 && picks <= experts, "experts_per_token must be in [1, 64] and at most num_experts");
  PPLX_REQUIRE(scores == PPLX_A2A_SOFTMAX || scores == PPLX_A2A_SIGMOID, "unknown scores");
  PPLX_REQUIRE(std::isfinite(scale), "weight_scale must be finite");
  if (m > kMaxTokens) return refuse(PPLX_A2A_UNSUPPORTED, "2^31 tokens or more");
  return PPLX_A2A_OK;
}

}  // namespace
}  // namespace pplx_amd

using namespace pplx_amd;

extern "C" int pplx_a2a_route_tokens(int device, const pplx_a2a_route_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_route_args_t &p = *args;
  const int st = check_picks(p.dtype, p.m, p.num_experts, p.experts_per_token, p.scores, p.weight_scale);
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
      typedef typename decltype(tag)::type T;
      const bool grouped = a.top_groups < a.groups;
      // Experts of a lane: as few as hold all of them, where no lane has some of two groups, whose lanes are a power of two.  (More
      // experts in a lane make its choice of the next one longer: 64 tokens of 256 experts 5.0 us, of 512 in 64 groups 8.0.)  What sixteen to
      // a lane do not hold is chosen for in LDS in 64 bits.
      const uint32_t size = a.experts / a.groups;
      uint32_t per = 1;
      auto lanes_of_group = [&] {
        uint32_t lanes = 1;
        while (lanes * per < size) lanes *= 2;
        return lanes;
      };
      while (per <= kMostExperts && (grouped ? (uint64_t)a.groups * lanes_of_group() > 64 : a.experts > 64 * per)) per *= 2;
      a.group_lanes = grouped ? lanes_of_group() : 64;
      a.lanes_shift = (uint32_t)__builtin_ctz(a.group_lanes);
      if (per > kMostExperts) {
        // (5461 experts in as many groups take 85 KiB)
        const uint32_t lds = 8 * (a.experts + (grouped ? a.groups : 0));
        auto kernel = pick_experts_exactly<T>;
        if (lds > 64 * 1024) {
          const hipError_t err =
              hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
          if (err != hipSuccess) (void)hipGetLastError();  // (the launch says so if it matters)
        }
        PPLX_LAUNCH(launch_groups(kernel, kernel, a.m, 64, lds, (hipStream_t)stream, a));
        return (int)PPLX_A2A_OK;
      }
      // (a choice in 64 bits that may follow one of sixteen logits in a lane takes more registers than there are: groups of so many go by scores)
      const bool scored = a.bias || (grouped && (a.group_top > 1 || per == kMostExperts));
      auto launch = [&](auto count) {
        constexpr int PER = decltype(count)::value;
        auto kernel = scored ? pick_experts<T, PER, true> : pick_experts<T, PER, false>;
        PPLX_LAUNCH(launch_groups(kernel, kernel, ((uint64_t)a.m + kTokensAtOnce - 1) / kTokensAtOnce, 64 * kTokensAtOnce, 0,
                                  (hipStream_t)stream, a));
        return (int)PPLX_A2A_OK;
      };
      switch (per) {
        case 1: return launch(std::integral_constant<int, 1>{});
        case 2: return launch(std::integral_constant<int, 2>{});
        case 4: return launch(std::integral_constant<int, 4>{});
        case 8: return launch(std::integral_constant<int, 8>{});
        default: return launch(std::integral_constant<int, kMostExperts>{});
      }
    });
  });
}

extern "C" int pplx_a2a_route_tokens_backward(int device, const pplx_a2a_route_backward_args_t *args, void *stream) {
  PPLX_REQUIRE(args, "args is NULL");
  const pplx_a2a_route_backward_args_t &p = *args;
  const int st = check_picks(p.dtype, p.m, p.num_experts, p.experts_per_token, p.scores, p.weight_scale);
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
      typedef typename decltype(tag)::type T;
      auto kernel = a.experts <= 64 ? pick_gradient<T, 1> : a.experts <= 256 ? pick_gradient<T, 4> : pick_gradient<T, 8>;
      const uint32_t lds = 4 * kTokensAtOnce * a.experts;
      if (lds > 64 * 1024) {
        const hipError_t err =
            hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (err != hipSuccess) (void)hipGetLastError();  // (the launch says so if it matters)
      }
      PPLX_LAUNCH(launch_groups(kernel, kernel, ((uint64_t)a.m + kTokensAtOnce - 1) / kTokensAtOnce, 64 * kTokensAtOnce, lds,
                                (hipStream_t)stream, a));
      return (int)PPLX_A2A_OK;
    });
  });
}
