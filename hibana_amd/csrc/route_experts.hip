// Routing of rows to experts, one wavefront a row: softmax or sigmoid scores, a bias for balance in the choice alone, groups of experts, top k,
// weights renormalized and scaled; and the gradient of the logits, given that of the weights.
//
//   s = softmax(l) or sigmoid(l);  c = s + bias;  a group's score = the sum of its best two c;  the best `kept` groups, equal ones by the lower;
//   the k largest c among their experts, equal ones by the lower expert;  w = s, with `renorm` s / sum of the chosen s, times `scale`.
//
// An expert whose logit is -inf or NaN, or whose c is (by its bias), is never chosen: slots left over name no expert (id e, weight 0). Scores of the chosen that
// are all too small for FP32 renormalize all the same (the sums are of scores relative to the largest chosen one's). A row with a NaN has NaN weights, with a +inf by the softmax too.
//
// The choice is not one of FP32's roundings: without a bias c grows with l, and the logits' own order decides. Else, and between groups, it is that of the
// formula in FP64; FP32 decides where it can: if two c next to each other in rank are nearer than its error can tell apart, the row is chosen again.
#include <type_traits>

#include "route.hpp"

namespace hb {

constexpr int ROUTE_MOST_K = 63;  // a selection a lane, and one more to compare the last with
constexpr int ROUTE_MOST_ROWS = 1 << 25;  // (a launch's lanes are counted in 32 bits)

struct RouteExperts {
  const void* logits;
  int64_t stride;        // elements
  const float* bias;     // or null
  const int32_t* slots;  // row r is real iff slots[r / steps] != 0 (null: every row)
  int m, e, k, steps;
  int groups, kept, size;  // size: experts a group
  int lanes, per, shift;   // lanes a group (a power of two, 2^shift), experts a lane
  int by_per;              // 2^16 / per, up: a tag (below 1024) times it is the tag's lane in units of 2^16
  int renorm;
  float scale;
  int32_t* ids;
  float* weights;
};

template <int KIND>
__device__ __forceinline__ float route_logit(const void* row, int e) {
  if constexpr (KIND == HB_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(row)[e]);
  if constexpr (KIND == HB_F16) return (float)static_cast<const _Float16*>(row)[e];
  return static_cast<const float*>(row)[e];
}

__device__ __forceinline__ float route_lane(float x, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane)); }
__device__ __forceinline__ double route_lane(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <typename T>
__device__ __forceinline__ T route_max(T a, T b) { return a > b ? a : b; }
template <typename T>
__device__ __forceinline__ T route_min(T a, T b) { return a < b ? a : b; }

// e^x and 1 / x. In FP32 by the device's own instructions: this is for the choice, whose error bound counts them (x log2(e) rounded: x 2^-24 of e^x, at most 2^-24 in all
// where e^x is below 1; the exponential and the reciprocal an ulp each).
__device__ __forceinline__ float route_exp(float x) { return __expf(x); }
__device__ __forceinline__ double route_exp(double x) { return exp(x); }
__device__ __forceinline__ float route_inverse(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ double route_inverse(double x) { return 1.0 / x; }
__device__ __forceinline__ float route_sum(float x) { return wave_sum(x); }
__device__ __forceinline__ double route_sum(double x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// Scores of the lane's experts (a softmax with an infinite logit: those that have one).
template <bool SIGMOID, typename T, int PER>
__device__ __forceinline__ void route_scores(const float (&l)[PER], uint32_t open, float most, T (&s)[PER]) {
  if (SIGMOID) {
#pragma unroll
    for (int j = 0; j < PER; j++) s[j] = route_inverse(T(1) + route_exp(-T(l[j])));
  } else {
    T sum = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      s[j] = !(open >> j & 1) ? T(0) : most == INFINITY ? T(l[j] == INFINITY ? 1 : 0) : route_exp(T(l[j]) - T(most));
      sum += s[j];
    }
    sum = route_sum(sum);
    const T by = sum > T(0) ? route_inverse(sum) : T(0);
#pragma unroll
    for (int j = 0; j < PER; j++) s[j] *= by;
  }
}

// A value of lane ^ D's (or, D = 4 and 8, its mirror's in eight and sixteen lanes, which holds the same where the smaller ones have been merged).
template <int D, typename T>
__device__ __forceinline__ T route_other(T x) {
  if constexpr (sizeof(T) == 4 && D <= 8) {
    constexpr int HOW = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x140;
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), HOW, 0xF, 0xF, false));
  } else {
    return __shfl_xor(x, D);
  }
}

// Whether the lane's group is among the `kept` best. `gap`: by how much the worst kept group is ahead of the best other (infinite without one).
template <typename T, int PER>
__device__ __forceinline__ bool route_groups(const RouteExperts& p, const T (&c)[PER], uint32_t open, int lane, T& gap) {
  const T none = -INFINITY;
  T b1 = none, b2 = none;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const T v = open >> j & 1 ? c[j] : none;
    b2 = route_max(b2, route_min(b1, v));
    b1 = route_max(b1, v);
  }
  auto merge = [&](auto d) {
    if (decltype(d)::value >= p.lanes) return;  // uniform
    const T o1 = route_other<decltype(d)::value>(b1), o2 = route_other<decltype(d)::value>(b2);
    b2 = route_max(route_min(b1, o1), route_max(b2, o2));
    b1 = route_max(b1, o1);
  };
  merge(std::integral_constant<int, 1>{}), merge(std::integral_constant<int, 2>{}), merge(std::integral_constant<int, 4>{});
  merge(std::integral_constant<int, 8>{}), merge(std::integral_constant<int, 16>{}), merge(std::integral_constant<int, 32>{});
  const T mine = b2 == none ? b1 : b1 + b2;
  const int group = lane >> p.shift;
  int ahead = 0;
  for (int g = 0; g < p.groups; g++) {
    const T other = route_lane(mine, g << p.shift);
    ahead += other > mine || (other == mine && g < group) ? 1 : 0;
  }
  // the ranks are a permutation: the last kept group and the first other one are there
  const uint64_t last = __ballot(group < p.groups && ahead == p.kept - 1), next = __ballot(group < p.groups && ahead == p.kept);
  const T worst = route_lane(mine, __builtin_ctzll(last)), best = route_lane(mine, __builtin_ctzll(next));
  gap = best == none || worst == T(INFINITY) ? T(INFINITY) : worst - best;
  return group < p.groups && ahead < p.kept;
}

// The row's choice in FP64: lane s < k gets selection s's tag (lane * per + register), or -1.
template <bool SIGMOID, int PER>
__device__ __forceinline__ int route_in_64_bits(const RouteExperts& p, const float (&l)[PER], const float (&bias)[PER], uint32_t counted, uint32_t open, float most, int lane) {
  double c[PER];
  route_scores<SIGMOID, double, PER>(l, counted, most, c);
#pragma unroll
  for (int j = 0; j < PER; j++) c[j] += (double)bias[j];
  if (p.kept < p.groups) {
    double gap;
    if (!route_groups<double, PER>(p, c, open, lane, gap)) open = 0;
  }
  if (!p.bias)  // inside the groups the logits' own order
#pragma unroll
    for (int j = 0; j < PER; j++) c[j] = l[j];
  int tag = -1;
  for (int s = 0; s < p.k; s++) {
    double best = -INFINITY;
    int at = 0;
#pragma unroll
    for (int j = 0; j < PER; j++)
      if ((open >> j & 1) && c[j] > best) best = c[j], at = j;
    double top = best;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = route_max(top, __shfl_xor(top, d));
    if (top == -INFINITY) break;
    const int winner = __builtin_ctzll(__ballot(best == top));
    const int from = __builtin_amdgcn_readlane(at, winner);
    if (lane == s) tag = winner * p.per + from;
    if (lane == winner) open &= ~(1u << from);
  }
  return tag;
}

// Lane l holds the experts l % lanes * per .. + per - 1 of group l / lanes: whole groups in neighbouring lanes, and experts in ascending order of lane, then register.
//
// Up to some thousand rows the launch's latency (one row of 512 BF16 logits, top 10: 5.1 us with nothing in the caches, 777 rows of 60 FP16 ones 5.5), then the instructions: 8192
// rows of 256 FP32 logits (8.4 MB, 1.7 us of reads), sigmoid, a bias, 4 of 8 groups, top 8: 17 us, 609 vector and 390 scalar instructions a row, of which the groups,
// the threshold and the ranks of the chosen (ballots and counts of them) are most. The library's exponential and division, and groups merged through LDS, were more of them.
template <int KIND, bool SIGMOID, int PER>
__global__ __launch_bounds__(256) void route_experts_kernel(RouteExperts p) {
  const int lane = threadIdx.x & 63, r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= p.m) return;
  if (p.slots && p.slots[r / p.steps] == 0) {
    if (lane < p.k) {
      p.ids[(int64_t)r * p.k + lane] = p.e;
      p.weights[(int64_t)r * p.k + lane] = 0.f;
    }
    return;
  }
  const char* row = static_cast<const char*>(p.logits) + (int64_t)r * p.stride * (KIND == HB_F32 ? 4 : 2);
  const int within = (lane & (p.lanes - 1)) * p.per, first = (lane >> p.shift) * p.size + within;
  const int have = (lane >> p.shift) < p.groups ? max(min(p.per, p.size - within), 0) : 0;
  float l[PER], bias[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) l[j] = route_logit<KIND>(row, min(first + j, p.e - 1)) + 0.f;  // (-0 counts as 0)
#pragma unroll
  for (int j = 0; j < PER; j++) bias[j] = p.bias ? p.bias[min(first + j, p.e - 1)] : 0.f;
  uint32_t open = 0;  // the lane's experts that can be chosen
  bool nan = false;
  float most = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    if (j >= have) continue;
    nan |= l[j] != l[j];
    if (l[j] > -INFINITY && bias[j] > -INFINITY) open |= 1u << j;
    most = fmaxf(most, l[j]);
  }
  nan = __ballot(nan) != 0;
  most = wave_max(most);
  // every logit counts in the softmax's sum, also those that a bias bars: a mask of its own
  uint32_t counted = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) counted |= j < have && l[j] > -INFINITY ? 1u << j : 0u;
  const bool by_logit = !p.bias;
  uint32_t key[PER];
  int tag;
  bool near = false;
  if (by_logit && p.kept >= p.groups) {
    uint32_t top;
#pragma unroll
    for (int j = 0; j < PER; j++) key[j] = open >> j & 1 ? score_key(l[j]) : 0u;
    top_ranked<true, PER>(key, p.per, p.k, lane, top, tag);
    if (top == 0u) tag = -1;
  } else {
    float c[PER];
    route_scores<SIGMOID, float, PER>(l, counted, most, c);
    float size = 0.f, largest = 0.f;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      size = fmaxf(size, c[j]);
      c[j] += bias[j];
      if (open >> j & 1) largest = fmaxf(largest, fabsf(c[j]));
    }
    // What two sums may seem apart, or in the wrong order, by FP32's roundings: a score is off by 2^-19 of the largest at most (its argument, the exponential, the sum over
    // PER registers and 64 lanes, the reciprocal and the product: 28 halves of an ulp), a sum with the bias by 2^-24 of itself; twice for two, and twice that. Of the largest
    // sum there is, not of the two: a bias of -1e9 on one expert sends every row to FP64, as equal logits of equal biases do. 8192 rows of 256 FP32 logits by sigmoid, 4 of 8 groups, in a
    // graph: 16.3 us, with such a bias 24.0 (without groups 12.5 and 19.1); BF16 logits 15.6, with a bias of zeros, whose ties are many, 23.6
    largest = wave_max(largest);
    const float off = 0x1p-17f * (SIGMOID ? 1.f : wave_max(size)) + 0x1p-22f * largest;
    uint32_t left = open;
    if (p.kept < p.groups) {
      float gap;
      if (!route_groups<float, PER>(p, c, open, lane, gap)) left = 0;
      near = gap <= 3.f * off || largest >= 0x1p126f;  // (the sum of two may be past FP32's range)
    }
    uint32_t top;
#pragma unroll
    for (int j = 0; j < PER; j++) key[j] = left >> j & 1 ? score_key(by_logit ? l[j] : c[j]) : 0u;
    if (by_logit) {
      top_ranked<true, PER>(key, p.per, p.k, lane, top, tag);
    } else {
      top_ranked<false, PER>(key, p.per, min(p.k + 1, 64), lane, top, tag);
      const uint32_t u = top ^ 0x80000000u;
      const float value = __builtin_bit_cast(float, u ^ (uint32_t)(((int32_t)u >> 31) & 0x7fffffff));
      const uint32_t under = __shfl_down(top, 1);
      const float below = __shfl_down(value, 1);
      near |= __ballot(lane < p.k && top != 0u && under != 0u && value - below <= off) != 0;
    }
    if (top == 0u) tag = -1;
    if (__builtin_expect(near, 0)) tag = route_in_64_bits<SIGMOID, PER>(p, l, bias, counted, open, most, lane);
  }
  if (lane >= p.k) tag = -1;
  const int holder = tag * p.by_per >> 16, id = tag < 0 ? p.e : (holder >> p.shift) * p.size + (holder & (p.lanes - 1)) * p.per + tag - holder * p.per;
  const float mine = tag < 0 ? -INFINITY : route_logit<KIND>(row, id);
  float w;
  if (p.renorm) {
    const float top = wave_max(mine);
    if (SIGMOID) {
      w = __builtin_amdgcn_readfirstlane(top < 0.f) ? expf(mine - top) / (1.f + expf(mine)) : 1.f / (1.f + expf(-mine));
    } else {
      w = expf(mine - top);
    }
    w = tag < 0 ? 0.f : w;
    const float sum = wave_sum(w);
    w = tag < 0 ? 0.f : w / sum;
  } else if (SIGMOID) {
    w = tag < 0 ? 0.f : 1.f / (1.f + expf(-mine));
  } else {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < PER; j++) sum += counted >> j & 1 ? expf(l[j] - most) : 0.f;
    sum = wave_sum(sum);
    w = tag < 0 ? 0.f : expf(mine - most) / sum;
  }
  if (lane < p.k) {
    p.ids[(int64_t)r * p.k + lane] = id;
    p.weights[(int64_t)r * p.k + lane] = tag < 0 ? 0.f : nan ? __builtin_nanf("") : w * p.scale;
  }
}

struct RouteGrad {
  const float* dweights;  // [m, k]
  const void* logits;
  int64_t stride;         // elements
  const int32_t* ids;     // [m, k]
  int m, e, k, renorm;
  float scale;
  void* out;              // [m, e]
};

// A wavefront a row: the chosen experts' values in its lanes, then the row's columns in 16-byte pieces, each piece the sum over the chosen of those that are its own. 8192 rows of 256
// FP32 with a sigmoid, which writes 8.4 MB and reads the chosen logits alone, 7.9 us with nothing in the caches; a softmax without `renorm`, which goes
// over the row three times, 2049 rows of 512 BF16 10.6: latency, of the passes one behind the other, or (the chosen alone, whose bytes are 1.7 us) of ids, their logits, the sums and
// the stores.
//
// With `renorm` dl = w (dw - sum of dw w) at the chosen experts (the sigmoid's: times 1 - s), zero elsewhere. Without: the sigmoid's dw s (1 - s) there; the softmax's
// s (dw - sum of dw s) at every expert, dw zero at those that were not chosen.
template <int KIND, bool SIGMOID>
__global__ __launch_bounds__(256) void route_grad_kernel(RouteGrad p) {
  constexpr int SIZE = KIND == HB_F32 ? 4 : 2, VEC = 16 / SIZE;
  const int lane = threadIdx.x & 63, r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= p.m) return;
  const char* row = static_cast<const char*>(p.logits) + (int64_t)r * p.stride * SIZE;
  int id = lane < p.k ? p.ids[(int64_t)r * p.k + lane] : -1;
  if (id < 0 || id >= p.e) id = -1;
  const float mine = id >= 0 ? route_logit<KIND>(row, id) : -INFINITY;
  const float dw = id >= 0 ? p.dweights[(int64_t)r * p.k + lane] * p.scale : 0.f;
  const bool dense = !SIGMOID && !p.renorm;
  float g, most = 0.f, sum = 0.f, all = 0.f;
  if (p.renorm) {
    const float top = wave_max(mine);
    float w = SIGMOID ? __builtin_amdgcn_readfirstlane(top < 0.f) ? expf(mine - top) / (1.f + expf(mine)) : 1.f / (1.f + expf(-mine)) : expf(mine - top);
    if (id < 0 || top == -INFINITY) w = 0.f;
    const float total = wave_sum(w);
    if (total > 0.f) w /= total;  // (a NaN stays one)
    else if (total != total) w = total;
    g = w * (dw - wave_sum(dw * w));
    if (SIGMOID) g *= 1.f / (1.f + expf(mine));
    if (id < 0) g = 0.f;
  } else if (SIGMOID) {
    const float s = 1.f / (1.f + expf(-mine));
    g = id < 0 ? 0.f : dw * s * (1.f / (1.f + expf(mine)));
  } else {
    float top = -INFINITY;
    for (int i = lane; i < p.e; i += 64) top = fmaxf(top, route_logit<KIND>(row, i));
    most = wave_max(top);
    for (int i = lane; i < p.e; i += 64) sum += expf(route_logit<KIND>(row, i) - most);
    sum = wave_sum(sum);
    g = dw;
    all = wave_sum(id < 0 ? 0.f : dw * (expf(mine - most) / sum));
  }
  char* out = static_cast<char*>(p.out) + (int64_t)r * p.e * SIZE;
  const bool whole = !(p.e % VEC);
  for (int v0 = 0; v0 * VEC < p.e; v0 += 64) {
    const int at = (v0 + lane) * VEC;
    float value[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) value[j] = 0.f;
    for (int s = 0; s < p.k; s++) {
      const int to = __builtin_amdgcn_readlane(id, s);
      const float add = route_lane(g, s);
#pragma unroll
      for (int j = 0; j < VEC; j++) value[j] += to == at + j ? add : 0.f;
    }
    if (at >= p.e) continue;
    if (dense) {
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float l = route_logit<KIND>(row, min(at + j, p.e - 1));
        const float score = most == -INFINITY ? 0.f : expf(l - most) / sum;
        value[j] = score * (value[j] - all);
      }
      if (most == -INFINITY)
#pragma unroll
        for (int j = 0; j < VEC; j++) value[j] = 0.f;
    }
    uint32_t bits[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      if constexpr (KIND == HB_BF16) bits[j] = f32_to_bf16_bits(value[j]);
      if constexpr (KIND == HB_F16) bits[j] = __builtin_bit_cast(uint16_t, (_Float16)value[j]);
      if constexpr (KIND == HB_F32) bits[j] = __float_as_uint(value[j]);
    }
    if (whole) {
      u32x4_t packed;
#pragma unroll
      for (int q = 0; q < 4; q++) packed[q] = SIZE == 4 ? bits[q] : bits[2 * q % VEC] | bits[(2 * q + 1) % VEC] << 16;
      *reinterpret_cast<u32x4_t*>(out + (int64_t)at * SIZE) = packed;
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++)
        if (at + j < p.e) {
          if constexpr (SIZE == 4) reinterpret_cast<uint32_t*>(out)[at + j] = bits[j];
          else reinterpret_cast<uint16_t*>(out)[at + j] = (uint16_t)bits[j];
        }
    }
  }
}

template <int KIND, bool SIGMOID>
static int route_experts_run(const RouteExperts& p, hipStream_t stream) {
  const unsigned blocks = (unsigned)((p.m + 3) / 4);
  if (p.per <= 4) HB_LAUNCH((route_experts_kernel<KIND, SIGMOID, 4>), dim3(blocks), dim3(256), 0, stream, p);
  else if (p.per <= 8) HB_LAUNCH((route_experts_kernel<KIND, SIGMOID, 8>), dim3(blocks), dim3(256), 0, stream, p);
  else HB_LAUNCH((route_experts_kernel<KIND, SIGMOID, 16>), dim3(blocks), dim3(256), 0, stream, p);
  return launch_status();
}

}  // namespace hb

using namespace hb;

extern "C" int hb_route_experts(const void* logits, int type, int64_t stride, int m, int e, int k, int scoring, const float* bias, int groups, int kept, int renorm, float scale,
                                const int32_t* slots, int steps, int32_t* ids, float* weights, void* stream) {
  if (!logits || !ids || !weights) return HB_ENULL;
  if (type < HB_BF16 || type > HB_F32 || (scoring != HB_SOFTMAX && scoring != HB_SIGMOID) || m <= 0 || m > ROUTE_MOST_ROWS || e <= 0 || e > 64 * ROUTE_PER_LANE || k <= 0 || k > ROUTE_MOST_K ||
      groups <= 0 || groups > 64 || e % groups || kept <= 0 || kept > groups || k > kept * (e / groups) || steps <= 0 || (m > 1 && stride < e))
    return HB_EINVAL;
  RouteExperts p{logits, stride, bias, slots, m, e, k, steps, groups, kept, e / groups, 1, 0, 0, 0, renorm != 0, scale, ids, weights};
  while (2 * p.lanes * groups <= 64) p.lanes *= 2, p.shift++;
  p.per = (p.size + p.lanes - 1) / p.lanes;
  if (p.per > ROUTE_PER_LANE) return HB_EINVAL;
  p.by_per = 65536 / p.per + 1;
  if (!aligned(logits, type == HB_F32 ? 4 : 2) || !aligned(bias, 4) || !aligned(slots, 4) || !aligned(ids, 4) || !aligned(weights, 4)) return HB_EINVAL;
  const hipStream_t s = as_stream(stream);
  if (scoring == HB_SIGMOID)
    return type == HB_BF16 ? route_experts_run<HB_BF16, true>(p, s) : type == HB_F16 ? route_experts_run<HB_F16, true>(p, s) : route_experts_run<HB_F32, true>(p, s);
  return type == HB_BF16 ? route_experts_run<HB_BF16, false>(p, s) : type == HB_F16 ? route_experts_run<HB_F16, false>(p, s) : route_experts_run<HB_F32, false>(p, s);
}

extern "C" int hb_route_experts_grad(const float* dweights, const void* logits, int type, int64_t stride, const int32_t* ids, int m, int e, int k, int scoring, int renorm,
                                     float scale, void* dlogits, void* stream) {
  if (!dweights || !logits || !ids || !dlogits) return HB_ENULL;
  if (type < HB_BF16 || type > HB_F32 || (scoring != HB_SOFTMAX && scoring != HB_SIGMOID) || m <= 0 || m > ROUTE_MOST_ROWS || e <= 0 || e > 64 * ROUTE_PER_LANE || k <= 0 || k > ROUTE_MOST_K ||
      (m > 1 && stride < e))
    return HB_EINVAL;
  if (!aligned(logits, type == HB_F32 ? 4 : 2) || !aligned(dweights, 4) || !aligned(ids, 4) || !aligned(dlogits, 16)) return HB_EINVAL;
  const RouteGrad p{dweights, logits, stride, ids, m, e, k, renorm != 0, scale, dlogits};
  const unsigned blocks = (unsigned)((m + 3) / 4);
  const hipStream_t s = as_stream(stream);
#define HB_RG(KIND) if (type == KIND) { if (scoring == HB_SIGMOID) HB_LAUNCH((route_grad_kernel<KIND, true>), dim3(blocks), dim3(256), 0, s, p); else HB_LAUNCH((route_grad_kernel<KIND, false>), dim3(blocks), dim3(256), 0, s, p); }
  HB_RG(HB_BF16) HB_RG(HB_F16) HB_RG(HB_F32)
#undef HB_RG
  return launch_status();
}
