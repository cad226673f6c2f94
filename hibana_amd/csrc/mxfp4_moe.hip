// Routed experts on microscaled four-bit weights and activations.
//
//   xq = the rows rounded to the format;  per routed pair (row, expert):
//   h = silu(gate xq) * (up xq) or relu(up xq)^2 in FP32, rounded to the format;  y = down h;  out = the weighted sum of a row's y.
#include <algorithm>

#include "mxfp4_ring.hpp"
#include "plan.hpp"
#include "stream_common.hpp"

namespace hb {

constexpr int MX_SCAN_PAIRS = 64;   // up to this many pairs every wavefront finds its workgroup's slot from the ids themselves
constexpr int MX_MOE_WAVES = 4;     // wavefronts a workgroup: small ones, so that several on a compute unit cover each other's starts and ends
constexpr int MX_MOE_TILES = 2;     // weight tiles a workgroup (wavefronts that share K) or a wavefront (that have their own)

// Rows' scales lie as the instruction takes them: a word a (quad of chunks, half), so a lane's scales of four chunks are one load.
constexpr int MX_STEP = 8;
__host__ __device__ constexpr int64_t mx_scale_row(int k) { return (k + 255) / 256 * 8; }
__device__ __forceinline__ int mx_scale_at(int group) { return (group >> 3) * 8 + (group & 1) * 4 + ((group >> 1) & 3); }

struct MxMoe {
  const uint8_t* w;        // the experts' stacked tile layouts
  int64_t expert_bytes;
  const void* x;           // few pairs, fc1: BF16 rows
  const uint8_t* aq;       // else activation codes by rows, [.., k / 2] ...
  const uint8_t* as;       // ... and scales [.., k / 32]
  const int32_t* ids;      // few pairs
  const float* weights;
  const int32_t* plan;     // many
  const int32_t* order;
  int base, experts, n, k, topk, pairs, inter;
  int span;                // many: units (of two tiles) a workgroup, or a wavefront
  uint8_t* hq;             // fc1: h by pair (few) or in sorted order (many)
  uint8_t* hs;
  void* y;                 // fc2: [pairs, n], or the rows' sums
};

// The slot of a call of few pairs that begins at pair `first`, found by every wavefront for itself: an expert's pairs in ascending order, cut
// into slots of 32; lane r of `list` holds the slot's pair r. 0 rows: another workgroup's.
__device__ __forceinline__ int mx_slot_of(const MxMoe& p, int id, int first, int& list) {
  const int lane = threadIdx.x & 63;
  const uint64_t same = __ballot(lane < p.pairs && p.ids[min(lane, p.pairs - 1)] == id);
  const int rank = __popcll(same & ((1ull << lane) - 1ull)), before = __popcll(same & ((1ull << first) - 1ull));
  if (before % MX_ROWS) return 0;
  // a pair of the slot hands its number to the lane of its place; the others theirs to places that nobody reads
  const bool mine = ((same >> lane) & 1) && rank >= before && rank < before + MX_ROWS;
  list = __builtin_amdgcn_ds_permute(4 * (mine ? rank - before : 32 + (lane & 31)), lane);
  return min(MX_ROWS, (int)__popcll(same) - before);
}

// h of 32 x 32 values (row r of the slot, 32 columns) from the joined sums of up (and gate), rounded to the format: of every 256 threads, thread
// i = 64 q + lane holds row lane % 32, columns 8 q + 4 (lane / 32) .. + 3. In two halves with a barrier between: a thread's largest magnitude goes to
// its word of `tops` (LDS), then the group's gives the scale.
template <bool GATED>
__device__ __forceinline__ float mx_h_of(float up, float gate) {
  const float u = fmaxf(up, 0.f);
  return GATED ? gate / (1.0f + expf(-gate)) * up : (up != up ? up : u * u);
}
template <bool GATED>
__device__ __forceinline__ f32x4_t mx_h(const f32x4_t& up, const f32x4_t& gate, uint32_t* tops) {
  f32x4_t h;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    h[j] = mx_h_of<GATED>(up[j], gate[j]);
    top = max(top, __float_as_uint(h[j]) & 0x7fffffffu);
  }
  tops[threadIdx.x] = top;
  return h;
}
__device__ __forceinline__ void mx_emit_h(const MxMoe& p, const f32x4_t& h, int column, bool real, int64_t pos, const uint32_t* tops) {
  const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5, q = (threadIdx.x >> 6) & 3;
  const uint32_t* of = tops + (threadIdx.x & ~255);
  uint32_t top = 0;
#pragma unroll
  for (int v = 0; v < 4; v++) top = max(top, max(of[v * 64 + r], of[v * 64 + 32 + r]));
  const uint32_t byte = mx_scale_byte(top);
  const float s = mx_scale_value(byte);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, h[0], h[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, h[2], h[3], s, 1);
  if (!real || column >= p.inter / 32) return;
  *reinterpret_cast<uint16_t*>(p.hq + pos * (p.inter / 2) + 16 * column + 4 * q + 2 * g) = byte == 255u ? 0 : (uint16_t)c;
  if (q || g) return;
  if (p.plan) {
    uint8_t* at = p.hs + pos * mx_scale_row(p.inter);
    at[mx_scale_at(column)] = (uint8_t)byte;
    if (column == p.inter / 32 - 1 && !(column & 1)) at[mx_scale_at(column + 1)] = 0;
  } else {
    p.hs[pos * (p.inter / 32) + column] = (uint8_t)byte;
  }
}

// ------------------------------------------------------------------------------------------------ few pairs
// fc1: a workgroup two weight tiles of the slot that begins at pair blockIdx.y (none: it leaves). The slot's expert is known from one
// id, so the weights are on their way while the slot's rows are looked for and their activations rounded into LDS. Latency bound: one row of 10 of 512
// experts (2048, 512) 5.8 us for 11 MB of weights.
constexpr int MX_FEW_WAVES = 8;
// PARTS lanes a group: values(acts, row of the slot, group, part, pair) puts it there.
template <int RUN, int PARTS, class Values>
__device__ __forceinline__ int mx_few_product(const MxMoe& p, f32x4_t* part, int& list, Values&& values) {
  const int first = blockIdx.y, id = p.ids[first], e = id - p.base;
  if (e < 0 || e >= p.experts) return 0;
  MxStream<MX_MOE_TILES, RUN> s;
  s.begin(p.w + e * p.expert_bytes, MxLayout(p.n, p.k), blockIdx.x * MX_MOE_TILES, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), MX_FEW_WAVES);
  const int rows = mx_slot_of(p, id, first, list);
  if (rows == 0) return 0;
  const MxActs acts(part, rows, p.k);
  const int all = rows * acts.groups * PARTS;
  for (int i = threadIdx.x; i < (all + 63) / 64 * 64; i += 64 * MX_FEW_WAVES) {  // whole wavefronts: `list` lies across the lanes
    const int r = i / PARTS / acts.groups, group = i / PARTS - r * acts.groups, pair = __shfl(list, min(r, rows - 1));
    if (i < all) values(acts, r, group, i % PARTS, pair);
  }
  __syncthreads();
  s.run(acts);
  mx_hand_over<MX_MOE_TILES>(part, s.acc);
  return rows;
}

template <bool GATED, int RUN>
__global__ __launch_bounds__(64 * MX_FEW_WAVES, RUN == 4 ? 2 : 4) void mx_fc1_few_kernel(MxMoe p) {
  extern __shared__ f32x4_t part[];
  int list = 0;
  const int rows = mx_few_product<RUN, 4>(p, part, list, [&](const MxActs& acts, int r, int group, int quarter, int pair) {
    Mx8<__bf16> v;
    v.load(static_cast<const __bf16*>(p.x) + (int64_t)(pair / p.topk) * p.k + MX_GROUP * group + 8 * quarter);
    acts.put(r, group, quarter, v);
  });
  if (rows == 0) return;
  const int r = threadIdx.x & 31, upper = threadIdx.x >> 8;  // the threads' upper half: the second tile where each is 32 columns
  const f32x4_t up = mx_joined<MX_MOE_TILES>(part, MX_FEW_WAVES, GATED ? threadIdx.x & 255 : threadIdx.x);
  const f32x4_t gate = GATED ? mx_joined<MX_MOE_TILES>(part, MX_FEW_WAVES, 256 + (threadIdx.x & 255)) : up;
  const int pair = __shfl(list, r);
  __syncthreads();  // the sums are read: their place takes the quarters' largest magnitudes
  uint32_t* tops = reinterpret_cast<uint32_t*>(part);
  const f32x4_t h = mx_h<GATED>(up, gate, tops);
  __syncthreads();
  mx_emit_h(p, h, GATED ? blockIdx.x : 2 * blockIdx.x + upper, r < rows && (!GATED || !upper), pair, tops);
}

// fc2 of the same slots, its results by pair.
template <typename Y, int RUN>
__global__ __launch_bounds__(64 * MX_FEW_WAVES, RUN == 4 ? 2 : 4) void mx_fc2_few_kernel(MxMoe p) {
  extern __shared__ f32x4_t part[];
  int list = 0;
  const int rows = mx_few_product<RUN, 1>(p, part, list, [&](const MxActs& acts, int r, int group, int, int pair) {
    acts.put(r, group, p.aq + (int64_t)pair * (p.k / 2), p.as + (int64_t)pair * acts.groups);
  });
  const int r = threadIdx.x & 31, pair = __shfl(list, r);
  if (r >= rows) return;
  const f32x4_t sum = mx_joined<MX_MOE_TILES>(part, MX_FEW_WAVES, threadIdx.x);
  const int n = (blockIdx.x * MX_MOE_TILES + (threadIdx.x >> 8)) * MX_ROWS + 8 * ((threadIdx.x >> 6) & 3) + 4 * ((threadIdx.x & 63) >> 5);
  typedef __attribute__((ext_vector_type(4))) Y y4_t;
  if (n < p.n) *reinterpret_cast<y4_t*>(static_cast<Y*>(p.y) + (int64_t)pair * p.n + n) = y4_t{(Y)sum[0], (Y)sum[1], (Y)sum[2], (Y)sum[3]};
}

// fc2 and the weighted sum of one row (blockIdx.y): a workgroup one tile of columns, its wavefronts the row's pairs in turn, their weighted
// results added in wavefront order. Reads a row's experts whether or not other rows name them too. 4.9 us behind the fc1 above, latency too.
constexpr int MX_ROW_WAVES = 8;
// ... where a wavefront's share is short: up to this many chunks of a row's pairs. One row of 10 of 512 experts (2048, 512), 80 chunks, fc2 so and as slots
// with a combine: 16.4 and 19.0 us the call, four rows 25.7 and 32.6; of 22 (1024, 2688), 924 chunks, one row 39.5 and 30.4.
constexpr int MX_ROW_CHUNKS = 128;
__global__ __launch_bounds__(64 * MX_ROW_WAVES, 2) void mx_fc2_row_kernel(MxMoe p) {
  __shared__ f32x4_t part[MX_ROW_WAVES * 4 * 8];
  const MxLayout at(p.n, p.k);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, groups = p.k / MX_GROUP;
  const int64_t row = blockIdx.y;
  constexpr int RUN = 8;
  f32x16_t total;
#pragma unroll
  for (int i = 0; i < 16; i++) total[i] = 0.f;
  for (int j = wave; j < p.topk; j += MX_ROW_WAVES) {
    const int64_t pair = row * p.topk + j;
    const int e = __builtin_amdgcn_readfirstlane(p.ids[pair]) - p.base;
    if (e < 0 || e >= p.experts) continue;
    const float weight = p.weights[pair];
    const uint8_t* codes = p.w + e * p.expert_bytes + (int64_t)blockIdx.x * at.chunks * 1024 + lane * 16;
    const uint8_t* scales = p.w + e * p.expert_bytes + at.codes() + (int64_t)blockIdx.x * at.quads * 256 + lane * 4;
    const uint8_t *hq = p.aq + pair * (p.k / 2), *hs = p.as + pair * groups;
    f32x16_t acc;
#pragma unroll
    for (int i = 0; i < 16; i++) acc[i] = 0.f;
    for (int c = 0; c < at.chunks; c += RUN) {
      i32x4_t b[RUN], a[RUN];
      uint32_t sb[RUN / 4], sa[RUN];
#pragma unroll
      for (int u = 0; u < RUN / 4; u++) sb[u] = *reinterpret_cast<const uint32_t*>(scales + ((c >> 2) + u) * 256);  // (quads come in pairs)
#pragma unroll
      for (int u = 0; u < RUN; u++) {
        const int in = min(c + u, at.chunks - 1), group = min(2 * in + half, groups - 1);
        b[u] = *reinterpret_cast<const i32x4_t*>(codes + in * 1024);
        a[u] = *reinterpret_cast<const i32x4_t*>(hq + 16 * group);
        sa[u] = hs[group];
      }
      mx_unrolled<RUN>([&](auto u) {
        if (c + u.value < at.chunks) acc = mx_mfma<u.value % 4, 0>(b[u.value], sb[u.value / 4], a[u.value], sa[u.value], acc);
      });
    }
#pragma unroll
    for (int i = 0; i < 16; i++) total[i] += weight * acc[i];
  }
  // every column of the product is the row's: lanes 0 and 32 hold all of it
  if ((lane & 31) == 0)
#pragma unroll
    for (int q = 0; q < 4; q++) part[wave * 8 + 2 * q + half] = mx_quarter(total, q);
  __syncthreads();
  if (threadIdx.x < 32) {
    const float* sums = reinterpret_cast<const float*>(part);
    float sum = sums[threadIdx.x];
    for (int w = 1; w < MX_ROW_WAVES; w++) sum += sums[w * 32 + threadIdx.x];
    const int n = blockIdx.x * MX_ROWS + threadIdx.x;
    if (n < p.n) static_cast<__bf16*>(p.y)[row * p.n + n] = (__bf16)sum;
  }
}

// ------------------------------------------------------------------------------------------------ many pairs
constexpr int MX_PLAN_PAIRS = 1024;  // from here the plan's launches share the pairs
// Workgroups of a product, about six a compute unit where there are so many: each has several units then, whose weights it asks for ahead. us, 1543 rows of 10
// of 512 experts (2048, 512), repeated on 2.5 GB of weights, pairs in BF16: 384 278, 768 251, 1536 240, twice that 250.
constexpr int MX_MANY_GROUPS = 1536;
// From this many pairs an expert slots have 64 rows, whose products share a weight tile's registers: 240 us against 292 for the call above, pairs in BF16 too (30 an
// expert), 71 and 74 for 300 rows of 8 of 64 (2048, 768); verify-sized calls are the same either way and keep the registers.
constexpr int MX_TALL_PAIRS = 24;
// x [rows, k] rounded for the products of many pairs, eight values a lane: codes by rows, scales as above (a last odd group's partner at 0). 1543 x 2048 4.8 us in a
// launch of its own.
struct MxRound {
  const __bf16* x;
  int64_t lanes;
  int k;
  uint8_t *codes, *scales;
};
__device__ __forceinline__ void mx_round_lane(const MxRound& job, int64_t i) {
  if (i >= job.lanes) return;  // whole groups leave together
  Mx8<__bf16> v;
  v.load(job.x + 8 * i);
  const uint32_t byte = mx_scale_byte(quad_max(v.amax()));
  reinterpret_cast<uint32_t*>(job.codes)[i] = byte == 255u ? 0u : v.codes(mx_scale_value(byte));
  if ((i & 3) == 0) {
    const uint32_t groups = (uint32_t)job.k / MX_GROUP, at_group = (uint32_t)(i >> 2);  // below 2^28: the codes are within a descriptor's reach
    const int64_t row = at_group / groups;
    const uint32_t group = at_group - (uint32_t)row * groups;
    uint8_t* at = job.scales + row * mx_scale_row(job.k);
    at[mx_scale_at(group)] = (uint8_t)byte;
    if (group == groups - 1 && (groups & 1)) at[mx_scale_at(groups)] = 0;
  }
}
__global__ __launch_bounds__(256) void mx_quantize_rows_kernel(MxRound job) { mx_round_lane(job, (int64_t)blockIdx.x * 256 + threadIdx.x); }
// The plan of a call of fewer pairs than its own launches share among workgroups, by the first workgroup, and the rounding beside it.
__global__ __launch_bounds__(PLAN_THREADS) void mx_plan_round_kernel(const int32_t* ids, int pairs, int e_lo, int e_n, int32_t* __restrict__ plan, int32_t* __restrict__ order,
                                                                     int slot_rows, int slot_cap, MxRound job) {
  extern __shared__ int plan_lds[];
  if (blockIdx.x == 0) {
    plan_work<false>(ids, pairs, e_lo, e_n, 0, plan, order, slot_rows, slot_cap, nullptr, 1, 0, 0, plan_lds);
  } else {
    mx_round_lane(job, (int64_t)(blockIdx.x - 1) * PLAN_THREADS + threadIdx.x);
  }
}
// Of a call whose plan counts the experts' pairs in a launch ahead of placing them: the first `groups` workgroups those counts, the others the rounding.
__global__ __launch_bounds__(PLAN_THREADS) void mx_count_round_kernel(const int32_t* ids, int pairs, int e_lo, int e_n, int32_t* __restrict__ plan, int32_t* __restrict__ order,
                                                                      int slot_rows, int slot_cap, int32_t* __restrict__ wide, int groups, MxRound job) {
  extern __shared__ int plan_lds[];
  if ((int)blockIdx.x < groups) {
    plan_work<true>(ids, pairs, e_lo, e_n, 0, plan, order, slot_rows, slot_cap, wide, groups, 1, blockIdx.x, plan_lds);
  } else {
    mx_round_lane(job, (int64_t)(blockIdx.x - groups) * PLAN_THREADS + threadIdx.x);
  }
}

// A wavefront's walk over steps of eight chunks of two weight tiles, for a slot of the plan (up to 32 MT rows of an expert). A step's weights, 16 KB
// a wavefront, are asked for as soon as the step before has taken its own out of the registers, so they are on their way while sums
// are joined, rounded and stored; a slot's activations (32 bytes of a row's chunk, read where they lie) stay in registers where one
// step covers the wavefront's K. Mostly reading the weights: 1543 rows of 10 of 512 experts (2048, 512) fc1 116 us, 4.9 TB/s where a plain read reaches 6.9, fc2 86 us, 4.8 with its
// results; 32 rows 24 and 13 us, 5.1 and 4.7; four rows of 22 of 512 ReLU^2 experts (1024, 2688) 23 and 23 us, 5.2.
template <int MT>
struct MxWalk {
  static constexpr int NT = MX_MOE_TILES;
  __amdgpu_buffer_rsrc_t w, ac, as;
  uint32_t code_at[MT], scale_at[MT];  // the lane's rows of activations, from the slot's first
  const MxLayout& at;
  int c0, c1;  // chunks of this wavefront's share of K: c0 a multiple of four
  i32x4_t b[MX_STEP][NT], a[MX_STEP][MT];
  uint32_t sb[MX_STEP / 4][NT], sa[MX_STEP / 4][MT];
  f32x16_t acc[MT][NT];
  // rows_of_x: how many rows the activations have (their descriptors end behind them)
  template <class Row>
  __device__ __forceinline__ MxWalk(const MxMoe& p, const MxLayout& at, const uint8_t* matrix, int rows, uint32_t rows_of_x, int share, int shares, Row&& row_of)
      : w(mx_rows(matrix, (uint32_t)at.bytes())), ac(mx_rows(p.aq, rows_of_x * (uint32_t)(p.k / 2))), as(mx_rows(p.as, rows_of_x * (uint32_t)mx_scale_row(p.k))), at(at) {
    const int quads = (at.chunks + 3) / 4, half = (threadIdx.x & 63) >> 5;
    c0 = 4 * (quads * share / shares);
    c1 = min(at.chunks, 4 * (quads * (share + 1) / shares));
#pragma unroll
    for (int i = 0; i < MT; i++) {
      const uint32_t row = row_of(min(32 * i + (int)(threadIdx.x & 31), rows - 1));  // (past the last: that one again, not to be stored)
      code_at[i] = row * (uint32_t)(p.k / 2) + 16 * half;
      scale_at[i] = row * (uint32_t)mx_scale_row(p.k) + 4 * half;
    }
  }
  __device__ __forceinline__ int steps() const { return max(1, (c1 - c0 + MX_STEP - 1) / MX_STEP); }
  // (chunks past the share's end: the last again, which costs no trip to memory, and not multiplied)
  __device__ __forceinline__ void ask_weights(int t0, int c) {
    const uint32_t lane = threadIdx.x & 63;
    const int last = max(c1 - 1, 0);
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int tile = min(t0 + t, at.tiles - 1), of = tile * at.chunks * 1024, s = (int)at.codes() + (tile * at.quads + (c >> 2)) * 256;
#pragma unroll
      for (int u = 0; u < MX_STEP; u++) b[u][t] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(w, lane * 16, of + min(c + u, last) * 1024, MX_NO_REUSE));
#pragma unroll
      for (int u = 0; u < MX_STEP / 4; u++) sb[u][t] = __builtin_amdgcn_raw_buffer_load_b32(w, lane * 4, s + u * 256, 0);
    }
  }
  __device__ __forceinline__ void ask_acts(int c) {
    const int last = max(c1 - 1, 0);
#pragma unroll
    for (int i = 0; i < MT; i++) {
#pragma unroll
      for (int u = 0; u < MX_STEP; u++) a[u][i] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(ac, code_at[i], min(c + u, last) * 32, 0));
#pragma unroll
      for (int u = 0; u < MX_STEP / 4; u++) sa[u][i] = __builtin_amdgcn_raw_buffer_load_b32(as, scale_at[i], ((c >> 2) + u) * 8, 0);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][t][e] = 0.f;
  }
  __device__ __forceinline__ void multiply(int c) {
    mx_unrolled<MX_STEP>([&](auto u) {
      if (c + u.value < c1) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int t = 0; t < NT; t++)
            acc[i][t] = mx_mfma<u.value % 4, u.value % 4>(b[u.value][t], sb[u.value / 4][t], a[u.value][i], sa[u.value / 4][i], acc[i][t]);
      }
    });
    __builtin_amdgcn_sched_barrier(0);  // the registers of b are free: what follows asks into them
  }
};

// The plan's slot of this workgroup and its span of units (two tiles each): p.span of them, from p.span blockIdx.x.
// fc1: KS wavefronts share a unit's K, as many as leave each about a step of it; the workgroup's 4 / KS groups of them have units of their own, whose
// sums become h together.
template <bool GATED, int MT, int KS>
__global__ __launch_bounds__(64 * MX_MOE_WAVES, MT == 1 ? 3 : 2) void mx_fc1_many_kernel(MxMoe p) {
  constexpr int SUBS = MX_MOE_WAVES / KS, PER = GATED ? 1 : 2;  // groups of wavefronts; 32 columns of h a unit
  __shared__ f32x4_t part[MX_MOE_WAVES * MX_MOE_TILES * 256];
  __shared__ uint32_t tops[SUBS * PER * 256];
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * (int)blockIdx.y;
  const int rows = entry[2], p0 = entry[1];
  if (rows == 0) return;
  const MxLayout at(p.n, p.k);
  const int units = (at.tiles + MX_MOE_TILES - 1) / MX_MOE_TILES, first = blockIdx.x * p.span * SUBS, last = min(first + p.span * SUBS, units);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = wave / KS;
  MxWalk<MT> walk(p, at, p.w + entry[0] * p.expert_bytes, rows, (uint32_t)(p.pairs / p.topk), wave % KS, KS, [&](int r) { return (uint32_t)(p.order[p0 + r] / p.topk); });
  const int steps = walk.steps();
  walk.ask_weights((first + sub) * MX_MOE_TILES, walk.c0);
  walk.ask_acts(walk.c0);
  for (int unit = first; unit < last; unit += SUBS) {
    walk.clear();
    for (int s = 0; s < steps; s++) {
      const int c = walk.c0 + s * MX_STEP;
      walk.multiply(c);
      if (s + 1 < steps) {
        walk.ask_weights((unit + sub) * MX_MOE_TILES, c + MX_STEP);
        walk.ask_acts(c + MX_STEP);
      } else if (unit + SUBS < last) {
        walk.ask_weights((unit + SUBS + sub) * MX_MOE_TILES, walk.c0);
        if (steps > 1) walk.ask_acts(walk.c0);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
      if (32 * i >= rows) break;
      mx_hand_over<MX_MOE_TILES>(part, walk.acc[i]);
      f32x4_t h[SUBS * PER];
#pragma unroll
      for (int e = 0; e < SUBS * PER; e++) {
        const f32x4_t* of = part + e / PER * KS * MX_MOE_TILES * 256;
        const f32x4_t up = mx_joined<MX_MOE_TILES>(of, KS, 256 * (e % PER) + threadIdx.x);
        h[e] = mx_h<GATED>(up, GATED ? mx_joined<MX_MOE_TILES>(of, KS, 256 + threadIdx.x) : up, tops + 256 * e);
      }
      __syncthreads();
      const int r = 32 * i + (threadIdx.x & 31);
#pragma unroll
      for (int e = 0; e < SUBS * PER; e++) mx_emit_h(p, h[e], PER * (unit + e / PER) + e % PER, r < rows, p0 + r, tops + 256 * e);
    }
  }
}

// fc2. SHARED: K split among the wavefronts as in fc1; else (short K) each wavefront has units of its own.
template <typename Y, int MT, bool SHARED>
__global__ __launch_bounds__(64 * MX_MOE_WAVES, MT == 1 ? 3 : 2) void mx_fc2_many_kernel(MxMoe p) {
  constexpr int NT = MX_MOE_TILES, PIECES = NT * MX_ROWS * (int)sizeof(Y) / 16, ROWS = 64 / PIECES;
  __shared__ f32x4_t part[SHARED ? MX_MOE_WAVES * NT * 256 : MX_MOE_WAVES * MX_ROWS * PIECES];
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * (int)blockIdx.y;
  const int rows = entry[2], p0 = entry[1];
  if (rows == 0) return;
  const MxLayout at(p.n, p.k);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, g = lane >> 5;
  const int units = (at.tiles + NT - 1) / NT, by = SHARED ? 1 : MX_MOE_WAVES;
  const int first = blockIdx.x * p.span * by + (SHARED ? 0 : wave), last = min((int)(blockIdx.x + 1) * p.span * by, units);
  if (first >= last) return;
  MxWalk<MT> walk(p, at, p.w + entry[0] * p.expert_bytes, rows, (uint32_t)p.pairs, SHARED ? wave : 0, SHARED ? MX_MOE_WAVES : 1, [&](int i) { return (uint32_t)(p0 + i); });
  const int steps = walk.steps();
  walk.ask_weights(first * NT, walk.c0);
  walk.ask_acts(walk.c0);
  typedef __attribute__((ext_vector_type(4))) Y y4_t;
  for (int unit = first; unit < last; unit += by) {
    walk.clear();
    for (int s = 0; s < steps; s++) {
      const int c = walk.c0 + s * MX_STEP;
      walk.multiply(c);
      if (s + 1 < steps) {
        walk.ask_weights(unit * NT, c + MX_STEP);
        walk.ask_acts(c + MX_STEP);
      } else if (unit + by < last) {
        walk.ask_weights((unit + by) * NT, walk.c0);
        if (steps > 1) walk.ask_acts(walk.c0);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
      if (32 * i >= rows) break;
      if constexpr (SHARED) {
        mx_hand_over<NT>(part, walk.acc[i]);
        if (32 * i + r < rows) {
          const int64_t pair = p.order[p0 + 32 * i + r];
#pragma unroll
          for (int t = 0; t < NT; t++) {
            const f32x4_t v = mx_joined<NT>(part, MX_MOE_WAVES, 256 * t + threadIdx.x);
            const int n = (unit * NT + t) * MX_ROWS + 8 * (threadIdx.x >> 6) + 4 * g;
            if (n < p.n) *reinterpret_cast<y4_t*>(static_cast<Y*>(p.y) + pair * p.n + n) = y4_t{(Y)v[0], (Y)v[1], (Y)v[2], (Y)v[3]};
          }
        }
      } else {  // a row's 64 results leave together, through the wavefront's own part of LDS (as mx_store_rows does it)
        i32x4_t* place = reinterpret_cast<i32x4_t*>(part) + wave * MX_ROWS * PIECES;
        uint8_t* bytes = reinterpret_cast<uint8_t*>(place);
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int in = (MX_ROWS * j + 8 * q + 4 * g) * (int)sizeof(Y), piece = (in / 16) ^ (r & (PIECES - 1));
            const f32x4_t v = mx_quarter(walk.acc[i][j], q);
            *reinterpret_cast<y4_t*>(bytes + (r * PIECES + piece) * 16 + in % 16) = y4_t{(Y)v[0], (Y)v[1], (Y)v[2], (Y)v[3]};
          }
#pragma unroll
        for (int from = 0; from < MX_ROWS; from += ROWS) {
          const int row = from + lane / PIECES, piece = lane % PIECES, n = unit * NT * MX_ROWS + piece * (16 / (int)sizeof(Y));
          const i32x4_t v = place[row * PIECES + (piece ^ (row & (PIECES - 1)))];
          if (32 * i + row < rows && n < p.n) *reinterpret_cast<i32x4_t*>(static_cast<Y*>(p.y) + (int64_t)p.order[p0 + 32 * i + row] * p.n + n) = v;
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ many pairs an expert
// The ring (mxfp4_ring.hpp) on the plan's slots of MX_RING_ROWS rows: the slot's rows of x rounded into the tile layout, fc1 with h rounded into it
// from the accumulators, fc2 with each row's results to its pair. 2048 rows of 8 of 64 experts (2560, 768), 256 rows each: gather 15 us, fc1 65
// (2.0 PFLOP/s, 9 TB/s into LDS), fc2 65 (1.0: six steps a workgroup, beside which its start and end are long, and 168 MB of results; 51 where they are BF16).
using MxMoeRing = MxRing<2, 2, 2, 2>;
constexpr int MX_RING_ROWS = MxMoeRing::TA * MX_ROWS;

// Rounding into the tile layout: a wavefront eight rows of a tile (`first` of them on) and a quad of chunks, eight lanes a row's 64 values, a quarter of a
// group each, so that a load instruction's lanes share eight whole lines and a store's two. (A lane a group, as the layout has it and a linear's rows are
// rounded, 16384 gathered rows of 2560 took 20 us, so 15.) x: the lane's row; groups past K have scale 0.
__device__ __forceinline__ void mx_round_quad(const __bf16* x, int k, int chunks, int quad, int first, uint8_t* tile_codes, uint8_t* quad_scales) {
  const int lane = threadIdx.x & 63, part = lane & 3, half = (lane >> 2) & 1, row = first + (lane >> 3), groups = k / MX_GROUP;
  Mx8<__bf16> v[4];
#pragma unroll
  for (int u = 0; u < 4; u++) v[u].load(x + MX_GROUP * (int64_t)min(2 * (4 * quad + u) + half, groups - 1) + 8 * part);
  uint32_t word = 0;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int c = 4 * quad + u;
    const bool in = 2 * c + half < groups;
    const uint32_t byte = in ? mx_scale_byte(quad_max(v[u].amax())) : 0u;
    word |= byte << (8 * u);
    if (c < chunks) reinterpret_cast<uint32_t*>(tile_codes + (int64_t)c * 1024 + (32 * half + row) * 16)[part] = in ? v[u].codes(mx_scale_value(byte)) : 0u;
  }
  if (part == 0) reinterpret_cast<uint32_t*>(quad_scales)[32 * half + row] = word;
}
// The slots' rows of x rounded into the tile layout, a workgroup a quad of a tile. The first workgroups of a tile also clear the scales of h behind its last
// group, which fc1 does not write: what they would multiply is scaled by 2^-127 on the weights' side, but has to be finite. (Rows rounded once and their
// codes gathered took a launch more: 5.4 and 10.6 us.)
__global__ __launch_bounds__(256) void mx_gather_kernel(MxMoe p, MxLayout xs, MxLayout hs) {
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * (int)blockIdx.y;
  const int rows = entry[2], p0 = entry[1], lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x % MxMoeRing::TA, quad = blockIdx.x / MxMoeRing::TA;
  if (MX_ROWS * tile >= rows) return;
  const int64_t at = (int64_t)blockIdx.y * MxMoeRing::TA + tile;
  const int r = min(MX_ROWS * tile + 8 * wave + (lane >> 3), rows - 1);  // (rows past the last: that one again)
  const __bf16* x = static_cast<const __bf16*>(p.x) + (int64_t)(p.order[p0 + r] / p.topk) * p.k;
  mx_round_quad(x, p.k, xs.chunks, quad, 8 * wave, const_cast<uint8_t*>(p.aq) + at * xs.chunks * 1024, const_cast<uint8_t*>(p.as) + (at * xs.quads + quad) * 256);
  if (quad == 0)
    for (int c = p.inter / MX_K + wave; c < hs.quads * 4; c += 4)
      if (2 * c + (lane >> 5) >= p.inter / MX_GROUP) p.hs[(at * hs.quads + (c >> 2)) * 256 + lane * 4 + (c & 3)] = 0;
}

// The slot and the tile of weight rows of a workgroup. Consecutive workgroups go to the eight dies in turn: a die takes two slots at a time, each with all
// columns, so that its L2 keeps a slot's activations, and the weights where both are one expert's.
struct MxPlace {
  int slot, column;
};
__device__ __forceinline__ MxPlace mx_place_of(int columns) {
  const int die = blockIdx.x % 8, at = blockIdx.x / 8, pair = at / (2 * columns), in = at - pair * 2 * columns, second = in >= columns;
  return {(pair * 8 + die) * 2 + second, in - second * columns};
}
__device__ __forceinline__ MxOperand mx_expert_tiles(const MxMoe& p, const MxLayout& at, int e, int tile) {
  const uint8_t* w = p.w + e * p.expert_bytes;
  return {w + (int64_t)tile * at.chunks * 1024, w + at.codes() + (int64_t)tile * at.quads * 256, at.tiles - tile};
}
__device__ __forceinline__ MxOperand mx_slot_tiles(const MxMoe& p, const MxLayout& at, int slot, int rows) {
  const int64_t tile = (int64_t)slot * MxMoeRing::TA;
  return {p.aq + tile * at.chunks * 1024, p.as + tile * at.quads * 256, (rows + MX_ROWS - 1) / MX_ROWS};
}

template <bool GATED>
__global__ __launch_bounds__(64 * MxMoeRing::WAVES, 2) void mx_fc1_ring_kernel(MxMoe p, int slots, int columns) {
  using Ring = MxMoeRing;
  constexpr int MT = 2, NT = 2;
  __shared__ i32x4_t buf0[Ring::BUFFER], buf1[Ring::BUFFER], buf2[Ring::BUFFER], buf3[Ring::BUFFER];
  const MxPlace place = mx_place_of(columns);
  if (place.slot >= slots) return;
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * place.slot;
  const int rows = entry[2];
  if (rows == 0) return;
  const MxLayout at(p.n, p.k), to(0, p.inter);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1, r = lane & 31, g = lane >> 5;
  f32x16_t acc[MT][NT];
  Ring::run(buf0, buf1, buf2, buf3, mx_slot_tiles(p, at, place.slot, rows), mx_expert_tiles(p, at, entry[0], place.column * Ring::TB), at.chunks, at.quads, 0, (at.chunks + 3) / 4, acc);
  // A lane holds 16 of the 32 values of a row's group, lane ^ 32 the others: columns 8 q + 4 g .. + 3 in registers 4 q .. 4 q + 3. Each lane ends with
  // eight bytes of the group's codes, columns 16 g .. 16 g + 15.
#pragma unroll
  for (int i = 0; i < MT; i++) {
    if (MX_ROWS * (wm * MT + i) >= rows) break;
#pragma unroll
    for (int j = 0; j < NT; j += GATED ? 2 : 1) {
      const int tile = place.column * Ring::TB + wn * NT + j, column = GATED ? tile >> 1 : tile;
      if (column >= p.inter / MX_GROUP) break;
      float h[16];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        h[e] = mx_h_of<GATED>(acc[i][j][e], acc[i][GATED ? j + 1 : j][e]);
        top = max(top, __float_as_uint(h[e]) & 0x7fffffffu);
      }
      top = max(top, (uint32_t)__shfl_xor((int)top, 32));
      const uint32_t byte = mx_scale_byte(top);
      const float s = mx_scale_value(byte);
      uint32_t c[4];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        c[q] = 0;
        c[q] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c[q], h[4 * q], h[4 * q + 1], s, 0);
        c[q] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c[q], h[4 * q + 2], h[4 * q + 3], s, 1);
      }
      const uint32_t lower = c[0] | c[1] << 16, upper = c[2] | c[3] << 16, other = (uint32_t)__shfl_xor((int)(g ? lower : upper), 32), own = g ? upper : lower;
      // g = 0: own is its q = 0, 1 and other the partner's; g = 1: other is the partner's (g = 0) q = 2, 3 and own its own
      const uint32_t first = g ? other : own, second = g ? own : other;  // of the lanes g = 0 and g = 1
      typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
      u32x2_t word = {(first & 0xffffu) | second << 16, first >> 16 | (second & 0xffff0000u)};
      if (byte == 255u) word = u32x2_t{0, 0};
      const int64_t row_tile = (int64_t)place.slot * Ring::TA + wm * MT + i;
      const int chunk = column >> 1, half = column & 1;
      *reinterpret_cast<u32x2_t*>(p.hq + ((row_tile * to.chunks + chunk) * 64 + 32 * half + r) * 16 + 8 * g) = word;
      if (g == 0) p.hs[(row_tile * to.quads + (chunk >> 2)) * 256 + (32 * half + r) * 4 + (chunk & 3)] = (uint8_t)byte;
    }
  }
}

template <typename Y>
__global__ __launch_bounds__(64 * MxMoeRing::WAVES, 2) void mx_fc2_ring_kernel(MxMoe p, int slots, int columns) {
  using Ring = MxMoeRing;
  constexpr int MT = 2, NT = 2;
  __shared__ i32x4_t buf0[Ring::BUFFER], buf1[Ring::BUFFER], buf2[Ring::BUFFER], buf3[Ring::BUFFER];
  const MxPlace place = mx_place_of(columns);
  if (place.slot >= slots) return;
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * place.slot;
  const int rows = entry[2];
  if (rows == 0) return;
  const MxLayout at(p.n, p.k);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  int pair[MT];  // of the wavefront's rows, on their way beside the product
#pragma unroll
  for (int i = 0; i < MT; i++) pair[i] = p.order[entry[1] + min(MX_ROWS * (wm * MT + i) + (int)(threadIdx.x & 31), rows - 1)];
  f32x16_t acc[MT][NT];
  Ring::run(buf0, buf1, buf2, buf3, mx_slot_tiles(p, at, place.slot, rows), mx_expert_tiles(p, at, entry[0], place.column * Ring::TB), at.chunks, at.quads, 0, (at.chunks + 3) / 4, acc);
  i32x4_t* own = wave == 0 ? buf0 : wave == 1 ? buf1 : wave == 2 ? buf2 : buf3;
#pragma unroll
  for (int i = 0; i < MT; i++) {
    const int row0 = MX_ROWS * (wm * MT + i);
    if (row0 >= rows) break;
    mx_store_rows<Y, NT>(own, p.n, (int64_t)(place.column * Ring::TB + wn * NT) * MX_ROWS, acc[i],
                         [&](int r) {
                           const int64_t to = __shfl(pair[i], r);
                           return row0 + r < rows ? static_cast<Y*>(p.y) + to * p.n : nullptr;
                         });
  }
}

namespace {
struct MxWorkspace {
  MoeWorkspace plan;
  uint8_t *xq, *xs, *hq, *hs;
  void* y;
  size_t bytes;
};

// Rows a pass of a call takes (more go in several, one behind the other): 2^18 pairs, which fill the device many times over and keep the workspace to a few
// GB, and what keeps the activations within a buffer descriptor's reach.
int most_rows(const hb_mxfp4_experts* ex, int topk) {
  const int64_t pairs = std::min<int64_t>((int64_t)1 << 18, (((int64_t)1 << 32) - 1) / (ex->inter / 2)), rows = (((int64_t)1 << 32) - 1) / (ex->hidden / 2);
  return (int)std::max<int64_t>(1, std::min(pairs / topk, rows));
}

bool few_pairs(int64_t pairs, int hidden, int inter) { return pairs <= MX_SCAN_PAIRS && MxActs::bytes(std::min<int64_t>(pairs, MX_ROWS), std::max(hidden, inter)) <= 64 * 1024; }

// From this many pairs an expert on (were they shared out evenly) a call runs on the ring: a slot of 128 rows of one expert half fills its tiles then, and
// the rows are worth being laid out. us, walk and ring, 64 experts (2048, 768): 48 pairs each 71 and 79, 64 94 and 82; 256 experts (2048, 512): 146 and
// 160, 181 and 168; 64 of ReLU^2 (1024, 2560), 62 each, 98 and 79.
constexpr int MX_RING_PAIRS = 56;
int fc1_rows(const hb_mxfp4_experts* ex) { return ex->gated ? 2 * ex->inter : ex->inter; }
int64_t ring_groups(int64_t slots, int columns) { return (slots + 15) / 16 * 16 * ((columns + 32 * MxMoeRing::TB - 1) / (32 * MxMoeRing::TB)); }
bool on_ring(int64_t pairs, const hb_mxfp4_experts* ex) {
  return pairs >= (int64_t)MX_RING_PAIRS * ex->experts &&
         ring_groups(moe_max_slots(pairs, ex->experts, 0, MX_RING_ROWS), std::max(fc1_rows(ex), ex->hidden_out)) < (int64_t)1 << 24;  // (a launch holds 2^32 threads)
}

MxWorkspace carve(const hb_mxfp4_experts* ex, void* base, int64_t m, int topk, bool sum) {
  m = std::min<int64_t>(m, most_rows(ex, topk));
  const int64_t pairs = m * topk;
  MxWorkspace w{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    uint8_t* ptr = base ? static_cast<uint8_t*>(base) + off : nullptr;
    off += (bytes + 255) & ~(size_t)255;
    return ptr;
  };
  if (!few_pairs(pairs, ex->hidden, ex->inter)) {
    w.plan.plan = reinterpret_cast<int32_t*>(take((PLAN_HEADER + (4 + DONE_PITCH) * moe_max_slots(pairs, ex->experts, 0, MX_ROWS) + 32) * sizeof(int32_t)));
    w.plan.plan_wide = reinterpret_cast<int32_t*>(take((size_t)64 * ex->experts * sizeof(int32_t)));
    w.plan.order = reinterpret_cast<int32_t*>(take((size_t)pairs * sizeof(int32_t)));
  }
  if (!few_pairs(pairs, ex->hidden, ex->inter) && on_ring(pairs, ex)) {
    const int64_t tiles = moe_max_slots(pairs, ex->experts, 0, MX_RING_ROWS) * MxMoeRing::TA;
    const MxLayout x(0, ex->hidden), h(0, ex->inter);
    w.xq = take((size_t)tiles * x.chunks * 1024);
    w.xs = take((size_t)tiles * x.quads * 256);
    w.hq = take((size_t)tiles * h.chunks * 1024);
    w.hs = take((size_t)tiles * h.quads * 256);
  } else {
    if (!few_pairs(pairs, ex->hidden, ex->inter)) {
      w.xq = take((size_t)m * (ex->hidden / 2));
      w.xs = take((size_t)m * mx_scale_row(ex->hidden));
    }
    w.hq = take((size_t)pairs * (ex->inter / 2));
    w.hs = take((size_t)pairs * mx_scale_row(ex->inter));
  }
  w.y = sum ? take((size_t)pairs * ex->hidden_out * sizeof(float)) : nullptr;
  w.bytes = off;
  return w;
}


size_t plan_lds_of(int experts) { return ((size_t)(PLAN_WAVES + 1) * experts + 3 * (PLAN_WAVES + 1)) * sizeof(int); }
constexpr int MX_MOST_TOPK = 4096;
constexpr int MX_MOST_EXPERTS = 960;  // the plan's counts of them lie in 64 KB of LDS

int check(const hb_mxfp4_experts* ex) {
  if (!ex || !ex->fc1 || !ex->fc2) return HB_ENULL;
  if (ex->experts <= 0 || ex->base < 0 || ex->hidden <= 0 || ex->inter <= 0 || ex->hidden_out <= 0 || ex->hidden % 32 || ex->inter % 32 || ex->hidden_out % 8 ||
      ex->hidden > 1 << 20 || ex->inter > 1 << 20 || ex->hidden_out > 1 << 20 || ex->experts > MX_MOST_EXPERTS || ex->base > 1 << 28)
    return HB_EINVAL;
  if (MxLayout(fc1_rows(ex), ex->hidden).bytes() >= (int64_t)1 << 31 || MxLayout(ex->hidden_out, ex->inter).bytes() >= (int64_t)1 << 31) return HB_EINVAL;  // offsets in one matrix
  return aligned(ex->fc1, 16) && aligned(ex->fc2, 16) ? HB_OK : HB_EINVAL;
}
}  // namespace

}  // namespace hb

using namespace hb;

static size_t workspace_of(const hb_mxfp4_experts* experts, int m, int topk, bool sum) {
  if (check(experts) != HB_OK || m <= 0 || topk <= 0 || topk > MX_MOST_TOPK || (int64_t)m * topk > 0x3fffffff) return 0;
  return carve(experts, nullptr, m, topk, sum).bytes;
}
extern "C" size_t hb_mxfp4_moe_workspace_bytes(const hb_mxfp4_experts* experts, int m, int topk) { return workspace_of(experts, m, topk, true); }
extern "C" size_t hb_mxfp4_moe_pairs_workspace_bytes(const hb_mxfp4_experts* experts, int m, int topk) { return workspace_of(experts, m, topk, false); }

// One pass: m <= most_rows. A sum's pairs lie in FP32 between fc2 and the combine, at any number of rows: in BF16 the largest tensor of a prefill would be half as
// large, but each pair would be rounded once more than the result is (1543 rows of 10 of 512 experts (2048, 512): relative
// error 2.4e-3 where FP32 pairs have 1.7e-3, the error of the result's own rounding; 212 us where they take 234, 126 MB more to write and read).
static int moe_pass(const hb_mxfp4_experts* experts, const void* x, const int32_t* ids, const float* weights, int m, int topk, int mode, void* out, void* workspace,
                    hipStream_t s) {
  const bool sum = mode == HB_MOE_SUM;
  const MxWorkspace ws = carve(experts, workspace, m, topk, sum);
  const int64_t pairs = (int64_t)m * topk;
  const MxLayout l1(fc1_rows(experts), experts->hidden), l2(experts->hidden_out, experts->inter);
  MxMoe p1{}, p2{};
  p1.w = static_cast<const uint8_t*>(experts->fc1);
  p1.expert_bytes = l1.bytes();
  p1.ids = ids;
  p1.weights = weights;
  p1.base = experts->base;
  p1.experts = experts->experts;
  p1.n = fc1_rows(experts);
  p1.k = experts->hidden;
  p1.topk = topk;
  p1.pairs = (int)pairs;
  p1.inter = experts->inter;
  p1.hq = ws.hq;
  p1.hs = ws.hs;
  p2 = p1;
  p2.w = static_cast<const uint8_t*>(experts->fc2);
  p2.expert_bytes = l2.bytes();
  p2.n = experts->hidden_out;
  p2.k = experts->inter;
  p2.aq = ws.hq;
  p2.as = ws.hs;
  p2.y = sum ? ws.y : out;
  const bool narrow = mode == HB_MOE_PAIRS_BF16;
  const unsigned groups1 = (unsigned)((l1.tiles + MX_MOE_TILES - 1) / MX_MOE_TILES), groups2 = (unsigned)((l2.tiles + MX_MOE_TILES - 1) / MX_MOE_TILES);
  auto combine = [&] {
    CombineParams c{};
    c.pairs = ws.y;
    c.ids = ids;
    c.weights = weights;
    c.e_lo = experts->base;
    c.e_n = experts->experts;
    c.m = m;
    c.topk = topk;
    c.h = experts->hidden_out;
    c.out = static_cast<uint16_t*>(out);
    moe_launch_combine(c, s);
  };
  if (few_pairs(pairs, experts->hidden, experts->inter)) {
    const int most = (int)std::min<int64_t>(MX_ROWS, pairs);
    const size_t room = (size_t)MX_FEW_WAVES * MX_MOE_TILES * 4096;
    p1.x = x;
    const size_t lds1 = std::max(room, MxActs::bytes(most, p1.k)), lds2 = std::max(room, MxActs::bytes(most, p2.k));
    const dim3 grid1(groups1, (unsigned)pairs), grid2(groups2, (unsigned)pairs), block(64 * MX_FEW_WAVES);
    const bool long1 = l1.chunks >= 4 * MX_FEW_WAVES, long2 = l2.chunks >= 4 * MX_FEW_WAVES;
    auto launch = [&](auto kernel, dim3 grid, size_t lds, const MxMoe& p) { HB_LAUNCH(kernel, grid, block, lds, s, p); };
    if (experts->gated) {
      launch(long1 ? mx_fc1_few_kernel<true, 4> : mx_fc1_few_kernel<true, 2>, grid1, lds1, p1);
    } else {
      launch(long1 ? mx_fc1_few_kernel<false, 4> : mx_fc1_few_kernel<false, 2>, grid1, lds1, p1);
    }
    if (sum && topk * l2.chunks <= MX_ROW_CHUNKS) {
      p2.y = out;
      HB_LAUNCH(mx_fc2_row_kernel, dim3((unsigned)l2.tiles, (unsigned)m), dim3(64 * MX_ROW_WAVES), 0, s, p2);
      return launch_status();
    }
    if (narrow) {
      launch(long2 ? mx_fc2_few_kernel<__bf16, 4> : mx_fc2_few_kernel<__bf16, 2>, grid2, lds2, p2);
    } else {
      launch(long2 ? mx_fc2_few_kernel<float, 4> : mx_fc2_few_kernel<float, 2>, grid2, lds2, p2);
    }
  } else {
    if (on_ring(pairs, experts)) {
      const int64_t slots = moe_max_slots(pairs, experts->experts, 0, MX_RING_ROWS);
      if (int e = moe_launch_plan(ids, pairs, experts->base, experts->experts, 0, ws.plan, s, MX_RING_ROWS)) return e;
      p1.x = x;
      p1.aq = ws.xq;
      p1.as = ws.xs;
      p1.plan = p2.plan = ws.plan.plan;
      p1.order = p2.order = ws.plan.order;
      HB_LAUNCH(mx_gather_kernel, dim3((unsigned)(l1.quads * MxMoeRing::TA), (unsigned)slots), dim3(256), 0, s, p1, l1, l2);
      auto launch = [&](auto kernel, const MxLayout& at, const MxMoe& p) {
        const int columns = (at.tiles + MxMoeRing::TB - 1) / MxMoeRing::TB;
        HB_LAUNCH(kernel, dim3((unsigned)ring_groups(slots, p.n)), dim3(64 * MxMoeRing::WAVES), 0, s, p, (int)slots, columns);
      };
      launch(experts->gated ? mx_fc1_ring_kernel<true> : mx_fc1_ring_kernel<false>, l1, p1);
      if (narrow) {
        launch(mx_fc2_ring_kernel<__bf16>, l2, p2);
      } else {
        launch(mx_fc2_ring_kernel<float>, l2, p2);
      }
      if (sum) combine();
      return launch_status();
    }
    const bool tall = pairs >= (int64_t)MX_TALL_PAIRS * experts->experts;
    const int slot_rows = tall ? 2 * MX_ROWS : MX_ROWS;
    const int64_t slots = moe_max_slots(pairs, experts->experts, 0, slot_rows);
    const MxRound job{static_cast<const __bf16*>(x), (int64_t)m * (experts->hidden / 8), experts->hidden, ws.xq, ws.xs};
    const size_t plan_lds = plan_lds_of(experts->experts);
    if (pairs < MX_PLAN_PAIRS) {
      HB_LAUNCH(mx_plan_round_kernel, dim3(1 + (unsigned)((job.lanes + PLAN_THREADS - 1) / PLAN_THREADS)), dim3(PLAN_THREADS), plan_lds, s, ids, (int)pairs, experts->base,
                experts->experts, ws.plan.plan, ws.plan.order, slot_rows, (int)slots, job);
    } else {
      const int counts = moe_plan_counts(pairs);
      const unsigned rounds = (unsigned)((job.lanes + PLAN_THREADS - 1) / PLAN_THREADS);
      if (counts)
        HB_LAUNCH(mx_count_round_kernel, dim3(counts + rounds), dim3(PLAN_THREADS), plan_lds, s, ids, (int)pairs, experts->base, experts->experts, ws.plan.plan, ws.plan.order,
                  slot_rows, (int)slots, ws.plan.plan_wide, counts, job);
      if (int e = moe_launch_plan(ids, pairs, experts->base, experts->experts, 0, ws.plan, s, slot_rows, nullptr, 0, counts > 0)) return e;
      if (!counts) HB_LAUNCH(mx_quantize_rows_kernel, dim3((unsigned)((job.lanes + 255) / 256)), dim3(256), 0, s, job);
    }
    p1.plan = p2.plan = ws.plan.plan;
    p1.order = p2.order = ws.plan.order;
    p1.aq = ws.xq;
    p1.as = ws.xs;
    const int64_t busy = std::min<int64_t>(slots, pairs / slot_rows + std::min<int64_t>(pairs, experts->experts) / 2 + 1);
    auto span_of = [&](int64_t units, int64_t by) {
      const int64_t spans = std::max<int64_t>(1, std::min<int64_t>((units + by - 1) / by, (MX_MANY_GROUPS + busy - 1) / busy));
      return (int)(((units + by - 1) / by + spans - 1) / spans);
    };
    auto launch = [&](auto kernel, unsigned units, unsigned by, MxMoe& p) {
      p.span = span_of(units, by);
      HB_LAUNCH(kernel, dim3((units + by * p.span - 1) / (by * p.span), (unsigned)slots), dim3(64 * MX_MOE_WAVES), 0, s, p);
    };
    auto fc1 = [&](auto gated) {
      constexpr bool G = decltype(gated)::value;
      if (l1.chunks <= MX_STEP) {
        launch(tall ? mx_fc1_many_kernel<G, 2, 1> : mx_fc1_many_kernel<G, 1, 1>, groups1, 4, p1);
      } else if (l1.chunks <= 2 * MX_STEP) {
        launch(tall ? mx_fc1_many_kernel<G, 2, 2> : mx_fc1_many_kernel<G, 1, 2>, groups1, 2, p1);
      } else {
        launch(tall ? mx_fc1_many_kernel<G, 2, 4> : mx_fc1_many_kernel<G, 1, 4>, groups1, 1, p1);
      }
    };
    if (experts->gated) {
      fc1(std::true_type());
    } else {
      fc1(std::false_type());
    }
    const bool own = l2.chunks <= 2 * MX_STEP;
    auto fc2 = [&](auto* type) {
      using Y = std::remove_pointer_t<decltype(type)>;
      if (own) {
        launch(tall ? mx_fc2_many_kernel<Y, 2, false> : mx_fc2_many_kernel<Y, 1, false>, groups2, MX_MOE_WAVES, p2);
      } else {
        launch(tall ? mx_fc2_many_kernel<Y, 2, true> : mx_fc2_many_kernel<Y, 1, true>, groups2, 1, p2);
      }
    };
    if (narrow) {
      fc2((__bf16*)nullptr);
    } else {
      fc2((float*)nullptr);
    }
  }
  if (sum) combine();
  return launch_status();
}

extern "C" int hb_mxfp4_moe(const hb_mxfp4_experts* experts, const void* x, const int32_t* ids, const float* weights, int m, int topk, int mode, void* out,
                            void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = check(experts)) return e;
  if (!x || !ids || !weights || !out || !workspace) return HB_ENULL;
  if (m <= 0 || topk <= 0 || topk > MX_MOST_TOPK || (int64_t)m * topk > 0x3fffffff || mode < HB_MOE_SUM || mode > HB_MOE_PAIRS_BF16) return HB_EINVAL;
  if (!aligned(x, 16) || !aligned(ids, 4) || !aligned(weights, 4) || !aligned(out, 16) || !aligned(workspace, 16)) return HB_EINVAL;
  if (workspace_bytes < carve(experts, nullptr, m, topk, mode == HB_MOE_SUM).bytes) return HB_EWORKSPACE;
  const int most = most_rows(experts, topk);
  const int64_t row = (int64_t)experts->hidden_out * (mode == HB_MOE_SUM ? 2 : mode == HB_MOE_PAIRS_F32 ? 4 * topk : 2 * topk);  // bytes
  for (int lo = 0; lo < m; lo += std::min(most, m - lo)) {
    if (int e = moe_pass(experts, static_cast<const uint16_t*>(x) + (int64_t)lo * experts->hidden, ids + (int64_t)lo * topk, weights + (int64_t)lo * topk, std::min(most, m - lo),
                         topk, mode, static_cast<uint8_t*>(out) + lo * row, workspace, as_stream(stream)))
      return e;
  }
  return HB_OK;
}
