// Routed experts on microscaled four-bit weights and activations.
//
//   xq = the rows rounded to the format;  per routed pair (row, expert):
//   h = silu(gate xq) * (up xq) or relu(up xq)^2 in FP32, rounded to the format;  y = down h;  out = the weighted sum of a row's y.
#include <algorithm>

#include "mxfp4.hpp"
#include "stream_common.hpp"

namespace hb {

constexpr int MX_SCAN_PAIRS = 512;  // up to this many pairs a workgroup finds its slot from the ids themselves
constexpr int MX_MOE_WAVES = 4;     // wavefronts a workgroup: small ones, so that several on a compute unit cover each other's starts and ends
constexpr int MX_MOE_TILES = 2;     // weight tiles a workgroup (wavefronts that share K) or a wavefront (that have their own)

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
  uint8_t* hq;             // fc1: h by pair (few) or in sorted order (many)
  uint8_t* hs;
  void* y;                 // fc2: [pairs, n], or the rows' sums
};

// The slot of a call of few pairs that begins at pair `first`, found by every workgroup for itself: an expert's pairs in ascending order,
// cut into slots of 32; `list` (LDS) receives the slot's pairs. 0 rows: another workgroup's. All of the workgroup's threads call it, past the
// barrier behind which `masks` (LDS) is written.
__device__ __forceinline__ void mx_scan(const MxMoe& p, int id, uint64_t* masks) {
  for (int i = threadIdx.x; i < MX_SCAN_PAIRS; i += 64 * MX_MOE_WAVES) {
    const uint64_t same = __ballot(i < p.pairs && p.ids[i < p.pairs ? i : 0] == id);
    if ((threadIdx.x & 63) == 0) masks[i >> 6] = same;
  }
}
__device__ __forceinline__ int mx_slot_of(const uint64_t* masks, int first, int* list) {
  int before = 0, total = 0, mine[MX_SCAN_PAIRS / (64 * MX_MOE_WAVES)];
#pragma unroll
  for (int v = 0; v < MX_SCAN_PAIRS / 64; v++) {
    const uint64_t m = masks[v];
    if (v == first >> 6) before = total + __popcll(m & ((1ull << (first & 63)) - 1ull));
#pragma unroll
    for (int j = 0; j < MX_SCAN_PAIRS / (64 * MX_MOE_WAVES); j++)
      if (v == j * MX_MOE_WAVES + (int)(threadIdx.x >> 6)) mine[j] = (m >> (threadIdx.x & 63)) & 1 ? total + __popcll(m & ((1ull << (threadIdx.x & 63)) - 1ull)) : -1;
    total += __popcll(m);
  }
  if (before % MX_ROWS) return 0;
#pragma unroll
  for (int j = 0; j < MX_SCAN_PAIRS / (64 * MX_MOE_WAVES); j++)
    if (mine[j] >= before && mine[j] < before + MX_ROWS) list[mine[j] - before] = j * 64 * MX_MOE_WAVES + threadIdx.x;
  return min(MX_ROWS, total - before);
}

// h of 32 x 32 values (row r of the slot, columns from 32 `column`) from the joined sums of up (and gate), rounded to the format: 256 threads, thread
// i = 64 q + lane holds row lane % 32, columns 8 q + 4 (lane / 32) .. + 3. `tops`: 256 words of LDS that nobody else uses up to the next barrier.
template <bool GATED>
__device__ __forceinline__ void mx_emit_h(const MxMoe& p, const f32x4_t& up, const f32x4_t& gate, int column, bool real, int64_t pos, uint32_t* tops) {
  const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5, q = threadIdx.x >> 6;
  float h[4];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float u = fmaxf(up[j], 0.f);
    h[j] = GATED ? gate[j] / (1.0f + expf(-gate[j])) * up[j] : (up[j] != up[j] ? up[j] : u * u);
    top = max(top, __float_as_uint(h[j]) & 0x7fffffffu);
  }
  tops[threadIdx.x] = top;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < 4; v++) top = max(top, max(tops[v * 64 + r], tops[v * 64 + 32 + r]));
  const uint32_t byte = mx_scale_byte(top);
  const float s = mx_scale_value(byte);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, h[0], h[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, h[2], h[3], s, 1);
  if (real && column < p.inter / 32) {
    *reinterpret_cast<uint16_t*>(p.hq + pos * (p.inter / 2) + 16 * column + 4 * q + 2 * g) = byte == 255u ? 0 : (uint16_t)c;
    if (q == 0 && g == 0) p.hs[pos * (p.inter / 32) + column] = (uint8_t)byte;
  }
}

// The two tiles of a workgroup as h: gated, an up and a gate tile are 32 columns; else each tile is 32. `part`: [waves][2 * 4][64], read by
// all behind a barrier that has passed.
template <bool GATED>
__device__ __forceinline__ void mx_finish_h(const MxMoe& p, f32x4_t* part, uint32_t* tops, bool real, int64_t pos) {
  const f32x4_t first = mx_joined<2>(part, MX_MOE_WAVES, threadIdx.x), second = mx_joined<2>(part, MX_MOE_WAVES, 256 + threadIdx.x);
  if (GATED) {
    mx_emit_h<true>(p, first, second, blockIdx.x, real, pos, tops);
  } else {
    mx_emit_h<false>(p, first, first, 2 * blockIdx.x, real, pos, tops);
    mx_emit_h<false>(p, second, second, 2 * blockIdx.x + 1, real, pos, tops + 256);
  }
}

// ------------------------------------------------------------------------------------------------ few pairs
// fc1: a workgroup two weight tiles of the slot that begins at pair blockIdx.y (none: it leaves). The slot's expert is known from one
// id, so the weights are on their way while the slot's rows are looked for and their activations rounded into LDS.
template <bool GATED, int RUN>
__global__ __launch_bounds__(64 * MX_MOE_WAVES, RUN == 4 ? 3 : 4) void mx_fc1_few_kernel(MxMoe p) {
  extern __shared__ f32x4_t part[];
  __shared__ uint64_t masks[MX_SCAN_PAIRS / 64];
  __shared__ int list[MX_ROWS];
  __shared__ uint32_t tops[GATED ? 256 : 512];
  const int first = blockIdx.y, id = p.ids[first], e = id - p.base;
  if (e < 0 || e >= p.experts) return;
  MxStream<MX_MOE_TILES, RUN> s(p.w + e * p.expert_bytes, MxLayout(p.n, p.k), blockIdx.x * MX_MOE_TILES, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), MX_MOE_WAVES);
  mx_scan(p, id, masks);
  __syncthreads();
  const int rows = mx_slot_of(masks, first, list);
  if (rows == 0) return;
  __syncthreads();
  const MxActs acts(part, rows, p.k);
  for (int i = threadIdx.x; i < rows * acts.groups; i += 64 * MX_MOE_WAVES) {
    const int r = i / acts.groups, group = i - r * acts.groups;
    acts.put(r, group, static_cast<const __bf16*>(p.x) + (int64_t)(list[r] / p.topk) * p.k + MX_GROUP * group);
  }
  __syncthreads();
  s.run(acts);
  mx_hand_over<MX_MOE_TILES>(part, s.acc);
  const int r = threadIdx.x & 31;
  mx_finish_h<GATED>(p, part, tops, r < rows, r < rows ? list[r] : 0);
}

// fc2 of the same slots, its results by pair.
template <typename Y, int RUN>
__global__ __launch_bounds__(64 * MX_MOE_WAVES, RUN == 4 ? 3 : 4) void mx_fc2_few_kernel(MxMoe p) {
  extern __shared__ f32x4_t part[];
  __shared__ uint64_t masks[MX_SCAN_PAIRS / 64];
  __shared__ int list[MX_ROWS];
  const int first = blockIdx.y, id = p.ids[first], e = id - p.base;
  if (e < 0 || e >= p.experts) return;
  MxStream<MX_MOE_TILES, RUN> s(p.w + e * p.expert_bytes, MxLayout(p.n, p.k), blockIdx.x * MX_MOE_TILES, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), MX_MOE_WAVES);
  mx_scan(p, id, masks);
  __syncthreads();
  const int rows = mx_slot_of(masks, first, list);
  if (rows == 0) return;
  __syncthreads();
  const MxActs acts(part, rows, p.k);
  for (int i = threadIdx.x; i < rows * acts.groups; i += 64 * MX_MOE_WAVES) {
    const int r = i / acts.groups, group = i - r * acts.groups;
    acts.put(r, group, p.aq + (int64_t)list[r] * (p.k / 2), p.as + (int64_t)list[r] * acts.groups);
  }
  __syncthreads();
  s.run(acts);
  mx_hand_over<MX_MOE_TILES>(part, s.acc);
  const int r = threadIdx.x & 31;
  if (r >= rows) return;
#pragma unroll
  for (int t = 0; t < MX_MOE_TILES; t++) {
    const f32x4_t sum = mx_joined<MX_MOE_TILES>(part, MX_MOE_WAVES, 256 * t + threadIdx.x);
    const int n = (blockIdx.x * MX_MOE_TILES + t) * MX_ROWS + 8 * (threadIdx.x >> 6) + 4 * ((threadIdx.x & 63) >> 5);
    typedef __attribute__((ext_vector_type(4))) Y y4_t;
    if (n < p.n) *reinterpret_cast<y4_t*>(static_cast<Y*>(p.y) + (int64_t)list[r] * p.n + n) = y4_t{(Y)sum[0], (Y)sum[1], (Y)sum[2], (Y)sum[3]};
  }
}

// fc2 and the weighted sum of one row (blockIdx.y): a workgroup one tile of columns, its wavefronts the row's pairs in turn, their weighted
// results added in wavefront order. Reads a row's experts whether or not other rows name them too.
constexpr int MX_ROW_WAVES = 8;
constexpr int MX_SINGLE_ROWS = 1;
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
// A slot of the plan (up to 32 MT rows of an expert) and its wavefronts' operands from memory: the activations' codes of a chunk are 32 bytes a
// row, read where they lie. RUN chunks are asked for, then multiplied: the other wavefronts of the compute unit cover the wait.
template <int MT>
struct MxRows {
  const uint8_t *codes[MT], *scales[MT];
  int groups;
  template <class Row>
  __device__ __forceinline__ MxRows(const MxMoe& p, int rows, Row&& row_of) : groups(p.k / MX_GROUP) {
#pragma unroll
    for (int i = 0; i < MT; i++) {
      const int64_t row = row_of(min(32 * i + (int)(threadIdx.x & 31), rows - 1));  // (past the last: that one again, not to be stored)
      codes[i] = p.aq + row * (p.k / 2);
      scales[i] = p.as + row * groups;
    }
  }
};
template <int MT, int RUN>
__device__ __forceinline__ void mx_gathered(const uint8_t* __restrict__ w, const MxLayout& at, int t0, int c0, int c1, const MxRows<MT>& rows, int tiles_of_rows,
                                            f32x16_t (&acc)[MT][MX_MOE_TILES]) {
  constexpr int NT = MX_MOE_TILES;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const uint8_t *codes[NT], *scales[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int tile = min(t0 + t, at.tiles - 1);
    codes[t] = w + (int64_t)tile * at.chunks * 1024 + lane * 16;
    scales[t] = w + at.codes() + (int64_t)tile * at.quads * 256 + lane * 4;
  }
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][t][e] = 0.f;
  for (int c = c0; c < c1; c += RUN) {
    i32x4_t b[RUN][NT], a[RUN][MT];
    uint32_t sb[NT], sa[RUN][MT];
#pragma unroll
    for (int t = 0; t < NT; t++) sb[t] = *reinterpret_cast<const uint32_t*>(scales[t] + (c >> 2) * 256);
#pragma unroll
    for (int u = 0; u < RUN; u++) {
      const int in = min(c + u, c1 - 1), group = min(2 * in + half, rows.groups - 1);
#pragma unroll
      for (int t = 0; t < NT; t++) b[u][t] = *reinterpret_cast<const i32x4_t*>(codes[t] + in * 1024);
#pragma unroll
      for (int i = 0; i < MT; i++) {
        a[u][i] = *reinterpret_cast<const i32x4_t*>(rows.codes[i] + 16 * group);
        sa[u][i] = rows.scales[i][group];
      }
    }
#pragma unroll
    for (int t = 0; t < NT; t++) sb[t] >>= 8 * (c & 3);
    mx_unrolled<RUN>([&](auto u) {
      if (c + u.value < c1) {
#pragma unroll
        for (int i = 0; i < MT; i++)
          if (i < tiles_of_rows) {
#pragma unroll
            for (int t = 0; t < NT; t++) acc[i][t] = mx_mfma<u.value, 0>(b[u.value][t], sb[t], a[u.value][i], sa[u.value][i], acc[i][t]);
          }
      }
    });
  }
}

// fc1: two weight tiles a workgroup, K split among its wavefronts.
template <bool GATED, int MT>
__global__ __launch_bounds__(64 * MX_MOE_WAVES, MT == 1 ? 4 : 3) void mx_fc1_many_kernel(MxMoe p) {
  __shared__ f32x4_t part[MX_MOE_WAVES * MX_MOE_TILES * 256];
  __shared__ uint32_t tops[GATED ? 256 : 512];
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * (int)blockIdx.y;
  const int rows = entry[2], p0 = entry[1];
  if (rows == 0) return;
  constexpr int RUN = 2;
  const MxLayout at(p.n, p.k);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), runs = (at.chunks + RUN - 1) / RUN;
  const MxRows<MT> from(p, rows, [&](int r) { return (int64_t)(p.order[p0 + r] / p.topk); });
  f32x16_t acc[MT][MX_MOE_TILES];
  mx_gathered<MT, RUN>(p.w + entry[0] * p.expert_bytes, at, blockIdx.x * MX_MOE_TILES, RUN * (runs * wave / MX_MOE_WAVES),
                       min(at.chunks, RUN * (runs * (wave + 1) / MX_MOE_WAVES)), from, (rows + 31) / 32, acc);
#pragma unroll
  for (int i = 0; i < MT; i++) {
    if (32 * i >= rows) break;
    mx_hand_over<MX_MOE_TILES>(part, acc[i]);
    const int r = 32 * i + (threadIdx.x & 31);
    mx_finish_h<GATED>(p, part, tops, r < rows, p0 + r);
  }
}

// fc2: each wavefront two tiles of its own, all of K; a row's 64 results leave together (as mx_store_rows does it, the rows found through `order`).
template <typename Y, int MT>
__global__ __launch_bounds__(64 * MX_MOE_WAVES, MT == 1 ? 4 : 3) void mx_fc2_many_kernel(MxMoe p) {
  constexpr int NT = MX_MOE_TILES, PIECES = NT * MX_ROWS * (int)sizeof(Y) / 16, ROWS = 64 / PIECES;
  __shared__ i32x4_t places[MX_MOE_WAVES][MX_ROWS * PIECES];
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * (int)blockIdx.y;
  const int rows = entry[2], p0 = entry[1];
  if (rows == 0) return;
  const MxLayout at(p.n, p.k);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t0 = (blockIdx.x * MX_MOE_WAVES + wave) * NT;
  if (t0 >= at.tiles) return;
  const MxRows<MT> from(p, rows, [&](int r) { return (int64_t)p0 + r; });
  f32x16_t acc[MT][NT];
  mx_gathered<MT, 2>(p.w + entry[0] * p.expert_bytes, at, t0, 0, at.chunks, from, (rows + 31) / 32, acc);
  i32x4_t* place = places[wave];
  uint8_t* bytes = reinterpret_cast<uint8_t*>(place);
  const int r = lane & 31, g = lane >> 5;
#pragma unroll
  for (int i = 0; i < MT; i++) {
    if (32 * i >= rows) break;
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int in = (MX_ROWS * j + 8 * q + 4 * g) * (int)sizeof(Y), piece = (in / 16) ^ (r & (PIECES - 1));
        const f32x4_t v = mx_quarter(acc[i][j], q);
        typedef __attribute__((ext_vector_type(4))) Y y4_t;
        *reinterpret_cast<y4_t*>(bytes + (r * PIECES + piece) * 16 + in % 16) = y4_t{(Y)v[0], (Y)v[1], (Y)v[2], (Y)v[3]};
      }
#pragma unroll
    for (int first = 0; first < MX_ROWS; first += ROWS) {
      const int row = first + lane / PIECES, piece = lane % PIECES, n = t0 * MX_ROWS + piece * (16 / (int)sizeof(Y));
      const i32x4_t v = place[row * PIECES + (piece ^ (row & (PIECES - 1)))];
      if (32 * i + row < rows && n < p.n) *reinterpret_cast<i32x4_t*>(static_cast<Y*>(p.y) + (int64_t)p.order[p0 + 32 * i + row] * p.n + n) = v;
    }
  }
}

namespace {
struct MxWorkspace {
  MoeWorkspace plan;
  uint8_t *xq, *xs, *hq, *hs;
  void* y;
  size_t bytes;
};

bool few_pairs(int64_t pairs, int hidden, int inter) { return pairs <= MX_SCAN_PAIRS && MxActs::bytes(std::min<int64_t>(pairs, MX_ROWS), std::max(hidden, inter)) <= 48 * 1024; }

MxWorkspace carve(const hb_mxfp4_experts* ex, void* base, int64_t m, int topk, bool sum) {
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
    w.xq = take((size_t)m * (ex->hidden / 2));
    w.xs = take((size_t)m * (ex->hidden / 32));
  }
  w.hq = take((size_t)pairs * (ex->inter / 2));
  w.hs = take((size_t)pairs * (ex->inter / 32));
  w.y = sum ? take((size_t)pairs * ex->hidden_out * sizeof(float)) : nullptr;
  w.bytes = off;
  return w;
}

int fc1_rows(const hb_mxfp4_experts* ex) { return ex->gated ? 2 * ex->inter : ex->inter; }

int check(const hb_mxfp4_experts* ex) {
  if (!ex || !ex->fc1 || !ex->fc2) return HB_ENULL;
  if (ex->experts <= 0 || ex->base < 0 || ex->hidden <= 0 || ex->inter <= 0 || ex->hidden_out <= 0 || ex->hidden % 32 || ex->inter % 32 || ex->hidden_out % 8 ||
      ex->hidden > 1 << 20 || ex->inter > 1 << 20 || ex->hidden_out > 1 << 20 || ex->experts > 1 << 20 || ex->base > 1 << 28)
    return HB_EINVAL;
  return aligned(ex->fc1, 16) && aligned(ex->fc2, 16) ? HB_OK : HB_EINVAL;
}
}  // namespace

}  // namespace hb

using namespace hb;

extern "C" size_t hb_mxfp4_moe_workspace_bytes(const hb_mxfp4_experts* experts, int m, int topk) {
  if (check(experts) != HB_OK || m <= 0 || topk <= 0 || (int64_t)m * topk > 0x3fffffff) return 0;
  return carve(experts, nullptr, m, topk, true).bytes;
}

extern "C" int hb_mxfp4_moe(const hb_mxfp4_experts* experts, const void* x, const int32_t* ids, const float* weights, int m, int topk, int mode, void* out,
                            void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = check(experts)) return e;
  if (!x || !ids || !weights || !out || !workspace) return HB_ENULL;
  if (m <= 0 || topk <= 0 || (int64_t)m * topk > 0x3fffffff || mode < HB_MOE_SUM || mode > HB_MOE_PAIRS_BF16) return HB_EINVAL;
  if (!aligned(x, 16) || !aligned(ids, 4) || !aligned(weights, 4) || !aligned(out, 16) || !aligned(workspace, 16)) return HB_EINVAL;
  const bool sum = mode == HB_MOE_SUM;
  const MxWorkspace ws = carve(experts, workspace, m, topk, sum);
  if (workspace_bytes < ws.bytes) return HB_EWORKSPACE;
  const int64_t pairs = (int64_t)m * topk;
  hipStream_t s = as_stream(stream);
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
  bool narrow = mode == HB_MOE_PAIRS_BF16;
  const unsigned groups1 = (unsigned)((l1.tiles + MX_MOE_TILES - 1) / MX_MOE_TILES), groups2 = (unsigned)((l2.tiles + MX_MOE_TILES - 1) / MX_MOE_TILES);
  if (few_pairs(pairs, experts->hidden, experts->inter)) {
    const int most = (int)std::min<int64_t>(MX_ROWS, pairs);
    const size_t room = (size_t)MX_MOE_WAVES * MX_MOE_TILES * 4096;
    p1.x = x;
    const size_t lds1 = std::max(room, MxActs::bytes(most, p1.k)), lds2 = std::max(room, MxActs::bytes(most, p2.k));
    const dim3 grid1(groups1, (unsigned)pairs), grid2(groups2, (unsigned)pairs), block(64 * MX_MOE_WAVES);
    const bool long1 = l1.chunks >= 4 * MX_MOE_WAVES, long2 = l2.chunks >= 4 * MX_MOE_WAVES;
    auto launch = [&](auto kernel, dim3 grid, size_t lds, const MxMoe& p) { HB_LAUNCH(kernel, grid, block, lds, s, p); };
    if (experts->gated) {
      launch(long1 ? mx_fc1_few_kernel<true, 4> : mx_fc1_few_kernel<true, 2>, grid1, lds1, p1);
    } else {
      launch(long1 ? mx_fc1_few_kernel<false, 4> : mx_fc1_few_kernel<false, 2>, grid1, lds1, p1);
    }
    if (sum && m <= MX_SINGLE_ROWS) {
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
    // a summed prefill-sized call keeps its pair outputs in BF16, half the traffic of its widest tensor, as the framework's other routed calls do
    narrow = narrow || (sum && m >= MOE_WIDE_ROWS);
    const bool tall = pairs >= (int64_t)experts->experts * 24;
    const int slot_rows = tall ? 2 * MX_ROWS : MX_ROWS;
    const int64_t slots = moe_max_slots(pairs, experts->experts, 0, slot_rows);
    if (slots > 65535) return HB_EINVAL;
    if (int e = moe_launch_plan(ids, pairs, experts->base, experts->experts, 0, ws.plan, s, slot_rows)) return e;
    if (int e = hb_mxfp4_quantize(x, HB_BF16, m, experts->hidden, ws.xq, ws.xs, stream)) return e;
    p1.plan = p2.plan = ws.plan.plan;
    p1.order = p2.order = ws.plan.order;
    p1.aq = ws.xq;
    p1.as = ws.xs;
    auto launch = [&](auto kernel, unsigned groups, const MxMoe& p) { HB_LAUNCH(kernel, dim3(groups, (unsigned)slots), dim3(64 * MX_MOE_WAVES), 0, s, p); };
    const unsigned own2 = (unsigned)((l2.tiles + MX_MOE_TILES * MX_MOE_WAVES - 1) / (MX_MOE_TILES * MX_MOE_WAVES));
    if (experts->gated) {
      launch(tall ? mx_fc1_many_kernel<true, 2> : mx_fc1_many_kernel<true, 1>, groups1, p1);
    } else {
      launch(tall ? mx_fc1_many_kernel<false, 2> : mx_fc1_many_kernel<false, 1>, groups1, p1);
    }
    if (narrow) {
      launch(tall ? mx_fc2_many_kernel<__bf16, 2> : mx_fc2_many_kernel<__bf16, 1>, own2, p2);
    } else {
      launch(tall ? mx_fc2_many_kernel<float, 2> : mx_fc2_many_kernel<float, 1>, own2, p2);
    }
  }
  if (sum) {
    CombineParams c{};
    c.pairs = ws.y;
    c.pairs_bf16 = narrow;
    c.ids = ids;
    c.weights = weights;
    c.e_lo = experts->base;
    c.e_n = experts->experts;
    c.m = m;
    c.topk = topk;
    c.h = experts->hidden_out;
    c.out = static_cast<uint16_t*>(out);
    moe_launch_combine(c, s);
  }
  return launch_status();
}
