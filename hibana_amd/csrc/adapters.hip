// Low-rank adapters of many requests at once beside a shared projection, and their gradients.
//
//   out[r] = y[r] + s_i (x[r] a_i^T) b_i,  i = index[r];   a [adapters, rank, k], b [adapters, rank, n]
//   g[r] = s_i dy[r] b_i^T;  dx[r] = g[r] a_i;  da_i = sum over i's rows of g[r]^T x[r];  db_i = sum of s_i (x[r] a_i^T)^T dy[r]
//
// Both matrices of an adapter lie rank by rank along their long axis, so the six products are of three kinds:
//   shrink   rows [m, long] times a matrix's rows: contraction over the long axis, [m, rank] FP32 sums, the long axis cut into `splits`
//   expand   [m, rank] times the matrix: contraction over the rank, added to y's rows (or alone: dx)
//   outer    [m, rank]^T times rows [m, long]: contraction over an adapter's rows, FP32
// Rows are grouped by adapter: a tile's rows are one adapter's, gathered by number. All of it is bound by memory (few operations a byte at
// any rank here); the matrix instructions are there so that one read of an adapter's matrix serves a tile's rows.
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace hb {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef uint32_t u32x4_loose __attribute__((ext_vector_type(4), aligned(2)));  // sixteen bytes at any element: rows of odd length

constexpr int AD_SELF_ROWS = 256;  // rows up to which a workgroup finds its tile from the index itself
constexpr int AD_CHUNK = 128;      // rows of an outer product's step: 32 a wavefront
constexpr int AD_MOST = 4096;      // adapters
constexpr int AD_RANK = 256;
constexpr int AD_MAX_ROWS = 1 << 24;
constexpr int AD_LONGEST = 1 << 22;  // of either axis

template <int KIND> struct AdType;
template <> struct AdType<HB_BF16> { static constexpr int SIZE = 2, PARTS = 2, OUTER = 3; };  // parts that FP32 values are cut into
template <> struct AdType<HB_F16> { static constexpr int SIZE = 2, PARTS = 2, OUTER = 2; };
template <> struct AdType<HB_F32> { static constexpr int SIZE = 4, PARTS = 1, OUTER = 1; };
template <int KIND> constexpr int AD_VEC = 16 / AdType<KIND>::SIZE;  // elements of a 16-byte load: the columns a lane holds

template <int KIND>
__device__ __forceinline__ float ad_value(uint32_t bits) {
  if constexpr (KIND == HB_BF16) return bf16_bits_to_f32((uint16_t)bits);
  if constexpr (KIND == HB_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  return __uint_as_float(bits);
}
template <int KIND>
__device__ __forceinline__ uint32_t ad_bits(float v) {
  if constexpr (KIND == HB_BF16) return f32_to_bf16_bits(v);
  if constexpr (KIND == HB_F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
  return __float_as_uint(v);
}

template <int KIND>
__device__ __forceinline__ uint32_t ad_elem(const u32x4_t& v, int j) {
  if constexpr (AdType<KIND>::SIZE == 4) return v[j];
  return (v[j >> 1] >> (16 * (j & 1))) & 0xffffu;
}

// Sixteen bytes from `at`, of which the first `left` elements are the row's (the rest zero).
template <int KIND>
__device__ __forceinline__ u32x4_t ad_load(const char* at, int64_t left) {
  if (left >= AD_VEC<KIND>) return *reinterpret_cast<const u32x4_loose*>(at);
  u32x4_t v{0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < AD_VEC<KIND>; j++) {
    if (j < left) {
      if constexpr (AdType<KIND>::SIZE == 4) v[j] = reinterpret_cast<const uint32_t*>(at)[j];
      else v[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(at)[j] << (16 * (j & 1));
    }
  }
  return v;
}
template <int KIND>
__device__ __forceinline__ void ad_store(char* at, const u32x4_t& v, int64_t left) {
  if (left >= AD_VEC<KIND>) {
    *reinterpret_cast<u32x4_loose*>(at) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < AD_VEC<KIND>; j++) {
    if (j < left) {
      if constexpr (AdType<KIND>::SIZE == 4) reinterpret_cast<uint32_t*>(at)[j] = v[j];
      else reinterpret_cast<uint16_t*>(at)[j] = (uint16_t)(v[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// acc += the 16 x 16 product of two operands whose lanes hold sixteen bytes along the contraction: 32 places of 16-bit types in one
// instruction, 16 of FP32 in four (instruction i contracts element i of every lane: any order serves that both operands have).
template <int KIND>
__device__ __forceinline__ f32x4_t ad_mma(const u32x4_t& a, const u32x4_t& b, f32x4_t acc) {
  if constexpr (KIND == HB_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc, 0, 0, 0);
  if constexpr (KIND == HB_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), acc, 0, 0, 0);
  if constexpr (KIND == HB_F32) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), acc, 0, 0, 0);
  }
  return acc;
}

// ------------------------------------------------------------------------------------------------ rows by adapter

// Classes 0 .. adapters - 1 are the adapters, `adapters` the rows without one (an index outside the pool, an adapter of rank 0).
struct AdIndex {
  const void* index;
  const int32_t* ranks;
  int wide;       // the index is int64
  int m, adapters, rank;
};
__device__ __forceinline__ int ad_rank(const AdIndex& p, int c) {
  return c >= p.adapters ? 0 : p.ranks ? min(max(p.ranks[c], 0), p.rank) : p.rank;
}
__device__ __forceinline__ int ad_class(const AdIndex& p, int row) {
  const int64_t i = p.wide ? reinterpret_cast<const int64_t*>(p.index)[row] : reinterpret_cast<const int32_t*>(p.index)[row];
  if (i < 0 || i >= p.adapters) return p.adapters;
  return p.ranks && p.ranks[i] <= 0 ? p.adapters : (int)i;
}

// The plan: int32 arrays [classes + 1] of where a class's rows, its tiles of two heights, its units (runs of `unit` rows, an outer
// product's share of the work) and its slots (partial sums: the units of classes that have more than one) begin, then the rows in order.
struct AdPlan {
  int32_t* at;
  int classes;
  __host__ __device__ int32_t* rows() const { return at; }
  __host__ __device__ int32_t* tiles(int which) const { return at + (1 + which) * (classes + 1); }
  __host__ __device__ int32_t* units() const { return at + 3 * (classes + 1); }
  __host__ __device__ int32_t* slots() const { return at + 4 * (classes + 1); }
  __host__ __device__ int32_t* order() const { return at + 5 * (classes + 1); }
  static size_t ints(int classes, int64_t m) { return 5 * ((size_t)classes + 1) + m; }
};

struct AdPlanParams {
  AdIndex in;
  AdPlan plan;
  int height[2];  // rows of the two kinds of tile
  int unit;
  int segments;   // wavefronts that count and place rows, each those of one stretch; segments * classes counters in LDS
};

// One workgroup: a stable counting sort (rows of a class stay in ascending order, so sums over them are the same every time).
__global__ __launch_bounds__(1024) void ad_plan_kernel(AdPlanParams p) {
  extern __shared__ int32_t counters[];  // [segment][class]
  __shared__ int32_t carry[16][5];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, classes = p.plan.classes, m = p.in.m;
  for (int i = threadIdx.x; i < p.segments * classes; i += 1024) counters[i] = 0;
  __syncthreads();
  const int stretch = ((m + p.segments - 1) / p.segments + 63) / 64 * 64;
  const int from = (int)min((int64_t)wave * stretch, (int64_t)m), upto = min(from + stretch, m);
  volatile int32_t* mine = counters + wave * classes;
  if (wave < p.segments)
    for (int r = from + lane; r < upto; r += 64) atomicAdd(const_cast<int32_t*>(mine) + ad_class(p.in, r), 1);
  __syncthreads();
  // each thread a run of classes: counts over the segments, then prefix sums over the threads
  const int per = (classes + 1023) / 1024, c0 = min((int)threadIdx.x * per, classes), c1 = min(c0 + per, classes);
  int sum[5] = {0, 0, 0, 0, 0};
  auto add = [&](int (&to)[5], int c, int rows) {
    const int units = c < p.in.adapters ? (rows + p.unit - 1) / p.unit : 0;
    to[0] += rows;
    to[1] += (rows + p.height[0] - 1) / p.height[0];
    to[2] += (rows + p.height[1] - 1) / p.height[1];
    to[3] += units;
    to[4] += units > 1 ? units : 0;
  };
  for (int c = c0; c < c1; c++) {
    int rows = 0;
    for (int s = 0; s < p.segments; s++) rows += counters[s * classes + c];
    add(sum, c, rows);
  }
  int before[5];
#pragma unroll
  for (int j = 0; j < 5; j++) {
    int x = sum[j];
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(x, d);
      if (lane >= d) x += up;
    }
    before[j] = x - sum[j];
    if (lane == 63) carry[wave][j] = x;
  }
  __syncthreads();
  for (int w = 0; w < wave; w++)
#pragma unroll
    for (int j = 0; j < 5; j++) before[j] += carry[w][j];
  int32_t* out[5] = {p.plan.rows(), p.plan.tiles(0), p.plan.tiles(1), p.plan.units(), p.plan.slots()};
  for (int c = c0; c < c1; c++) {
    int at = before[0], rows = 0;
    for (int s = 0; s < p.segments; s++) {
      const int n = counters[s * classes + c];
      counters[s * classes + c] = at + rows;
      rows += n;
    }
#pragma unroll
    for (int j = 0; j < 5; j++) out[j][c] = before[j];
    add(before, c, rows);
    if (c == classes - 1)
#pragma unroll
      for (int j = 0; j < 5; j++) out[j][classes] = before[j];
  }
  __syncthreads();
  if (wave < p.segments) {
    int32_t* order = p.plan.order();
    for (int r0 = from; r0 < upto; r0 += 64) {
      const int r = r0 + lane, c = r < upto ? ad_class(p.in, r) : -1;
      uint64_t left = __ballot(c >= 0);
      while (left) {
        const int v = __builtin_amdgcn_readlane(c, __builtin_ctzll(left));
        const uint64_t same = __ballot(c == v);
        const int base = mine[v];
        if (c == v) order[base + __popcll(same & ((1ull << lane) - 1ull))] = r;
        if (lane == 0) mine[v] = base + __popcll(same);
        left &= ~same;
      }
    }
  }
}

// The class that place t of an ascending array [classes + 1] of first places is in (by every wavefront for itself).
__device__ __forceinline__ int ad_find(const int32_t* first, int classes, int t) {
  const int lane = threadIdx.x & 63;
  int c = -1;
  for (int i = 0; i <= classes; i += 64) {
    const int n = __popcll(__ballot(i + lane <= classes && first[min(i + lane, classes)] <= t));
    c += n;
    if (n < 64) break;
  }
  return c;
}

// Tile t: its class, its rows' numbers in LDS and how many they are (0: no such tile). Without a plan, t is a row: a tile begins at every
// T-th row of a class.
template <int T>
__device__ __forceinline__ int ad_tile(const AdIndex& p, const AdPlan& plan, int which, int t, int32_t* rows, int& c) {
  const int lane = threadIdx.x & 63;
  int count;
  if (plan.at) {
    if (t >= plan.tiles(which)[plan.classes]) return 0;
    c = ad_find(plan.tiles(which), plan.classes, t);
    const int start = plan.rows()[c] + (t - plan.tiles(which)[c]) * T;
    count = min(T, plan.rows()[c + 1] - start);
    if (threadIdx.x < T) rows[threadIdx.x] = plan.order()[start + min((int)threadIdx.x, count - 1)];
  } else {
    c = ad_class(p, t);
    uint64_t same[AD_SELF_ROWS / 64];
    int ahead = 0, all = 0;
#pragma unroll
    for (int j = 0; j < AD_SELF_ROWS / 64; j++) {
      same[j] = 0;
      if (64 * j < p.m) same[j] = __ballot(64 * j + lane < p.m && ad_class(p, min(64 * j + lane, p.m - 1)) == c);
      if (64 * j + 63 < t) ahead += __popcll(same[j]);
      else if (64 * j <= t) ahead += __popcll(same[j] & ((1ull << (t - 64 * j)) - 1ull));
      all += __popcll(same[j]);
    }
    if (ahead % T) return 0;
    count = min(T, all - ahead);
    int at = 0;
#pragma unroll
    for (int j = 0; j < AD_SELF_ROWS / 64; j++) {
      const int place = at + __popcll(same[j] & ((1ull << lane) - 1ull)) - ahead;
      if ((same[j] >> lane & 1) && place >= 0 && place < T) rows[place] = 64 * j + lane;  // (every wavefront the same)
      at += __popcll(same[j]);
    }
    if ((int)threadIdx.x >= count && threadIdx.x < T) rows[threadIdx.x] = t;  // places behind the last row repeat the first: t itself
  }
  __syncthreads();
  return count;
}

// ------------------------------------------------------------------------------------------------ shrink

struct AdShrinkJob {
  const char* v;      // rows, `stride` bytes apart
  int64_t stride;
  const char* w;      // [adapters, rank, length]
  int length, share;  // units of 128 bytes a split
  float* sums;        // [splits, m, rank]
};
struct AdShrink {
  AdIndex in;
  AdPlan plan;
  AdShrinkJob job[2];
  int chunks;  // of RT x 16 ranks
};

// A workgroup: a tile's rows times RT x 16 ranks over one split of the long axis, the four wavefronts taking units of 128 bytes in turn (a
// whole cache line of every row) and joining their sums in LDS.
template <int KIND, int TM, int RT>
__global__ __launch_bounds__(256) void ad_shrink_kernel(AdShrink p) {
  constexpr int VEC = AD_VEC<KIND>, SIZE = AdType<KIND>::SIZE, UNIT = 128 / SIZE;
  __shared__ int32_t rows[16 * TM];
  __shared__ f32x4_t part[4][TM * RT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4, col = lane & 15;
  int c;
  const int count = ad_tile<16 * TM>(p.in, p.plan, 0, blockIdx.x, rows, c);
  if (count == 0 || c >= p.in.adapters) return;
  const AdShrinkJob& job = p.job[blockIdx.z / p.chunks];
  const int rank = ad_rank(p.in, c), r0 = (blockIdx.z % p.chunks) * 16 * RT;
  if (r0 >= rank) return;
  const int units = (job.length + UNIT - 1) / UNIT, whole = job.length / UNIT, u0 = blockIdx.y * job.share, u1 = min(u0 + job.share, units);
  const char* x[TM];
  const char* w[RT];
#pragma unroll
  for (int i = 0; i < TM; i++) x[i] = job.v + rows[16 * i + col] * job.stride + group * 16;
#pragma unroll
  for (int i = 0; i < RT; i++) w[i] = job.w + ((int64_t)c * p.in.rank + min(r0 + 16 * i + col, rank - 1)) * job.length * SIZE + group * 16;  // (ranks behind the last: nobody reads the sums)
  f32x4_t acc[TM][RT] = {};
  for (int u = u0 + wave; u < min(u1, whole); u += 4) {
    u32x4_t xv[TM][2], wv[RT][2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int i = 0; i < RT; i++) wv[i][h] = *reinterpret_cast<const u32x4_loose*>(w[i] + (int64_t)u * 128 + 64 * h);
#pragma unroll
      for (int i = 0; i < TM; i++) xv[i][h] = *reinterpret_cast<const u32x4_loose*>(x[i] + (int64_t)u * 128 + 64 * h);
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < RT; j++) acc[i][j] = ad_mma<KIND>(xv[i][h], wv[j][h], acc[i][j]);
  }
  if (u0 <= whole && u1 > whole && (whole - u0) % 4 == wave) {  // the row's last, cut unit, by the wavefront whose turn it is
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int64_t left = job.length - ((int64_t)whole * UNIT + h * (UNIT / 2) + group * VEC);
      u32x4_t wv[RT];
#pragma unroll
      for (int i = 0; i < RT; i++) wv[i] = ad_load<KIND>(w[i] + (int64_t)whole * 128 + 64 * h, left);
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const u32x4_t xv = ad_load<KIND>(x[i] + (int64_t)whole * 128 + 64 * h, left);
#pragma unroll
        for (int j = 0; j < RT; j++) acc[i][j] = ad_mma<KIND>(xv, wv[j], acc[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < RT; j++) part[wave][i * RT + j][lane] = acc[i][j];
  __syncthreads();
  float* sums = job.sums + (int64_t)blockIdx.y * p.in.m * p.in.rank;
  for (int t = wave; t < TM * RT; t += 4) {
    const f32x4_t s = part[0][t][lane] + part[1][t][lane] + part[2][t][lane] + part[3][t][lane];
    const int r = r0 + 16 * (t % RT) + col;
    if (r >= rank) continue;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int place = 16 * (t / RT) + 4 * group + i;
      if (place < count) sums[(int64_t)rows[place] * p.in.rank + r] = s[i];
    }
  }
}

// ------------------------------------------------------------------------------------------------ FP32 sums as matrix operands

// The sums are operands of the second product. To keep what FP32 holds of them, a value goes in as the sum of two or three of the type's:
// BF16 by cutting (8 bits a part, never past the value's size: no overflow; two parts 2^-16 of it, three all of it), FP16 by rounding what a power of two
// has brought below 2^15 (two parts: 2^-22, or 2^-40 of the largest).
template <int KIND, int PARTS>
__device__ __forceinline__ void ad_cut(float v, uint16_t (&part)[PARTS]) {
  const bool finite = fabsf(v) < INFINITY;
  if constexpr (KIND == HB_BF16) {
    float rest = v;
#pragma unroll
    for (int i = 0; i < PARTS; i++) {
      if (i == PARTS - 1) {
        part[i] = finite || i == 0 ? f32_to_bf16_bits(rest) : 0;
      } else {
        const uint32_t top = __float_as_uint(rest) & 0xffff0000u;
        part[i] = finite ? (uint16_t)(top >> 16) : i == 0 ? f32_to_bf16_bits(v) : 0;
        rest -= __uint_as_float(top);
      }
    }
  } else {
    const _Float16 high = (_Float16)v;
    part[0] = __builtin_bit_cast(uint16_t, high);
    part[1] = finite ? __builtin_bit_cast(uint16_t, (_Float16)(v - (float)high)) : 0;
  }
}

// The power of two that brings a largest magnitude to 2^14 .. 2^15, and its inverse.
__device__ __forceinline__ int ad_exponent(float most) { return most > 0.f ? max((int)(__float_as_uint(most) >> 23) - 127, -100) - 14 : -100; }
__device__ __forceinline__ float ad_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Lane's operands along the contraction from eight rows of sixteen bytes: element j of the eight, for each j.
template <int KIND>
__device__ __forceinline__ void ad_turn(const u32x4_t (&v)[8], u32x4_t (&out)[AD_VEC<KIND>]) {
  if constexpr (AdType<KIND>::SIZE == 2) {
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
      for (int q = 0; q < 4; q++) out[j][q] = __builtin_amdgcn_perm(v[2 * q + 1][j >> 1], v[2 * q][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
  }
}

// ------------------------------------------------------------------------------------------------ expand

struct AdExpand {
  AdIndex in;
  AdPlan plan;
  const float* sums;   // [splits, m, rank]
  const float* scale;  // [adapters] or null
  int splits, n, padded;  // padded: the rank in LDS, a multiple of 32
  const char* w;       // [adapters, rank, n]
  const char* y;       // null: zeros
  int64_t y_stride;    // bytes
  char* out;
  int64_t out_stride;
};

// A workgroup: a tile's rows times four wavefronts' columns, sixteen lanes of sixteen bytes each. Lane l's operand for instruction j is column
// l * VEC + j: eight rows of the matrix, turned in registers, give it all of them, and the results are whole 16-byte pieces of out's rows.
template <int KIND, int TM>
__global__ __launch_bounds__(256) void ad_expand_kernel(AdExpand p) {
  constexpr int VEC = AD_VEC<KIND>, SIZE = AdType<KIND>::SIZE, PARTS = AdType<KIND>::PARTS;
  extern __shared__ __align__(16) char staged[];  // [part][row][padded + 16 bytes]
  __shared__ int32_t rows[16 * TM];
  __shared__ int32_t power[16 * TM];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4, col = lane & 15;
  int c;
  const int count = ad_tile<16 * TM>(p.in, p.plan, 1, blockIdx.x, rows, c);
  if (count == 0) return;
  const int64_t first = ((int64_t)blockIdx.y * 4 + wave) * 16 * VEC + col * VEC, left = p.n - first;
  if (c >= p.in.adapters) {  // no adapter: the rows as they are
    if (p.y == p.out) return;
#pragma unroll
    for (int i = 0; i < 4 * TM; i++) {
      const int place = 4 * i + group;
      if (place < count && left > 0) {
        const u32x4_t v = p.y ? ad_load<KIND>(p.y + rows[place] * p.y_stride + first * SIZE, left) : u32x4_t{0u, 0u, 0u, 0u};
        ad_store<KIND>(p.out + rows[place] * p.out_stride + first * SIZE, v, left);
      }
    }
    return;
  }
  const int rank = ad_rank(p.in, c), pitch = p.padded + (SIZE == 2 ? 8 : 4);  // elements
  u32x4_t yv[TM][4];
#pragma unroll
  for (int t = 0; t < TM; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int place = 16 * t + 4 * group + i;
      yv[t][i] = p.y && place < count && left > 0 ? ad_load<KIND>(p.y + rows[place] * p.y_stride + first * SIZE, left) : u32x4_t{0u, 0u, 0u, 0u};
    }
  {  // the rows' sums, joined over the splits and scaled
    constexpr int EACH = 256 / (16 * TM);  // threads a row
    const int place = threadIdx.x / EACH, lane_of = threadIdx.x % EACH;
    const float* sums = p.sums + (int64_t)rows[place] * p.in.rank;
    const float scale = p.scale ? p.scale[c] : 1.0f;
    auto sum = [&](int r) {
      float v = 0.f;
      for (int s = 0; s < p.splits; s++) v += sums[(int64_t)s * p.in.m * p.in.rank + r];
      return v * scale;
    };
    float unit = 1.0f;
    if constexpr (KIND == HB_F16) {
      float most = 0.f;
      for (int r = lane_of; r < rank; r += EACH) {
        const float v = fabsf(sum(r));
        most = v < INFINITY ? fmaxf(most, v) : most;
      }
#pragma unroll
      for (int d = 1; d < EACH; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
      const int e = ad_exponent(most);
      if (lane_of == 0) power[place] = e;
      unit = ad_pow2(-e);
    }
    const int used = (rank + 31) & ~31;
    for (int r = lane_of; r < used; r += EACH) {
      const float v = r < rank ? sum(r) * unit : 0.f;
      if constexpr (SIZE == 4) {
        reinterpret_cast<float*>(staged)[place * pitch + r] = v;
      } else {
        uint16_t part[PARTS];
        ad_cut<KIND, PARTS>(v, part);
#pragma unroll
        for (int i = 0; i < PARTS; i++) reinterpret_cast<uint16_t*>(staged)[(i * 16 * TM + place) * pitch + r] = part[i];
      }
    }
  }
  __syncthreads();
  if (first - col * VEC >= p.n) return;  // a wavefront behind the last column (idle lanes of the others take part in the products)
  f32x4_t acc[TM][VEC] = {};
  for (int r0 = 0; r0 < rank; r0 += 32) {
    u32x4_t v[8];
#pragma unroll
    for (int s = 0; s < 8; s++) {
      const char* at = p.w + (((int64_t)c * p.in.rank + min(r0 + 8 * group + s, rank - 1)) * p.n + first) * SIZE;
      v[s] = left > 0 ? ad_load<KIND>(at, left) : u32x4_t{0u, 0u, 0u, 0u};
    }
    if constexpr (SIZE == 2) {
      u32x4_t w[VEC];
      ad_turn<KIND>(v, w);
#pragma unroll
      for (int t = 0; t < TM; t++)
#pragma unroll
        for (int i = 0; i < PARTS; i++) {
          const u32x4_t s = *reinterpret_cast<const u32x4_t*>(staged + ((i * 16 * TM + 16 * t + col) * pitch + r0 + 8 * group) * 2);
#pragma unroll
          for (int j = 0; j < VEC; j++) acc[t][j] = ad_mma<KIND>(s, w[j], acc[t][j]);
        }
    } else {
#pragma unroll
      for (int t = 0; t < TM; t++) {
        const float* s = reinterpret_cast<const float*>(staged) + (16 * t + col) * pitch + r0 + 8 * group;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
          for (int j = 0; j < VEC; j++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[i], __uint_as_float(v[i][j]), acc[t][j], 0, 0, 0);
      }
    }
  }
  if (left <= 0) return;
#pragma unroll
  for (int t = 0; t < TM; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int place = 16 * t + 4 * group + i;
      if (place >= count) continue;
      float unit = 1.0f;
      if constexpr (KIND == HB_F16) unit = ad_pow2(power[place]);
      u32x4_t v{0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float to = ad_value<KIND>(ad_elem<KIND>(yv[t][i], j)) + (KIND == HB_F16 ? acc[t][j][i] * unit : acc[t][j][i]);
        if constexpr (SIZE == 4) v[j] = __float_as_uint(to);
        else v[j >> 1] |= ad_bits<KIND>(to) << (16 * (j & 1));
      }
      ad_store<KIND>(p.out + rows[place] * p.out_stride + first * SIZE, v, left);
    }
}

// ------------------------------------------------------------------------------------------------ outer

struct AdOuterJob {
  const float* sums;   // [splits, m, rank]: of the other side's shrink
  const char* v;       // rows
  int64_t stride;      // bytes
  int length;
  float* to;           // [adapters, rank, length]
  float* parts;        // [slots, rank, length]
};
struct AdOuter {
  AdIndex in;
  AdPlan plan;
  AdOuterJob job[2];
  const float* scale;
  int splits, unit, chunks;
};

// A workgroup: RT x 16 ranks times sixteen lanes' columns over a unit of an adapter's rows, the four wavefronts taking 32 rows of every 128 and joining
// their sums in LDS. An adapter's only unit writes the gradient, several write partial sums.
template <int KIND, int RT>
__global__ __launch_bounds__(256) void ad_outer_kernel(AdOuter p) {
  constexpr int VEC = AD_VEC<KIND>, SIZE = AdType<KIND>::SIZE, PARTS = AdType<KIND>::OUTER, PITCH = AD_CHUNK + (SIZE == 2 ? 8 : 4);
  constexpr int STAGED = PARTS * 16 * RT * PITCH * SIZE, JOINED = 4 * VEC * 64 * 16;
  __shared__ __align__(16) char staged[STAGED > JOINED ? STAGED : JOINED];  // [part][rank][row of the chunk]; at the end [wavefront][column of a lane][lane]
  __shared__ int32_t rows[AD_CHUNK];
  __shared__ float most_of[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4, col = lane & 15;
  const AdOuterJob& job = p.job[blockIdx.z / p.chunks];
  const int r0 = (blockIdx.z % p.chunks) * 16 * RT, u = blockIdx.y;
  if (u >= p.plan.units()[p.plan.classes]) return;
  const int64_t first = (int64_t)blockIdx.x * 16 * VEC + col * VEC, left = job.length - first;
  if ((int64_t)blockIdx.x * 16 * VEC >= job.length) return;
  const int c = ad_find(p.plan.units(), p.plan.classes, u);
  const int which = u - p.plan.units()[c], units = p.plan.units()[c + 1] - p.plan.units()[c];
  const int start = p.plan.rows()[c] + which * p.unit, end = min(start + p.unit, p.plan.rows()[c + 1]);
  const int rank = ad_rank(p.in, c);
  float* to = (units > 1 ? job.parts + (int64_t)(p.plan.slots()[c] + which) * p.in.rank * job.length : job.to + (int64_t)c * p.in.rank * job.length);
  const float scale = p.scale ? p.scale[c] : 1.0f;
  f32x4_t acc[RT][VEC] = {};
  int power = -200;  // FP16: the sums are in units of 2^power
  for (int at = start; r0 < rank && at < end; at += AD_CHUNK) {
    const int count = min(AD_CHUNK, end - at);
    __syncthreads();  // the last chunk's operands are read
    if (threadIdx.x < AD_CHUNK) rows[threadIdx.x] = p.plan.order()[at + min((int)threadIdx.x, count - 1)];
    __syncthreads();
    u32x4_t v[8];
#pragma unroll
    for (int s = 0; s < 8; s++) {
      const int place = 32 * wave + 8 * group + s;
      v[s] = left > 0 && place < count ? ad_load<KIND>(job.v + rows[place] * job.stride + first * SIZE, left) : u32x4_t{0u, 0u, 0u, 0u};
    }
    {  // thread: row t % 128 of the chunk, half of the ranks
      const int place = threadIdx.x & (AD_CHUNK - 1), from = (threadIdx.x >> 7) * 8 * RT;
      const float* sums = job.sums + (int64_t)rows[place] * p.in.rank + r0 + from;
      float g[8 * RT];
#pragma unroll
      for (int i = 0; i < 8 * RT; i++) g[i] = 0.f;
      if (place < count)
        for (int s = 0; s < p.splits; s++)
#pragma unroll
          for (int i = 0; i < 8 * RT; i++) g[i] += r0 + from + i < rank ? sums[(int64_t)s * p.in.m * p.in.rank + i] : 0.f;
      float unit = 1.0f;
      if constexpr (KIND == HB_F16) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 8 * RT; i++) {
          const float size = fabsf(g[i] * scale);
          most = size < INFINITY ? fmaxf(most, size) : most;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
        if (lane == 0) most_of[wave] = most;
        __syncthreads();
        const int e = max(power, ad_exponent(fmaxf(fmaxf(most_of[0], most_of[1]), fmaxf(most_of[2], most_of[3]))));
        if (e != power) {  // the sums so far in the new units
          const float by = power <= -200 ? 0.f : ad_pow2(max(power - e, -126));
#pragma unroll
          for (int i = 0; i < RT; i++)
#pragma unroll
            for (int j = 0; j < VEC; j++) acc[i][j] *= by;
          power = e;
        }
        unit = ad_pow2(-power);
      }
#pragma unroll
      for (int i = 0; i < 8 * RT; i++) {
        const float value = g[i] * scale * unit;
        if constexpr (SIZE == 4) {
          reinterpret_cast<float*>(staged)[(from + i) * PITCH + place] = value;
        } else {
          uint16_t part[PARTS];
          ad_cut<KIND, PARTS>(value, part);
#pragma unroll
          for (int q = 0; q < PARTS; q++) reinterpret_cast<uint16_t*>(staged)[(q * 16 * RT + from + i) * PITCH + place] = part[q];
        }
      }
    }
    __syncthreads();
    if constexpr (SIZE == 2) {
      u32x4_t w[VEC];
      ad_turn<KIND>(v, w);
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int i = 0; i < PARTS; i++) {
          const u32x4_t s = *reinterpret_cast<const u32x4_t*>(staged + ((i * 16 * RT + 16 * t + col) * PITCH + 32 * wave + 8 * group) * 2);
#pragma unroll
          for (int j = 0; j < VEC; j++) acc[t][j] = ad_mma<KIND>(s, w[j], acc[t][j]);
        }
    } else {
#pragma unroll
      for (int t = 0; t < RT; t++) {
        const float* s = reinterpret_cast<const float*>(staged) + (16 * t + col) * PITCH + 32 * wave + 8 * group;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
          for (int j = 0; j < VEC; j++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[i], __uint_as_float(v[i][j]), acc[t][j], 0, 0, 0);
      }
    }
  }
  // D: this lane's columns first .. first + VEC - 1 of ranks 4 group .. + 3 of every sixteen
  f32x4_t* join = reinterpret_cast<f32x4_t*>(staged);
#pragma unroll
  for (int t = 0; t < RT; t++) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VEC; j++) join[(wave * VEC + j) * 64 + lane] = acc[t][j];
    __syncthreads();
    // thread: rank t * 16 + 4 group + wave of the columns of its lane
    const int r = r0 + 16 * t + 4 * group + wave;
    if (r < p.in.rank && left > 0) {
      float* row = to + (int64_t)r * job.length + first;
      const float unit = KIND == HB_F16 && power > -200 ? ad_pow2(power) : 1.0f;
      float sum[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) v += reinterpret_cast<const float*>(&join[(w * VEC + j) * 64 + lane])[wave];
        sum[j] = r < rank ? v * unit : 0.f;
      }
#pragma unroll
      for (int j = 0; j < VEC; j++)
        if (j < left) row[j] = sum[j];
    }
  }
}

// The partial sums of adapters with several units, in the units' order; zeros for adapters that have no row.
__global__ __launch_bounds__(256) void ad_join_kernel(AdOuter p) {
  const AdOuterJob& job = p.job[blockIdx.z];
  const int c = blockIdx.y, units = p.plan.units()[c + 1] - p.plan.units()[c];
  if (units == 1) return;
  const int64_t size = (int64_t)p.in.rank * job.length;
  const float* from = job.parts + (int64_t)p.plan.slots()[c] * size;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int u = 0; u < units; u++) v += from[u * size + i];
    job.to[(int64_t)c * size + i] = v;
  }
}

// ------------------------------------------------------------------------------------------------ host

struct AdShape {
  int64_t m;
  int adapters, rank, k, n, kind, size;
  bool grads, self;
  int tm0, tm1, rt, splits, unit;  // tile heights / 16 of shrink and expand, rank tiles a shrink's workgroup, splits of the long axis, rows a unit
  int64_t tiles0, tiles1, units, slots;
  size_t plan_bytes, sums_bytes, parts_bytes;  // plan | sums (x) | sums (dy) | parts (da) | parts (db)
  size_t bytes() const { return plan_bytes + sums_bytes * (grads ? 2 : 1) + parts_bytes; }
};
static size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
static int64_t cut(int64_t a, int64_t b) { return (a + b - 1) / b; }

static bool ad_shape(const hb_adapters* a, int64_t m, bool grads, AdShape& s) {
  if (a->type < HB_BF16 || a->type > HB_F32 || a->adapters <= 0 || a->adapters > AD_MOST || a->rank <= 0 || a->rank > AD_RANK || a->k <= 0 || a->n <= 0 ||
      a->k > AD_LONGEST || a->n > AD_LONGEST || m <= 0 || m > AD_MAX_ROWS)
    return false;
  s = AdShape{};
  s.m = m, s.adapters = a->adapters, s.rank = a->rank, s.k = a->k, s.n = a->n, s.kind = a->type, s.size = a->type == HB_F32 ? 4 : 2;
  s.grads = grads;
  s.self = !grads && m <= AD_SELF_ROWS;
  const int64_t classes = std::min<int64_t>(a->adapters + 1, m);
  s.tm0 = s.self || m < 2048 ? 1 : 2;
  s.tm1 = s.self || m < 2048 ? 1 : 2;
  s.tiles0 = s.self ? m : cut(m, 16 * s.tm0) + classes;
  s.tiles1 = s.self ? m : cut(m, 16 * s.tm1) + classes;
  s.rt = s.self || a->rank <= 16 ? 1 : a->rank <= 32 ? 2 : 4;
  const int64_t longest = grads ? std::max(a->k, a->n) : a->k, units = cut(longest, 128 / s.size), chunks = cut(a->rank, 16 * s.rt);
  const int64_t groups = (s.self ? std::min<int64_t>(m, a->adapters + cut(m, 16)) : cut(m, 16 * s.tm0)) * chunks * (grads ? 2 : 1);
  s.splits = (int)std::max<int64_t>(1, std::min<int64_t>(cut(1024, groups), cut(units, 16)));
  s.sums_bytes = up256((size_t)s.splits * m * a->rank * 4);
  s.plan_bytes = s.self ? 0 : up256(AdPlan::ints(a->adapters + 1, m) * 4);
  if (grads) {
    const int64_t blocks = (cut(a->k, 16 * 16 / s.size) + cut(a->n, 16 * 16 / s.size)) * cut(a->rank, 64);
    s.unit = (int)std::min<int64_t>(std::max<int64_t>(AD_CHUNK, cut(cut(m * blocks, 2048), AD_CHUNK) * AD_CHUNK), 1 << 20);
    s.units = cut(m, s.unit) + classes;
    s.slots = 2 * (m / s.unit);  // an adapter of more than one unit has fewer than two for every `unit` of its rows
    s.parts_bytes = up256((size_t)s.slots * a->rank * a->k * 4) + up256((size_t)s.slots * a->rank * a->n * 4);
  } else {
    s.unit = AD_CHUNK;
  }
  return true;
}

static int ad_run_plan(const AdShape& s, const AdIndex& in, const AdPlan& plan, hipStream_t stream) {
  AdPlanParams p{in, plan, {16 * s.tm0, 16 * s.tm1}, s.unit, 1};
  while (p.segments < 16 && (int64_t)(2 * p.segments) * plan.classes <= 12288) p.segments *= 2;
  ad_plan_kernel<<<1, 1024, (size_t)p.segments * plan.classes * 4, stream>>>(p);
  return launch_status();
}

template <int KIND>
static int ad_run_shrink(const AdShape& s, AdShrink& p, int jobs, hipStream_t stream) {
  p.chunks = (int)cut(s.rank, 16 * s.rt);
  for (int j = 0; j < jobs; j++) p.job[j].share = (int)cut(cut(p.job[j].length, 128 / s.size), s.splits);
  const dim3 grid((unsigned)s.tiles0, (unsigned)s.splits, (unsigned)(p.chunks * jobs));
#define HB_AD(TM, RT) if (s.tm0 == TM && s.rt == RT) ad_shrink_kernel<KIND, TM, RT><<<grid, 256, 0, stream>>>(p)
  HB_AD(1, 1); HB_AD(1, 2); HB_AD(1, 4); HB_AD(2, 1); HB_AD(2, 2); HB_AD(2, 4);
#undef HB_AD
  return launch_status();
}

template <int KIND>
static int ad_run_expand(const AdShape& s, AdExpand& p, hipStream_t stream) {
  p.splits = s.splits;
  p.padded = (int)cut(s.rank, 32) * 32;
  const dim3 grid((unsigned)s.tiles1, (unsigned)cut(p.n, 4 * 16 * AD_VEC<KIND>));
  const size_t lds = (size_t)AdType<KIND>::PARTS * 16 * s.tm1 * (p.padded * AdType<KIND>::SIZE + 16);
  if (s.tm1 == 1) ad_expand_kernel<KIND, 1><<<grid, 256, lds, stream>>>(p);
  else ad_expand_kernel<KIND, 2><<<grid, 256, lds, stream>>>(p);
  return launch_status();
}

template <int KIND>
static int ad_run_outer(const AdShape& s, AdOuter& p, hipStream_t stream) {
  const int rt = s.rank <= 16 ? 1 : s.rank <= 32 ? 2 : 4;
  p.chunks = (int)cut(s.rank, 16 * rt);
  const int longest = std::max(p.job[0].length, p.job[1].length);
  const dim3 grid((unsigned)cut(longest, 16 * AD_VEC<KIND>), (unsigned)s.units, (unsigned)(2 * p.chunks));
  if (rt == 1) ad_outer_kernel<KIND, 1><<<grid, 256, 0, stream>>>(p);
  if (rt == 2) ad_outer_kernel<KIND, 2><<<grid, 256, 0, stream>>>(p);
  if (rt == 4) ad_outer_kernel<KIND, 4><<<grid, 256, 0, stream>>>(p);
  int code = launch_status();
  if (code) return code;
  const unsigned blocks = (unsigned)std::min<int64_t>(cut((int64_t)s.rank * longest, 256), 1024);
  ad_join_kernel<<<dim3(blocks, (unsigned)s.adapters, 2), 256, 0, stream>>>(p);
  return launch_status();
}

template <int KIND>
static int ad_add(const hb_adapters* a, const AdShape& s, const AdIndex& in, const void* x, int64_t x_stride, const void* y, int64_t y_stride, void* out, int64_t out_stride,
                  char* ws, hipStream_t stream) {
  const AdPlan plan{s.self ? nullptr : reinterpret_cast<int32_t*>(ws), s.adapters + 1};
  float* sums = reinterpret_cast<float*>(ws + s.plan_bytes);
  int code = s.self ? HB_OK : ad_run_plan(s, in, plan, stream);
  if (code) return code;
  AdShrink down{in, plan, {{static_cast<const char*>(x), x_stride * s.size, static_cast<const char*>(a->a), s.k, 0, sums}, {}}, 0};
  if ((code = ad_run_shrink<KIND>(s, down, 1, stream))) return code;
  AdExpand up{in, plan, sums, a->scale, 0, s.n, 0, static_cast<const char*>(a->b), static_cast<const char*>(y), y_stride * s.size, static_cast<char*>(out), out_stride * s.size};
  return ad_run_expand<KIND>(s, up, stream);
}

template <int KIND>
static int ad_grads(const hb_adapters* a, const AdShape& s, const AdIndex& in, const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, void* dx, float* da, float* db,
                    char* ws, hipStream_t stream) {
  const AdPlan plan{reinterpret_cast<int32_t*>(ws), s.adapters + 1};
  float* of_x = reinterpret_cast<float*>(ws + s.plan_bytes);
  float* of_dy = reinterpret_cast<float*>(ws + s.plan_bytes + s.sums_bytes);
  float* parts_a = reinterpret_cast<float*>(ws + s.plan_bytes + 2 * s.sums_bytes);
  float* parts_b = reinterpret_cast<float*>(ws + s.plan_bytes + 2 * s.sums_bytes + up256((size_t)s.slots * s.rank * s.k * 4));
  int code = ad_run_plan(s, in, plan, stream);
  if (code) return code;
  const char *xr = static_cast<const char*>(x), *dyr = static_cast<const char*>(dy);
  AdShrink down{in, plan, {{xr, x_stride * s.size, static_cast<const char*>(a->a), s.k, 0, of_x}, {dyr, dy_stride * s.size, static_cast<const char*>(a->b), s.n, 0, of_dy}}, 0};
  if ((code = ad_run_shrink<KIND>(s, down, 2, stream))) return code;
  AdExpand up{in, plan, of_dy, a->scale, 0, s.k, 0, static_cast<const char*>(a->a), nullptr, 0, static_cast<char*>(dx), (int64_t)s.k * s.size};
  if ((code = ad_run_expand<KIND>(s, up, stream))) return code;
  AdOuter outer{in, plan, {{of_dy, xr, x_stride * s.size, s.k, da, parts_a}, {of_x, dyr, dy_stride * s.size, s.n, db, parts_b}}, a->scale, s.splits, s.unit, 0};
  return ad_run_outer<KIND>(s, outer, stream);
}

static int ad_check(const hb_adapters* a, const void* index, int index_bytes, int64_t m, bool grads, AdShape& s) {
  if (!a || !a->a || !a->b || !index) return HB_ENULL;
  if ((index_bytes != 4 && index_bytes != 8) || !ad_shape(a, m, grads, s)) return HB_EINVAL;
  if (!aligned(a->a, s.size) || !aligned(a->b, s.size) || !aligned(a->scale, 4) || !aligned(a->ranks, 4) || !aligned(index, index_bytes)) return HB_EINVAL;
  return HB_OK;
}

}  // namespace hb

using namespace hb;

extern "C" size_t hb_adapters_workspace_bytes(const hb_adapters* adapters, int64_t m, int grads) {
  AdShape s;
  return adapters && ad_shape(adapters, m, grads != 0, s) ? s.bytes() : 0;
}

extern "C" int hb_adapters_add(const hb_adapters* adapters, const void* x, int64_t x_stride, const void* y, int64_t y_stride, const void* index, int index_bytes, int64_t m,
                               void* out, int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
  AdShape s;
  if (!x || !y || !out || !workspace) return HB_ENULL;
  if (int code = ad_check(adapters, index, index_bytes, m, false, s)) return code;
  if (x_stride < s.k || y_stride < s.n || out_stride < s.n || !aligned(x, s.size) || !aligned(y, s.size) || !aligned(out, s.size) || !aligned(workspace, 16)) return HB_EINVAL;
  if (y == out && y_stride != out_stride) return HB_EINVAL;
  if (workspace_bytes < s.bytes()) return HB_EWORKSPACE;
  const AdIndex in{index, adapters->ranks, index_bytes == 8, (int)m, s.adapters, s.rank};
  auto run = [&](auto kind) {
    return ad_add<decltype(kind)::value>(adapters, s, in, x, x_stride, y, y_stride, out, out_stride, static_cast<char*>(workspace), as_stream(stream));
  };
  if (s.kind == HB_BF16) return run(std::integral_constant<int, HB_BF16>{});
  if (s.kind == HB_F16) return run(std::integral_constant<int, HB_F16>{});
  return run(std::integral_constant<int, HB_F32>{});
}

extern "C" int hb_adapters_grads(const hb_adapters* adapters, const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* index, int index_bytes, int64_t m,
                                 void* dx, float* da, float* db, void* workspace, size_t workspace_bytes, void* stream) {
  AdShape s;
  if (!x || !dy || !dx || !da || !db || !workspace) return HB_ENULL;
  if (int code = ad_check(adapters, index, index_bytes, m, true, s)) return code;
  if (x_stride < s.k || dy_stride < s.n || !aligned(x, s.size) || !aligned(dy, s.size) || !aligned(dx, s.size) || !aligned(da, 4) || !aligned(db, 4) || !aligned(workspace, 16))
    return HB_EINVAL;
  if (workspace_bytes < s.bytes()) return HB_EWORKSPACE;
  const AdIndex in{index, adapters->ranks, index_bytes == 8, (int)m, s.adapters, s.rank};
  auto run = [&](auto kind) {
    return ad_grads<decltype(kind)::value>(adapters, s, in, x, x_stride, dy, dy_stride, dx, da, db, static_cast<char*>(workspace), as_stream(stream));
  };
  if (s.kind == HB_BF16) return run(std::integral_constant<int, HB_BF16>{});
  if (s.kind == HB_F16) return run(std::integral_constant<int, HB_F16>{});
  return run(std::integral_constant<int, HB_F32>{});
}
