// Low-rank adapters of many requests at once beside a shared projection, and their gradients.
//
//   out[r] = y[r] + s_i (x[r] a_i^T) b_i,  i = index[r];   a [adapters, rank, k], b [adapters, rank, n]
//   g[r] = s_i dy[r] b_i^T;  dx[r] = g[r] a_i;  da_i = sum over i's rows of g[r]^T x[r];  db_i = sum of s_i (x[r] a_i^T)^T dy[r]
//
// Both matrices of an adapter lie rank by rank along their long axis, so the six products are of three kinds:
//   shrink   rows [m, long] times a matrix's rows: contraction over the long axis, [m, rank] FP32 sums, the long axis cut into splits
//            that other workgroups have
//   expand   [m, rank] times the matrix: contraction over the rank, added to y's rows (or alone: dx)
//   outer    [m, rank]^T times rows [m, long]: contraction over an adapter's rows, FP32
// Rows are grouped by adapter: a tile's rows are one adapter's, gathered by number. All of it is bound by memory (few operations a byte at
// any rank here); the matrix instructions are there so that one read of an adapter's matrix serves a tile's rows.
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "route.hpp"

namespace hb {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef uint32_t u32x4_loose __attribute__((ext_vector_type(4), aligned(2)));  // sixteen bytes at any element: rows of odd length

// Splits of the long axis, at most, in a call of few rows; its readers join them. One row of 5120 at rank 16, both kernels with nothing in the caches: one split 16.2 us, five
// 11.9, ten 10.4; 64 rows of 32 adapters of up to 64 ranks do not care.
constexpr int AD_SPLITS = 12;
// Rows up to which a workgroup finds its tile from the index itself, in two launches for three. 256 rows of 5120 x 5120, eight adapters, rank 16: 13.3 us a call in a graph, with a
// plan 17.8; of 32 adapters 15.0 and 19.7; 512 rows of 32 adapters 26 and 21.
constexpr int AD_SELF_ROWS = 256;
constexpr int AD_TILE = 32;        // rows of a planned call's tile: the places of a matrix instruction's contraction in an outer product
constexpr int AD_MOST = 4096;      // adapters
constexpr int AD_RANK = 256;
constexpr int AD_MAX_ROWS = 1 << 24;
constexpr int AD_LONGEST = 1 << 22;  // of either axis
constexpr int64_t AD_STRIDE = 0xffffffffll;  // bytes from row to row

template <int KIND> struct AdType;
template <> struct AdType<HB_BF16> { static constexpr int SIZE = 2, PARTS = 3; };  // parts that FP32 values are cut into
template <> struct AdType<HB_F16> { static constexpr int SIZE = 2, PARTS = 3; };
template <> struct AdType<HB_F32> { static constexpr int SIZE = 4, PARTS = 1; };
template <int KIND> constexpr int AD_VEC = 16 / AdType<KIND>::SIZE;  // elements of a 16-byte load: the columns a lane holds

template <int KIND>
__device__ __forceinline__ float ad_value(uint32_t bits) {
  if constexpr (KIND == HB_BF16) return bf16_bits_to_f32((uint16_t)bits);
  if constexpr (KIND == HB_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  return __uint_as_float(bits);
}
template <int KIND>
__device__ __forceinline__ uint32_t ad_bits(float v) {
  if constexpr (KIND == HB_BF16) return bf16_of(v);
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

// Row r of rows `pitch` bytes apart: one multiply-add of 64 bits (three of a 64-bit pitch's, sixteen cycles each).
__device__ __forceinline__ const char* ad_row(const char* rows, int r, uint32_t pitch) { return rows + (uint64_t)(uint32_t)r * pitch; }
__device__ __forceinline__ char* ad_row(char* rows, int r, uint32_t pitch) { return rows + (uint64_t)(uint32_t)r * pitch; }

// A lane's sixteen bytes of a row of n elements, of which `first` is the lane's first: behind the row's end its last sixteen bytes, so that no load is behind a
// branch (the compiler waits for all that is under way where it does not know how many loads are). AD_TINY: rows shorter than that, element by element.
enum { AD_NEAR = 0, AD_TINY = 1, AD_PAST = 2 };  // AD_PAST: past the caches
template <int KIND, int HOW>
__device__ __forceinline__ u32x4_t ad_take(const char* row, int first, int n) {
  if constexpr (HOW == AD_TINY) return ad_load<KIND>(row + first * AdType<KIND>::SIZE, n - first);
  const u32x4_loose* at = reinterpret_cast<const u32x4_loose*>(row + (int64_t)min(first, n - AD_VEC<KIND>) * AdType<KIND>::SIZE);
  if constexpr (HOW == AD_PAST) return __builtin_nontemporal_load(at);
  return *at;
}
// The elements of the row that `ad_take` was asked for, and no others.
template <int KIND, int HOW>
__device__ __forceinline__ void ad_put(char* row, const u32x4_t& v, int first, int n) {
  if (first + AD_VEC<KIND> <= n) {
    u32x4_loose* at = reinterpret_cast<u32x4_loose*>(row + (int64_t)first * AdType<KIND>::SIZE);
    if constexpr (HOW == AD_PAST) __builtin_nontemporal_store(v, at);
    else *at = v;
    return;
  }
  const int from = HOW == AD_TINY ? first : n - AD_VEC<KIND>;
#pragma unroll
  for (int j = 0; j < AD_VEC<KIND>; j++) {
    if (from + j >= first && from + j < n) {
      if constexpr (AdType<KIND>::SIZE == 4) reinterpret_cast<uint32_t*>(row)[from + j] = v[j];
      else reinterpret_cast<uint16_t*>(row)[from + j] = (uint16_t)ad_elem<KIND>(v, j);
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

// Classes 0 .. adapters - 1 are the adapters, `adapters` the rows without one (an index outside the pool).
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
  return i < 0 || i >= p.adapters ? p.adapters : (int)i;
}

// The plan: int32 arrays [classes + 1] of where a class's rows, its tiles, its units (runs of `unit` rows, an outer product's share of the work) and
// its slots (partial sums: the units of classes that have more than one) begin, then the rows in order.
struct AdPlan {
  int32_t* at;
  int classes;
  __host__ __device__ int32_t* rows() const { return at; }
  __host__ __device__ int32_t* tiles() const { return at + (classes + 1); }
  __host__ __device__ int32_t* units() const { return at + 2 * (classes + 1); }
  __host__ __device__ int32_t* slots() const { return at + 3 * (classes + 1); }
  __host__ __device__ int32_t* order() const { return at + 4 * (classes + 1); }
  static size_t ints(int classes, int64_t m) { return 4 * ((size_t)classes + 1) + m; }
};

struct AdPlanParams {
  AdIndex in;
  AdPlan plan;
  int unit;
  int segments;   // wavefronts that count and place rows, each those of one stretch; segments * classes counters in LDS
  int32_t* tickets;  // the shrink's arrival counters, to be cleared
  int64_t clear;
};

// The classes' first places from their numbers of rows: each thread a run of classes, prefix sums over the threads. `rows_of`(class, first row): its rows.
template <typename Rows>
__device__ __forceinline__ void ad_plan_classes(const AdPlanParams& p, int32_t (*carry)[4], Rows&& rows_of) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, classes = p.plan.classes;
  const int per = (classes + 1023) / 1024, c0 = min((int)threadIdx.x * per, classes), c1 = min(c0 + per, classes);
  int sum[4] = {0, 0, 0, 0}, before[4];
  auto add = [&](int (&to)[4], int c, int n) {
    const int units = c < p.in.adapters ? max((n + p.unit - 1) / p.unit, 1) : 0;  // (an adapter without rows has one, of none: it writes the zeros)
    to[0] += n;
    to[1] += (n + AD_TILE - 1) / AD_TILE;
    to[2] += units;
    to[3] += units > 1 ? units : 0;
  };
  for (int c = c0; c < c1; c++) add(sum, c, rows_of(c, -1));
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int x = wave_inclusive_sum(sum[j]);
    before[j] = x - sum[j];
    if (lane == 63) carry[wave][j] = x;
  }
  __syncthreads();
  if (c0 < c1)
    for (int w = 0; w < wave; w++)
#pragma unroll
      for (int j = 0; j < 4; j++) before[j] += carry[w][j];
  int32_t* out[4] = {p.plan.rows(), p.plan.tiles(), p.plan.units(), p.plan.slots()};
  for (int c = c0; c < c1; c++) {
    const int n = rows_of(c, before[0]);
#pragma unroll
    for (int j = 0; j < 4; j++) out[j][c] = before[j];
    add(before, c, n);
    if (c == classes - 1)
#pragma unroll
      for (int j = 0; j < 4; j++) out[j][classes] = before[j];
  }
  __syncthreads();
}

// The lanes of the same class, of up to eight times 64 rows side by side, by the ballots of its bits: as many steps for rows of one class as of 64. (A lane without a row,
// c < 0, gets nothing to use.)
__device__ __forceinline__ void ad_same(const int (&c)[8], int bits, int pieces, uint64_t (&same)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) same[i] = __ballot(c[i] >= 0);
  for (int b = 0; b < bits; b++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (i >= pieces) break;  // uniform
      const int mine = __builtin_amdgcn_sbfe(c[i], b, 1);  // 0 or -1
      const uint64_t on = __ballot(mine != 0);
      same[i] &= (uint64_t)(~((uint32_t)(on >> 32) ^ mine)) << 32 | (~((uint32_t)on ^ mine));
    }
}

// One workgroup: a stable counting sort (rows of a class stay in ascending order, so sums over them are the same every time). What it takes is latency, so the
// steps are few and side by side. Up to AD_HELD rows whose 64-row pieces have a counter each for every class: a wavefront has up to eight pieces, each lane their
// classes and its places among them in registers; a wavefront a class adds the pieces' counts up. 8192 rows of 4 adapters 7.6 us, of 64 11, 4096 of 4 5.4 (through the
// other kernel's one counter a class and wavefront: 8192 rows of 64 adapters 15.7).
constexpr int AD_HELD = 8192;
constexpr int AD_COUNTERS = 15360;  // of 64 KB of LDS, less the prefix sums'
__global__ __launch_bounds__(1024) void ad_plan_pieces_kernel(AdPlanParams p) {
  extern __shared__ int32_t counters[];  // [piece][class], then [class]
  __shared__ int32_t carry[16][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, classes = p.plan.classes, m = p.in.m, pieces = (m + 63) / 64, bits = 32 - __builtin_clz(classes - 1);
  int32_t* all = counters + pieces * classes;
  int c[8], place[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int r = (wave + 16 * i) * 64 + lane;
    c[i] = r < m ? ad_class(p.in, r) : -1;
  }
  for (int64_t i = threadIdx.x; i < p.clear; i += 1024) p.tickets[i] = 0;
  for (int i = threadIdx.x; i < pieces * classes; i += 1024) counters[i] = 0;
  __syncthreads();
  uint64_t same[8];
  ad_same(c, bits, (pieces - wave + 15) / 16, same);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    place[i] = __popcll(same[i] & ((1ull << lane) - 1ull));
    if (c[i] >= 0 && place[i] == 0) counters[(wave + 16 * i) * classes + c[i]] = __popcll(same[i]);
  }
  __syncthreads();
  for (int v = wave; v < classes; v += 16) {
    const int n0 = 2 * lane < pieces ? counters[2 * lane * classes + v] : 0, n1 = 2 * lane + 1 < pieces ? counters[(2 * lane + 1) * classes + v] : 0;
    const int upto = wave_inclusive_sum(n0 + n1);
    if (2 * lane < pieces) counters[2 * lane * classes + v] = upto - n1 - n0;
    if (2 * lane + 1 < pieces) counters[(2 * lane + 1) * classes + v] = upto - n1;
    if (lane == 63) all[v] = upto;
  }
  __syncthreads();
  ad_plan_classes(p, carry, [&](int v, int first) {
    const int n = all[v];
    if (first >= 0) all[v] = first;
    return n;
  });
  int32_t* order = p.plan.order();
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (c[i] >= 0) order[all[c[i]] + counters[(wave + 16 * i) * classes + c[i]] + place[i]] = (wave + 16 * i) * 64 + lane;
}

// Any number of rows: `segments` wavefronts with a stretch of the rows each, 512 after 512, twice over, the next ones' classes under way. What one compute unit can read: 65536
// rows of 4 adapters 57 us, of 512 100, and of 4096 (three wavefronts' counters are all that fit) 280.
__global__ __launch_bounds__(1024) void ad_plan_kernel(AdPlanParams p) {
  extern __shared__ int32_t counters[];  // [segment][class]
  __shared__ int32_t carry[16][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, classes = p.plan.classes, m = p.in.m, bits = 32 - __builtin_clz(classes - 1);
  const int stretch = ((m + p.segments - 1) / p.segments + 63) / 64 * 64;
  const int from = wave < p.segments ? (int)min((int64_t)wave * stretch, (int64_t)m) : m, upto = min(from + stretch, m);
  for (int64_t i = threadIdx.x; i < p.clear; i += 1024) p.tickets[i] = 0;
  for (int i = threadIdx.x; i < p.segments * classes; i += 1024) counters[i] = 0;
  __syncthreads();
  volatile int32_t* mine = counters + wave * classes;  // (of a wavefront that has rows)
  // f(row, its place among the rows of its class) for the wavefront's rows; the classes' counters move up by them
  auto each = [&](auto&& f) {
    int next[8];
    auto load = [&](int r0) {  // (behind the last row it again: no load behind a branch)
#pragma unroll
      for (int i = 0; i < 8; i++) next[i] = ad_class(p.in, min(r0 + 64 * i + lane, m - 1));
    };
    load(from);
    for (int r0 = from; r0 < upto; r0 += 512) {
      int c[8];
      uint64_t same[8];
#pragma unroll
      for (int i = 0; i < 8; i++) c[i] = r0 + 64 * i + lane < upto ? next[i] : -1;
      load(min(r0 + 512, m - 1));
      ad_same(c, bits, 8, same);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (c[i] < 0) continue;
        const int have = mine[c[i]], before = __popcll(same[i] & ((1ull << lane) - 1ull));
        if (before == 0) mine[c[i]] = have + __popcll(same[i]);  // (behind every lane's read: a wavefront's come in order)
        f(r0 + 64 * i + lane, have + before);
      }
    }
  };
  each([](int, int) {});
  __syncthreads();
  ad_plan_classes(p, carry, [&](int c, int first) {
    int n = 0;
    for (int s = 0; s < p.segments; s++) {
      const int here = counters[s * classes + c];
      if (first >= 0) counters[s * classes + c] = first + n;
      n += here;
    }
    return n;
  });
  int32_t* order = p.plan.order();
  each([&](int r, int place) { order[place] = r; });
}

// The class whose tiles (or units), which begin at first[class], number t is of, or `classes` if there is none; its first one and its first row and the next class's
// (one load each for up to 63 classes, side by side). By every wavefront for itself.
struct AdPlace {
  int c, first, row, next_row;
};
__device__ __forceinline__ AdPlace ad_find(const AdPlan& plan, const int32_t* first, int t) {
  const int lane = threadIdx.x & 63, classes = plan.classes;
  AdPlace at{-1, 0, 0, 0};
  for (int i = 0; i <= classes; i += 64) {
    const int mine = first[min(i + lane, classes)], row = plan.rows()[min(i + lane, classes)];
    const int n = __popcll(__ballot(i + lane <= classes && mine <= t));
    if (n) {
      at.first = __builtin_amdgcn_readlane(mine, n - 1);
      at.row = __builtin_amdgcn_readlane(row, n - 1);
    }
    at.c += n;
    if (n < 64) {
      if (n) at.next_row = __builtin_amdgcn_readlane(row, n);
      break;
    }
    at.next_row = plan.rows()[min(i + 64, classes)];
  }
  return at;
}

// A plan's tile t: its class, its rows' first place in the order and how many they are (0: no such tile).
__device__ __forceinline__ int ad_tile(const AdPlan& plan, int t, int& c, int& start) {
  const AdPlace at = ad_find(plan, plan.tiles(), t);
  c = at.c;
  if (c >= plan.classes) return 0;
  start = at.row + (t - at.first) * AD_TILE;
  return min(AD_TILE, at.next_row - start);
}

// Few rows, no plan: a tile of up to sixteen begins at every sixteenth row of a class, and every wavefront finds tile t from the index itself, by the ballots of the
// classes' bits. Lane l gets the number of the tile's row l % 16 (behind the last one the first again); 0 rows: no such tile.
template <int GROUPS>
__device__ __forceinline__ int ad_tile_of(const AdIndex& p, int t, int& c, int& row) {  // of up to GROUPS times 64 rows
  const int lane = threadIdx.x & 63, groups = (p.m + 63) / 64;
  int mine[GROUPS], ahead[GROUPS];  // a row's class, how many rows of it are ahead of it
  uint64_t there[GROUPS], same[GROUPS][GROUPS];
#pragma unroll
  for (int j = 0; j < GROUPS; j++) {
    mine[j] = j < groups ? ad_class(p, min(64 * j + lane, p.m - 1)) : 0;
    there[j] = __ballot(64 * j + lane < p.m);
#pragma unroll
    for (int i = 0; i <= j; i++) same[j][i] = there[i];
  }
  for (int b = 0; b < 32 - __builtin_clz(p.adapters); b++) {
    uint64_t on[GROUPS];
#pragma unroll
    for (int j = 0; j < GROUPS; j++) {
      if (j >= groups) break;  // uniform
      const int bit = __builtin_amdgcn_sbfe(mine[j], b, 1);  // 0 or -1
      on[j] = __ballot(bit != 0);
#pragma unroll
      for (int i = 0; i <= j; i++) same[j][i] &= (uint64_t)(~((uint32_t)(on[i] >> 32) ^ bit)) << 32 | (~((uint32_t)on[i] ^ bit));
    }
  }
  int before = 0, first = -1;
#pragma unroll
  for (int j = 0; j < GROUPS; j++) {
    ahead[j] = __popcll(same[j][j] & ((1ull << lane) - 1ull));
#pragma unroll
    for (int i = 0; i < j; i++) ahead[j] += __popcll(same[j][i]);
    const uint64_t begin = __ballot(64 * j + lane < p.m && ahead[j] % 16 == 0);
    const uint64_t hit = __ballot((begin >> lane & 1) && before + __popcll(begin & ((1ull << lane) - 1ull)) == t);
    if (hit) {
      c = __builtin_amdgcn_readlane(mine[j], __builtin_ctzll(hit));
      first = __builtin_amdgcn_readlane(ahead[j], __builtin_ctzll(hit));
    }
    before += __popcll(begin);
  }
  if (first < 0) return 0;
  int all = 0;
  row = 0;
#pragma unroll
  for (int j = 0; j < GROUPS; j++) {  // the rows hand their numbers to the lanes of their places, all others theirs to lanes that nobody reads
    const bool of = 64 * j + lane < p.m && mine[j] == c;
    const int place = ahead[j] - first;
    const int got = __builtin_amdgcn_ds_permute(4 * (of && place >= 0 && place < 16 ? place : 16 + (lane & 31)), 64 * j + lane + 1);  // (0: nothing came)
    if (lane < 16 && got) row = got - 1;
    all += __popcll(__ballot(of));
  }
  const int count = min(16, all - first);
  row = __shfl(row, (lane & 15) < count ? lane & 15 : 0);
  return count;
}
__device__ __forceinline__ int ad_tile_at(const AdIndex& p, int t, int& c, int& row) {
  if (p.m > 128) return ad_tile_of<AD_SELF_ROWS / 64>(p, t, c, row);
  if (p.m > 64) return ad_tile_of<2>(p, t, c, row);
  return ad_tile_of<1>(p, t, c, row);
}

// ------------------------------------------------------------------------------------------------ FP32 sums as matrix operands

// The sums are operands of the second product. To keep what FP32 holds of them, a value goes in as the sum of three of the type's: BF16 by cutting (8 bits a
// part, never past the value's size: no overflow; three parts are all of it), FP16 by rounding what a power of two has brought below 2^15 (all of it down to 2^-39 of the
// largest, half of FP16's smallest step; 2^-37 where `ad_lower` brings the parts to a larger unit). Two parts hold 2^-16 of a BF16 sum, 2^-22 of an FP16 one.
template <int KIND>
__device__ __forceinline__ void ad_cut(float v, uint16_t (&part)[AdType<KIND>::PARTS]) {
  constexpr int PARTS = AdType<KIND>::PARTS;
  const bool finite = fabsf(v) < INFINITY;
  float rest = v;
  if constexpr (KIND == HB_BF16) {
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
#pragma unroll
    for (int i = 0; i < PARTS; i++) {
      const _Float16 top = (_Float16)rest;
      part[i] = finite || i == 0 ? __builtin_bit_cast(uint16_t, top) : 0;
      rest -= (float)top;
    }
  }
}

// The power of two that brings a largest magnitude to 2^14 .. 2^15 (its exponent, -100 or more).
__device__ __forceinline__ int ad_exponent(float most) { return most > 0.f ? max((int)(__float_as_uint(most) >> 23) - 127, -86) - 14 : -100; }
__device__ __forceinline__ float ad_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// FP16 parts times 2^e, e <= 0 (what falls below FP16's smallest step, 2^-38 of the unit's largest, is gone)
__device__ __forceinline__ u32x4_t ad_lower(const u32x4_t& v, int e) {
  f16x8_t f = __builtin_bit_cast(f16x8_t, v);
  f = f * (_Float16)ad_pow2(max(e, -24));
  if (__builtin_expect(__ballot(e < -24) != 0, 0)) f = f * (_Float16)ad_pow2(max(min(e + 24, 0), -24));
  return __builtin_bit_cast(u32x4_t, f);
}

// Lane's operand j along the contraction from eight rows of sixteen bytes: their elements j.
__device__ __forceinline__ u32x4_t ad_turn(const u32x4_t (&v)[8], int j) {
  u32x4_t out;
#pragma unroll
  for (int q = 0; q < 4; q++) out[q] = __builtin_amdgcn_perm(v[2 * q + 1][j >> 1], v[2 * q][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
  return out;
}

// ------------------------------------------------------------------------------------------------ shrink

// acc[i][j] += units u0, u0 + step, .. below u1 of TM x 16 rows times RT x 16 rows of a matrix; the last, cut unit of a row is taken if it is among them.
// Units of 128 bytes (a whole cache line of every row), DEPTH of them under way.
template <int KIND, int TM, int RT, int LIMIT = RT>
__device__ __forceinline__ void ad_shrink_units(const char* const (&x)[TM], const char* const (&w)[LIMIT], int length, int u0, int u1, int step, f32x4_t (&acc)[TM][LIMIT]) {
  constexpr int VEC = AD_VEC<KIND>, SIZE = AdType<KIND>::SIZE, UNIT = 128 / SIZE, DEPTH = TM == 1 ? 4 : 2;
  const int whole = length / UNIT, end = min(u1, whole), group = (threadIdx.x & 63) >> 4;
  u32x4_t xv[DEPTH][TM][2], wv[DEPTH][RT][2];
  auto load = [&](int d, int u) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int i = 0; i < TM; i++) xv[d][i][h] = *reinterpret_cast<const u32x4_loose*>(x[i] + (int64_t)u * 128 + 64 * h);
#pragma unroll
      for (int i = 0; i < RT; i++) wv[d][i][h] = *reinterpret_cast<const u32x4_loose*>(w[i] + (int64_t)u * 128 + 64 * h);
    }
  };
  auto products = [&](int d) {
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < RT; j++) acc[i][j] = ad_mma<KIND>(xv[d][i][h], wv[d][j][h], acc[i][j]);
  };
  // (no load behind a branch while others are to stay under way: see ad_take)
  int u = u0, left = u0 < end ? (end - u0 + step - 1) / step : 0;
  if (left >= DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; d++) load(d, u + d * step);
    for (; left >= 2 * DEPTH; left -= DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; d++) {
        products(d);
        load(d, u + (d + DEPTH) * step);
      }
      u += DEPTH * step;
    }
#pragma unroll
    for (int d = 0; d < DEPTH; d++) products(d);
    u += DEPTH * step;
    left -= DEPTH;
  }
#pragma unroll
  for (int d = 0; d < DEPTH - 1; d++)
    if (d < left) load(d, u + d * step);
#pragma unroll
  for (int d = 0; d < DEPTH - 1; d++)
    if (d < left) products(d);
  u += left * step;
  if (u == whole && u < u1) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int64_t left = length - ((int64_t)whole * UNIT + h * (UNIT / 2) + group * VEC);
#pragma unroll
      for (int i = 0; i < RT; i++) wv[0][i][h] = ad_load<KIND>(w[i] + (int64_t)whole * 128 + 64 * h, left);
#pragma unroll
      for (int i = 0; i < TM; i++) xv[0][i][h] = ad_load<KIND>(x[i] + (int64_t)whole * 128 + 64 * h, left);
    }
    products(0);
  }
}

// Few rows: a workgroup's four wavefronts share one split of the long axis of a tile's rows and sixteen ranks, and join their sums in LDS; the splits' sums
// are joined by their readers (no arrival counters, which a launch would have to clear). Latency bounds it: 64 rows of 5120, 32 adapters of up to 64 ranks (10 MB of matrices), 8.0 us
// with nothing in the caches, one row of rank 16 5.0.
struct AdFew {
  AdIndex in;
  const char* x;
  uint32_t x_stride;   // bytes
  const char* a;       // [adapters, rank, k]
  int k, n, splits, share;  // share: units of 128 bytes a split
  float* sums;         // [splits, m, rank]
  const float* scale;
  const char* b;       // [adapters, rank, n]
  const char* y;
  uint32_t y_stride;
  char* out;
  uint32_t out_stride;
  int padded;          // the rank in LDS, a multiple of 32
};

template <int KIND>
__global__ __launch_bounds__(256) void ad_shrink_few_kernel(AdFew p) {
  constexpr int SIZE = AdType<KIND>::SIZE, UNIT = 128 / SIZE;
  __shared__ f32x4_t part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4, col = lane & 15;
  int c, row;
  const int count = ad_tile_at(p.in, blockIdx.x, c, row);
  if (count == 0 || c >= p.in.adapters) return;
  const int rank = ad_rank(p.in, c), r0 = blockIdx.z * 16;
  if (r0 >= rank) return;
  const char* const x[1] = {ad_row(p.x, row, p.x_stride) + group * 16};
  const char* const w[1] = {p.a + ((int64_t)c * p.in.rank + min(r0 + col, rank - 1)) * p.k * SIZE + group * 16};  // (ranks behind the last: nobody reads the sums)
  const int u0 = blockIdx.y * p.share;
  f32x4_t acc[1][1] = {};
  ad_shrink_units<KIND, 1, 1>(x, w, p.k, u0 + wave, min(u0 + p.share, (p.k + UNIT - 1) / UNIT), 4, acc);
  part[wave][lane] = acc[0][0];
  __syncthreads();
  const int place = 4 * group + wave;  // thread: row 4 group + wave, rank r0 + col
  const int to = __shfl(row, place);
  if (place < count && r0 + col < rank) {
    float s = 0.f;
#pragma unroll
    for (int w4 = 0; w4 < 4; w4++) s += reinterpret_cast<const float*>(&part[w4][lane])[wave];
    p.sums[((int64_t)blockIdx.y * p.in.m + to) * p.in.rank + r0 + col] = s;
  }
}

// A plan's tiles: a workgroup has one split of the long axis for a tile's 32 rows and RT x 16 ranks, its wavefronts taking units in turn. Of a tile's workgroups the last one to
// arrive adds the splits' sums up, in their order, and leaves them, scaled, as the operands that the second products take: by rows (for the expansion), and with
// rows and ranks changed over (for the outer product).
//
// The splits are there to keep every compute unit at it: one alone reads some 20 GB/s. Both shrinks of 2048 rows of 5120 at rank 16 (42 MB) take 17.7 us in 1024 workgroups, of
// which the data 9, the way to it and the joining of the splits the rest (in 128 workgroups of the whole axis each: 24 us). Where the rank is high the matrices' own reads count:
// every tile reads its adapter's again, from the die's cache (8192 rows of 12800 and 2560, ranks 8 .. 64, 252 MB: 96 us, 63 of them with the matrices' loads left out).
struct AdShrinkJob {
  const char* v;      // rows, `stride` bytes apart
  uint32_t stride;
  const char* w;      // [adapters, rank, length]
  int length, splits, share;  // units of 128 bytes a split
  float* parts;       // [tile][chunk][split][row][rank] of sums (several splits), and an arrival counter [tile][chunk]
  int32_t* tickets;
  char* by_row;       // [tile][32 ranks][part][row][rank], or null
  char* by_rank;      // [tile][16 ranks][part][rank][row], or null
  int8_t* row_power;  // FP16: the exponents that the values are in, [tile][16 ranks][row] ...
  int8_t* rank_power; // ... and [tile][16 ranks]
};
struct AdShrink {
  AdIndex in;
  AdPlan plan;
  AdShrinkJob job[2];
  const float* scale;
  int chunks;  // of RT x 16 ranks
};
constexpr int AD_WAVES = 4;
constexpr int AD_EXPANDS = 768;   // workgroups of an expansion, about: 4096 rows of 5120 26.6 us (in 256: 36.2, in 2048: 26.5)
// Results of this many bytes are stored past the caches: half of what the dies' hold. Through them they push out what is still to be read. Add of 4096 rows of 5120 at rank 32
// (42 MB of results) 52 -> 45 us a call (y's rows read so too: 48 us). Rows of 2560 x 5120, rank 16, in a graph, through the caches and past them: 1600 (16 MB) 27.2 and 26.3 us, 2400
// 31.6 and 30.2, 4096 44.8 and 41.2, 8192 75.9 and 76.7; with a reader of the results behind it (silu_and_mul of them) 35.7 and 35.5, 43.0 and 42.8, 62.9 and 65.0, 107 and
// 113.6: a reader of a fresh 42 MB loses more than the call gains. Into y itself, as the linears and blocks call it, the two are the same with and without the reader. Gradients of 2048 rows
// of 5120 (21 MB of dx) 43.5 and 42.4, of 4096 74.0 and 72.6, of 8192 118.4 and 115.0.
constexpr int64_t AD_PAST_BYTES = 16 << 20;
// Rows of this many bytes, both sides' together, are read past the caches by the outer products, after which nobody reads them: half of the last-level cache's. 8192 rows of
// 12800 and 2560 (252 MB, and 210 MB of dx past the caches) 274 -> 227 us the call. Rows of 5120 and 5120 in a graph, through the caches and past them: 42 MB 42.2 and 43.9 us, 61 55.7
// and 57.2, 84 72.6 and 70.3, 123 96.2 and 92.8, 168 126.5 and 115.5: the two meet near 70 MB.
constexpr int64_t AD_PAST_ROWS = 128ll << 20;
__host__ __device__ constexpr int ad_sixteens(int rank) { return (rank + 15) / 16; }
__host__ __device__ constexpr int ad_thirties(int rank) { return (rank + 31) / 32; }

template <int KIND, int RT>
__global__ __launch_bounds__(64 * AD_WAVES) void ad_shrink_kernel(AdShrink p) {
  constexpr int SIZE = AdType<KIND>::SIZE, UNIT = 128 / SIZE, PARTS = AdType<KIND>::PARTS, WIDE = 16 * RT, PITCH = WIDE + 1;
  constexpr int JOINED = AD_WAVES / 2 * 2 * RT * 64 * 16, SUMS = 32 * PITCH * 4;
  __shared__ __align__(16) char shared[JOINED > SUMS ? JOINED : SUMS];
  __shared__ int32_t row_power[AD_TILE * RT], rank_power[RT], last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4, col = lane & 15, tile = blockIdx.x;
  int c, start;
  const int count = ad_tile(p.plan, tile, c, start);
  if (count == 0 || c >= p.in.adapters) return;
  const int chunk = blockIdx.y % p.chunks, of_both = blockIdx.y / p.chunks, second = of_both >= p.job[0].splits, split = second ? of_both - p.job[0].splits : of_both;
  const AdShrinkJob& job = p.job[second];
  const int rank = ad_rank(p.in, c), r0 = chunk * WIDE;
  if (r0 >= rank) return;
  const float scale = p.scale ? p.scale[c] : 1.0f;
  const char* x[2];
  const char* w[RT];
#pragma unroll
  for (int i = 0; i < 2; i++) x[i] = ad_row(job.v, p.plan.order()[start + min(16 * i + col, count - 1)], job.stride) + group * 16;  // (rows behind the last: not used)
#pragma unroll
  for (int i = 0; i < RT; i++) w[i] = job.w + ((int64_t)c * p.in.rank + min(r0 + 16 * i + col, rank - 1)) * job.length * SIZE + group * 16;
  f32x4_t acc[2][RT] = {};
  const int first = split * job.share + wave, units = min((split + 1) * job.share, (job.length + UNIT - 1) / UNIT);
  // an adapter of a lower rank than the pool's: only the sixteens that it has
  if (RT == 4 && rank - r0 > 32) ad_shrink_units<KIND, 2, 4, RT>(x, w, job.length, first, units, AD_WAVES, acc);
  else if (RT >= 2 && rank - r0 > 16) ad_shrink_units<KIND, 2, 2, RT>(x, w, job.length, first, units, AD_WAVES, acc);
  else ad_shrink_units<KIND, 2, 1, RT>(x, w, job.length, first, units, AD_WAVES, acc);
  // the wavefronts' sums: the upper half of them to the lower half, again and again
  f32x4_t* join = reinterpret_cast<f32x4_t*>(shared);
#pragma unroll
  for (int half = AD_WAVES / 2; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int i = 0; i < 2 * RT; i++) join[((wave - half) * 2 * RT + i) * 64 + lane] = acc[i / RT][i % RT];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int i = 0; i < 2 * RT; i++) acc[i / RT][i % RT] += join[(wave * 2 * RT + i) * 64 + lane];
    __syncthreads();
  }
  float* sums = reinterpret_cast<float*>(shared);
  if (wave == 0) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < RT; j++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int place = 16 * i + 4 * group + q, r = 16 * j + col;
          sums[place * PITCH + r] = place < count && r0 + r < rank ? acc[i][j][q] * scale : 0.f;
        }
  }
  __syncthreads();
  const int t = threadIdx.x, sixteens = ad_sixteens(p.in.rank);
  if (job.splits > 1) {  // the sums to memory past this die's cache, and the ticket behind them
    const int64_t mine = (int64_t)tile * p.chunks + chunk;
    float* parts = job.parts + mine * job.splits * (AD_TILE * WIDE);
    for (int i = t; i < AD_TILE * WIDE; i += 64 * AD_WAVES) store_through(&parts[split * (AD_TILE * WIDE) + i], sums[i / WIDE * PITCH + i % WIDE]);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0) last = __hip_atomic_fetch_add(&job.tickets[mine], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == job.splits - 1;
    __syncthreads();
    if (!last) return;
    for (int i = t; i < AD_TILE * WIDE; i += 64 * AD_WAVES) {
      float v = 0.f;
#pragma unroll 8
      for (int s = 0; s < job.splits; s++) v += load_through(&parts[s * (AD_TILE * WIDE) + i]);
      sums[i / WIDE * PITCH + i % WIDE] = v;
    }
    __syncthreads();
  }
  if constexpr (KIND == HB_F16) {
    if (t < AD_TILE * RT) {  // thread: sixteen ranks of a row
      const int place = t % AD_TILE, j = t / AD_TILE;
      float most = 0.f;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const float size = fabsf(sums[place * PITCH + 16 * j + r]);
        most = size < INFINITY ? fmaxf(most, size) : most;
      }
      const int e = ad_exponent(most);
      row_power[j * AD_TILE + place] = e;
      int high = e;
#pragma unroll
      for (int d = 1; d < AD_TILE; d <<= 1) high = max(high, __shfl_xor(high, d));
      if (place == 0) rank_power[j] = high;
      if (r0 / 16 + j < sixteens) {
        const int64_t at = (int64_t)tile * sixteens + r0 / 16 + j;
        if (job.by_row) job.row_power[at * AD_TILE + place] = (int8_t)e;
        if (job.by_rank && place == 0) job.rank_power[at] = (int8_t)high;
      }
    }
    __syncthreads();
  }
  if (job.by_row) {
    constexpr int ROW = RT == 1 ? 32 : WIDE;  // (up to sixteen ranks: zeros behind them to 32)
    for (int i = t; i < AD_TILE * ROW; i += 64 * AD_WAVES) {
      const int r = i % 32, place = i / 32 % AD_TILE, step = i / (32 * AD_TILE);
      if (r0 + 32 * step >= p.in.rank) break;
      const float v = 32 * step + r < WIDE ? sums[place * PITCH + 32 * step + r] : 0.f;
      const int64_t at = ((int64_t)tile * ad_thirties(p.in.rank) + r0 / 32 + step) * PARTS * 1024 + place * 32 + r;
      if constexpr (SIZE == 4) {
        reinterpret_cast<float*>(job.by_row)[at] = v;
      } else {
        uint16_t part[PARTS];
        const float unit = KIND == HB_F16 && 32 * step + r < WIDE ? ad_pow2(-row_power[(32 * step + r) / 16 * AD_TILE + place]) : 1.0f;
        ad_cut<KIND>(v * unit, part);
#pragma unroll
        for (int q = 0; q < PARTS; q++) reinterpret_cast<uint16_t*>(job.by_row)[at + q * 1024] = part[q];
      }
    }
  }
  if (job.by_rank) {
    for (int i = t; i < AD_TILE * WIDE; i += 64 * AD_WAVES) {
      const int place = i % AD_TILE, r = i / AD_TILE % 16, j = i / (AD_TILE * 16);
      if (r0 / 16 + j >= sixteens) break;
      const float v = sums[place * PITCH + 16 * j + r];
      const int64_t at = ((int64_t)tile * sixteens + r0 / 16 + j) * PARTS * 512 + r * 32 + place;
      if constexpr (SIZE == 4) {
        reinterpret_cast<float*>(job.by_rank)[at] = v;
      } else {
        uint16_t part[PARTS];
        ad_cut<KIND>(KIND == HB_F16 ? v * ad_pow2(-rank_power[j]) : v, part);
#pragma unroll
        for (int q = 0; q < PARTS; q++) reinterpret_cast<uint16_t*>(job.by_rank)[at + q * 512] = part[q];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ expand

// acc[j] of TM x 16 rows += 32 ranks: `s` their parts (or FP32 values), v eight ranks of the matrix a lane, sixteen bytes each. Lane l's operand for instruction j
// is column l * VEC + j: the eight rows, turned in registers, give it all of them, and the results are whole 16-byte pieces of out's rows.
template <int KIND, int TM, int LIMIT, int WORDS>
__device__ __forceinline__ void ad_products(const u32x4_t (&s)[LIMIT][WORDS], const u32x4_t (&v)[8], f32x4_t (&acc)[LIMIT][AD_VEC<KIND>]) {  // (of LIMIT, the first TM)
  if constexpr (KIND == HB_F32) {
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int t = 0; t < TM; t++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(s[t][i >> 2][i & 3]), __uint_as_float(v[i][j]), acc[t][j], 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < AD_VEC<KIND>; j++) {
      const u32x4_t w = ad_turn(v, j);
#pragma unroll
      for (int i = 0; i < WORDS; i++)
#pragma unroll
        for (int t = 0; t < TM; t++) acc[t][j] = ad_mma<KIND>(s[t][i], w, acc[t][j]);
    }
  }
}

// y + the lane's VEC sums of row i of its four (times 2^e), rounded.
template <int KIND>
__device__ __forceinline__ u32x4_t ad_result(const u32x4_t& y, const f32x4_t (&acc)[AD_VEC<KIND>], int i, float unit) {
  u32x4_t v;
  auto value = [&](int j) { return ad_value<KIND>(ad_elem<KIND>(y, j)) + (KIND == HB_F16 ? acc[j][i] * unit : acc[j][i]); };
#pragma unroll
  for (int q = 0; q < 4; q++) {
    if constexpr (KIND == HB_F32) v[q] = __float_as_uint(value(q));
    else if constexpr (KIND == HB_BF16) v[q] = bf16_pair(value(2 * q), value(2 * q + 1));
    else v[q] = ad_bits<KIND>(value(2 * q)) | ad_bits<KIND>(value(2 * q + 1)) << 16;
  }
  return v;
}

// Few rows: a workgroup joins the splits' sums of its tile in LDS, then a tile's rows times four wavefronts' columns, sixteen lanes of sixteen bytes each. 64 rows of 25600, 32
// adapters of up to 64 ranks (55 MB of matrices and rows): 21 us with nothing in the caches, 2.6 TB/s: a wavefront has few steps behind its start, and its 230 registers,
// most of them matrix rows under way, leave room for two a SIMD. One row of 5120 at rank 16 5.6 us.
template <int KIND, int HOW>
__global__ __launch_bounds__(256) void ad_expand_few_kernel(AdFew p) {
  constexpr int VEC = AD_VEC<KIND>, SIZE = AdType<KIND>::SIZE, PARTS = AdType<KIND>::PARTS;
  extern __shared__ __align__(16) char staged[];  // [part][row][padded + 16 bytes]
  __shared__ int32_t power[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4, col = lane & 15;
  int c, row;
  const int count = ad_tile_at(p.in, blockIdx.x, c, row);
  if (count == 0) return;
  const int rank = ad_rank(p.in, c), pitch = p.padded + (SIZE == 2 ? 8 : 4);  // elements
  if (rank == 0 && p.y == p.out) return;
  const int stride = gridDim.y * 4;
  int block = blockIdx.y * 4 + wave;
  u32x4_t y[4], v[2][8];
  int rows[4];
#pragma unroll
  for (int i = 0; i < 4; i++) rows[i] = __shfl(row, 4 * group + i);
  auto base = [&](int first) {  // (rows behind the last: the first again)
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = ad_take<KIND, HOW>(ad_row(p.y, rows[i], p.y_stride), first, p.n);
  };
  // what is under way: (block, 32 ranks) one after another, two ahead of the products (behind the last block the row's end: no load behind a branch)
  const char* matrix = p.b + (int64_t)c * p.in.rank * p.n * SIZE;  // (a class without an adapter reads none)
  int ahead = block * 16 * VEC + col * VEC, ahead_rank = 0;
  auto load = [&](u32x4_t (&to)[8]) {
#pragma unroll
    for (int s = 0; s < 8; s++) to[s] = ad_take<KIND, HOW == AD_TINY ? AD_TINY : AD_NEAR>(ad_row(matrix, min(ahead_rank + 8 * group + s, rank - 1), (uint32_t)p.n * SIZE), min(ahead, p.n), p.n);
    ahead_rank += 32;
    if (ahead_rank >= rank) ahead_rank = 0, ahead += stride * 16 * VEC;
  };
  base(block * 16 * VEC + col * VEC);
  if (rank == 0) {  // no adapter: the rows as they are
    for (; block * (16 * VEC) < p.n; block += stride) {
      const int first = block * 16 * VEC + col * VEC;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (4 * group + i < count) ad_put<KIND, HOW>(ad_row(p.out, rows[i], p.out_stride), y[i], first, p.n);
      base(min(first + stride * 16 * VEC, p.n));
    }
    return;
  }
  load(v[0]);
  load(v[1]);
  {  // the rows' sums, joined over the splits and scaled: sixteen threads a row
    const int place = threadIdx.x / 16, lane_of = threadIdx.x % 16;
    const float* sums = p.sums + (int64_t)__shfl(row, place) * p.in.rank;
    const float scale = p.scale ? p.scale[c] : 1.0f;
    auto sum = [&](int r) {  // every split's load under way before the first is used
      float part[AD_SPLITS], to = 0.f;
#pragma unroll
      for (int s = 0; s < AD_SPLITS; s++) part[s] = s < p.splits ? sums[(int64_t)s * p.in.m * p.in.rank + r] : 0.f;
#pragma unroll
      for (int s = 0; s < AD_SPLITS; s++) to += part[s];
      return to * scale;
    };
    float unit = 1.0f;
    if constexpr (KIND == HB_F16) {
      float most = 0.f;
      for (int r = lane_of; r < rank; r += 16) {
        const float size = fabsf(sum(r));
        most = size < INFINITY ? fmaxf(most, size) : most;
      }
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
      const int e = ad_exponent(most);
      if (lane_of == 0) power[place] = e;
      unit = ad_pow2(-e);
    }
    const int used = (rank + 31) & ~31;
#pragma unroll 2
    for (int r = lane_of; r < used; r += 16) {
      const float to = r < rank && place < count ? sum(r) * unit : 0.f;
      if constexpr (SIZE == 4) {
        reinterpret_cast<float*>(staged)[place * pitch + r] = to;
      } else {
        uint16_t part[PARTS];
        ad_cut<KIND>(to, part);
#pragma unroll
        for (int i = 0; i < PARTS; i++) reinterpret_cast<uint16_t*>(staged)[(i * 16 + place) * pitch + r] = part[i];
      }
    }
  }
  __syncthreads();
  f32x4_t acc[1][VEC] = {};
  int r0 = 0;
  for (bool more = block * (16 * VEC) < p.n; more;) {  // (idle lanes behind the last column take part in the products)
#pragma unroll
    for (int d = 0; d < 2; d++) {
      if (!more) break;
      constexpr int WORDS = SIZE == 4 ? 2 : PARTS;
      u32x4_t s[1][WORDS];
#pragma unroll
      for (int i = 0; i < WORDS; i++)
        s[0][i] = *reinterpret_cast<const u32x4_t*>(SIZE == 4 ? staged + (col * pitch + r0 + 8 * group + 4 * i) * 4 : staged + ((i * 16 + col) * pitch + r0 + 8 * group) * 2);
      ad_products<KIND, 1, 1, WORDS>(s, v[d], acc);
      load(v[d]);
      r0 += 32;
      if (r0 < rank) continue;
      const int first = block * 16 * VEC + col * VEC;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (4 * group + i < count)
          ad_put<KIND, HOW>(ad_row(p.out, rows[i], p.out_stride), ad_result<KIND>(y[i], acc[0], i, KIND == HB_F16 ? ad_pow2(power[4 * group + i]) : 1.0f), first, p.n);
#pragma unroll
      for (int j = 0; j < VEC; j++) acc[0][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      r0 = 0;
      block += stride;
      more = block * (16 * VEC) < p.n;
      base(min(first + stride * 16 * VEC, p.n));
    }
  }
}

// The partial sums of adapters with several units, in the units' order: block `block` of `blocks` for the adapter whose first slot is `slot`. (dx's expansion has them as
// further workgroups: a launch of their own for so little is 5 us.)
struct AdJoinJob {
  int length;
  float* to;           // [adapters, rank, length]
  const float* parts;  // [slots, rank, length]
};
struct AdJoin {
  AdJoinJob job[2];
  int slots, blocks;
};
__device__ __forceinline__ void ad_join(const AdIndex& in, const AdPlan& plan, const AdJoinJob& job, int slot, int block, int blocks) {
  if (slot >= plan.slots()[plan.classes]) return;
  const AdPlace at = ad_find(plan, plan.slots(), slot);
  if (at.first != slot) return;
  const int units = plan.slots()[at.c + 1] - slot;
  const int64_t size = (int64_t)in.rank * job.length;
  const float* from = job.parts + slot * size;
  for (int64_t i = ((int64_t)block * 256 + threadIdx.x) * 4; i < size; i += (int64_t)blocks * 1024) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int u = 0; u < units; u++) {
      const u32x4_t part = ad_load<HB_F32>(reinterpret_cast<const char*>(from + u * size + i), size - i);
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] += __uint_as_float(part[j]);
    }
    u32x4_t out;
#pragma unroll
    for (int j = 0; j < 4; j++) out[j] = __float_as_uint(v[j]);
    ad_store<HB_F32>(reinterpret_cast<char*>(job.to + (int64_t)at.c * size + i), out, size - i);
  }
}

// A plan's tiles, sixteen rows a workgroup: every wavefront for itself, over every (4 x share)-th block of sixteen lanes' columns. It is bound by what it stores and y's
// rows: 4096 rows of 5120 at rank 32 (84 MB) 26.6 us with nothing in the caches, 3.2 TB/s, in three wavefronts a SIMD (with two tiles of
// rows a wavefront the matrix is turned in registers half as often, and there is room for two: slower); dx of 2048 rows of 5120 (21 MB and the join) 9.8.
struct AdExpand {
  AdIndex in;
  AdPlan plan;
  const char* by_row;  // the shrink's
  const int8_t* row_power;
  int n;
  const char* w;       // [adapters, rank, n]
  const char* y;       // null: zeros
  uint32_t y_stride;   // bytes
  char* out;
  uint32_t out_stride;
  int share;           // workgroups a tile (gridDim.y, less those that join)
  AdJoin join;
};
template <int KIND, int HOW>
__global__ __launch_bounds__(256, 3) void ad_expand_kernel(AdExpand p) {
  if ((int)blockIdx.y >= p.share) {
    const int i = (blockIdx.y - p.share) * gridDim.x + blockIdx.x, of = p.join.slots * p.join.blocks;
    if (i < 2 * of) ad_join(p.in, p.plan, p.join.job[i >= of], i % of / p.join.blocks, i % p.join.blocks, p.join.blocks);
    return;
  }
  constexpr int VEC = AD_VEC<KIND>, SIZE = AdType<KIND>::SIZE, PARTS = AdType<KIND>::PARTS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4, col = lane & 15, tile = blockIdx.x >> 1, half = blockIdx.x & 1;
  int c, start;
  int count = ad_tile(p.plan, tile, c, start) - 16 * half;
  if (count <= 0) return;
  start += 16 * half;
  count = min(count, 16);
  const int rank = ad_rank(p.in, c);
  if (rank == 0 && p.y == p.out) return;
  int rows[4];
#pragma unroll
  for (int i = 0; i < 4; i++) rows[i] = p.plan.order()[start + min(4 * group + i, count - 1)];
  const int sixteens = ad_sixteens(p.in.rank), steps = ad_thirties(rank);
  int power = 0;  // FP16: of row col, the largest over the ranks
  const int8_t* powers = p.row_power + (int64_t)tile * sixteens * AD_TILE + 16 * half;  // (the wavefront's)
  if constexpr (KIND == HB_F16) {
    power = -128;
    for (int j = 0; j < ad_sixteens(rank); j++) power = max(power, (int)powers[j * AD_TILE + col]);
  }
  const char* sums = p.by_row + (int64_t)tile * ad_thirties(p.in.rank) * PARTS * 1024 * SIZE + ((16 * half + col) * 32 + 8 * group) * SIZE;
  constexpr int WORDS = SIZE == 4 ? 2 : PARTS;
  u32x4_t s[1][WORDS], y[4], v[8];
  auto parts = [&](int step) {
#pragma unroll
    for (int i = 0; i < WORDS; i++) {
      s[0][i] = *reinterpret_cast<const u32x4_t*>(sums + (int64_t)step * PARTS * 1024 * SIZE + (SIZE == 4 ? 16 * i : i * 2048));
      if constexpr (KIND == HB_F16) {
        const int j = 2 * step + (group >> 1);  // (ranks behind the last sixteen are zero)
        s[0][i] = ad_lower(s[0][i], j < ad_sixteens(rank) ? powers[j * AD_TILE + col] - power : 0);
      }
    }
  };
  const char* mine = p.w + (int64_t)c * p.in.rank * p.n * SIZE;
  auto matrix = [&](int first, int step) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = ad_take<KIND, HOW == AD_TINY ? AD_TINY : AD_NEAR>(ad_row(mine, min(32 * step + 8 * group + i, rank - 1), (uint32_t)p.n * SIZE), first, p.n);
  };
  auto base = [&](int first) {  // (rows behind the last: it again)
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = p.y ? ad_take<KIND, HOW == AD_TINY ? AD_TINY : AD_NEAR>(ad_row(p.y, rows[i], p.y_stride), first, p.n) : u32x4_t{0u, 0u, 0u, 0u};
  };
  // the wavefront's blocks, the next one's matrix under way while one is added; a rank of up to 32 keeps its sums in registers
  const int stride = p.share * 4;
  int block = blockIdx.y * 4 + wave;
  if (block * 16 * VEC >= p.n) return;
  base(block * 16 * VEC + col * VEC);
  if (steps) {
    matrix(block * 16 * VEC + col * VEC, 0);
    parts(0);
  }
  float unit[4];
#pragma unroll
  for (int i = 0; i < 4; i++) unit[i] = KIND == HB_F16 ? ad_pow2(max(__shfl(power, 4 * group + i), -126)) : 1.0f;
  for (; block * 16 * VEC < p.n; block += stride) {
    const int first = block * 16 * VEC + col * VEC;
    const bool more = (block + stride) * 16 * VEC < p.n;
    f32x4_t acc[1][VEC] = {};
    for (int step = 0; step < steps; step++) {
      ad_products<KIND, 1, 1, WORDS>(s, v, acc);
      if (step + 1 < steps) {
        matrix(first, step + 1);
        parts(step + 1);
      }
    }
    if (more) {
      if (steps) matrix(first + stride * 16 * VEC, 0);
      if (steps > 1) parts(0);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (4 * group + i < count)  // (without an adapter the rows as they are: -0 too)
        ad_put<KIND, HOW>(ad_row(p.out, rows[i], p.out_stride), rank == 0 ? y[i] : ad_result<KIND>(y[i], acc[0], i, unit[i]), first, p.n);
    if (more) base(first + stride * 16 * VEC);
  }
}

// ------------------------------------------------------------------------------------------------ outer

struct AdOuterJob {
  const char* by_rank;  // of the other side's shrink
  const int8_t* rank_power;
  const char* v;        // rows
  uint32_t stride;      // bytes
  int length;
  float* to;            // [adapters, rank, length]
  float* parts;         // [slots, rank, length]
};
struct AdOuter {
  AdIndex in;
  AdPlan plan;
  AdOuterJob job[2];
  int unit, chunks;
};

// A workgroup: RT x 16 ranks times sixteen lanes' columns over a unit of an adapter's rows, the four wavefronts taking its tiles in turn and joining
// their sums in LDS. A lane's eight rows of sixteen bytes are turned as in the expansion; the next tile's are under way while one is
// multiplied. An adapter's only unit writes the gradient (zeros, if it has no rows), several write partial sums for ad_join. (Joined by the last of them to
// arrive instead, whose sums must pass the dies' caches in words: 28 us for the 16 of both kernels at 2048 rows of 5120 x 5120, rank 16.) The rows' reads bound it: there 11.1 us
// for 42 MB that the shrink has just read, 3.8 TB/s; 8192 rows of 12800 and 2560, FP16, ranks up to 64, 77 us for 252 MB, past the last-level cache, 3.3 TB/s
// (64 at the least; of two parts a sum 66).
// A unit has 512 rows or more: of 128 the parts cost their join more (10.4 us for 9.4 of the launch that has it), of 2048 the products are in too few workgroups (15.3 for 11.1).
template <int KIND, int RT, int HOW>
__global__ __launch_bounds__(256, RT == 1 ? 3 : 2) void ad_outer_kernel(AdOuter p) {
  constexpr int VEC = AD_VEC<KIND>, SIZE = AdType<KIND>::SIZE, PARTS = AdType<KIND>::PARTS, WORDS = SIZE == 4 ? 2 : PARTS;
  __shared__ f32x4_t join[4 * VEC * 64];  // [wavefront][column of a lane][lane]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4, col = lane & 15;
  const AdOuterJob& job = p.job[blockIdx.z / p.chunks];
  const int r0 = (blockIdx.z % p.chunks) * 16 * RT, u = blockIdx.y, sixteens = ad_sixteens(p.in.rank);
  if (u >= p.plan.units()[p.plan.classes] || (int64_t)blockIdx.x * 16 * VEC >= job.length) return;
  const int first = blockIdx.x * 16 * VEC + col * VEC, left = job.length - first;
  const AdPlace at = ad_find(p.plan, p.plan.units(), u);
  const int c = at.c, which = u - at.first, units = p.plan.units()[c + 1] - at.first;
  const int start = at.row + which * p.unit, end = min(start + p.unit, at.next_row);
  const int rank = ad_rank(p.in, c), tile0 = p.plan.tiles()[c] + which * (p.unit / AD_TILE), tiles = r0 < rank ? (end - start + AD_TILE - 1) / AD_TILE : 0;
  const int have = max(min(RT, ad_sixteens(rank - r0)), 1);  // sixteens of ranks (those behind the adapter's rank are not written)
  float* to = units > 1 ? job.parts + (int64_t)(p.plan.slots()[c] + which) * p.in.rank * job.length : job.to + (int64_t)c * p.in.rank * job.length;
  f32x4_t acc[RT][VEC] = {};
  int power[RT];  // FP16: the sums are in units of 2^power, the largest of the unit's tiles
  const int8_t* powers = job.rank_power + (int64_t)tile0 * sixteens + r0 / 16;
#pragma unroll
  for (int t = 0; t < RT; t++) {
    power[t] = 0;
    if constexpr (KIND == HB_F16) {
      power[t] = -128;
      for (int i = lane; i < tiles && t < have; i += 64) power[t] = max(power[t], (int)powers[(int64_t)i * sixteens + t]);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) power[t] = max(power[t], __shfl_xor(power[t], d));
    }
  }
  // The tiles, for USED of the RT sixteens: a loop of its own for each (one that chose inside moved its sums between the register files every time, 450 registers for 240). Under
  // way: the rows and their sums one tile ahead, the rows' numbers two.
  auto run = [&](auto used) {
    constexpr int USED = decltype(used)::value;
    int rows[8], shift[USED];
    u32x4_t next[8], ahead[USED][WORDS];
    f32x4_t sum[USED][VEC] = {};
    auto number = [&](int tile) {
      const int from = start + tile * AD_TILE + 8 * group;
#pragma unroll
      for (int s = 0; s < 8; s++) rows[s] = p.plan.order()[min(from + s, end - 1)];
    };
    auto load = [&](int tile) {
#pragma unroll
      for (int s = 0; s < 8; s++) next[s] = ad_take<KIND, HOW>(ad_row(job.v, rows[s], job.stride), first, job.length);
#pragma unroll
      for (int t = 0; t < USED; t++) {  // (behind the adapter's sixteens its last one again)
        const int j = min(t, have - 1);
        const char* from = job.by_rank + ((int64_t)(tile0 + tile) * sixteens + r0 / 16 + j) * PARTS * 512 * SIZE + (col * 32 + 8 * group) * SIZE;
#pragma unroll
        for (int i = 0; i < WORDS; i++) ahead[t][i] = *reinterpret_cast<const u32x4_t*>(from + (SIZE == 4 ? 16 * i : i * 1024));
        if constexpr (KIND == HB_F16) shift[t] = powers[(int64_t)tile * sixteens + j];
      }
    };
    const int last = tiles - 1;  // (behind the last tile it again: no load behind a branch)
    number(wave);
    load(wave);
    number(min(wave + 4, last));
    for (int tile = wave; tile < tiles; tile += 4) {
      u32x4_t v[8], s[USED][WORDS];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = next[i];
      if (start + (tile + 1) * AD_TILE > end)  // the last tile's rows behind the end: what they repeat may be infinite
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = start + tile * AD_TILE + 8 * group + i < end ? v[i] : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
      for (int t = 0; t < USED; t++)
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
          s[t][i] = ahead[t][i];
          if constexpr (KIND == HB_F16) s[t][i] = ad_lower(s[t][i], shift[t] - power[t]);
        }
      load(min(tile + 4, last));
      number(min(tile + 8, last));
      ad_products<KIND, USED, USED, WORDS>(s, v, sum);
    }
#pragma unroll
    for (int t = 0; t < USED; t++)
#pragma unroll
      for (int j = 0; j < VEC; j++) acc[t][j] = sum[t][j];
  };
  if (wave < tiles) {
    if (RT == 4 && have > 2) run(std::integral_constant<int, RT>{});
    else if (RT >= 2 && have == 2) run(std::integral_constant<int, RT < 2 ? 1 : 2>{});
    else run(std::integral_constant<int, 1>{});
  }
  // D: this lane's columns first .. first + VEC - 1 of ranks 4 group .. + 3 of every sixteen
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const float unit = KIND == HB_F16 ? ad_pow2(max(power[t], -126)) : 1.0f;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VEC; j++) join[(wave * VEC + j) * 64 + lane] = KIND == HB_F16 ? acc[t][j] * unit : acc[t][j];
    __syncthreads();
    // thread: rank t * 16 + 4 group + wave of the columns of its lane
    const int r = r0 + 16 * t + 4 * group + wave;
    if (r < p.in.rank && left > 0) {
      float* row = to + (int64_t)r * job.length;
      float sum[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) v += reinterpret_cast<const float*>(&join[(w * VEC + j) * 64 + lane])[wave];
        sum[j] = r < rank ? v : 0.f;
      }
      const bool whole = first + VEC <= job.length;
#pragma unroll
      for (int q = 0; q < VEC; q += 4) {
        u32x4_t v;
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = __float_as_uint(sum[q + j]);
        if (whole) *reinterpret_cast<u32x4_loose*>(row + first + q) = v;
      }
      if (!whole) {
        const int from = HOW == AD_TINY ? first : job.length - VEC;  // the lane's columns, of which the ones before `first` are another's
#pragma unroll
        for (int j = 0; j < VEC; j++)
          if (from + j >= first && from + j < job.length) row[from + j] = sum[j];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host

static size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
static int64_t cut(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct AdShape {
  int64_t m;
  int adapters, rank, k, n, kind, size;
  bool grads, few;
  int splits, rt, unit;  // few: splits of the long axis. Else rank tiles a shrink's workgroup, rows a unit
  int share, splits_x, splits_dy, chunks;  // units of 128 bytes a split of the shrinks (x alone without gradients), chunks of ranks
  int64_t tiles, units, slots, tickets;
  // few: sums. Else plan | tickets | splits' sums | the x side by row or by rank | its powers | the dy side by row | by rank | its powers of both | parts of da | of db
  size_t sums_bytes, plan_bytes, ticket_bytes, split_bytes, row_bytes, rank_bytes, row_power_bytes, rank_power_bytes, part_a_bytes, part_b_bytes;
  size_t bytes() const {
    if (few) return sums_bytes;
    if (!grads) return plan_bytes + ticket_bytes + split_bytes + row_bytes + row_power_bytes;
    return plan_bytes + ticket_bytes + split_bytes + row_bytes + row_power_bytes + 2 * (rank_bytes + rank_power_bytes) + part_a_bytes + part_b_bytes;
  }
};

static bool ad_shape(const hb_adapters* a, int64_t m, bool grads, AdShape& s) {
  if (a->type < HB_BF16 || a->type > HB_F32 || a->adapters <= 0 || a->adapters > AD_MOST || a->rank <= 0 || a->rank > AD_RANK || a->k <= 0 || a->n <= 0 ||
      a->k > AD_LONGEST || a->n > AD_LONGEST || m <= 0 || m > AD_MAX_ROWS)
    return false;
  s = AdShape{};
  s.m = m, s.adapters = a->adapters, s.rank = a->rank, s.k = a->k, s.n = a->n, s.kind = a->type, s.size = a->type == HB_F32 ? 4 : 2;
  s.grads = grads;
  s.few = !grads && m <= AD_SELF_ROWS;
  const int64_t classes = std::min<int64_t>(a->adapters + 1, m);
  if (s.few) {
    s.tiles = std::min<int64_t>(m, a->adapters + cut(m, 16));  // at most: p classes of m rows have (m - p) / 16 + p of them or fewer
    const int64_t groups = s.tiles * cut(a->rank, 16);
    s.splits = (int)std::max<int64_t>(1, std::min<int64_t>({cut(1024, groups), cut(cut(a->k, 128 / s.size), 8), AD_SPLITS}));
    s.sums_bytes = up256((size_t)s.splits * m * a->rank * 4);
    return true;
  }
  s.tiles = cut(m, AD_TILE) + classes;
  s.rt = a->rank <= 16 ? 1 : a->rank <= 32 ? 2 : 4;
  s.plan_bytes = up256(AdPlan::ints(a->adapters + 1, m) * 4);
  s.chunks = (int)cut(a->rank, 16 * s.rt);
  const int64_t units_x = cut(a->k, 128 / s.size), units_dy = grads ? cut(a->n, 128 / s.size) : 0;
  s.share = (int)std::max<int64_t>(2 * AD_WAVES, cut((units_x + units_dy) * cut(m, AD_TILE) * s.chunks, 1024));
  s.splits_x = (int)cut(units_x, s.share), s.splits_dy = (int)cut(units_dy, s.share);
  s.tickets = s.tiles * s.chunks * (grads ? 2 : 1);
  s.split_bytes = up256((size_t)s.tiles * s.chunks * ((s.splits_x > 1 ? s.splits_x : 0) + (s.splits_dy > 1 ? s.splits_dy : 0)) * AD_TILE * 16 * s.rt * 4);
  const int parts = a->type == HB_F32 ? AdType<HB_F32>::PARTS : AdType<HB_BF16>::PARTS;
  s.row_bytes = up256((size_t)s.tiles * ad_thirties(a->rank) * parts * 1024 * s.size);
  s.rank_bytes = up256((size_t)s.tiles * ad_sixteens(a->rank) * parts * 512 * s.size);
  s.row_power_bytes = a->type == HB_F16 ? up256((size_t)s.tiles * ad_sixteens(a->rank) * AD_TILE) : 0;
  s.rank_power_bytes = a->type == HB_F16 ? up256((size_t)s.tiles * ad_sixteens(a->rank)) : 0;
  s.unit = 4 * AD_TILE;
  if (grads) {
    const int64_t blocks = (cut(a->k, 256 / s.size) + cut(a->n, 256 / s.size)) * cut(a->rank, 64);
    s.unit = (int)std::min<int64_t>(std::max<int64_t>(16 * AD_TILE, cut(cut(m * blocks, 512), 4 * AD_TILE) * 4 * AD_TILE), 1 << 20);
    s.units = cut(m, s.unit) + a->adapters;
    s.slots = 2 * (m / s.unit);  // an adapter of more than one unit has at most two for every whole `unit` of its rows
    s.part_a_bytes = up256((size_t)s.slots * a->rank * a->k * 4);
    s.part_b_bytes = up256((size_t)s.slots * a->rank * a->n * 4);
  }
  s.ticket_bytes = up256((size_t)s.tickets * 4);
  return true;
}

static int ad_run_plan(const AdShape& s, const AdIndex& in, const AdPlan& plan, char* ws, hipStream_t stream) {
  AdPlanParams p{in, plan, s.unit, 1, reinterpret_cast<int32_t*>(ws + s.plan_bytes), s.tickets};
  const int64_t pieces = cut(s.m, 64);
  if (s.m <= AD_HELD && (pieces + 1) * plan.classes <= AD_COUNTERS) {
    HB_LAUNCH((ad_plan_pieces_kernel), dim3(1), dim3(1024), (size_t)(pieces + 1) * plan.classes * 4, stream, p);
  } else {
    p.segments = std::max(1, std::min(16, AD_COUNTERS / plan.classes));
    HB_LAUNCH((ad_plan_kernel), dim3(1), dim3(1024), (size_t)p.segments * plan.classes * 4, stream, p);
  }
  return launch_status();
}

template <int KIND>
static int ad_run_shrink(const AdShape& s, AdShrink& p, char* ws, hipStream_t stream) {
  p.chunks = s.chunks;
  int32_t* tickets = reinterpret_cast<int32_t*>(ws + s.plan_bytes);
  float* parts = reinterpret_cast<float*>(ws + s.plan_bytes + s.ticket_bytes);
  for (int j = 0; j < (s.grads ? 2 : 1); j++) {
    p.job[j].splits = j ? s.splits_dy : s.splits_x;
    p.job[j].share = s.share;
    p.job[j].tickets = tickets + j * s.tiles * s.chunks;
    p.job[j].parts = parts + (j && s.splits_x > 1 ? s.tiles * s.chunks * s.splits_x * AD_TILE * 16 * s.rt : 0);
  }
  const dim3 grid((unsigned)s.tiles, (unsigned)(p.chunks * (s.splits_x + s.splits_dy)));
  if (s.rt == 1) HB_LAUNCH((ad_shrink_kernel<KIND, 1>), grid, dim3(64 * AD_WAVES), 0, stream, p);
  if (s.rt == 2) HB_LAUNCH((ad_shrink_kernel<KIND, 2>), grid, dim3(64 * AD_WAVES), 0, stream, p);
  if (s.rt == 4) HB_LAUNCH((ad_shrink_kernel<KIND, 4>), grid, dim3(64 * AD_WAVES), 0, stream, p);
  return launch_status();
}

template <int KIND>
static int ad_run_expand(const AdShape& s, AdExpand& p, hipStream_t stream) {
  const int64_t groups = cut(p.n, 4 * 16 * AD_VEC<KIND>);
  const int64_t share = std::max<int64_t>(1, std::min<int64_t>(groups, cut(s.m, 16) * groups / AD_EXPANDS));
  p.share = (int)cut(groups, share);
  const dim3 grid((unsigned)(2 * s.tiles), (unsigned)(p.share + cut(2ll * p.join.slots * p.join.blocks, 2 * s.tiles)));
  if (p.n < AD_VEC<KIND>) HB_LAUNCH((ad_expand_kernel<KIND, AD_TINY>), grid, dim3(256), 0, stream, p);
  else if (s.m * p.n * s.size >= AD_PAST_BYTES) HB_LAUNCH((ad_expand_kernel<KIND, AD_PAST>), grid, dim3(256), 0, stream, p);
  else HB_LAUNCH((ad_expand_kernel<KIND, AD_NEAR>), grid, dim3(256), 0, stream, p);
  return launch_status();
}

template <int KIND>
static int ad_run_outer(const AdShape& s, AdOuter& p, hipStream_t stream) {
  p.chunks = s.chunks;
  const int longest = std::max(p.job[0].length, p.job[1].length);
  const dim3 grid((unsigned)cut(longest, 16 * AD_VEC<KIND>), (unsigned)s.units, (unsigned)(2 * p.chunks));
  const bool tiny = std::min(p.job[0].length, p.job[1].length) < AD_VEC<KIND>;
#define HB_AD(RT) \
  if (s.rt == RT) { \
    if (tiny) HB_LAUNCH((ad_outer_kernel<KIND, RT, AD_TINY>), grid, dim3(256), 0, stream, p); \
    else if (s.m * (s.k + s.n) * s.size >= AD_PAST_ROWS) HB_LAUNCH((ad_outer_kernel<KIND, RT, AD_PAST>), grid, dim3(256), 0, stream, p); \
    else HB_LAUNCH((ad_outer_kernel<KIND, RT, AD_NEAR>), grid, dim3(256), 0, stream, p); \
  }
  HB_AD(1) HB_AD(2) HB_AD(4)
#undef HB_AD
  return launch_status();
}

template <int KIND>
static int ad_add(const hb_adapters* a, const AdShape& s, const AdIndex& in, const void* x, int64_t x_stride, const void* y, int64_t y_stride, void* out, int64_t out_stride,
                  char* ws, hipStream_t stream) {
  const char *xr = static_cast<const char*>(x), *yr = static_cast<const char*>(y);
  char* to = static_cast<char*>(out);
  if (s.few) {
    AdFew p{in, xr, (uint32_t)(x_stride * s.size), static_cast<const char*>(a->a), s.k, s.n, s.splits, (int)cut(cut(s.k, 128 / s.size), s.splits), reinterpret_cast<float*>(ws),
            a->scale, static_cast<const char*>(a->b), yr, (uint32_t)(y_stride * s.size), to, (uint32_t)(out_stride * s.size), ad_thirties(s.rank) * 32};
    HB_LAUNCH((ad_shrink_few_kernel<KIND>), dim3((unsigned)s.tiles, (unsigned)s.splits, (unsigned)ad_sixteens(s.rank)), dim3(256), 0, stream, p);
    if (int code = launch_status()) return code;
    const size_t lds = (size_t)AdType<KIND>::PARTS * 16 * (p.padded * AdType<KIND>::SIZE + 16);
    // workgroups enough for every compute unit twice: what finds its rows and joins their sums has then several blocks of columns to do it for. 64 rows of 25600, 36 tiles:
    // 21 us in 17 workgroups a tile, 25 in 8 or 50
    const int64_t groups = cut(s.n, 4 * 16 * AD_VEC<KIND>), share = std::max<int64_t>(1, std::min<int64_t>(groups, s.tiles * groups / 512));
    const dim3 grid((unsigned)s.tiles, (unsigned)cut(groups, share));
    if (s.n < AD_VEC<KIND>) HB_LAUNCH((ad_expand_few_kernel<KIND, AD_TINY>), grid, dim3(256), lds, stream, p);
    else HB_LAUNCH((ad_expand_few_kernel<KIND, AD_NEAR>), grid, dim3(256), lds, stream, p);
    return launch_status();
  }
  const AdPlan plan{reinterpret_cast<int32_t*>(ws), s.adapters + 1};
  char* by_row = ws + s.plan_bytes + s.ticket_bytes + s.split_bytes;
  int8_t* power = reinterpret_cast<int8_t*>(by_row + s.row_bytes);
  int code = ad_run_plan(s, in, plan, ws, stream);
  if (code) return code;
  AdShrink down{in, plan, {{xr, (uint32_t)(x_stride * s.size), static_cast<const char*>(a->a), s.k, 0, 0, nullptr, nullptr, by_row, nullptr, power, nullptr}, {}}, a->scale, 0};
  if ((code = ad_run_shrink<KIND>(s, down, ws, stream))) return code;
  AdExpand up{in, plan, by_row, power, s.n, static_cast<const char*>(a->b), yr, (uint32_t)(y_stride * s.size), to, (uint32_t)(out_stride * s.size), 0, {}};
  return ad_run_expand<KIND>(s, up, stream);
}

template <int KIND>
static int ad_grads(const hb_adapters* a, const AdShape& s, const AdIndex& in, const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, void* dx, float* da, float* db,
                    char* ws, hipStream_t stream) {
  const AdPlan plan{reinterpret_cast<int32_t*>(ws), s.adapters + 1};
  char* at = ws + s.plan_bytes + s.ticket_bytes + s.split_bytes;
  auto take = [&](size_t bytes) { char* here = at; at += bytes; return here; };
  char* dy_rows = take(s.row_bytes);
  int8_t* dy_row_power = reinterpret_cast<int8_t*>(take(s.row_power_bytes));
  char *x_ranks = take(s.rank_bytes), *dy_ranks = take(s.rank_bytes);
  int8_t *x_power = reinterpret_cast<int8_t*>(take(s.rank_power_bytes)), *dy_power = reinterpret_cast<int8_t*>(take(s.rank_power_bytes));
  float *part_a = reinterpret_cast<float*>(take(s.part_a_bytes)), *part_b = reinterpret_cast<float*>(take(s.part_b_bytes));
  int code = ad_run_plan(s, in, plan, ws, stream);
  if (code) return code;
  const char *xr = static_cast<const char*>(x), *dyr = static_cast<const char*>(dy);
  AdShrink down{in, plan,
                {{xr, (uint32_t)(x_stride * s.size), static_cast<const char*>(a->a), s.k, 0, 0, nullptr, nullptr, nullptr, x_ranks, nullptr, x_power},
                 {dyr, (uint32_t)(dy_stride * s.size), static_cast<const char*>(a->b), s.n, 0, 0, nullptr, nullptr, dy_rows, dy_ranks, dy_row_power, dy_power}},
                a->scale, 0};
  if ((code = ad_run_shrink<KIND>(s, down, ws, stream))) return code;
  // the outer products ahead of dx: they read x and dy again while the last-level cache holds what it can of them
  AdOuter outer{in, plan, {{dy_ranks, dy_power, xr, (uint32_t)(x_stride * s.size), s.k, da, part_a}, {x_ranks, x_power, dyr, (uint32_t)(dy_stride * s.size), s.n, db, part_b}}, s.unit, 0};
  if ((code = ad_run_outer<KIND>(s, outer, stream))) return code;
  AdExpand up{in, plan, dy_rows, dy_row_power, s.k, static_cast<const char*>(a->a), nullptr, 0, static_cast<char*>(dx), (uint32_t)(s.k * s.size), 0,
              {{{s.k, da, part_a}, {s.n, db, part_b}}, (int)s.slots, (int)std::min<int64_t>(cut((int64_t)s.rank * std::max(s.k, s.n), 1024), 1024)}};
  return ad_run_expand<KIND>(s, up, stream);
}

// Whether two sets of m rows of `width` bytes share any: y's rows are read while others of out's are written, so these are y's own or none of them.
static bool ad_rows_meet(int64_t y, int64_t y_stride, int64_t out, int64_t out_stride, int64_t m, int64_t width) {
  if (out >= y + (m - 1) * y_stride + width || y >= out + (m - 1) * out_stride + width) return false;
  if (y_stride == out_stride) {  // out's row r begins `in` bytes behind y's row r + ahead begins
    int64_t ahead = (out - y) / y_stride, in = (out - y) % y_stride;
    if (in < 0) in += y_stride, ahead--;
    return (in < width && std::abs(ahead) < m) || (y_stride - in < width && std::abs(ahead + 1) < m);
  }
  for (int64_t r = 0; r < m; r++) {  // y's row r and the first of out's that ends behind its begin
    const int64_t at = y + r * y_stride, behind = at - out - width;
    const int64_t row = behind < 0 ? 0 : behind / out_stride + 1;
    if (row < m && out + row * out_stride < at + width) return true;
  }
  return false;
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
  if (x_stride < s.k || y_stride < s.n || out_stride < s.n || std::max({x_stride, y_stride, out_stride}) > AD_STRIDE / s.size || !aligned(x, s.size) || !aligned(y, s.size) || !aligned(out, s.size) || !aligned(workspace, 16)) return HB_EINVAL;
  if (y == out && y_stride != out_stride) return HB_EINVAL;
  if (workspace_bytes < s.bytes()) return HB_EWORKSPACE;
  if (y != out && ad_rows_meet(reinterpret_cast<int64_t>(y), y_stride * s.size, reinterpret_cast<int64_t>(out), out_stride * s.size, m, (int64_t)s.n * s.size)) return HB_EINVAL;
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
  if (x_stride < s.k || dy_stride < s.n || std::max(x_stride, dy_stride) > AD_STRIDE / s.size || !aligned(x, s.size) || !aligned(dy, s.size) || !aligned(dx, s.size) || !aligned(da, 4) || !aligned(db, 4) || !aligned(workspace, 16))
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
