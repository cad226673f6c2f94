// The microscaled four-bit format: rounding to it (alone, and behind a gated activation), the values back, the weights' tile
// layout, and the linear.
#include <algorithm>
#include <atomic>

#include "mxfp4_ring.hpp"
#include "stream_common.hpp"

namespace hb {

// ------------------------------------------------------------------------------------------------ rounding, and back
// x [rows, k] -> codes [rows, k / 2], scales [rows, k / 32]. A lane takes eight consecutive values, four lanes a group: loads and
// stores of a wavefront are consecutive, and the group's largest magnitude is two lane exchanges. Memory bound: 1543 x 5120 of FP32 6.9 us, 5.2 TB/s
// read and written; one row is 1.5 us, and the call its host work (6.2).
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t lanes, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= lanes) return;  // whole groups leave together: `lanes` is a multiple of four
  Mx8<T> v;
  v.load(x + 8 * i);
  const uint32_t byte = mx_scale_byte(quad_max(v.amax()));
  reinterpret_cast<uint32_t*>(codes)[i] = byte == 255u ? 0u : v.codes(mx_scale_value(byte));
  if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
}

__device__ __forceinline__ void mx_values(uint32_t c, float s, __bf16* out) {
  bf16x2_t v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1),
                   __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3)};
  u32x4_t w;
#pragma unroll
  for (int j = 0; j < 4; j++) w[j] = __builtin_bit_cast(uint32_t, v[j]);
  *reinterpret_cast<u32x4_t*>(out) = w;
}
__device__ __forceinline__ void mx_values(uint32_t c, float s, _Float16* out) {  // through FP32: what a half does not hold rounds once
  const f32x2_t v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3)};
  typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
  f16x8_t w;
#pragma unroll
  for (int j = 0; j < 8; j++) w[j] = (_Float16)v[j >> 1][j & 1];
  *reinterpret_cast<f16x8_t*>(out) = w;
}
__device__ __forceinline__ void mx_values(uint32_t c, float s, float* out) {
  const f32x2_t v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3)};
#pragma unroll
  for (int h = 0; h < 2; h++) *reinterpret_cast<f32x4_t*>(out + 4 * h) = f32x4_t{v[2 * h][0], v[2 * h][1], v[2 * h + 1][0], v[2 * h + 1][1]};
}

// The values that codes and scales stand for, eight a lane. Memory bound: 2048 x 25600 to BF16 20 us, 6.6 TB/s, most of it written.
template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t lanes, T* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= lanes) return;
  mx_values(reinterpret_cast<const uint32_t*>(codes)[i], mx_scale_value(scales[i >> 2]), out + 8 * i);
}

// The lower end of silu(g) u in FP32, for g between -80 and 2^100 whose magnitude, where it is not zero, is 2^-100 and more or that of a 16-bit type: exp(-g) as exp2 of hi = -g log2(e) rounded, times 1 + r with r = -g - hi ln2
// (the product exact, in one multiply-add), one reciprocal, whose argument is scaled by 1 + MX_SILU_OFF. Without that scaling it is off by
// less than MX_SILU_OFF of its value: 2^-23 each for exp2 and the reciprocal, 2^-24 each for the correction, the sum and the two products,
// 80 x 2^-28.4 = 2^-22.1 for ln2 in FP32, together 0.73 x 2^-20 (and 2^-24 for the scaling's rounding); so the exact value lies between
// this and this (1 + 2 MX_SILU_OFF) (1 + 2^-23), which MX_SILU_SPAN is above. (A smaller FP32 gate's half is subnormal and loses bits that a large u brings
// back. BF16's smallest gates have eight bits at most, whose half FP32 holds exactly; FP16's are normal here.)
constexpr float MX_SILU_OFF = 0x1p-20f, MX_SILU_SPAN = 0x1.2p-19f;
__device__ __forceinline__ float mx_silu_mul(float g, float u) {
  const float hi = g * -1.44269504088896340736f;
  const float r = __builtin_fmaf(hi, -0.693147180559945309f, -g);
  const float e = __builtin_amdgcn_exp2f(hi);
  const float t = __builtin_fmaf(e, r, e);
  return g * __builtin_amdgcn_rcpf(__builtin_fmaf(t, 1.0f + MX_SILU_OFF, 1.0f + MX_SILU_OFF)) * u;
}

// silu(gate) * up of [rows, 2 half] rounded to the format in one pass; gate | up, or both in alternating blocks of `pairs` columns.
// A product within FP32's error of a border between two codes, or a group whose largest is that near a power of two, would
// round by that error: such a group (a few in a million values) is computed again in 64 bits, and so is one
// whose gates or products leave FP32's comfortable range. Mostly reading: 2048 x 51200 of FP16 49 us, 4.8 TB/s (a plain read of data that is not
// in the Infinity Cache reaches 6.9); with a 64-bit division a lane and a longer exponential 52.
template <typename T>
__global__ __launch_bounds__(256) void mx_silu_quantize_kernel(const T* __restrict__ x, int64_t rows, int half, int pairs, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales) {
  // A launch has 2^31 lanes at most. The row of the workgroup's first lane is one scalar division; the others are in that row or, where a row has 256 lanes
  // and more, in the next.
  const uint32_t per_row = (uint32_t)half >> 3, first = blockIdx.x * 256u, i = first + threadIdx.x;
  if (i >= (uint32_t)rows * per_row) return;  // whole groups leave together: half is a multiple of 32
  uint32_t r = first / per_row, c8 = first - r * per_row + threadIdx.x;
  if (per_row >= 256u) {
    const uint32_t over = c8 >= per_row;
    r += over;
    c8 -= over * per_row;
  } else {
    const uint32_t more = c8 / per_row;
    r += more;
    c8 -= more * per_row;
  }
  const uint32_t c = 8 * c8, gate_at = pairs ? (c / (uint32_t)pairs) * 2 * (uint32_t)pairs + c % (uint32_t)pairs : c, up_at = gate_at + (uint32_t)(pairs ? pairs : half);
  Mx8<T> g, u;
  x += (int64_t)r * 2 * half;
  g.load(x + gate_at);
  u.load(x + up_at);
  Mx8<float> p, q;
  float least = 0.f, most_g = 0.f;  // (a NaN passes by: its product is one)
  uint32_t small_g = 0xffffffffu;   // the bits of the smallest gate that is not zero, less one
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float gj = g.at(j);
    p.v[j >> 2][j & 3] = mx_silu_mul(gj, u.at(j));
    least = __builtin_fminf(least, gj);
    if (!std::is_same_v<T, _Float16>) most_g = __builtin_fmaxf(most_g, gj);
    if (std::is_same_v<T, float>) small_g = min(small_g, (__float_as_uint(gj) & 0x7fffffffu) - 1u);
  }
  bool far = least < -80.0f || most_g > 0x1p100f || small_g < 0x0d800000u - 1u;  // 2^-100
  const uint32_t top = quad_max(p.amax());
  uint32_t byte = mx_scale_byte(top);
  const float s = mx_scale_value(byte);
#pragma unroll
  for (int j = 0; j < 8; j++) q.v[j >> 2][j & 3] = p.v[j >> 2][j & 3] * (1.0f + MX_SILU_SPAN);
  uint32_t code = p.codes(s);
  constexpr uint32_t SPAN = 36;  // ulps: MX_SILU_SPAN of a value is 18 to 36
  far |= code != q.codes(s);
  far |= byte != 255u && ((top ^ (top + SPAN)) >> 23) != 0;
  far |= top != 0 && top < 0x0d800000u;  // below 2^-100
  if (byte == 255u) code = 0;
  if (quad_max(far)) {
    double v[8];
    double most = 0;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double gj = g.at(j);
      v[j] = gj / (1.0 + exp(-gj)) * (double)u.at(j);
      most = fmax(most, fabs(v[j]));  // (passes over a NaN)
      finite &= fabs(v[j]) < 0x1p128;
    }
    most = fmax(most, __shfl_xor(most, 1));
    most = fmax(most, __shfl_xor(most, 2));
    const int e = (int)((__double_as_longlong(most) >> 52) & 0x7ff) - 1023;  // floor(log2), or far below
    byte = quad_max(!finite) ? 255u : e < -125 ? 0u : (uint32_t)(e + 125);
    const double unit = __longlong_as_double((int64_t)(1023 + 127 - (int)byte) << 52);  // 2^(127 - byte)
    code = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double a = fabs(v[j]) * unit;
      uint32_t one = (uint32_t)(a > 0.25) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0);
      one |= signbit(v[j]) ? 8u : 0u;
      code |= one << (4 * j);
    }
    if (byte == 255u) code = 0;
  }
  reinterpret_cast<uint32_t*>(codes)[i] = code;
  if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
}

// ------------------------------------------------------------------------------------------------ the weights' layout
// The matrix row that row `r` of tile `t` holds. `gated_inter` (a gated pair [up; gate] of that many rows each): up and gate
// tiles alternate, so that two consecutive tiles are the two factors of 32 consecutive columns of their product.
__device__ __forceinline__ int64_t mx_source_row(int t, int r, int gated_inter) {
  return gated_inter ? (int64_t)(t & 1) * gated_inter + (t >> 1) * MX_ROWS + r : (int64_t)t * MX_ROWS + r;
}

// Row-major codes and scales of `matrices` matrices -> their tile layouts (UNPACK: the way back). A thread a (tile, lane): 16
// bytes of codes and one scale. Once a matrix, and for activations that come rounded into a product on the ring; 25600 x 5120 28 us, 5.0 TB/s read and written.
template <bool UNPACK>
__global__ __launch_bounds__(256) void mx_repack_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t n, int k, int gated_inter,
                                                        uint8_t* __restrict__ tiled) {
  const MxLayout at(n, k);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, lane_chunks = (int64_t)at.tiles * at.quads * 4 * 64;
  if (i >= lane_chunks) return;
  codes += (int64_t)blockIdx.y * n * (k / 2);
  scales += (int64_t)blockIdx.y * n * (k / 32);
  tiled += (int64_t)blockIdx.y * at.bytes();
  const int lane = (int)(i & 63);
  const uint32_t tc = (uint32_t)(i >> 6);  // below 2^26
  const int t = (int)(tc / (uint32_t)(at.quads * 4)), c = (int)tc - t * at.quads * 4;  // chunks past the last only have scales
  const int64_t row = mx_source_row(t, lane & 31, gated_inter);
  const int group = 2 * c + (lane >> 5);
  const bool in = row < n && group < k / 32;
  uint8_t* scale_at = tiled + at.codes() + ((int64_t)t * at.quads + (c >> 2)) * 256 + lane * 4 + (c & 3);
  i32x4_t* code_at = reinterpret_cast<i32x4_t*>(tiled + (((int64_t)t * at.chunks + c) * 64 + lane) * 16);
  if (UNPACK) {
    if (!in) return;
    scales[row * (k / 32) + group] = *scale_at;
    *reinterpret_cast<i32x4_t*>(codes + row * (k / 2) + 16 * group) = *code_at;
  } else {
    *scale_at = in ? scales[row * (k / 32) + group] : 0;
    if (c < at.chunks) *code_at = in ? *reinterpret_cast<const i32x4_t*>(codes + row * (k / 2) + 16 * group) : i32x4_t{0, 0, 0, 0};
  }
}

// ------------------------------------------------------------------------------------------------ the linear
struct MxLinear {
  const void* x;            // [m, k] values, or row-major codes
  const uint8_t* x_scales;  // row-major scales of the codes
  const uint8_t* w;         // tile layout
  void* y;
  int64_t m, n;
  int k, waves;
};

// Few rows: a workgroup NT tiles of weight rows, its wavefronts the chunks of K. The first weights are asked for, then the workgroup puts
// the activations into LDS, rounded on the way: each workgroup all of them, which costs less than a launch. (32 x 32 x 64 products of which up to 31 columns are
// idle: the matrix cores have nothing else to do.) One row of 5120 x 5120 5.4 us (on cold weights 6.5): latency of the launch, the activations, ten chunks of weights a wavefront
// and the join. Eight rows of 25600 x 5120 14.2 us where part of the weights are in the Infinity Cache, 17.6 on cold ones: 4.0 TB/s.
template <typename T, typename Y, int NT, int RUN>
__global__ __launch_bounds__(512) void mx_few_rows_kernel(MxLinear p) {
  extern __shared__ f32x4_t part[];  // the activations, then [waves][NT * 4][64]
  constexpr int AT_ONCE = std::is_same_v<T, float> ? 4 : 8;
  MxStream<NT, RUN> s;
  const MxLayout at(p.n, p.k);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t0 = blockIdx.x * NT, groups = p.k / MX_GROUP;
  const int64_t row0 = (int64_t)blockIdx.y * MX_ROWS;
  const int rows = (int)min((int64_t)MX_ROWS, p.m - row0);
  const MxActs acts(part, rows, p.k);
  // Loads return in order: the first activations are asked for ahead of the weights, or they would stand behind all of them while nothing else is on its way.
  if constexpr (std::is_same_v<T, uint8_t>) {
    const int all = rows * groups;
    const uint8_t *x = static_cast<const uint8_t*>(p.x) + row0 * (p.k / 2), *x_scales = p.x_scales + row0 * groups;
    auto source = [&](int i, i32x4_t& code, uint32_t& scale) {
      code = *reinterpret_cast<const i32x4_t*>(x + 16 * (int64_t)i);
      scale = x_scales[i];
    };
    auto put = [&](int i, const i32x4_t& code, uint32_t scale) {
      const int r = i / groups, at = (i - r * groups) * rows + r;
      acts.codes[at] = code;
      acts.scales[at] = (uint8_t)scale;
    };
    i32x4_t code[AT_ONCE];
    uint32_t scale[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; j++) source(min((int)(threadIdx.x + j * blockDim.x), all - 1), code[j], scale[j]);
    __builtin_amdgcn_sched_barrier(0);
    s.begin(p.w, at, t0, wave, p.waves);
#pragma unroll
    for (int j = 0; j < AT_ONCE; j++)
      if (threadIdx.x + j * blockDim.x < all) put(threadIdx.x + j * blockDim.x, code[j], scale[j]);
    for (int i = threadIdx.x + AT_ONCE * blockDim.x; i < all; i += blockDim.x) {
      source(i, code[0], scale[0]);
      put(i, code[0], scale[0]);
    }
  } else {
    const int all = rows * groups * 4;  // eight values from 8 i of the contiguous rows a lane
    const uint32_t inverse = 0xffffffffu / (uint32_t)groups + 1u;  // i / groups = the upper half of i inverse: i below 32 groups, groups below 2^13
    const T* x = static_cast<const T*>(p.x) + row0 * p.k;
    auto source = [&](Mx8<T>& v, int i) { v.load(x + 8 * (int64_t)min(i, all - 1)); };
    auto put = [&](int i, const Mx8<T>& v) {
      const int r = groups == 1 ? i >> 2 : (int)__umulhi((uint32_t)i >> 2, inverse);
      if (i < all) acts.put(r, (i >> 2) - r * groups, i & 3, v);
    };
    Mx8<T> v[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; j++) source(v[j], threadIdx.x + j * blockDim.x);
    __builtin_amdgcn_sched_barrier(0);
    s.begin(p.w, at, t0, wave, p.waves);
#pragma unroll
    for (int j = 0; j < AT_ONCE; j++) put(threadIdx.x + j * blockDim.x, v[j]);
    for (int i0 = threadIdx.x + AT_ONCE * blockDim.x; i0 < all; i0 += AT_ONCE * blockDim.x) {
#pragma unroll
      for (int j = 0; j < AT_ONCE; j++) source(v[j], i0 + j * blockDim.x);
#pragma unroll
      for (int j = 0; j < AT_ONCE; j++) put(i0 + j * blockDim.x, v[j]);
    }
  }
  __syncthreads();
  s.run(acts);
  mx_hand_over<NT>(part, s.acc);
  for (int i = threadIdx.x; i < NT * 256; i += blockDim.x) {
    const f32x4_t sum = mx_joined<NT>(part, p.waves, i);
    const int l = i & 63, q = (i >> 6) & 3, t = t0 + (i >> 8);
    const int64_t row = row0 + (l & 31), n = (int64_t)t * MX_ROWS + 8 * q + 4 * (l >> 5);
    if (row < p.m && n < p.n) mx_store4<Y>(static_cast<Y*>(p.y) + row * p.n + n, sum, p.n - n, p.n % 4 == 0);
  }
}

// More rows, on the ring (mxfp4_ring.hpp). Many take 2 x 2 wavefronts of 4 x 4 tiles: 256 accumulator registers, one wavefront a SIMD, and a matrix
// instruction's operands come from LDS at half of the 128 bytes a cycle that it gives, what is asked for at a quarter. 2048 rows of 25600 x 5120:
// three rounds of the device in 122 us, 4.2 PFLOP/s (the products alone 6.6 on random data, at the clock that the card's power leaves them;
// without any loads into LDS 15 % less time, with loads from the L2 alone 6 %), the last columns 17. Up to 128 rows a wavefront has all of
// the workgroup's rows and its own weights: 77 rows 15.3 us, the weights at 4.6 TB/s, half of them from the Infinity Cache; on cold ones 20.9.
struct MxTiles {
  const uint8_t* a;
  const uint8_t* w;
  void* y;               // K shared by gridDim.y workgroups: their FP32 sums [shares, m, n]
  int64_t m, n;
  int k, rows_of_tiles;  // workgroups along m
  int first, last;       // the tiles of weight rows that this launch covers
};
template <typename Y, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(64 * WM * WN, 1) void mx_ring_kernel(MxTiles p) {
  using Ring = MxRing<WM, WN, MT, NT>;
  __shared__ i32x4_t buf0[Ring::BUFFER], buf1[Ring::BUFFER], buf2[Ring::BUFFER], buf3[Ring::BUFFER];
  const MxLayout la(p.m, p.k), lw(p.n, p.k);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  // consecutive workgroups go to the eight dies in turn: each die walks a run of tiles, rows fastest, so that its L2 keeps a run of weights
  const int total = gridDim.x, per = (total + 7) / 8, die = blockIdx.x % 8, whole = total % 8 ? total % 8 : 8;  // the first `whole` dies have `per` workgroups, the others one less
  const int at = die * per - (die > whole ? die - whole : 0) + (int)(blockIdx.x / 8);
  const int a0 = at % p.rows_of_tiles * Ring::TA, b0 = p.first + at / p.rows_of_tiles * Ring::TB;
  const int quads = (la.chunks + 3) / 4, q0 = (int)((int64_t)quads * blockIdx.y / gridDim.y), q1 = (int)((int64_t)quads * (blockIdx.y + 1) / gridDim.y);
  Y* y = static_cast<Y*>(p.y) + (int64_t)blockIdx.y * p.m * p.n;
  const MxOperand a{p.a + (int64_t)a0 * la.chunks * 1024, p.a + la.codes() + (int64_t)a0 * la.quads * 256, la.tiles - a0};
  const MxOperand b{p.w + (int64_t)b0 * lw.chunks * 1024, p.w + lw.codes() + (int64_t)b0 * lw.quads * 256, lw.tiles - b0};
  f32x16_t acc[MT][NT];
  Ring::run(buf0, buf1, buf2, buf3, a, b, la.chunks, la.quads, q0, q1, acc);
  i32x4_t* place = wave == 0 ? buf0 : wave == 1 ? buf1 : wave == 2 ? buf2 : buf3;  // each wavefront takes one of the ring's buffers
#pragma unroll
  for (int i = 0; i < MT; i++) {
    const int64_t row0 = (int64_t)(a0 + wm * MT + i) * MX_ROWS;
    mx_store_rows<Y, NT>(place, p.n, (int64_t)(b0 + wn * NT) * MX_ROWS, acc[i], [&](int r) { return row0 + r < p.m ? y + (row0 + r) * p.n : nullptr; });
  }
}

// x [rows, k] rounded into the tile layout, a wavefront a tile: it reads 32 rows of 128 (FP32: 256) bytes, a lane its group,
// whose codes are the 16 bytes that it owns. Rows past the last are left as they are (their results are not stored). 2048 x 5120 of BF16 7.6 us, 3.5 TB/s:
// a lane's 64 bytes are a read of their own.
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_tiles_kernel(const T* __restrict__ x, int64_t rows, int k, uint8_t* __restrict__ tiled) {
  const MxLayout at(rows, k);
  const int lane = threadIdx.x & 63, all = at.quads * 4;  // K's chunks in whole quads: those past the last only have scales
  const uint32_t i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // below 2^26
  const int64_t t = i / (uint32_t)all;
  const int c = (int)(i - (uint32_t)t * all), group = 2 * c + (lane >> 5);
  const int64_t row = t * MX_ROWS + (lane & 31);
  if (row >= rows) return;
  uint32_t byte = 0;
  i32x4_t code = {0, 0, 0, 0};
  if (group < k / MX_GROUP) {
    MxGroup<T> v;
    v.load(x + row * k + MX_GROUP * (int64_t)group);
    code = v.codes(byte);
  }
  if (c < at.chunks) *reinterpret_cast<i32x4_t*>(tiled + ((t * at.chunks + c) * 64 + lane) * 16) = code;
  tiled[at.codes() + (t * at.quads + (c >> 2)) * 256 + lane * 4 + (c & 3)] = (uint8_t)byte;
}

// The shares' sums added in their order and rounded, four columns a thread (`whole`) or one. 64 rows of 5120 x 5120, five shares: ring 8.2 us, this 3.1.
template <typename Y>
__global__ __launch_bounds__(256) void mx_join_kernel(const float* __restrict__ sums, int64_t count, int shares, int whole, Y* __restrict__ y) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (whole) {
    if (4 * i >= count) return;
    f32x4_t sum = reinterpret_cast<const f32x4_t*>(sums)[i];
    for (int s = 1; s < shares; s++) sum += *reinterpret_cast<const f32x4_t*>(sums + s * count + 4 * i);
    mx_store4<Y>(y + 4 * i, sum, 4, true);
  } else {
    if (i >= count) return;
    float sum = sums[i];
    for (int s = 1; s < shares; s++) sum += sums[s * count + i];
    y[i] = mx_out<Y>(sum);
  }
}

// How a call is made.
struct MxPlan {
  enum { FEW_ROUNDING, FEW, RING } way;
  int mt, shares;    // RING: row tiles a wavefront (4 wide: 4 of the 2 x 2 form; 2 wide: its half), workgroups that share K
  bool square;       // RING: the 2 x 2 forms
  size_t tiles, bytes;  // workspace: of the activations, of all
};
// Few rows (their activations fit LDS): one tile of weight rows a workgroup, or two, which share a workgroup's activations, where that does not give the busiest
// compute unit more tiles. us in a graph on cold weights, eight rows of 5120 k, one and two: 256 tiles 8.8 and 9.8, 257 10.7 and 9.8, 384 11.4 and 11.2, 512 12.5
// and 12.6, 513 14.1 and 15.0, 640 15.7 and 17.5, 768 16.5 and 17.9, 769 18.1 and 17.9, 800 19.9 and 18.0, 1024 21.3 and 19.4, 1280 25.6 and 26.0, 1600 31.9 and
// 32.5; 32 rows of 1024 k, 320 tiles, 7.1 and 5.9; 128 rows of 4000 x 832 in passes 6.3 and 5.5, 160 rows 7.6 and 7.7.
constexpr int MX_DEVICE = 256;  // compute units
static bool two_tiles(int64_t tiles, int64_t passes) {
  auto busiest = [&](int64_t workgroups) { return (workgroups * passes + MX_DEVICE - 1) / MX_DEVICE; };
  return 2 * busiest((tiles + 1) / 2) <= busiest(tiles);
}
// The rounding rides in that launch, each workgroup all rows, while they are not more than so many values; past it the rounding is a launch of its own. us in a graph and
// called one by one, inside and ahead: 20 rows of 4000 x 4096 (80 K values) 9.4 and 8.7, 8.6 and 11.9; 31 rows of it (124 K) 11.5 and 10.7, 9.0 and 11.7. More tiles
// than compute units, cold weights, 5120 k: two tiles a workgroup, 320 tiles, 12 rows (60 K) 11.2 and 11.0, 11.2 and 10.7, 16 rows (80 K) 12.5 and 12.3, 11.4 and 10.8; 800
// tiles 18.7 and 18.4, 18.9 and 18.3, then 21.1 and 20.7, 19.2 and 18.7; one tile, 640, 8 rows (40 K) 15.7 and 15.3, 16.2 and 15.6, 12 rows 17.3 and 17.0, 16.7 and 16.1.
static int64_t round_values(int64_t tiles) { return (tiles <= MX_DEVICE ? 80 : two_tiles(tiles, 1) ? 64 : 48) * 1024; }
// Past that size a matrix of more than four tiles a compute unit goes to the ring. us as above, ahead and ring, 5120 k: 16 rows of 800 tiles 19.2 and 18.7, 20.6 and 20.0, 24 rows
// 19.8 and 19.1, 20.9 and 20.4; 16 rows of 1280 26.5 and 25.5, 26.7 and 25.7, 24 rows 29.1 and 28.2, 26.9 and 26.0; of 1600 33.0 and 31.8, 31.2 and 30.1.
constexpr int MX_RING_TILES = 4 * MX_DEVICE;
// More rows of a small matrix are passes of 32 rows beside one another, which read its weights again: one launch where the ring takes two, or three with K shared.
// Up to MX_PASS_VALUES values a pass, and MX_PASSES_WORK of tiles x passes x k. us as above, passes and ring: 128 rows of 4000 x 832 (416 K) 5.6 and 6.9, 8.1 and 10.7; 64
// rows of 4000 x 1664 (416 K) 7.2 and 7.2, 10.5 and 14.2; 128 rows of 1000 x 4000 (512 K) 10.4 and 10.3, 11.5 and 14.2; 256 rows of 12000 x 256 (768 K) 9.2 and 9.1, 7.2
// and 10.8.
constexpr int64_t MX_PASS_VALUES = 128 * 1024, MX_PASSES_WORK = 768 * 1024;
static MxPlan plan_of(int64_t m, int64_t n, int k, int x_type) {
  const MxLayout rows(m, k), w(n, k);
  MxPlan p{};
  const size_t acts = MxActs::bytes(m, k);
  const bool small = m * k <= round_values(w.tiles);
  if (m > MX_ROWS && (int64_t)MX_ROWS * k <= MX_PASS_VALUES && (int64_t)rows.tiles * w.tiles * k <= MX_PASSES_WORK) {
    p.way = MxPlan::FEW_ROUNDING;
    return p;
  }
  if (m <= MX_ROWS && acts <= (w.tiles <= 256 ? 144 : 64) * 1024 && (small || w.tiles <= MX_RING_TILES)) {
    const bool rounds = x_type != HB_MXFP4 && !small;
    p.way = rounds ? MxPlan::FEW : MxPlan::FEW_ROUNDING;
    p.tiles = p.bytes = rounds ? (size_t)m * (k / 2 + k / MX_GROUP) : 0;
    return p;
  }
  p.way = MxPlan::RING;
  p.square = m > 128;
  auto groups = [&](int mt) {
    const int64_t high = p.square ? 2 * mt : mt, wide = p.square ? 2 * mt : 4;
    return (rows.tiles + high - 1) / high * ((w.tiles + wide - 1) / wide);
  };
  // 256 x 256 a workgroup where such tiles fill the device well enough, and past a round of it where padding the rows to 256 costs no more than an
  // eighth. us, large and small tiles, 5120 k: 2048 rows of 5120 42 and 45, of 25600 145 and 181; 777 rows of 25600 78 and 74; 1100 rows 88 and 96.
  p.mt = !p.square ? rows.tiles : groups(4) >= 160 && (groups(4) <= MX_DEVICE || 32 * groups(4) <= 9 * groups(2)) ? 4 : 2;
  // K is shared where the tiles leave half the device idle, by up to eight workgroups of at least eight steps
  p.shares = (int)std::max<int64_t>(1, std::min<int64_t>({MX_DEVICE / groups(p.mt), rows.quads / 4, 8}));
  p.tiles = (size_t)(rows.bytes() + 255) / 256 * 256;
  p.bytes = p.tiles + (p.shares > 1 ? (size_t)p.shares * m * n * sizeof(float) : 0);
  return p;
}

template <typename Y, int WM, int WN, int MT, int NT>
static int launch_ring(MxTiles p, const MxPlan& plan, float* sums, hipStream_t stream) {
  const MxLayout la(p.m, p.k), lw(p.n, p.k);
  if (!p.last) p.last = lw.tiles;
  p.rows_of_tiles = (la.tiles + WM * MT - 1) / (WM * MT);
  const dim3 grid((unsigned)(p.rows_of_tiles * ((p.last - p.first + WN * NT - 1) / (WN * NT))), (unsigned)plan.shares);
  if (plan.shares == 1) {
    HB_LAUNCH((mx_ring_kernel<Y, WM, WN, MT, NT>), grid, dim3(64 * WM * WN), 0, stream, p);
    return HB_OK;
  }
  Y* y = static_cast<Y*>(p.y);
  p.y = sums;
  HB_LAUNCH((mx_ring_kernel<float, WM, WN, MT, NT>), grid, dim3(64 * WM * WN), 0, stream, p);
  const int64_t count = p.m * p.n;
  const int whole = count % 4 == 0, each = whole ? 1024 : 256;
  HB_LAUNCH((mx_join_kernel<Y>), dim3((unsigned)((count + each - 1) / each)), dim3(256), 0, stream, sums, count, plan.shares, whole, y);
  return HB_OK;
}

template <typename T, typename Y, int NT, int RUN>
static int launch_few(const MxLinear& p, const MxLayout& at, hipStream_t stream) {
  const size_t lds = std::max(MxActs::bytes(std::min<int64_t>(p.m, MX_ROWS), p.k), (size_t)p.waves * NT * 4096);
  if (lds > 64 * 1024) {
    // set for a device once: the attribute is the loaded kernel's, and each device has its own
    static std::atomic<uint64_t> raised{0};
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess) return HB_ELAUNCH;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (!(raised.load(std::memory_order_acquire) & bit)) {
      if (hipFuncSetAttribute(reinterpret_cast<const void*>(&mx_few_rows_kernel<T, Y, NT, RUN>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) return HB_ELAUNCH;
      raised.fetch_or(bit, std::memory_order_release);
    }
  }
  HB_LAUNCH((mx_few_rows_kernel<T, Y, NT, RUN>), dim3((unsigned)((at.tiles + NT - 1) / NT), (unsigned)((p.m + MX_ROWS - 1) / MX_ROWS)), dim3(64 * p.waves), lds, stream, p);
  return HB_OK;
}

template <typename T, typename Y>
static int launch_linear(MxLinear p, uint8_t* workspace, hipStream_t stream) {
  constexpr bool held = std::is_same_v<T, uint8_t>;
  const MxPlan plan = plan_of(p.m, p.n, p.k, held ? HB_MXFP4 : HB_F32);
  if (plan.way == MxPlan::FEW) {
    const int64_t lanes = p.m * (p.k / 8);
    if constexpr (!held) {
      uint8_t* scales = workspace + p.m * (p.k / 2);
      HB_LAUNCH((mx_quantize_kernel<T>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, stream, static_cast<const T*>(p.x), lanes, workspace, scales);
      p.x = workspace;
      p.x_scales = scales;
    }
  }
  if (plan.way != MxPlan::RING) {
    const MxLayout at(p.n, p.k);
    p.waves = std::min(at.chunks, 8);
    auto few = [&](auto* type) {
      using X = std::remove_pointer_t<decltype(type)>;
      if (two_tiles(at.tiles, (p.m + MX_ROWS - 1) / MX_ROWS)) return launch_few<X, Y, 2, 4>(p, at, stream);
      return at.chunks >= 32 ? launch_few<X, Y, 1, 4>(p, at, stream) : launch_few<X, Y, 1, 1>(p, at, stream);
    };
    return plan.way == MxPlan::FEW ? few((uint8_t*)nullptr) : few((T*)nullptr);
  }
  if constexpr (held) {
    if (int e = hb_mxfp4_repack(p.x, p.x_scales, 1, p.m, p.k, 0, workspace, stream)) return e;
  } else {
    const MxLayout rows(p.m, p.k);
    HB_LAUNCH((mx_quantize_tiles_kernel<T>), dim3((unsigned)((int64_t)rows.tiles * rows.quads)), dim3(256), 0, stream, static_cast<const T*>(p.x), p.m, p.k, workspace);
  }
  MxTiles q{workspace, p.w, p.y, p.m, p.n, p.k, 0, 0, 0};
  float* sums = reinterpret_cast<float*>(workspace + plan.tiles);
  if (plan.square && plan.mt == 4) {
    // The last columns of workgroups, those past whole rounds of the device, as four workgroups of 128 x 128 each in a launch behind: a
    // round of a few large ones costs as much as a full one. 2048 rows of 25600 x 5120 (3.125 rounds): 162 us as one launch, 152 so.
    const MxLayout rows(p.m, p.k), w(p.n, p.k);
    const int high = (rows.tiles + 7) / 8, wide = (w.tiles + 7) / 8, whole = high * wide / MX_DEVICE * MX_DEVICE / high;
    const int rest = (high * wide - whole * high) * 4;
    if (whole && rest && rest <= 2 * MX_DEVICE) {
      q.last = whole * 8;
      if (int e = launch_ring<Y, 2, 2, 4, 4>(q, plan, sums, stream)) return e;
      q.first = whole * 8;
      q.last = w.tiles;
      return launch_ring<Y, 2, 2, 2, 2>(q, plan, sums, stream);
    }
  }
  if (plan.square) return plan.mt == 4 ? launch_ring<Y, 2, 2, 4, 4>(q, plan, sums, stream) : launch_ring<Y, 2, 2, 2, 2>(q, plan, sums, stream);
  switch (plan.mt) {
    case 1: return launch_ring<Y, 1, 4, 1, 1>(q, plan, sums, stream);
    case 2: return launch_ring<Y, 1, 4, 2, 1>(q, plan, sums, stream);
    case 3: return launch_ring<Y, 1, 4, 3, 1>(q, plan, sums, stream);
  }
  return launch_ring<Y, 1, 4, 4, 1>(q, plan, sums, stream);
}

template <typename F>
static int by_type(int type, F&& f) {
  switch (type) {
    case HB_BF16: return f((__bf16*)nullptr);
    case HB_F16: return f((_Float16*)nullptr);
    case HB_F32: return f((float*)nullptr);
  }
  return HB_EINVAL;
}
// launch(first row, rows): a launch holds 2^32 threads, so 2^31 lanes of eight values at a time.
template <typename F>
static void by_rows(int64_t rows, int lanes, F&& launch) {
  const int64_t most = std::max<int64_t>(1, ((int64_t)1 << 31) / lanes);
  for (int64_t lo = 0; lo < rows; lo += most) launch(lo, std::min(most, rows - lo));
}

}  // namespace hb

using namespace hb;

extern "C" int hb_mxfp4_quantize(const void* x, int type, int64_t rows, int k, void* codes, void* scales, void* stream) {
  if (!x || !codes || !scales) return HB_ENULL;
  if (rows <= 0 || k <= 0 || k % MX_GROUP || rows > (int64_t)1 << 40 || rows * (k / 8) > (int64_t)255 << 31) return HB_EINVAL;
  if (!aligned(x, 16) || !aligned(codes, 16)) return HB_EINVAL;
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_rows(rows, k / 8, [&](int64_t lo, int64_t count) {
      const int64_t lanes = count * (k / 8);
      HB_LAUNCH((mx_quantize_kernel<T>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, as_stream(stream), static_cast<const T*>(x) + lo * k, lanes,
                static_cast<uint8_t*>(codes) + lo * (k / 2), static_cast<uint8_t*>(scales) + lo * (k / MX_GROUP));
    });
    return launch_status();
  });
}

extern "C" int hb_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int k, int type, void* out, void* stream) {
  if (!codes || !scales || !out) return HB_ENULL;
  if (rows <= 0 || k <= 0 || k % MX_GROUP || rows > (int64_t)1 << 40 || rows * (k / 8) > (int64_t)255 << 31) return HB_EINVAL;
  if (!aligned(codes, 16) || !aligned(out, 16)) return HB_EINVAL;
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_rows(rows, k / 8, [&](int64_t lo, int64_t count) {
      const int64_t lanes = count * (k / 8);
      HB_LAUNCH((mx_dequantize_kernel<T>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, as_stream(stream), static_cast<const uint8_t*>(codes) + lo * (k / 2),
                static_cast<const uint8_t*>(scales) + lo * (k / MX_GROUP), lanes, static_cast<T*>(out) + lo * k);
    });
    return launch_status();
  });
}

extern "C" int hb_silu_mul_quant_mxfp4(const void* gate_up, int type, int64_t rows, int half, int pairs, void* codes, void* scales, void* stream) {
  if (!gate_up || !codes || !scales) return HB_ENULL;
  if (rows <= 0 || half <= 0 || half % MX_GROUP || half > 1 << 29 || pairs < 0 || (pairs && (pairs % 8 || half % pairs)) || rows > (int64_t)1 << 40 ||
      rows * (half / 8) > (int64_t)255 << 31)
    return HB_EINVAL;
  if (!aligned(gate_up, 16) || !aligned(codes, 16)) return HB_EINVAL;
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_rows(rows, half / 8, [&](int64_t lo, int64_t count) {
      HB_LAUNCH((mx_silu_quantize_kernel<T>), dim3((unsigned)((count * (half / 8) + 255) / 256)), dim3(256), 0, as_stream(stream),
                static_cast<const T*>(gate_up) + lo * 2 * half, count, half, pairs, static_cast<uint8_t*>(codes) + lo * (half / 2),
                static_cast<uint8_t*>(scales) + lo * (half / MX_GROUP));
    });
    return launch_status();
  });
}

constexpr int64_t MX_MOST_ROWS = (int64_t)1 << 24;
// Sizes that the layout's indices and a launch's 2^32 threads hold (a matrix of 2^37 values).
static bool layout_holds(int64_t n, int k) { return n > 0 && k > 0 && k <= 1 << 23 && k % MX_GROUP == 0 && n <= (int64_t)1 << 30 && (n + 31) / 32 * ((k + 511) / 512) < (int64_t)1 << 23; }

extern "C" size_t hb_mxfp4_tiled_bytes(int64_t n, int k) { return layout_holds(n, k) ? (size_t)MxLayout(n, k).bytes() : 0; }

static int repack(bool unpack, void* codes, void* scales, int matrices, int64_t n, int k, int gated, void* tiled, void* stream) {
  if (!codes || !scales || !tiled) return HB_ENULL;
  if (!layout_holds(n, k) || matrices <= 0 || matrices > 65535 || (gated && n % 64)) return HB_EINVAL;
  if (!aligned(codes, 16) || !aligned(tiled, 16)) return HB_EINVAL;
  const MxLayout at(n, k);
  const dim3 grid((unsigned)(((int64_t)at.tiles * at.quads * 4 * 64 + 255) / 256), (unsigned)matrices);
  const int inter = gated ? (int)(n / 2) : 0;
  if (unpack) {
    HB_LAUNCH((mx_repack_kernel<true>), grid, dim3(256), 0, as_stream(stream), static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), n, k, inter,
              static_cast<uint8_t*>(tiled));
  } else {
    HB_LAUNCH((mx_repack_kernel<false>), grid, dim3(256), 0, as_stream(stream), static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), n, k, inter,
              static_cast<uint8_t*>(tiled));
  }
  return launch_status();
}
extern "C" int hb_mxfp4_repack(const void* codes, const void* scales, int matrices, int64_t n, int k, int gated, void* tiled, void* stream) {
  return repack(false, const_cast<void*>(codes), const_cast<void*>(scales), matrices, n, k, gated, tiled, stream);
}
extern "C" int hb_mxfp4_unpack(const void* tiled, int matrices, int64_t n, int k, int gated, void* codes, void* scales, void* stream) {
  return repack(true, codes, scales, matrices, n, k, gated, const_cast<void*>(tiled), stream);
}

extern "C" size_t hb_mxfp4_linear_workspace_bytes(int64_t m, int64_t n, int k, int x_type) {
  return m > 0 && m <= MX_MOST_ROWS && layout_holds(n, k) && layout_holds(m, k) ? plan_of(m, n, k, x_type).bytes : 0;
}

extern "C" int hb_mxfp4_linear(const void* x, const void* x_scales, int x_type, int64_t m, const void* tiled, int64_t n, int k, void* y, int y_type,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (!x || !tiled || !y || (x_type == HB_MXFP4 && !x_scales)) return HB_ENULL;
  if (m <= 0 || m > MX_MOST_ROWS || !layout_holds(n, k) || y_type < HB_BF16 || y_type > HB_F32 || x_type < HB_BF16 || x_type > HB_MXFP4) return HB_EINVAL;
  if (x_type != HB_MXFP4 && x_type != y_type) return HB_EINVAL;
  if (!aligned(x, 16) || !aligned(tiled, 16) || !aligned(y, 16)) return HB_EINVAL;
  const size_t need = hb_mxfp4_linear_workspace_bytes(m, n, k, x_type);
  if (need && !workspace) return HB_ENULL;
  if (!aligned(workspace, 16) || !layout_holds(m, k)) return HB_EINVAL;
  if (workspace_bytes < need) return HB_EWORKSPACE;
  const MxLinear p{x, static_cast<const uint8_t*>(x_scales), static_cast<const uint8_t*>(tiled), y, m, n, k, 0};
  const int code = by_type(y_type, [&](auto* t) {
    using Y = std::remove_pointer_t<decltype(t)>;
    return x_type == HB_MXFP4 ? launch_linear<uint8_t, Y>(p, static_cast<uint8_t*>(workspace), as_stream(stream)) : launch_linear<Y, Y>(p, static_cast<uint8_t*>(workspace), as_stream(stream));
  });
  return code ? code : launch_status();
}
