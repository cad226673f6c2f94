// The microscaled four-bit format: rounding to it (alone, and behind a gated activation), the values back, the weights' tile
// layout, and the linear.
#include <algorithm>

#include "mxfp4.hpp"
#include "stream_common.hpp"

namespace hb {

// ------------------------------------------------------------------------------------------------ rounding, and back
// x [rows, k] -> codes [rows, k / 2], scales [rows, k / 32]. A lane takes eight consecutive values, four lanes a group: loads and
// stores of a wavefront are consecutive, and the group's largest magnitude is two lane exchanges. Memory bound.
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

// The values that codes and scales stand for, eight a lane.
template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t lanes, T* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= lanes) return;
  mx_values(reinterpret_cast<const uint32_t*>(codes)[i], mx_scale_value(scales[i >> 2]), out + 8 * i);
}

// silu(g) u in FP32, g not below -80: exp2 of -g log2(e) as a product's two halves, one reciprocal. Off by less than
// MX_SILU_OFF of its value: an ulp each for exp2 and the reciprocal, half of one for the correction, the sum and the two products.
constexpr float MX_SILU_OFF = 0x1p-20f;  // (twice the sum of those)
__device__ __forceinline__ float mx_silu_mul(float g, float u) {
  constexpr float L = 1.44269504088896340736f, L_LO = (float)(1.44269504088896340736 - (double)1.44269504088896340736f);
  const float z = __builtin_fminf(__builtin_fmaxf(g, -80.0f), 200.0f);  // (past 200 exp2 is 0 all the same)
  const float hi = -z * L, lo = __builtin_fmaf(-z, L, -hi) - z * L_LO;
  const float e = __builtin_amdgcn_exp2f(hi);
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_fmaf(e, 0.693147180559945309f * lo, e)) * u;
}

// silu(gate) * up of [rows, 2 half] rounded to the format in one pass; gate | up, or both in alternating blocks of `pairs` columns.
// A product within FP32's error of a border between two codes, or a group whose largest is that near a power of two, would
// round by that error: such a group (a few in a million values) is computed again in 64 bits, and so is one
// whose products leave FP32's comfortable range.
template <typename T>
__global__ __launch_bounds__(256) void mx_silu_quantize_kernel(const T* __restrict__ x, int64_t rows, int half, int pairs, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per_row = half >> 3;
  if (i >= rows * per_row) return;  // whole groups leave together: half is a multiple of 32
  const int64_t r = i / per_row;
  const int c = 8 * (int)(i - r * per_row);
  const int gate_at = pairs ? (c / pairs) * 2 * pairs + c % pairs : c, up_at = pairs ? gate_at + pairs : half + c;
  Mx8<T> g, u;
  g.load(x + r * 2 * half + gate_at);
  u.load(x + r * 2 * half + up_at);
  Mx8<float> p, q;
  bool far = false;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    p.v[j >> 2][j & 3] = mx_silu_mul(g.at(j), u.at(j));
    far |= g.at(j) < -80.0f;
  }
  const uint32_t top = quad_max(p.amax());
  uint32_t byte = mx_scale_byte(top);
  const float s = mx_scale_value(byte);
#pragma unroll
  for (int j = 0; j < 8; j++) {
    q.v[j >> 2][j & 3] = p.v[j >> 2][j & 3] * (1.0f + MX_SILU_OFF);
    p.v[j >> 2][j & 3] *= 1.0f - MX_SILU_OFF;
  }
  uint32_t code = p.codes(s);
  constexpr uint32_t OFF = 16;  // ulps of MX_SILU_OFF
  far |= code != q.codes(s);
  far |= byte != 255u && (((top - OFF) ^ (top + OFF)) >> 23) != 0 && top != 0;
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
// tiles alternate, so that four consecutive tiles are the two factors of 32 consecutive columns of their product.
__device__ __forceinline__ int64_t mx_source_row(int t, int r, int gated_inter) {
  return gated_inter ? (int64_t)(t & 1) * gated_inter + (t >> 1) * 16 + r : (int64_t)t * 16 + r;
}

// Row-major codes and scales of `matrices` matrices -> their tile layouts (UNPACK: the way back). A thread a (tile, lane): 16
// bytes of codes and one scale.
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
  const int64_t tc = i >> 6;
  const int t = (int)(tc / (at.quads * 4)), c = (int)(tc - (int64_t)t * at.quads * 4);  // chunks past the last only have scales
  const int64_t row = mx_source_row(t, lane & 15, gated_inter);
  const int group = 4 * c + (lane >> 4);
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

// A row's group as the product's operand: rounded on the way (T: a value type), or read (uint8_t: row-major codes).
template <typename T>
__device__ __forceinline__ i32x4_t mx_acts(const void* x, const uint8_t*, int64_t row, int k, int group, uint32_t& byte) {
  return mx_round_group<T>(static_cast<const T*>(x) + row * k + 32 * (int64_t)group, byte);
}
template <>
__device__ __forceinline__ i32x4_t mx_acts<uint8_t>(const void* x, const uint8_t* scales, int64_t row, int k, int group, uint32_t& byte) {
  byte = scales[row * (k / 32) + group];
  return *reinterpret_cast<const i32x4_t*>(static_cast<const uint8_t*>(x) + row * (k / 2) + 16 * (int64_t)group);
}

// Up to sixteen rows: a workgroup NT tiles of weight rows, its wavefronts the chunks of K, their sums added through LDS in
// wavefront order.
template <typename T, typename Y, int NT>
__global__ __launch_bounds__(1024) void mx_few_rows_kernel(MxLinear p) {
  extern __shared__ f32x4_t part[];  // [waves][NT][64]
  const MxLayout at(p.n, p.k);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.x * NT, groups = p.k / 32;
  const int64_t row0 = (int64_t)blockIdx.y * 16;
  const int c0 = (int)((int64_t)at.chunks * wave / p.waves), c1 = (int)((int64_t)at.chunks * (wave + 1) / p.waves);
  const bool real = row0 + r < p.m;
  f32x4_t acc[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int c = c0; c < c1; c++) {
    i32x4_t w[NT], a = {0, 0, 0, 0};
    uint32_t sw[NT], sa = 0;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int tile = min(t0 + t, at.tiles - 1);  // past the last: its product is not stored
      w[t] = *reinterpret_cast<const i32x4_t*>(p.w + (((int64_t)tile * at.chunks + c) * 64 + lane) * 16);
      sw[t] = *reinterpret_cast<const uint32_t*>(p.w + at.codes() + ((int64_t)tile * at.quads + (c >> 2)) * 256 + lane * 4) >> (8 * (c & 3));
    }
    if (real && 4 * c + g < groups) a = mx_acts<T>(p.x, p.x_scales, row0 + r, p.k, 4 * c + g, sa);
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = mx_mfma(w[t], sw[t], a, sa, acc[t]);
  }
#pragma unroll
  for (int t = 0; t < NT; t++) part[(wave * NT + t) * 64 + lane] = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 64; i += blockDim.x) {
    f32x4_t sum = part[i];
    for (int w = 1; w < p.waves; w++) sum += part[w * NT * 64 + i];
    const int l = i & 63, t = t0 + (i >> 6);
    const int64_t row = row0 + (l & 15), n = (int64_t)t * 16 + 4 * (l >> 4);
    if (row < p.m)
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (n + j < p.n) static_cast<Y*>(p.y)[row * p.n + n + j] = mx_out<Y>(sum[j]);
  }
}

// More than sixteen rows: both operands in the tile layout. A workgroup's WM x WN wavefronts hold WM MT x WN NT output tiles of 16 x 16;
// two chunks of K of its rows of both operands are a stage, asked for while the stage before is multiplied, written to LDS (a tile as
// it lies: a wavefront reads and writes 1024 consecutive bytes, no bank twice) when that is done, one barrier a stage. k past the matrix
// has scale 0 on both sides: 2^-254 of anything is nothing in FP32, so what the codes hold there does not matter.
struct MxTiles {
  const uint8_t* a;
  const uint8_t* w;
  void* y;
  int64_t m, n;
  int k, rows_of_tiles;  // workgroups along m
};

template <typename Y>
__device__ __forceinline__ void mx_store4(Y* out, const f32x4_t& v, int64_t left, bool whole) {
  if (whole) {
    typedef __attribute__((ext_vector_type(4))) Y y4_t;
    *reinterpret_cast<y4_t*>(out) = y4_t{mx_out<Y>(v[0]), mx_out<Y>(v[1]), mx_out<Y>(v[2]), mx_out<Y>(v[3])};
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < left) out[j] = mx_out<Y>(v[j]);
  }
}

template <int WM, int WN, int MT, int NT>
struct MxTileCore {
  static constexpr int WAVES = WM * WN, TA = WM * MT, TB = WN * NT, STAGE = 2 * (TA + TB), HELD = STAGE / WAVES;
  static constexpr int LDS_BYTES = 2 * STAGE * 1024;
  static_assert(STAGE % WAVES == 0, "whole tiles a wavefront");
};

template <typename Y, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(64 * WM * WN) void mx_tile_kernel(MxTiles p) {
  using Core = MxTileCore<WM, WN, MT, NT>;
  constexpr int WAVES = Core::WAVES, TA = Core::TA, TB = Core::TB, HELD = Core::HELD, STAGE = Core::STAGE;
  extern __shared__ i32x4_t lds[];  // [2][2 chunks][TA + TB][64]
  const MxLayout la(p.m, p.k), lw(p.n, p.k);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  // consecutive workgroups go to the eight dies in turn: each die walks a run of tiles, rows fastest, so that its L2 keeps a run of weights
  const int total = gridDim.x, per = (total + 7) / 8, id = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
  const int whole_runs = total % 8 ? total % 8 : 8;  // dies with `per` workgroups; the others have one less
  const int at = (int)(blockIdx.x % 8) < whole_runs ? id : id - ((int)(blockIdx.x % 8) - whole_runs);
  const int tm = at % p.rows_of_tiles, tn = at / p.rows_of_tiles;
  const int a0 = tm * TA, b0 = tn * TB, stages = (la.chunks + 1) / 2;

  const uint8_t* src[HELD];  // this wavefront's tiles of a stage, at chunk 0
#pragma unroll
  for (int j = 0; j < HELD; j++) {
    const int t = (wave + j * WAVES) % (TA + TB);
    const bool act = t < TA;
    const int tile = act ? min(a0 + t, la.tiles - 1) : min(b0 + t - TA, lw.tiles - 1);
    src[j] = (act ? p.a : p.w) + (int64_t)tile * la.chunks * 1024;
  }
  i32x4_t held[HELD];
  auto ask = [&](int s) {
#pragma unroll
    for (int j = 0; j < HELD; j++) {
      const int c = min(2 * s + (wave + j * WAVES) / (TA + TB), la.chunks - 1);
      held[j] = *reinterpret_cast<const i32x4_t*>(src[j] + c * 1024 + lane * 16);
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int j = 0; j < HELD; j++) lds[(buf * STAGE + wave + j * WAVES) * 64 + lane] = held[j];
  };
  uint32_t sa[MT], sb[NT];
  auto scales = [&](int q) {
#pragma unroll
    for (int t = 0; t < MT; t++)
      sa[t] = *reinterpret_cast<const uint32_t*>(p.a + la.codes() + ((int64_t)min(a0 + wm * MT + t, la.tiles - 1) * la.quads + q) * 256 + lane * 4);
#pragma unroll
    for (int t = 0; t < NT; t++)
      sb[t] = *reinterpret_cast<const uint32_t*>(p.w + lw.codes() + ((int64_t)min(b0 + wn * NT + t, lw.tiles - 1) * lw.quads + q) * 256 + lane * 4);
  };
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NT; j++) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  ask(0);
  scales(0);
  put(0);
  __syncthreads();
#define MX_CHUNK(BUF, C, OP)                                                                                                              \
  {                                                                                                                                       \
    const i32x4_t* at_a = lds + ((BUF) * STAGE + (C) * (TA + TB) + wm * MT) * 64 + lane;                                                   \
    const i32x4_t* at_b = lds + ((BUF) * STAGE + (C) * (TA + TB) + TA + wn * NT) * 64 + lane;                                              \
    i32x4_t fa[MT];                                                                                                                       \
    _Pragma("unroll") for (int i = 0; i < MT; i++) fa[i] = at_a[i * 64];                                                                   \
    _Pragma("unroll") for (int j = 0; j < NT; j++) {                                                                                       \
      const i32x4_t fb = at_b[j * 64];                                                                                                    \
      const i32x8_t wb = __builtin_shufflevector(fb, fb, 0, 1, 2, 3, -1, -1, -1, -1);                                                      \
      _Pragma("unroll") for (int i = 0; i < MT; i++) {                                                                                     \
        const i32x8_t wa = __builtin_shufflevector(fa[i], fa[i], 0, 1, 2, 3, -1, -1, -1, -1);                                              \
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wb, wa, acc[i][j], 4, 4, OP, (int)sb[j], OP, (int)sa[i]);             \
      }                                                                                                                                   \
    }                                                                                                                                     \
  }
  for (int s = 0; s < stages; s += 2) {
    if (s + 1 < stages) ask(s + 1);
    MX_CHUNK(0, 0, 0)
    MX_CHUNK(0, 1, 1)
    if (s + 1 < stages) {
      put(1);
      __syncthreads();
      if (s + 2 < stages) ask(s + 2);
      MX_CHUNK(1, 0, 2)
      MX_CHUNK(1, 1, 3)
      if (s + 2 < stages) {
        scales((s + 2) / 2);
        put(0);
        __syncthreads();
      }
    }
  }
#undef MX_CHUNK
  const int r = lane & 15, g = lane >> 4;
  const bool aligned4 = p.n % 4 == 0;
#pragma unroll
  for (int i = 0; i < MT; i++) {
    const int64_t row = (int64_t)(a0 + wm * MT + i) * 16 + r;
    if (row >= p.m) continue;
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const int64_t n = (int64_t)(b0 + wn * NT + j) * 16 + 4 * g;
      if (n < p.n) mx_store4<Y>(static_cast<Y*>(p.y) + row * p.n + n, acc[i][j], p.n - n, aligned4);
    }
  }
}

// Many rows: 256 x 256 outputs a workgroup, 128 x 128 a wavefront (256 accumulator registers, one wavefront a SIMD), so that a matrix
// instruction's operands come from LDS at 48 of the 128 bytes a cycle it gives ... Four buffers of one chunk of K; a chunk's 32 tiles come by
// LDS-direct loads, asked for three steps ahead and waited for one step before they are read, so that a step can fetch the next
// one's first fragments ahead of the barrier between them. A separate array a buffer: the compiler then knows that reading one
// does not wait for the loads into another.
struct MxBig {
  static constexpr int TA = 16, TB = 16;
};
typedef __attribute__((address_space(3))) uint8_t* mx_lds_t;

// mx_mfma with the sum staying in its accumulator registers (left to itself the compiler moves 256 of them about) and the scales in byte
// OP of their words. The two wait states in front cover an operand that a vector instruction has just written, and hide behind the matrix
// instruction before (16 cycles); mx_sums_done stands before the sums are read.
template <int OP>
__device__ __forceinline__ void mx_mfma_in_place(f32x4_t& acc, i32x4_t a, i32x4_t b, uint32_t sa, uint32_t sb) {
#define MX_MFMA(SELECT) \
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " SELECT " cbsz:4 blgp:4" : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb))
  if constexpr (OP == 0) MX_MFMA("op_sel_hi:[0,0,0]");
  if constexpr (OP == 1) MX_MFMA("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  if constexpr (OP == 2) MX_MFMA("op_sel_hi:[1,1,0]");
  if constexpr (OP == 3) MX_MFMA("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef MX_MFMA
}
__device__ __forceinline__ void mx_sums_done() { asm volatile("s_nop 15\n\ts_nop 7" ::: "memory"); }

// A buffer descriptor in scalar registers: what is read past `bytes` is zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_rows(const uint8_t* base, int bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)at), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(hi << 32 | lo), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

template <typename Y>
__global__ __launch_bounds__(256, 1) void mx_big_kernel(MxTiles p) {
  constexpr int T = MxBig::TA + MxBig::TB, ASKS = T / 4;
  __shared__ i32x4_t buf0[T * 64], buf1[T * 64], buf2[T * 64], buf3[T * 64];
  const MxLayout la(p.m, p.k), lw(p.n, p.k);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  const int total = gridDim.x, per = (total + 7) / 8, die = blockIdx.x % 8;
  const int whole_runs = total % 8 ? total % 8 : 8;
  const int at = die * per - (die > whole_runs ? die - whole_runs : 0) + (int)(blockIdx.x / 8);
  const int tm = at % p.rows_of_tiles, tn = at / p.rows_of_tiles;
  const int a0 = tm * MxBig::TA, b0 = tn * MxBig::TB, chunks = la.chunks;

  // this wavefront's eight tiles of a chunk: of A for the first two wavefronts, of B for the others (past the last: the last again)
  const bool act = wave < 2;
  const int tiles = act ? la.tiles : lw.tiles, first = min((act ? a0 : b0) + (wave & 1) * 8, tiles - 1), left = min(8, tiles - first), row_bytes = chunks * 1024;
  const __amdgpu_buffer_rsrc_t rows = mx_rows((act ? p.a : p.w) + (int64_t)first * row_bytes, left * row_bytes);
#define MX_ASK(BUF, C)                                                                                                                    \
  {                                                                                                                                       \
    const int in_row = min((C), chunks - 1) * 1024;                                                                                       \
    _Pragma("unroll") for (int j = 0; j < ASKS; j++)                                                                                      \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (mx_lds_t)(BUF + (wave * ASKS + j) * 64), 16, lane * 16, min(j, left - 1) * row_bytes + in_row, 0, 0); \
  }

  uint32_t sa[8], sb[8], na[8], nb[8];
  auto scales = [&](int q) {
#pragma unroll
    for (int t = 0; t < 8; t++) {
      na[t] = *reinterpret_cast<const uint32_t*>(p.a + la.codes() + ((int64_t)min(a0 + wm * 8 + t, la.tiles - 1) * la.quads + q) * 256 + lane * 4);
      nb[t] = *reinterpret_cast<const uint32_t*>(p.w + lw.codes() + ((int64_t)min(b0 + wn * 8 + t, lw.tiles - 1) * lw.quads + q) * 256 + lane * 4);
    }
  };
  f32x4_t acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  scales(0);
  MX_ASK(buf0, 0)
  MX_ASK(buf1, 1)
  MX_ASK(buf2, 2)
  asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  i32x4_t fa[2][8], fb[4];
#pragma unroll
  for (int i = 0; i < 8; i++) fa[0][i] = buf0[(wm * 8 + i) * 64 + lane];
  fb[0] = buf0[(16 + wn * 8) * 64 + lane];
  fb[1] = buf0[(16 + wn * 8 + 1) * 64 + lane];
#define MX_STEP(CUR, NEXT, ASKED, C, OP)                                                                                                   \
  {                                                                                                                                       \
    MX_ASK(ASKED, (C) + 3)                                                                                                               \
    __builtin_amdgcn_sched_barrier(0);                                                                                                    \
    _Pragma("unroll") for (int j = 0; j < 8; j++) {                                                                                       \
      fb[(j + 2) & 3] = j < 6 ? CUR[(16 + wn * 8 + j + 2) * 64 + lane] : NEXT[(16 + wn * 8 + j - 6) * 64 + lane];                          \
      fa[1 - ((OP) & 1)][j] = NEXT[(wm * 8 + j) * 64 + lane];                                                                             \
      _Pragma("unroll") for (int i = 0; i < 8; i++) mx_mfma_in_place<OP>(acc[i][j], fb[j & 3], fa[(OP) & 1][i], sb[j], sa[i]);               \
      __builtin_amdgcn_sched_barrier(0);                                                                                                  \
    }                                                                                                                                     \
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");                                                                                      \
    __builtin_amdgcn_s_barrier();                                                                                                         \
    __builtin_amdgcn_sched_barrier(0);                                                                                                    \
  }
  for (int q = 0; q < la.quads; q++) {
#pragma unroll
    for (int t = 0; t < 8; t++) sa[t] = na[t], sb[t] = nb[t];
    scales(min(q + 1, la.quads - 1));
    MX_STEP(buf0, buf1, buf3, 4 * q, 0)
    MX_STEP(buf1, buf2, buf0, 4 * q + 1, 1)
    MX_STEP(buf2, buf3, buf1, 4 * q + 2, 2)
    MX_STEP(buf3, buf0, buf2, 4 * q + 3, 3)
  }
#undef MX_STEP
#undef MX_ASK
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was asked for past the end arrives before the workgroup leaves its LDS
  mx_sums_done();
#pragma unroll
  for (int i = 0; i < 8; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) asm volatile("" : "+a"(acc[i][j]));
  const int r = lane & 15, g = lane >> 4;
  const bool aligned4 = p.n % 4 == 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int64_t row = (int64_t)(a0 + wm * 8 + i) * 16 + r;
    if (row >= p.m) continue;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int64_t n = (int64_t)(b0 + wn * 8 + j) * 16 + 4 * g;
      if (n < p.n) mx_store4<Y>(static_cast<Y*>(p.y) + row * p.n + n, acc[i][j], p.n - n, aligned4);
    }
  }
}

// x [rows, k] rounded into the tile layout (rows past the last are left as they are: their results are not stored).
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_tiles_kernel(const T* __restrict__ x, int64_t rows, int k, uint8_t* __restrict__ tiled) {
  const MxLayout at(rows, k);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per_row = at.quads * 64;  // lanes of eight values, K in whole quads
  const int64_t row = i / per_row;
  if (row >= rows) return;  // whole groups leave together
  const int e = (int)(i - row * per_row), group = e >> 2, c = group >> 2, lane = (group & 3) * 16 + (int)(row & 15);
  const int64_t t = row >> 4;
  uint32_t byte = 0, code = 0;
  if (group < k / 32) {
    Mx8<T> v;
    v.load(x + row * k + 8 * e);
    byte = mx_scale_byte(quad_max(v.amax()));
    code = byte == 255u ? 0u : v.codes(mx_scale_value(byte));
  }
  if (c < at.chunks) *reinterpret_cast<uint32_t*>(tiled + ((t * at.chunks + c) * 64 + lane) * 16 + 4 * (e & 3)) = code;
  if ((e & 3) == 0) tiled[at.codes() + (t * at.quads + (c >> 2)) * 256 + lane * 4 + (c & 3)] = (uint8_t)byte;
}

constexpr int MX_FEW_ROWS = 16;

template <typename Y, int WM, int WN, int MT, int NT>
static int launch_tiles(MxTiles p, hipStream_t stream) {
  using Core = MxTileCore<WM, WN, MT, NT>;
  static const hipError_t raised = hipFuncSetAttribute(reinterpret_cast<const void*>(&mx_tile_kernel<Y, WM, WN, MT, NT>), hipFuncAttributeMaxDynamicSharedMemorySize, Core::LDS_BYTES);
  if (raised != hipSuccess) return HB_ELAUNCH;
  const MxLayout la(p.m, p.k), lw(p.n, p.k);
  p.rows_of_tiles = (la.tiles + Core::TA - 1) / Core::TA;
  const int64_t groups = (int64_t)p.rows_of_tiles * ((lw.tiles + Core::TB - 1) / Core::TB);
  HB_LAUNCH((mx_tile_kernel<Y, WM, WN, MT, NT>), dim3((unsigned)groups), dim3(64 * WM * WN), Core::LDS_BYTES, stream, p);
  return HB_OK;
}

template <typename Y>
static int launch_big(MxTiles p, hipStream_t stream) {
  const MxLayout la(p.m, p.k), lw(p.n, p.k);
  p.rows_of_tiles = (la.tiles + MxBig::TA - 1) / MxBig::TA;
  HB_LAUNCH((mx_big_kernel<Y>), dim3((unsigned)(p.rows_of_tiles * ((lw.tiles + MxBig::TB - 1) / MxBig::TB))), dim3(256), 0, stream, p);
  return HB_OK;
}

template <typename T, typename Y>
static int launch_many(const MxLinear& p, uint8_t* tiles, hipStream_t stream) {
  const MxLayout at(p.m, p.k);
  if constexpr (std::is_same_v<T, uint8_t>) {
    if (int e = hb_mxfp4_repack(p.x, p.x_scales, 1, p.m, p.k, 0, tiles, stream)) return e;
  } else {
    HB_LAUNCH((mx_quantize_tiles_kernel<T>), dim3((unsigned)((p.m * at.quads * 64 + 255) / 256)), dim3(256), 0, stream, static_cast<const T*>(p.x), p.m, p.k, tiles);
  }
  const MxTiles q{tiles, p.w, p.y, p.m, p.n, p.k, 0};
  if (p.m <= 32) return launch_tiles<Y, 1, 4, 2, 2>(q, stream);
  if (p.m <= 64) return launch_tiles<Y, 1, 4, 4, 2>(q, stream);
  if (p.m <= 96) return launch_tiles<Y, 1, 4, 6, 2>(q, stream);
  if (p.m <= 128) return launch_tiles<Y, 1, 4, 8, 2>(q, stream);
  return launch_big<Y>(q, stream);
}

template <typename T, typename Y>
static int launch_linear(const MxLinear& p0, uint8_t* tiles, hipStream_t stream) {
  if (p0.m > MX_FEW_ROWS) return launch_many<T, Y>(p0, tiles, stream);
  MxLinear p = p0;
  const MxLayout at(p.n, p.k);
  constexpr int NT = 4;
  p.waves = std::min(at.chunks, 8);
  const unsigned passes = (unsigned)((p.m + 15) / 16);
  HB_LAUNCH((mx_few_rows_kernel<T, Y, NT>), dim3((unsigned)((at.tiles + NT - 1) / NT), passes), dim3(64 * p.waves), (size_t)p.waves * NT * 64 * 16, stream, p);
  return HB_OK;
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
static size_t type_bytes(int type) { return type == HB_F32 ? 4 : 2; }

}  // namespace hb

using namespace hb;

extern "C" int hb_mxfp4_quantize(const void* x, int type, int64_t rows, int k, void* codes, void* scales, void* stream) {
  if (!x || !codes || !scales) return HB_ENULL;
  if (rows <= 0 || k <= 0 || k % MX_GROUP || rows > (int64_t)1 << 40 || rows * (k / 8) > (int64_t)255 << 31) return HB_EINVAL;
  if (!aligned(x, 16) || !aligned(codes, 16)) return HB_EINVAL;
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int64_t lanes = rows * (k / 8);
    HB_LAUNCH((mx_quantize_kernel<T>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, as_stream(stream), static_cast<const T*>(x), lanes,
              static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales));
    return launch_status();
  });
}

extern "C" int hb_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int k, int type, void* out, void* stream) {
  if (!codes || !scales || !out) return HB_ENULL;
  if (rows <= 0 || k <= 0 || k % MX_GROUP || rows > (int64_t)1 << 40 || rows * (k / 8) > (int64_t)255 << 31) return HB_EINVAL;
  if (!aligned(codes, 16) || !aligned(out, 16)) return HB_EINVAL;
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int64_t lanes = rows * (k / 8);
    HB_LAUNCH((mx_dequantize_kernel<T>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, as_stream(stream), static_cast<const uint8_t*>(codes),
              static_cast<const uint8_t*>(scales), lanes, static_cast<T*>(out));
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
    const int64_t lanes = rows * (half / 8);
    HB_LAUNCH((mx_silu_quantize_kernel<T>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, as_stream(stream), static_cast<const T*>(gate_up), rows, half,
              pairs, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales));
    return launch_status();
  });
}

// Sizes that the layout's indices and a launch's grid hold.
static bool layout_holds(int64_t n, int k) { return n > 0 && k > 0 && k <= 1 << 25 && k % MX_GROUP == 0 && n <= (int64_t)1 << 30 && (n + 15) / 16 * ((k + 511) / 512) <= (int64_t)1 << 28; }

extern "C" size_t hb_mxfp4_tiled_bytes(int64_t n, int k) { return layout_holds(n, k) ? (size_t)MxLayout(n, k).bytes() : 0; }

static int repack(bool unpack, void* codes, void* scales, int matrices, int64_t n, int k, int gated, void* tiled, void* stream) {
  if (!codes || !scales || !tiled) return HB_ENULL;
  if (!layout_holds(n, k) || matrices <= 0 || matrices > 65535 || (gated && n % 64)) return HB_EINVAL;
  if (!aligned(codes, 16) || !aligned(tiled, 16)) return HB_EINVAL;
  const MxLayout at(n, k);
  const dim3 grid((unsigned)(((int64_t)at.tiles * at.quads * 256 + 255) / 256), (unsigned)matrices);
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
  (void)x_type;
  return m > MX_FEW_ROWS && layout_holds(n, k) && layout_holds(m, k) ? (size_t)MxLayout(m, k).bytes() : 0;
}

extern "C" int hb_mxfp4_linear(const void* x, const void* x_scales, int x_type, int64_t m, const void* tiled, int64_t n, int k, void* y, int y_type,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (!x || !tiled || !y || (x_type == HB_MXFP4 && !x_scales)) return HB_ENULL;
  if (m <= 0 || m > (int64_t)1 << 19 || !layout_holds(n, k) || y_type < HB_BF16 || y_type > HB_F32 || x_type < HB_BF16 || x_type > HB_MXFP4) return HB_EINVAL;
  if (x_type != HB_MXFP4 && x_type != y_type) return HB_EINVAL;
  if (!aligned(x, 16) || !aligned(tiled, 16) || !aligned(y, type_bytes(y_type))) return HB_EINVAL;
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
