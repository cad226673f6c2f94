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

template <typename T, typename Y>
static int launch_linear(const MxLinear& p0, hipStream_t stream) {
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
static bool layout_holds(int64_t n, int k) { return n > 0 && k > 0 && k % MX_GROUP == 0 && n <= (int64_t)1 << 30 && (n + 15) / 16 * ((k + 511) / 512) <= (int64_t)1 << 28; }

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
  (void)m, (void)n, (void)k, (void)x_type;
  return 0;
}

extern "C" int hb_mxfp4_linear(const void* x, const void* x_scales, int x_type, int64_t m, const void* tiled, int64_t n, int k, void* y, int y_type,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (!x || !tiled || !y || (x_type == HB_MXFP4 && !x_scales)) return HB_ENULL;
  if (m <= 0 || m > (int64_t)1 << 19 || !layout_holds(n, k) || y_type < HB_BF16 || y_type > HB_F32 || x_type < HB_BF16 || x_type > HB_MXFP4) return HB_EINVAL;
  if (x_type != HB_MXFP4 && x_type != y_type) return HB_EINVAL;
  if (!aligned(x, 16) || !aligned(tiled, 16) || !aligned(y, type_bytes(y_type))) return HB_EINVAL;
  if (workspace_bytes < hb_mxfp4_linear_workspace_bytes(m, n, k, x_type)) return HB_EWORKSPACE;
  const MxLinear p{x, static_cast<const uint8_t*>(x_scales), static_cast<const uint8_t*>(tiled), y, m, n, k, 0};
  const int code = by_type(y_type, [&](auto* t) {
    using Y = std::remove_pointer_t<decltype(t)>;
    return x_type == HB_MXFP4 ? launch_linear<uint8_t, Y>(p, as_stream(stream)) : launch_linear<Y, Y>(p, as_stream(stream));
  });
  return code ? code : launch_status();
}
