// The microscaled four-bit format (MXFP4) on gfx950: what its kernels share.
//
// Values come in groups of 32 along K. A group has one power-of-two scale, an E8M0 byte b standing for 2^(b - 127) (255: NaN),
// and 32 E2M1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign), two a byte, element 2 i in the low nibble. The rounding of a group:
//   b = max(floor(log2 amax) + 127 - 2, 0),  code = the nearest E2M1 of x / 2^(b - 127), ties to the even code, beyond 6 to 6;
// a group that holds an infinity or a NaN has b = 255 and codes 0. The scale is the power of two that puts the largest magnitude
// into [4, 8): what lies in (6, 8) is cut to 6, and the whole group costs one exponent field. x / 2^(b - 127) is exact, so the codes
// are the rounding's whatever computes them; v_cvt_scalef32_pk_fp4_* does it for two values at a time (its ties, its saturation and
// its scales down to 2^-127 were checked over every BF16 and FP16 value).
#pragma once

#include "common.hpp"

namespace hb {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;

constexpr int MX_GROUP = 32;
constexpr int MX_ROWS = 16, MX_K = 128;  // a tile: what one matrix instruction takes of either operand

// ------------------------------------------------------------------------------------------------ tile layout
// A matrix [n, k] as the products read it: tiles of 16 rows x 128 k, [ceil(n / 16)][ceil(k / 128)], 1024 bytes of codes each, lane
// l = 16 g + r of a wavefront owning the 16 bytes of row r, k = 32 g .. 32 g + 31: its operand of one
// v_mfma_scale_f32_16x16x128_f8f6f4, so a tile is one 128-bit load a lane, 1024 consecutive bytes a wavefront. Behind the codes the
// scales: four tiles' along K together, 256 bytes, lane l owning the four bytes of its row and its group in each of them.
// Rows and k past the matrix hold code 0 and scale 0.
struct MxLayout {
  int tiles, chunks, quads;  // 16-row tiles, 128-k chunks, groups of four chunks
  __host__ __device__ MxLayout(int64_t n, int64_t k) : tiles((int)((n + MX_ROWS - 1) / MX_ROWS)), chunks((int)((k + MX_K - 1) / MX_K)), quads((chunks + 3) / 4) {}
  __host__ __device__ int64_t codes() const { return (int64_t)tiles * chunks * 1024; }
  __host__ __device__ int64_t bytes() const { return codes() + (int64_t)tiles * quads * 256; }
};

// ------------------------------------------------------------------------------------------------ rounding
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {  // the FP32 bits of the group's largest magnitude
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : e < 2u ? 0u : e - 2u;
}
// 2^(b - 127) as FP32; b = 255: NaN
__device__ __forceinline__ float mx_scale_value(uint32_t b) { return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7fc00000u : b << 23); }

// The two 16-bit values of a word (by value: a bit cast of a vector's element written in place reads element 0).
__device__ __forceinline__ bf16x2_t bf16_pair_of(uint32_t w) { return __builtin_bit_cast(bf16x2_t, w); }
__device__ __forceinline__ f16x2_t f16_pair_of(uint32_t w) { return __builtin_bit_cast(f16x2_t, w); }
__device__ __forceinline__ u16x2_t magnitudes_of(uint32_t w) { return __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu); }

// Eight consecutive values of a type: loaded, their largest magnitude as FP32 bits, their codes under a scale.
template <typename T>
struct Mx8;
template <>
struct Mx8<__bf16> {
  u32x4_t v;
  __device__ __forceinline__ void load(const __bf16* p) { v = *reinterpret_cast<const u32x4_t*>(p); }
  __device__ __forceinline__ uint32_t amax() const {
    u16x2_t m = magnitudes_of(v[0]);
#pragma unroll
    for (int j = 1; j < 4; j++) m = __builtin_elementwise_max(m, magnitudes_of(v[j]));
    return (uint32_t)(m[0] > m[1] ? m[0] : m[1]) << 16;
  }
  __device__ __forceinline__ uint32_t codes(float s) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, bf16_pair_of(v[0]), s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, bf16_pair_of(v[1]), s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, bf16_pair_of(v[2]), s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, bf16_pair_of(v[3]), s, 3);
  }
  __device__ __forceinline__ float at(int j) const { return __uint_as_float((j & 1) ? v[j >> 1] & 0xffff0000u : v[j >> 1] << 16); }
};
template <>
struct Mx8<_Float16> {
  u32x4_t v;
  __device__ __forceinline__ void load(const _Float16* p) { v = *reinterpret_cast<const u32x4_t*>(p); }
  __device__ __forceinline__ uint32_t amax() const {
    u16x2_t m = magnitudes_of(v[0]);
#pragma unroll
    for (int j = 1; j < 4; j++) m = __builtin_elementwise_max(m, magnitudes_of(v[j]));
    const unsigned short top = m[0] > m[1] ? m[0] : m[1];
    return __float_as_uint((float)__builtin_bit_cast(_Float16, top)) & 0x7fffffffu;  // a half's subnormals are normal here
  }
  __device__ __forceinline__ uint32_t codes(float s) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, f16_pair_of(v[0]), s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, f16_pair_of(v[1]), s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, f16_pair_of(v[2]), s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, f16_pair_of(v[3]), s, 3);
  }
  __device__ __forceinline__ float at(int j) const { return (float)f16_pair_of(v[j >> 1])[j & 1]; }
};
template <>
struct Mx8<float> {
  f32x4_t v[2];
  __device__ __forceinline__ void load(const float* p) {
    v[0] = *reinterpret_cast<const f32x4_t*>(p);
    v[1] = *reinterpret_cast<const f32x4_t*>(p + 4);
  }
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t u = __float_as_uint(v[j >> 2][j & 3]) & 0x7fffffffu;
      m = u > m ? u : m;
    }
    return m;
  }
  __device__ __forceinline__ uint32_t codes(float s) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0][0], v[0][1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0][2], v[0][3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[1][0], v[1][1], s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[1][2], v[1][3], s, 3);
  }
  __device__ __forceinline__ float at(int j) const { return v[j >> 2][j & 3]; }
};

// The largest of a word over the four lanes of a quad (a group of 32 at eight values a lane), in each of them.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  uint32_t o = __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, false);  // lane ^ 1
  x = o > x ? o : x;
  o = __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, false);  // lane ^ 2
  return o > x ? o : x;
}

// One lane's whole group of 32: the 16 bytes of codes, and the scale byte.
template <typename T>
__device__ __forceinline__ i32x4_t mx_round_group(const T* p, uint32_t& byte) {
  Mx8<T> x[4];
#pragma unroll
  for (int j = 0; j < 4; j++) x[j].load(p + 8 * j);
  uint32_t m = x[0].amax();
#pragma unroll
  for (int j = 1; j < 4; j++) {
    const uint32_t o = x[j].amax();
    m = o > m ? o : m;
  }
  byte = mx_scale_byte(m);
  const float s = mx_scale_value(byte);
  const uint32_t finite = byte == 255u ? 0u : ~0u;
  i32x4_t c;
#pragma unroll
  for (int j = 0; j < 4; j++) c[j] = (int)(x[j].codes(s) & finite);
  return c;
}

// acc += (16 rows of a) x (16 rows of b)^T over 128 k, codes and scale bytes (in the low byte) in the lanes that own them. In the result
// lane 16 g + r holds rows 4 g .. 4 g + 3 of a for row r of b.
__device__ __forceinline__ f32x4_t mx_mfma(i32x4_t a, uint32_t sa, i32x4_t b, uint32_t sb, f32x4_t acc) {
  const i32x8_t wa = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1), wb = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, acc, 4, 4, 0, (int)sa, 0, (int)sb);  // 4: E2M1
}

// An FP32 sum in the result's type: one rounding.
template <typename T>
__device__ __forceinline__ T mx_out(float v) {
  return (T)v;
}

}  // namespace hb
