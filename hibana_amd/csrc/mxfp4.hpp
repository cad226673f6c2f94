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

#include <type_traits>

#include "common.hpp"

namespace hb {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;

constexpr int MX_GROUP = 32;
constexpr int MX_ROWS = 32, MX_K = 64;  // a tile: what one matrix instruction takes of either operand

// ------------------------------------------------------------------------------------------------ tile layout
// A matrix [n, k] as the products read it: tiles of 32 rows x 64 k, [ceil(n / 32)][ceil(k / 64)], 1024 bytes of codes each, lane
// l = 32 g + r of a wavefront owning the 16 bytes of row r, k = 32 g .. 32 g + 31: its operand of one
// v_mfma_scale_f32_32x32x64_f8f6f4, so a tile is one 128-bit load a lane, 1024 consecutive bytes a wavefront. Behind the codes the
// scales: four tiles along K together (a quad), 256 bytes, lane l owning the four bytes of its row and its group in each of them; K in
// whole pairs of quads. Rows and k past the matrix hold scale 0 (and code 0).
// (32 x 32 x 64 and not 16 x 16 x 128: one wavefront a SIMD gets 9.2 PFLOP/s out of the former, 3.1 of the latter, four 9.5 and 4.6.)
struct MxLayout {
  int tiles, chunks, quads;  // 32-row tiles, 64-k chunks, groups of four chunks
  __host__ __device__ MxLayout(int64_t n, int64_t k) : tiles((int)((n + MX_ROWS - 1) / MX_ROWS)), chunks((int)((k + MX_K - 1) / MX_K)), quads((chunks + 7) / 8 * 2) {}
  __host__ __device__ int64_t codes() const { return (int64_t)tiles * chunks * 1024; }
  __host__ __device__ int64_t bytes() const { return codes() + (int64_t)tiles * quads * 256; }
};

constexpr int MX_NO_REUSE = 2;  // the cache policy of loads whose bytes are not read again soon
// A buffer descriptor in scalar registers: what is read past `bytes` is zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_rows(const uint8_t* base, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)at), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(hi << 32 | lo), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}

// f(0), f(1) .. f(N - 1), each with its number as a constant.
template <int N, int I = 0, class F>
__device__ __forceinline__ void mx_unrolled(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    mx_unrolled<N, I + 1>(f);
  }
}

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

// A lane's whole group of 32 values: loaded, then the 16 bytes of codes and the scale byte (of a group that is not finite any codes: its scale
// is NaN).
template <typename T>
struct MxGroup {
  Mx8<T> x[4];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int j = 0; j < 4; j++) x[j].load(p + 8 * j);
  }
  __device__ __forceinline__ i32x4_t codes(uint32_t& byte) const {
    uint32_t m = x[0].amax();
#pragma unroll
    for (int j = 1; j < 4; j++) m = max(m, x[j].amax());
    byte = mx_scale_byte(m);
    const float s = mx_scale_value(byte);
    i32x4_t c;
#pragma unroll
    for (int j = 0; j < 4; j++) c[j] = (int)x[j].codes(s);
    return c;
  }
};

// The activations of a product of few rows, in LDS: codes [group][rows][16 bytes], scales [group][rows] behind them, so that the lanes of a
// fragment read consecutive addresses.
struct MxActs {
  i32x4_t* codes;
  uint8_t* scales;
  int rows, groups;
  __device__ __forceinline__ MxActs(void* lds, int rows, int k) : codes(static_cast<i32x4_t*>(lds)), scales(static_cast<uint8_t*>(lds) + (size_t)rows * (k / 2)), rows(rows), groups(k / MX_GROUP) {}
  static __host__ __device__ size_t bytes(int64_t rows, int k) { return ((size_t)rows * (k / 2 + k / MX_GROUP) + 15) / 16 * 16; }
  // Eight values, quarter `part` of group `group` of row r, rounded with the three lanes beside that hold the others (a lane a group would
  // read 64 bytes of its own at a time, twice as many lines an instruction as there are bytes for) ...
  template <typename T>
  __device__ __forceinline__ void put(int r, int group, int part, const Mx8<T>& v) const {
    const uint32_t byte = mx_scale_byte(quad_max(v.amax()));
    reinterpret_cast<uint32_t*>(codes)[(group * rows + r) * 4 + part] = v.codes(mx_scale_value(byte));
    if (part == 0) scales[group * rows + r] = (uint8_t)byte;
  }
  // ... or codes as they are.
  __device__ __forceinline__ void put(int r, int group, const uint8_t* row_codes, const uint8_t* row_scales) const {
    codes[group * rows + r] = *reinterpret_cast<const i32x4_t*>(row_codes + 16 * group);
    scales[group * rows + r] = row_scales[group];
  }
};

// acc += (32 rows of a) x (32 rows of b)^T over 64 k, codes and scale bytes (byte OP_A / OP_B of the words) in the lanes that own them. In the
// result lane 32 g + r holds, in registers 4 q .. 4 q + 3, rows 8 q + 4 g .. + 3 of a for row r of b.
template <int OP_A, int OP_B>
__device__ __forceinline__ f32x16_t mx_mfma(i32x4_t a, uint32_t sa, i32x4_t b, uint32_t sb, f32x16_t acc) {
  const i32x8_t wa = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1), wb = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, wb, acc, 4, 4, OP_A, (int)sa, OP_B, (int)sb);  // 4: E2M1
}
__device__ __forceinline__ f32x4_t mx_quarter(const f32x16_t& v, int q) { return f32x4_t{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]}; }

// A wavefront's sums over chunks c0 .. c1 - 1 (c0 a multiple of RUN: 1, 2 or 4) of NT tiles of weight rows from tile t0 (past the last: the
// last again, not to be stored) and up to 32 activation rows: RUN chunks of weights are asked for ahead of the RUN that are multiplied.
template <int NT, int RUN>
struct MxStream {
  __amdgpu_buffer_rsrc_t codes, scales;  // of the NT tiles
  int code_at[NT], scale_at[NT];
  i32x4_t b[RUN][NT];
  uint32_t sb[NT];
  int c0, c1;
  f32x16_t acc[NT];
  // The first run is on its way from here.
  __device__ __forceinline__ void begin(const uint8_t* matrix, const MxLayout& at, int t0, int wave, int waves) {
    const int tiles = min(NT, at.tiles - t0);
    codes = mx_rows(matrix + (int64_t)t0 * at.chunks * 1024, (uint32_t)tiles * at.chunks * 1024);
    scales = mx_rows(matrix + at.codes() + (int64_t)t0 * at.quads * 256, (uint32_t)tiles * at.quads * 256);
    const int runs = (at.chunks + RUN - 1) / RUN;
    c0 = RUN * (runs * wave / waves);
    c1 = min(at.chunks, RUN * (runs * (wave + 1) / waves));
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int tile = min(t, at.tiles - 1 - t0);
      code_at[t] = tile * at.chunks * 1024;
      scale_at[t] = tile * at.quads * 256;
    }
    ask(min(c0, at.chunks - 1));
  }
  // (chunks past the end are asked for again and not multiplied) The weights take their place in the Infinity Cache: eight rows of 25600 x 5120 14.0 us where three such
  // matrices are read in turn, 19.3 where ten are; with MX_NO_REUSE 15.8 and 17.8.
  __device__ __forceinline__ void ask(int c) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int t = 0; t < NT; t++) sb[t] = __builtin_amdgcn_raw_buffer_load_b32(scales, lane * 4, scale_at[t] + (c >> 2) * 256, 0);
#pragma unroll
    for (int u = 0; u < RUN; u++)
#pragma unroll
      for (int t = 0; t < NT; t++)
        b[u][t] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(codes, lane * 16, code_at[t] + min(c + u, max(c1 - 1, 0)) * 1024, 0));
  }
  template <int U>
  __device__ __forceinline__ void step(const i32x4_t (&w)[RUN][NT], const uint32_t (&sw)[NT], const i32x4_t& a, uint32_t sa) {
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = mx_mfma<U, 0>(w[U][t], sw[t], a, sa, acc[t]);
  }
  __device__ __forceinline__ void run(const MxActs& acts) {
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int i = 0; i < 16; i++) acc[t][i] = 0.f;
    const int half = (threadIdx.x & 63) >> 5, r = min((int)(threadIdx.x & 31), acts.rows - 1);  // (rows past the last: that one again, not to be stored)
    for (int c = c0; c < c1; c += RUN) {
      i32x4_t now[RUN][NT], a[RUN];
      uint32_t sw[NT], sa[RUN];
#pragma unroll
      for (int t = 0; t < NT; t++) sw[t] = RUN == 4 ? sb[t] : sb[t] >> (8 * (c & 3));
#pragma unroll
      for (int u = 0; u < RUN; u++) {
        // (k past the matrix: the last group again; the weights' codes there are 0)
        const int at = min(2 * (c + u) + half, acts.groups - 1) * acts.rows + r;
        a[u] = acts.codes[at];
        sa[u] = acts.scales[at];
#pragma unroll
        for (int t = 0; t < NT; t++) now[u][t] = b[u][t];
      }
      if (c + RUN < c1) ask(c + RUN);
      step<0>(now, sw, a[0], sa[0]);
      if constexpr (RUN > 1)
        if (c + 1 < c1) step<1>(now, sw, a[1], sa[1]);
      if constexpr (RUN > 2) {
        if (c + 2 < c1) step<2>(now, sw, a[2], sa[2]);
        if (c + 3 < c1) step<3>(now, sw, a[3], sa[3]);
      }
    }
  }
};

// The wavefronts' sums of a workgroup added in wavefront order, through LDS: part [waves][NT * 4][64]. Entry i of NT * 256 is quarter
// (i / 64) % 4 of tile i / 256, lane i % 64.
template <int NT>
__device__ __forceinline__ void mx_hand_over(f32x4_t* part, const f32x16_t (&acc)[NT]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();  // the activations' place
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int q = 0; q < 4; q++) part[((wave * NT + t) * 4 + q) * 64 + lane] = mx_quarter(acc[t], q);
  __syncthreads();
}
template <int NT>
__device__ __forceinline__ f32x4_t mx_joined(const f32x4_t* part, int waves, int i) {
  f32x4_t sum = part[i];
  for (int w = 1; w < waves; w++) sum += part[w * NT * 256 + i];
  return sum;
}

// An FP32 sum in the result's type: one rounding.
template <typename T>
__device__ __forceinline__ T mx_out(float v) {
  return (T)v;
}

}  // namespace hb
