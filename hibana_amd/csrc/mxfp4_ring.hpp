// The matrix products of many rows on microscaled four-bit operands: both in the tile layout, a workgroup a rectangle of output tiles.
#pragma once

#include "mxfp4.hpp"

namespace hb {

typedef __attribute__((address_space(3))) uint8_t* mx_lds_t;

// mx_mfma with the sum staying in its accumulator registers (left to itself the compiler moves 256 of them about) and the scales in byte
// OP of their words. The compiler does not know it for a matrix instruction, so what it has to wait for is waited for here: the two wait states in front cover
// an operand that a vector instruction has just written, and hide behind the matrix instruction before (32 cycles); mx_sums_done ends every
// block that the products stand in, so that whatever the compiler does to the sums between blocks comes after them.
template <int OP>
__device__ __forceinline__ void mx_mfma_in_place(f32x16_t& acc, i32x4_t a, i32x4_t b, uint32_t sa, uint32_t sb) {
#define MX_MFMA(SELECT) \
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 " SELECT " cbsz:4 blgp:4" : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb))
  if constexpr (OP == 0) MX_MFMA("op_sel_hi:[0,0,0]");
  if constexpr (OP == 1) MX_MFMA("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  if constexpr (OP == 2) MX_MFMA("op_sel_hi:[1,1,0]");
  if constexpr (OP == 3) MX_MFMA("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef MX_MFMA
}
__device__ __forceinline__ void mx_sums_done() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// A vector that starts where its elements do.
template <typename V, typename E>
struct __attribute__((packed, aligned(sizeof(E)), may_alias)) MxLoose {
  V v;
};
// Four neighbouring results of a row, `left` of them inside the matrix; `whole`: rows start on four.
template <typename Y>
__device__ __forceinline__ void mx_store4(Y* out, const f32x4_t& v, int64_t left, bool whole) {
  typedef __attribute__((ext_vector_type(4))) Y y4_t;
  const y4_t y = {mx_out<Y>(v[0]), mx_out<Y>(v[1]), mx_out<Y>(v[2]), mx_out<Y>(v[3])};
  if (whole) {
    *reinterpret_cast<y4_t*>(out) = y;
  } else if (left >= 4) {
    reinterpret_cast<MxLoose<y4_t, Y>*>(out)->v = y;
  } else {
#pragma unroll
    for (int j = 0; j < 3; j++)
      if (j < left) out[j] = y[j];
  }
}

// Both operands in the tile layout. A workgroup's WM x WN wavefronts hold MT x NT output tiles of 32 x 32 each; 128 k of the
// workgroup's rows of both operands are a step. LDS holds RING = 4 steps: a step's tiles come by LDS-direct loads (a tile as it lies: a
// wavefront reads and writes 1024 consecutive bytes, no bank twice), asked for three steps ahead and waited for before the step ahead of
// theirs (a second chunk: before theirs), so that a step can fetch the next one's first fragments ahead of the barrier between them. A separate array a step: the
// compiler then knows that reading one does not wait for the loads into another. k past the matrix has scale 0 on both sides: 2^-254 of
// anything is nothing in FP32, so what is read in the place of its codes does not matter.
struct MxOperand {  // tiles from the workgroup's first, `left` of them there (those behind: the last again, not to be stored)
  const uint8_t *codes, *scales;
  int left;
};
template <int WM, int WN, int MT, int NT>
struct MxRing {
  static constexpr int WAVES = WM * WN, TA = WM * MT, TB = WN * NT, T = TA + TB, SCALES = MT + NT;
  static constexpr int BUFFER = 2 * T * 64;  // [2 chunks][A tiles, B tiles][64]
  static_assert(TB % WAVES == 0);
  static constexpr bool IN_PLACE = MT * NT > 8;  // the products in asm, which the compiler does not see
  static constexpr int ASKS_A = (2 * TA + WAVES - 1) / WAVES, ASKS_B = (2 * TB + WAVES - 1) / WAVES, ASKS = ASKS_A + ASKS_B;  // tiles a wavefront asks for a step
  static constexpr int LATE = ASKS_B / 2 + (TA % WAVES == 0 ? ASKS_A / 2 : 0);  // of those, what is of a step's second chunk for certain

  // acc = the sums over quads q0 .. q1 - 1 of the matrices' chunks and quads. The buffers are separate arrays of LDS, free
  // again when it returns.
  static __device__ __forceinline__ void run(i32x4_t (&buf0)[BUFFER], i32x4_t (&buf1)[BUFFER], i32x4_t (&buf2)[BUFFER], i32x4_t (&buf3)[BUFFER], const MxOperand& a,
                                             const MxOperand& b, int chunks, int quads, int q0, int q1, f32x16_t (&acc)[MT][NT]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    const int row_bytes = chunks * 1024, left_a = min(TA, a.left), left_b = min(TB, b.left);
    const __amdgpu_buffer_rsrc_t rows_a = mx_rows(a.codes, left_a * row_bytes), rows_b = mx_rows(b.codes, left_b * row_bytes);
    // piece `wave + j * WAVES` of a step's 2 TA (2 TB): tile (that % TA) of chunk (that / TA); past the last piece, tile or chunk: the last again
#define MX_ASK_OF(ROWS, TILES, LEFT, FIRST, BUF, S, J)                                                                                    \
    {                                                                                                                                       \
      const int piece = min(wave + (J) * WAVES, 2 * TILES - 1), chunk = piece / TILES, tile = piece - chunk * TILES;                          \
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ROWS, (mx_lds_t)(BUF + (chunk * T + FIRST + tile) * 64), 16, lane * 16,                       \
                                               min(tile, LEFT - 1) * row_bytes + min(2 * (S) + chunk, chunks - 1) * 1024, 0, 0);            \
    }
    // The pieces of chunk 0 first, B's and A's; then the LATE ones, which are of chunk 1 alone. (Where A's are not whole pieces a wavefront and chunk,
    // all of them go with the first.)
#define MX_ASK(BUF, S, J)                                                                  \
    if constexpr ((J) < ASKS_B / 2) {                                                        \
      MX_ASK_OF(rows_b, TB, left_b, TA, BUF, S, J)                                           \
    } else if constexpr ((J) < ASKS - LATE) {                                                \
      MX_ASK_OF(rows_a, TA, left_a, 0, BUF, S, (J) - ASKS_B / 2)                             \
    } else if constexpr ((J) < ASKS - LATE + ASKS_B / 2) {                                   \
      MX_ASK_OF(rows_b, TB, left_b, TA, BUF, S, (J) - (ASKS - LATE) + ASKS_B / 2)            \
    } else {                                                                                 \
      MX_ASK_OF(rows_a, TA, left_a, 0, BUF, S, (J) - (ASKS - LATE) - ASKS_B / 2 + ASKS_A / 2) \
    }

    // the scales of this wavefront's tiles, a quad at a time
    const int scale_bytes = quads * 256, first_sa = min(wm * MT, left_a - 1), first_sb = min(wn * NT, left_b - 1);
    const int left_sa = min(MT, left_a - first_sa), left_sb = min(NT, left_b - first_sb);
    const __amdgpu_buffer_rsrc_t scales_a = mx_rows(a.scales + (int64_t)first_sa * scale_bytes, left_sa * scale_bytes);
    const __amdgpu_buffer_rsrc_t scales_b = mx_rows(b.scales + (int64_t)first_sb * scale_bytes, left_sb * scale_bytes);
    uint32_t now[SCALES], next[SCALES];  // A's, then B's
    auto scale = [&](int t, int q) {
      next[t] = t < MT ? __builtin_amdgcn_raw_buffer_load_b32(scales_a, lane * 4, min(t, left_sa - 1) * scale_bytes + q * 256, 0)
                       : __builtin_amdgcn_raw_buffer_load_b32(scales_b, lane * 4, min(t - MT, left_sb - 1) * scale_bytes + q * 256, 0);
    };
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

#pragma unroll
    for (int t = 0; t < SCALES; t++) scale(t, q0);
    mx_unrolled<ASKS>([&](auto j) { MX_ASK(buf0, 2 * q0, j.value) });
    mx_unrolled<ASKS>([&](auto j) { MX_ASK(buf1, 2 * q0 + 1, j.value) });
    mx_unrolled<ASKS>([&](auto j) { MX_ASK(buf2, 2 * q0 + 2, j.value) });
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ASKS + LATE) : "memory");
    __builtin_amdgcn_s_barrier();
    // a step: for each of its two chunks and each tile of B, the products with all tiles of A. Fragments come ahead of their use: B's two
    // groups of products, A's a chunk.
    constexpr int GROUPS = 2 * NT, AHEAD = GROUPS < 3 ? 1 : 2;
    i32x4_t fa[2][MT], fb[4];
    auto a_at = [&](const i32x4_t* buf, int chunk, int i) { return buf[(chunk * T + wm * MT + i) * 64 + lane]; };
    auto b_at = [&](const i32x4_t* buf, int group) { return buf[(group / NT * T + TA + wn * NT + group % NT) * 64 + lane]; };
#pragma unroll
    for (int i = 0; i < MT; i++) fa[0][i] = a_at(buf0, 0, i);
#pragma unroll
    for (int j = 0; j < AHEAD; j++) fb[j] = b_at(buf0, j);
    // What the step asks of memory (at a quad's first step the next quad's scales, then its tiles three steps on) goes out between the products: in
    // front of them all, it and the barrier would leave the matrix cores idle for a fifth of the step. At its end what may still be on its way is
    // the step's own and the step's before LATE ones: the next step reads its own tiles, asked for two steps ago, and chunk 0 of the one behind it. (All of
    // that one waited for: 2048 rows of 25600 x 5120 148 us, so 144.5.) The wait counts loads, so every load of the step has to be made: the scales of a quad that no
    // step takes (MORE = 0) are not asked for, where the compiler would drop them and the wait leave LATE tiles of the next step on their way
    // (tests/test_mxfp4_ring_waits.py counts them in the machine code).
#define MX_STEP(CUR, NEXT, ASKED, S, ODD, MORE)                                                                                                         \
    mx_unrolled<GROUPS>([&](auto group) {                                                                                                               \
      constexpr int v = group.value, u = v / NT, j = v % NT, ring = (ODD) * GROUPS + v;                                                                 \
      fb[(ring + AHEAD) & 3] = v + AHEAD < GROUPS ? b_at(CUR, v + AHEAD) : b_at(NEXT, v + AHEAD - GROUPS);                                              \
      _Pragma("unroll") for (int i = j * MT / NT; i < (j + 1) * MT / NT; i++) fa[1 - u][i] = u == 0 ? a_at(CUR, 1, i) : a_at(NEXT, 0, i);               \
      mx_unrolled<MT>([&](auto tile) {                                                                                                                  \
        constexpr int i = tile.value, at = v * MT + i;  /* the step's product */                                                                        \
        if constexpr (IN_PLACE) {                                                                                                                       \
          mx_mfma_in_place<2 * (ODD) + u>(acc[i][j], fb[ring & 3], fa[u][i], now[MT + j], now[i]);                                                      \
        } else {                                                                                                                                        \
          acc[i][j] = mx_mfma<2 * (ODD) + u, 2 * (ODD) + u>(fb[ring & 3], now[MT + j], fa[u][i], now[i], acc[i][j]);                                    \
        }                                                                                                                                               \
        constexpr int ALL = GROUPS * MT, FIRST = (ALL + 3) / 4, H = (ODD) ? 0 : FIRST, W = ALL - FIRST;  /* asked for behind products H .. H + W - 1 */ \
        constexpr int before = at < H ? 0 : at - H >= W ? ASKS : (at - H) * ASKS / W;                                                                   \
        constexpr int after = at < H ? 0 : at + 1 - H >= W ? ASKS : (at + 1 - H) * ASKS / W;                                                            \
        if constexpr (!(ODD) && (MORE)) {                                                                                                               \
          constexpr int from = at >= H ? SCALES : at * SCALES / H, to = at >= H ? SCALES : (at + 1) * SCALES / H;                                       \
          mx_unrolled<to - from>([&](auto k) { scale(from + k.value, min((S) / 2 + 1, quads - 1)); });                                                  \
        }                                                                                                                                               \
        mx_unrolled<after - before>([&](auto k) { MX_ASK(ASKED, (S) + 3, before + k.value) });                                                          \
        __builtin_amdgcn_sched_barrier(0);                                                                                                              \
      });                                                                                                                                               \
    });                                                                                                                                                 \
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ODD) || !(MORE) ? ASKS + LATE : ASKS + LATE + SCALES) : "memory");                                        \
    __builtin_amdgcn_s_barrier();                                                                                                                       \
    __builtin_amdgcn_sched_barrier(0);
#define MX_QUAD                                                               \
    _Pragma("unroll") for (int t = 0; t < SCALES; t++) now[t] = next[t];
    int q = q0;
    for (; q + 1 < q1; q += 2) {
      MX_QUAD
      MX_STEP(buf0, buf1, buf3, 2 * q, 0, 1)
      MX_STEP(buf1, buf2, buf0, 2 * q + 1, 1, 1)
      MX_QUAD
      MX_STEP(buf2, buf3, buf1, 2 * q + 2, 0, 1)
      MX_STEP(buf3, buf0, buf2, 2 * q + 3, 1, 1)
      if (IN_PLACE) mx_sums_done();
    }
    if (q < q1) {
      MX_QUAD
      MX_STEP(buf0, buf1, buf3, 2 * q, 0, 0)
      MX_STEP(buf1, buf2, buf0, 2 * q + 1, 1, 0)
      if (IN_PLACE) mx_sums_done();
    }
#undef MX_QUAD
#undef MX_STEP
#undef MX_ASK
#undef MX_ASK_OF
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was asked for past the end arrives before the workgroup leaves its LDS
    if constexpr (IN_PLACE) {
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) asm volatile("" : "+a"(acc[i][j]));
    }
    __builtin_amdgcn_s_barrier();  // every wavefront has left the ring
  }
};

// 32 rows x NT tiles of a wavefront's sums, stored. A lane holds four columns of one row, 8 or 16 bytes: stored as they are, an instruction
// would touch 32 rows' lines. They go through the wavefront's own part of LDS and leave as whole rows of NT x 32 columns, 16 bytes a
// lane; a row's 16-byte pieces are XORed with its number so that neither way meets a bank twice. Where rows do not start on 16 bytes the stores do not either, and a
// row's last piece is stored by columns. (Each lane its four columns, one by one, there: 2000 rows of 2049 x 2048 30.4 us, so 17.4.) row_at(r):
// where column 0 of the tile's row r goes, or null.
template <typename Y, int NT, class RowAt>
__device__ __forceinline__ void mx_store_rows(i32x4_t* place, int64_t columns, int64_t n0, const f32x16_t (&sums)[NT], RowAt&& row_at) {
  constexpr int PIECES = NT * MX_ROWS * (int)sizeof(Y) / 16, ROWS = 64 / PIECES > 0 ? 64 / PIECES : 1, EACH = 16 / (int)sizeof(Y);
  const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
  uint8_t* bytes = reinterpret_cast<uint8_t*>(place);
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int at = (MX_ROWS * j + 8 * q + 4 * g) * (int)sizeof(Y), piece = (at / 16) ^ (r & (PIECES - 1));
      mx_store4<Y>(reinterpret_cast<Y*>(bytes + (r * PIECES + piece) * 16 + at % 16), mx_quarter(sums[j], q), 4, true);
    }
  auto store = [&](auto whole) {
#pragma unroll
    for (int first = 0; first < MX_ROWS; first += ROWS) {
      const int row = first + lane / PIECES, piece = lane % PIECES;
      const int64_t n = n0 + piece * EACH;
      const i32x4_t v = place[row * PIECES + (piece ^ (row & (PIECES - 1)))];
      Y* to = row_at(row);
      if (!to || n >= columns) continue;
      if constexpr (decltype(whole)::value) {
        *reinterpret_cast<i32x4_t*>(to + n) = v;
      } else if (n + EACH <= columns) {
        reinterpret_cast<MxLoose<i32x4_t, Y>*>(to + n)->v = v;
      } else {
        typedef __attribute__((ext_vector_type(EACH))) Y ys_t;
        const ys_t y = __builtin_bit_cast(ys_t, v);
#pragma unroll
        for (int e = 0; e < EACH - 1; e++)
          if (n + e < columns) to[n + e] = y[e];
      }
    }
  };
  if (columns % EACH == 0) {
    store(std::true_type());
  } else {
    store(std::false_type());
  }
}

}  // namespace hb
