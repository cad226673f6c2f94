// Routed experts on microscaled four-bit weights and activations.
//
//   xq = the rows rounded to the format;  per routed pair (row, expert):
//   h = silu(gate xq) * (up xq) or relu(up xq)^2 in FP32, rounded to the format;  y = down h;  out = the weighted sum of a row's y.
#include <algorithm>

#include "mxfp4.hpp"
#include "stream_common.hpp"

namespace hb {

struct MxMoe {
  const uint8_t* w;        // the experts' stacked tile layouts
  int64_t expert_bytes;
  const uint8_t* aq;       // activation codes by rows, [.., k / 2] ...
  const uint8_t* as;       // ... and scales [.., k / 32]
  const int32_t* plan;
  const int32_t* order;
  int n, k, topk, waves;
  uint8_t* hq;             // fc1: h in sorted order
  uint8_t* hs;
  void* y;                 // fc2: [pairs, n]
};

// One slot's (up to sixteen rows of an expert) product with NT tiles of weight rows; K split among the workgroup's wavefronts, their
// sums added through LDS in wavefront order: sums[i] of the first NT * 64 threads, tile i / 64, lane i % 64.
template <int NT>
__device__ __forceinline__ f32x4_t mx_slot_sums(const MxMoe& p, const uint8_t* w, int t0, const uint8_t* codes, const uint8_t* scales, bool real, f32x4_t* part) {
  const MxLayout at(p.n, p.k);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
  const int c0 = at.chunks * wave / p.waves, c1 = at.chunks * (wave + 1) / p.waves;
  f32x4_t acc[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int c = c0; c < c1; c++) {
    i32x4_t b[NT], a = {0, 0, 0, 0};
    uint32_t sb[NT], sa = 0;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int tile = min(t0 + t, at.tiles - 1);  // past the last: not stored
      b[t] = *reinterpret_cast<const i32x4_t*>(w + (((int64_t)tile * at.chunks + c) * 64 + lane) * 16);
      sb[t] = *reinterpret_cast<const uint32_t*>(w + at.codes() + ((int64_t)tile * at.quads + (c >> 2)) * 256 + lane * 4) >> (8 * (c & 3));
    }
    if (real && 4 * c + g < p.k / 32) {
      sa = scales[4 * c + g];
      a = *reinterpret_cast<const i32x4_t*>(codes + 16 * (4 * c + g));
    }
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = mx_mfma(b[t], sb[t], a, sa, acc[t]);
  }
#pragma unroll
  for (int t = 0; t < NT; t++) part[(wave * NT + t) * 64 + lane] = acc[t];
  __syncthreads();
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  if (threadIdx.x < NT * 64) {
    sum = part[threadIdx.x];
    for (int v = 1; v < p.waves; v++) sum += part[v * NT * 64 + threadIdx.x];
  }
  return sum;
}

// fc1: a workgroup 32 columns of h (gated: two pairs of an up and a gate tile) of a slot; h leaves rounded to the format.
template <bool GATED>
__global__ __launch_bounds__(1024) void mx_fc1_kernel(MxMoe p) {
  constexpr int NT = GATED ? 4 : 2;
  extern __shared__ f32x4_t part[];
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * (int)blockIdx.y;
  const int rows = entry[2], p0 = entry[1];
  if (rows == 0) return;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int64_t row = r < rows ? p.order[p0 + r] / p.topk : 0;
  const f32x4_t sum = mx_slot_sums<NT>(p, p.w + entry[0] * p.expert_bytes, blockIdx.x * NT, p.aq + row * (p.k / 2), p.as + row * (p.k / 32), r < rows, part);
  __syncthreads();
  if (threadIdx.x < NT * 64) part[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  // a lane: row r, columns 4 g .. 4 g + 3 and 16 + 4 g .. of the 32
  float h[8];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const f32x4_t up = part[(GATED ? 2 * t : t) * 64 + lane], gate = GATED ? part[(2 * t + 1) * 64 + lane] : up;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float u = fmaxf(up[j], 0.f);
      h[4 * t + j] = GATED ? gate[j] / (1.0f + expf(-gate[j])) * up[j] : (up[j] != up[j] ? up[j] : u * u);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(h[j]) & 0x7fffffffu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 16));
  top = max(top, (uint32_t)__shfl_xor((int)top, 32));
  const uint32_t byte = mx_scale_byte(top);
  const float s = mx_scale_value(byte);
  if (r >= rows) return;
  const int64_t inter = GATED ? p.n / 2 : p.n, pos = p0 + r;
#pragma unroll
  for (int t = 0; t < 2; t++) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, h[4 * t], h[4 * t + 1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, h[4 * t + 2], h[4 * t + 3], s, 1);
    *reinterpret_cast<uint16_t*>(p.hq + pos * (inter / 2) + 16 * blockIdx.x + 8 * t + 2 * g) = byte == 255u ? 0 : (uint16_t)c;
  }
  if (g == 0) p.hs[pos * (inter / 32) + blockIdx.x] = (uint8_t)byte;
}

// fc2: a workgroup 64 output columns of a slot, written by pair.
template <typename Y>
__global__ __launch_bounds__(1024) void mx_fc2_kernel(MxMoe p) {
  constexpr int NT = 4;
  extern __shared__ f32x4_t part[];
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * (int)blockIdx.y;
  const int rows = entry[2], p0 = entry[1];
  if (rows == 0) return;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int64_t pos = p0 + min(r, rows - 1);
  const f32x4_t sum = mx_slot_sums<NT>(p, p.w + entry[0] * p.expert_bytes, blockIdx.x * NT, p.aq + pos * (p.k / 2), p.as + pos * (p.k / 32), r < rows, part);
  const int n = (blockIdx.x * NT + (threadIdx.x >> 6)) * 16 + 4 * g;
  if (threadIdx.x >= NT * 64 || r >= rows || n >= p.n) return;  // n and p.n are multiples of four
  Y* out = static_cast<Y*>(p.y) + (int64_t)p.order[p0 + r] * p.n + n;
#pragma unroll
  for (int j = 0; j < 4; j++) out[j] = (Y)sum[j];
}

namespace {
struct MxWorkspace {
  MoeWorkspace plan;
  uint8_t *xq, *xs, *hq, *hs;
  void* y;
  size_t bytes;
};

MxWorkspace carve(const hb_mxfp4_experts* ex, void* base, int64_t m, int topk, bool sum) {
  const int64_t pairs = m * topk;
  MxWorkspace w{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    uint8_t* ptr = base ? static_cast<uint8_t*>(base) + off : nullptr;
    off += (bytes + 255) & ~(size_t)255;
    return ptr;
  };
  w.plan.plan = reinterpret_cast<int32_t*>(take((PLAN_HEADER + (4 + DONE_PITCH) * moe_max_slots(pairs, ex->experts, 0) + 32) * sizeof(int32_t)));
  w.plan.plan_wide = reinterpret_cast<int32_t*>(take((size_t)64 * ex->experts * sizeof(int32_t)));
  w.plan.order = reinterpret_cast<int32_t*>(take((size_t)pairs * sizeof(int32_t)));
  w.xq = take((size_t)m * (ex->hidden / 2));
  w.xs = take((size_t)m * (ex->hidden / 32));
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
  const int64_t pairs = (int64_t)m * topk, slots = moe_max_slots(pairs, experts->experts, 0);
  if (slots > 65535) return HB_EINVAL;
  hipStream_t s = as_stream(stream);
  if (int e = moe_launch_plan(ids, pairs, experts->base, experts->experts, 0, ws.plan, s)) return e;
  if (int e = hb_mxfp4_quantize(x, HB_BF16, m, experts->hidden, ws.xq, ws.xs, stream)) return e;
  const MxLayout l1(fc1_rows(experts), experts->hidden), l2(experts->hidden_out, experts->inter);
  MxMoe p1{static_cast<const uint8_t*>(experts->fc1), l1.bytes(), ws.xq, ws.xs, ws.plan.plan, ws.plan.order, fc1_rows(experts), experts->hidden, topk,
           std::min(l1.chunks, 8), ws.hq, ws.hs, nullptr};
  MxMoe p2{static_cast<const uint8_t*>(experts->fc2), l2.bytes(), ws.hq, ws.hs, ws.plan.plan, ws.plan.order, experts->hidden_out, experts->inter, topk,
           std::max(4, std::min(l2.chunks, 8)), nullptr, nullptr, sum ? ws.y : out};
  const dim3 grid1((unsigned)(experts->inter / 32), (unsigned)slots), grid2((unsigned)((l2.tiles + 3) / 4), (unsigned)slots);
  p1.waves = std::max(4, p1.waves);
  if (experts->gated) {
    HB_LAUNCH((mx_fc1_kernel<true>), grid1, dim3(64 * p1.waves), (size_t)p1.waves * 4 * 1024, s, p1);
  } else {
    HB_LAUNCH((mx_fc1_kernel<false>), grid1, dim3(64 * p1.waves), (size_t)p1.waves * 2 * 1024, s, p1);
  }
  if (mode == HB_MOE_PAIRS_BF16) {
    HB_LAUNCH((mx_fc2_kernel<__bf16>), grid2, dim3(64 * p2.waves), (size_t)p2.waves * 4 * 1024, s, p2);
  } else {
    HB_LAUNCH((mx_fc2_kernel<float>), grid2, dim3(64 * p2.waves), (size_t)p2.waves * 4 * 1024, s, p2);
  }
  if (sum) {
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
  }
  return launch_status();
}
