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

constexpr int MX_SLOT_ROWS = MX_ROWS;

// A slot's (up to 32 rows of an expert) product with NT tiles of weight rows, K split among the workgroup's wavefronts: their sums in LDS.
// row_of: the row of the activations that is the slot's row r.
template <int NT, int RUN, class Row>
__device__ __forceinline__ void mx_slot_product(const MxMoe& p, const uint8_t* w, int t0, int rows, Row&& row_of, f32x4_t* part) {
  MxStream<NT, RUN> s(w, MxLayout(p.n, p.k), t0, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), p.waves);
  const MxActs acts(part, rows, p.k);
  for (int i = threadIdx.x; i < rows * acts.groups; i += blockDim.x) {
    const int r = i / acts.groups, group = i - r * acts.groups;
    const int64_t row = row_of(r);
    acts.put(r, group, p.aq + row * (p.k / 2), p.as + row * acts.groups);
  }
  __syncthreads();
  s.run(acts);
  mx_hand_over<NT>(part, s.acc);
}

// fc1: a workgroup 32 columns of h of a slot (gated: the up tile and its gate tile); h leaves rounded to the format. Four lanes share a
// row's group: wavefront q holds its columns 8 q + 4 g .. + 3 (g: the lane's half) ... joined through LDS.
template <bool GATED>
__global__ __launch_bounds__(512) void mx_fc1_kernel(MxMoe p) {
  constexpr int NT = GATED ? 2 : 1;
  extern __shared__ f32x4_t part[];
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * (int)blockIdx.y;
  const int rows = entry[2], p0 = entry[1];
  if (rows == 0) return;
  const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
  mx_slot_product<NT, 4>(p, p.w + entry[0] * p.expert_bytes, blockIdx.x * NT, rows, [&](int i) { return (int64_t)(p.order[p0 + i] / p.topk); }, part);
  const int q = threadIdx.x >> 6;  // the launch has at least four wavefronts
  float h[4];
  uint32_t top = 0;
  if (q < 4) {
    const f32x4_t up = mx_joined<NT>(part, p.waves, threadIdx.x), gate = GATED ? mx_joined<NT>(part, p.waves, 256 * (NT - 1) + threadIdx.x) : up;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float u = fmaxf(up[j], 0.f);
      h[j] = GATED ? gate[j] / (1.0f + expf(-gate[j])) * up[j] : (up[j] != up[j] ? up[j] : u * u);
      top = max(top, __float_as_uint(h[j]) & 0x7fffffffu);
    }
  }
  __syncthreads();  // the sums are read: their place takes the quarters' largest magnitudes
  uint32_t* tops = reinterpret_cast<uint32_t*>(part);
  if (q < 4) tops[q * 64 + lane] = top;
  __syncthreads();
  if (q >= 4 || r >= rows) return;
#pragma unroll
  for (int v = 0; v < 4; v++) top = max(top, max(tops[v * 64 + r], tops[v * 64 + 32 + r]));
  const uint32_t byte = mx_scale_byte(top);
  const float s = mx_scale_value(byte);
  const int64_t inter = GATED ? p.n / 2 : p.n, pos = p0 + r;
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, h[0], h[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, h[2], h[3], s, 1);
  *reinterpret_cast<uint16_t*>(p.hq + pos * (inter / 2) + 16 * blockIdx.x + 4 * q + 2 * g) = byte == 255u ? 0 : (uint16_t)c;
  if (q == 0 && g == 0) p.hs[pos * (inter / 32) + blockIdx.x] = (uint8_t)byte;
}

// fc2: a workgroup NT tiles of output columns of a slot, written by pair.
template <typename Y, int NT>
__global__ __launch_bounds__(512) void mx_fc2_kernel(MxMoe p) {
  extern __shared__ f32x4_t part[];
  const int32_t* entry = p.plan + PLAN_HEADER + 4 * (int)blockIdx.y;
  const int rows = entry[2], p0 = entry[1];
  if (rows == 0) return;
  const int r = threadIdx.x & 31;
  mx_slot_product<NT, 2>(p, p.w + entry[0] * p.expert_bytes, blockIdx.x * NT, rows, [&](int i) { return (int64_t)p0 + i; }, part);
  const int64_t pair = r < rows ? p.order[p0 + r] : 0;
  for (int i = threadIdx.x; i < NT * 256; i += blockDim.x) {
    const f32x4_t sum = mx_joined<NT>(part, p.waves, i);
    const int n = (blockIdx.x * NT + (i >> 8)) * MX_ROWS + 8 * ((i >> 6) & 3) + 4 * ((i & 63) >> 5);
    if (r >= rows || n >= p.n) continue;  // n and p.n are multiples of four
    typedef __attribute__((ext_vector_type(4))) Y y4_t;
    *reinterpret_cast<y4_t*>(static_cast<Y*>(p.y) + pair * p.n + n) = y4_t{(Y)sum[0], (Y)sum[1], (Y)sum[2], (Y)sum[3]};
  }
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
  const int64_t pairs = (int64_t)m * topk, slots = moe_max_slots(pairs, experts->experts, 0, MX_SLOT_ROWS);
  if (slots > 65535) return HB_EINVAL;
  hipStream_t s = as_stream(stream);
  if (int e = moe_launch_plan(ids, pairs, experts->base, experts->experts, 0, ws.plan, s, MX_SLOT_ROWS)) return e;
  if (int e = hb_mxfp4_quantize(x, HB_BF16, m, experts->hidden, ws.xq, ws.xs, stream)) return e;
  const MxLayout l1(fc1_rows(experts), experts->hidden), l2(experts->hidden_out, experts->inter);
  MxMoe p1{static_cast<const uint8_t*>(experts->fc1), l1.bytes(), ws.xq, ws.xs, ws.plan.plan, ws.plan.order, fc1_rows(experts), experts->hidden, topk,
           8, ws.hq, ws.hs, nullptr};
  MxMoe p2{static_cast<const uint8_t*>(experts->fc2), l2.bytes(), ws.hq, ws.hs, ws.plan.plan, ws.plan.order, experts->hidden_out, experts->inter, topk,
           4, nullptr, nullptr, sum ? ws.y : out};
  const int most = (int)std::min<int64_t>(MX_SLOT_ROWS, pairs);
  const size_t acts1 = MxActs::bytes(most, experts->hidden), acts2 = MxActs::bytes(most, experts->inter);
  if (acts1 > 64 * 1024 || acts2 > 64 * 1024) return HB_EINVAL;
  const dim3 grid1((unsigned)(experts->inter / 32), (unsigned)slots), grid2((unsigned)((l2.tiles + 1) / 2), (unsigned)slots);
  if (experts->gated) {
    HB_LAUNCH((mx_fc1_kernel<true>), grid1, dim3(64 * p1.waves), std::max(acts1, (size_t)p1.waves * 2 * 4096), s, p1);
  } else {
    HB_LAUNCH((mx_fc1_kernel<false>), grid1, dim3(64 * p1.waves), std::max(acts1, (size_t)p1.waves * 4096), s, p1);
  }
  if (mode == HB_MOE_PAIRS_BF16) {
    HB_LAUNCH((mx_fc2_kernel<__bf16, 2>), grid2, dim3(64 * p2.waves), std::max(acts2, (size_t)p2.waves * 2 * 4096), s, p2);
  } else {
    HB_LAUNCH((mx_fc2_kernel<float, 2>), grid2, dim3(64 * p2.waves), std::max(acts2, (size_t)p2.waves * 2 * 4096), s, p2);
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
