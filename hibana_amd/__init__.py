"""MI355X-native quantized-weight linear and MoE expert kernels behind the reference's `hibana.kernels` op signatures.

  hibana_amd.kernels.w3       W3Weight, pack / pack_codes / codes / group_scales / dequantize / w3_linear / attach
  hibana_amd.kernels.w3_moe   W3Experts, w3_moe, fc1_order, moe layer
  hibana_amd.kernels.ops      nvfp4_linear, w3_decode, silu_and_mul, moe_combine(_pairs), route_topk, route_experts(_grad), adapted_linear
  hibana_amd.kernels.mxfp4    Mxfp4, quantize / dequantize: the microscaled four-bit format (with ops.mxfp4_linear, silu_mul_quant_mxfp4)
  hibana_amd.kernels.mxfp4_moe  Mxfp4Experts, mxfp4_moe: routed experts in it
  hibana_amd.kernels.adapters Adapters, add / grads: low-rank adapters of many requests beside a shared projection
  hibana_amd.weights          Nvfp4Linear, Mxfp4Linear, unpack_fp4, block-scale swizzle, the Linear protocol

The compute is hand-written HIP for gfx950 in hibana_amd/csrc, loaded through a C ABI (include/hibana_hip.h).
There is no CPU fallback: calling an op without the built library or without a GPU raises.
"""
__version__ = "0.1.0"
