"""helexa_amd: MI355X (gfx950) implementation of helexa neuron's Qwen3-Next
sparse-MoE block behind a C ABI (include/hx_moe.h, libhxmoe.so)."""
from .moe import (BF16, F16, F32, F8_E4M3, HX_DEVICE, HX_HOST, MXFP4, Q4_K, Q6_K, Q8_0, F8Linear, HxError,
                  Qwen3_5MoeBlock, TextConfig, balance_loss, balance_workspace_size, dequantize, expert_counts, lib,
                  quantize, quantize_activations, quantize_f8, row_bytes)

__all__ = ["BF16", "F16", "F32", "F8_E4M3", "F8Linear", "HX_DEVICE", "HX_HOST", "MXFP4", "Q4_K", "Q6_K", "Q8_0",
           "HxError", "Qwen3_5MoeBlock", "TextConfig", "balance_loss", "balance_workspace_size", "dequantize",
           "expert_counts", "lib", "quantize", "quantize_activations", "quantize_f8", "row_bytes"]
