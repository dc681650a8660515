"""helion_b200: B200-native (sm_100a) FP8 GEMM and FP8 attention behind Helion's example signatures.

Public surface:
    fp8_gemm, fp8_attention         -- operators on torch CUDA tensors (helion_b200.ops)
    preprocess_fp8_attention_inputs -- q, k, v -> e4m3 in one kernel, with the reference's views
    int8_gemm                       -- int8 sibling of fp8_gemm (scales for each token and channel)
    rms_norm_quantize               -- RMS norm with the residual's addition, 8-bit codes and row scales out
    quantize_rows                   -- 16- / 32-bit rows -> 8-bit codes (e4m3 or int8) and row scales
    gated_matmul                    -- act(x Wg) * (x Wu) in one kernel, fp16 / bf16 with gradients
    gated_gemm                      -- the same with e4m3 / int8 operands and scales
    HostGemm                        -- fp8_gemm on pinned host buffers with overlapped PCIe copies
    matmul                          -- fp16 / bf16 sibling of fp8_gemm with the bias / ReLU epilogues
    attention                       -- fp16 / bf16 sibling of fp8_attention (examples/attention.py)
    DropInKernel                    -- object with the protocol of helion.runtime.kernel.Kernel
                                       that the reference's test and benchmark harness touch
There is no CPU, Triton or PyTorch fallback: calls fail loudly when the CUDA library is missing.
"""
from __future__ import annotations

from ._lib import DeviceWaitTimeout, LibraryNotBuiltError
from .gated import gated_gemm, gated_matmul
from .host_io import HostGemm
from .ops import (
    attention,
    attention_into,
    fp8_attention,
    fp8_gemm,
    int8_gemm,
    matmul,
    preprocess_fp8_attention_inputs,
    quantize_rows,
    rms_norm_quantize,
)

__all__ = [
    "fp8_gemm",
    "fp8_attention",
    "attention_into",
    "preprocess_fp8_attention_inputs",
    "int8_gemm",
    "rms_norm_quantize",
    "quantize_rows",
    "gated_matmul",
    "gated_gemm",
    "HostGemm",
    "matmul",
    "attention",
    "DeviceWaitTimeout",
    "LibraryNotBuiltError",
]
