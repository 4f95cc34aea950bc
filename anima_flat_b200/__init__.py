"""anima_flat_b200 — the fused DiT layer ops of anima-flat, hand-written for B200 (sm_100a).

Public functions mirror src/kernels/{adaln,fp8,rope,ctx_scale,rms}.py of the reference:

    adaln, residual_adaln                         (AdaLN modulate, gated residual)
    adaln_fp8, residual_adaln_fp8, rowquant       (per-row FP8 e4m3 quantisation)
    qkv_norm_rope, head_norm                      (q/k RMSNorm + 3D RoPE)
    ctx_scale                                     (trimmed cross-attention gain)
    ctx_scale_rowquant                            (the gain and FP8 quantisation in one pass)
    rms_silu, add_rms_silu, shuffle_rms_silu      (VAE channel RMS norm + SiLU)

and, without a counterpart there:

    rowquant_int8, quantize_weight_int8, int8_linear, int8_linear_dx
                                                  (8-bit integer linear layers)
    gelu_int8, gelu_int8_bwd, int8_wgrad, int8_restore (8-bit activation checkpoints)
    int8_lora_mlp                                 (an MLP on these, with adapters)
    sandwich_norm, sandwich_norm_int8, sandwich_norm_bwd
                                                  (norms before and after a block)

All run through the C-ABI library ``lib/libanima_flat_b200.so`` (see
``include/anima_flat_b200.h``); there is no CPU fallback.
"""

from .kernels.adaln import adaln, residual_adaln
from .kernels.ctx_scale import ctx_scale, ctx_scale_rowquant
from .kernels.fp8 import FP8, FP8_MAX, adaln_fp8, residual_adaln_fp8, rowquant
from .kernels.int8 import (
    Int8Weight,
    gelu_int8,
    gelu_int8_bwd,
    int8_linear,
    int8_linear_dx,
    int8_restore,
    int8_wgrad,
    quantize_weight_int8,
    rowquant_int8,
)
from .kernels.int8_mlp import LoRA, int8_lora_mlp
from .kernels.rms import add_rms_silu, rms_silu, shuffle_rms_silu
from .kernels.rope import head_norm, qkv_norm_rope
from .kernels.sandwich import sandwich_norm, sandwich_norm_bwd, sandwich_norm_int8
from .tables import rope_tables

__all__ = [
    "FP8",
    "FP8_MAX",
    "Int8Weight",
    "LoRA",
    "adaln",
    "adaln_fp8",
    "add_rms_silu",
    "ctx_scale",
    "ctx_scale_rowquant",
    "gelu_int8",
    "gelu_int8_bwd",
    "head_norm",
    "int8_linear",
    "int8_linear_dx",
    "int8_lora_mlp",
    "int8_restore",
    "int8_wgrad",
    "qkv_norm_rope",
    "quantize_weight_int8",
    "residual_adaln",
    "residual_adaln_fp8",
    "rms_silu",
    "rope_tables",
    "rowquant",
    "rowquant_int8",
    "sandwich_norm",
    "sandwich_norm_bwd",
    "sandwich_norm_int8",
    "shuffle_rms_silu",
]
