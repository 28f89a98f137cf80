"""HIP (gfx950) kernels behind the reference's ``slipstream.kernels`` call signatures."""

from slipstream_amd.kernels.block_copy import copy_blocks, swap_blocks
from slipstream_amd.kernels.fp8_gemm import fp8_gemm
from slipstream_amd.kernels.fp8_rows import quantize_fp8
from slipstream_amd.kernels.int8_gemm import w8a8_gemm
from slipstream_amd.kernels.int8_rows import fused_rmsnorm_int8, fused_swiglu_int8, quantize_int8
from slipstream_amd.kernels.latent_attention import (
    latent_attention_decode,
    latent_attention_expanded,
    latent_attention_varlen,
)
from slipstream_amd.kernels.latent_cache import latent_rope_and_cache
from slipstream_amd.kernels.paged_attention import (
    attention_status,
    paged_attention,
    paged_attention_decode,
    paged_attention_prefill,
    paged_attention_shared_prefix,
    paged_attention_varlen,
)
from slipstream_amd.kernels.norm_act import fused_rmsnorm, fused_swiglu
from slipstream_amd.kernels.packed_step import packed_attention
from slipstream_amd.kernels.quant_gemm import w4a16_gemm
from slipstream_amd.kernels.reshape_and_cache import reshape_and_cache
from slipstream_amd.kernels.rope_cache import rope_and_cache

__all__ = [
    "attention_status",
    "copy_blocks",
    "fp8_gemm",
    "fused_rmsnorm",
    "fused_rmsnorm_int8",
    "fused_swiglu",
    "fused_swiglu_int8",
    "latent_attention_decode",
    "latent_attention_expanded",
    "latent_attention_varlen",
    "latent_rope_and_cache",
    "packed_attention",
    "paged_attention",
    "paged_attention_decode",
    "paged_attention_prefill",
    "paged_attention_shared_prefix",
    "paged_attention_varlen",
    "quantize_fp8",
    "quantize_int8",
    "reshape_and_cache",
    "rope_and_cache",
    "swap_blocks",
    "w4a16_gemm",
    "w8a8_gemm",
]
