"""MI355X skinny decode GEMM kernels and the cache operators between them
(import surface mirrors the reference's engine/kernels/__init__.py:1-8)."""

from .attention import CacheAttention, CacheEviction, qk_norm_rope, rope_table
from .cache import DecodeCache
from .gemm import (Gemv, SkinnyGateUp, SkinnyMatmul, SkinnySelect, add_rms_norm, gemm_into, normed_fused, pick_gateup, pick_matmul,
                   pick_normed, plan, select_fused, select_plan, tune_projection)

__all__ = ["CacheAttention", "CacheEviction", "DecodeCache", "Gemv", "SkinnyGateUp", "SkinnyMatmul", "SkinnySelect", "add_rms_norm",
           "gemm_into", "normed_fused", "pick_gateup", "pick_matmul", "pick_normed", "plan", "qk_norm_rope", "rope_table",
           "select_fused", "select_plan", "tune_projection"]
