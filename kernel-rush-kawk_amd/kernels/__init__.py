"""MI355X skinny decode GEMM kernels, the cache operators between them, the paged
cache of many requests and their low-rank adapters (import surface mirrors the
reference's engine/kernels/__init__.py:1-8)."""

from .adapters import LowRankAdapters
from .attention import CacheAttention, CacheEviction, qk_norm_rope, rope_table
from .cache import DecodeCache
from .gemm import (Gemv, SkinnyGateUp, SkinnyMatmul, SkinnySelect, add_rms_norm, gemm_into, normed_fused, pick_gateup, pick_matmul,
                   pick_normed, plan, select_fused, select_plan, tune_projection)
from .paged import PagedAttention, PageTables, paged_qk_norm_rope, paged_workspace_bytes
from .serve import AdapterSet, PagedCache

__all__ = ["AdapterSet", "CacheAttention", "CacheEviction", "DecodeCache", "Gemv", "LowRankAdapters", "PagedAttention", "PagedCache",
           "PageTables", "SkinnyGateUp", "SkinnyMatmul", "SkinnySelect", "add_rms_norm", "gemm_into", "normed_fused", "paged_qk_norm_rope",
           "paged_workspace_bytes", "pick_gateup", "pick_matmul", "pick_normed", "plan", "qk_norm_rope", "rope_table", "select_fused",
           "select_plan", "tune_projection"]
