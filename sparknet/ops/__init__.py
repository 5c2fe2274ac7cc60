"""Hand-written sm_100a ops: tcgen05 GEMM (bf16 and block-scaled fp8), the decode GEMM
(few tokens, split-K, fused SwiGLU / RoPE epilogues), the fused prefill collectives
(all-gather -> GEMM, GEMM -> reduce-scatter), split-KV decode attention, the fused
decode all-reduce + RMSNorm, and the paged 8-bit KV cache (page planning, append, read and
decode attention)."""

from .attention import decode_attention
from .decode_gemm import DecodeGemm, interleave_gate_up, linear, split_gate_up
from .gemm import gemm
from .kv_cache import Fp8KVCache, kv_append, kv_read, rope_kv_append
from .paged_attention import paged_decode_attention
from .paging import PagePlan, PageTable, plan_pages
from .prefill import ag_gemm, ag_gemm_fp8, ag_gemm_reference, gemm_rs, gemm_rs_fp8, gemm_rs_reference

__all__ = ["DecodeGemm", "ag_gemm", "ag_gemm_fp8", "ag_gemm_reference", "gemm", "gemm_rs", "gemm_rs_fp8",
           "gemm_rs_reference",
           "decode_attention", "interleave_gate_up", "linear", "split_gate_up",
           "Fp8KVCache", "PagePlan", "PageTable", "kv_append", "kv_read", "paged_decode_attention", "plan_pages",
           "rope_kv_append"]
