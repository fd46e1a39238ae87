"""torch bridge: the hot-path ops as ``torch.library`` custom ops with fake (meta) kernels,
following the reference's bridge (arke/integration/torch_bridge.py:140-181) but without its eager
fallback — the op body always runs the sm_100a kernel.

    register_ops()                      # idempotent
    q, s   = torch.ops.arke.quantize_per_token(x)
    y      = torch.ops.arke.w8a8_gemm(q, s, w, sw)
    yq, s2 = torch.ops.arke.swiglu_fp8(x2)
    o, lse = torch.ops.arke.gqa_fwd(q, k, v, True)
    y      = torch.ops.arke.rope(x4, cos, sin)
    q, k, v = torch.ops.arke.qkv_rope_split(qkv, cos, sin, B, S, Hq, Hkv, D)
    tok, m = torch.ops.arke.fused_linear_ce(h, w_lm, labels, -100)
    q      = torch.ops.arke.qkv_rope_paged_append(qkv, cos, sin, k_cache, v_cache, table, kv_lens, cu_q, Hq)
    o, lse = torch.ops.arke.paged_gqa_fwd(q, k_cache, v_cache, table, kv_lens, cu_q, prefix)
    tok    = torch.ops.arke.sample_tokens(logits, u, 0.8, 50, 0.95, 0.0)
    tok, lp = torch.ops.arke.sample_tokens_logprob(logits, u, temperature_rows=t, top_p_rows=p)
"""
from __future__ import annotations

from typing import Optional

import torch

_REGISTERED = False


def register_ops() -> bool:
    """Registers ``arke::rmsnorm``, ``arke::rmsnorm_quant``, ``arke::quantize_per_token``, ``arke::w8a8_gemm``, ``arke::swiglu_fp8``,
    ``arke::gqa_fwd``, ``arke::rope``, ``arke::qkv_rope_split``, ``arke::fused_linear_ce``, ``arke::qkv_rope_paged_append``,
    ``arke::paged_gqa_fwd``, ``arke::sample_tokens`` and ``arke::sample_tokens_logprob``; returns True when (already) registered."""
    global _REGISTERED
    if _REGISTERED:
        return True
    from . import ops

    @torch.library.custom_op("arke::quantize_per_token", mutates_args=())
    def quantize_per_token(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return ops.quantize_per_token(x)

    @quantize_per_token.register_fake
    def _(x):
        return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)

    @torch.library.custom_op("arke::rmsnorm", mutates_args=())
    def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
        return ops.rmsnorm(x, w, eps=eps)

    @rmsnorm.register_fake
    def _(x, w, eps):
        return torch.empty_like(x)

    @torch.library.custom_op("arke::rmsnorm_quant", mutates_args=())
    def rmsnorm_quant(x: torch.Tensor, residual: torch.Tensor, w: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
        return ops.rmsnorm(x, w, eps=eps, residual=residual, quantize="int8", return_y=False)

    @rmsnorm_quant.register_fake
    def _(x, residual, w, eps):
        return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)

    @torch.library.custom_op("arke::w8a8_gemm", mutates_args=())
    def w8a8_gemm(xq: torch.Tensor, sx: torch.Tensor, w: torch.Tensor, sw: torch.Tensor) -> torch.Tensor:
        return ops.w8a8_gemm(xq, sx, w, sw)

    @w8a8_gemm.register_fake
    def _(xq, sx, w, sw):
        return xq.new_empty((xq.shape[0], w.shape[1]), dtype=torch.bfloat16)

    @torch.library.custom_op("arke::swiglu_fp8", mutates_args=())
    def swiglu_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return ops.swiglu_fp8(x)

    @swiglu_fp8.register_fake
    def _(x):
        return (x.new_empty((*x.shape[:-1], x.shape[-1] // 2), dtype=torch.float8_e4m3fn),
                x.new_empty(x.shape[:-1], dtype=torch.float32))

    @torch.library.custom_op("arke::gqa_fwd", mutates_args=())
    def gqa_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool) -> tuple[torch.Tensor, torch.Tensor]:
        return ops.gqa_fwd(q, k, v, causal=causal)

    @gqa_fwd.register_fake
    def _(q, k, v, causal):
        return torch.empty_like(q), q.new_empty(q.shape[:-1], dtype=torch.float32)

    @torch.library.custom_op("arke::rope", mutates_args=())
    def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        return ops.rope(x, cos, sin)

    @rope.register_fake
    def _(x, cos, sin):
        return torch.empty_like(x, memory_format=torch.contiguous_format)

    @torch.library.custom_op("arke::qkv_rope_split", mutates_args=())
    def qkv_rope_split(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, B: int, S: int, Hq: int, Hkv: int,
                       D: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        return ops.qkv_rope_split(qkv, cos, sin, B, S, Hq, Hkv, D)

    @qkv_rope_split.register_fake
    def _(qkv, cos, sin, B, S, Hq, Hkv, D):
        return (qkv.new_empty((B, Hq, S, D)), qkv.new_empty((B, Hkv, S, D)), qkv.new_empty((B, Hkv, S, D)))

    @torch.library.custom_op("arke::fused_linear_ce", mutates_args=())
    def fused_linear_ce(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor,
                        ignore_index: int) -> tuple[torch.Tensor, torch.Tensor]:
        return ops.fused_linear_ce(x, w, labels, ignore_index=ignore_index)

    @fused_linear_ce.register_fake
    def _(x, w, labels, ignore_index):
        return x.new_empty((x.shape[0],), dtype=torch.float32), x.new_empty((), dtype=torch.float32)

    @torch.library.custom_op("arke::qkv_rope_paged_append", mutates_args=("k_cache", "v_cache"))
    def qkv_rope_paged_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                              block_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: Optional[torch.Tensor], Hq: int,
                              positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        return ops.qkv_rope_paged_append(qkv, cos, sin, k_cache, v_cache, block_table, kv_lens, Hq, cu_q=cu_q, positions=positions)

    @qkv_rope_paged_append.register_fake
    def _(qkv, cos, sin, k_cache, v_cache, block_table, kv_lens, cu_q, Hq, positions=None):
        return qkv.new_empty((qkv.shape[0], Hq, k_cache.shape[3]))

    @torch.library.custom_op("arke::paged_gqa_fwd", mutates_args=())
    def paged_gqa_fwd(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                      cu_q: Optional[torch.Tensor], shared_prefix: int, causal: bool = True, softmax_scale: Optional[float] = None,
                      max_new: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
        return ops.paged_gqa_fwd(q, k_cache, v_cache, block_table, kv_lens, cu_q=cu_q, shared_prefix=shared_prefix, causal=causal,
                                 softmax_scale=softmax_scale, max_new=max_new)

    @paged_gqa_fwd.register_fake
    def _(q, k_cache, v_cache, block_table, kv_lens, cu_q, shared_prefix, causal=True, softmax_scale=None, max_new=0):
        return torch.empty_like(q, memory_format=torch.contiguous_format), q.new_empty(q.shape[:-1], dtype=torch.float32)

    # a setting is the number, or the vector of one value per row where it is given
    def either(rows, number):
        return number if rows is None else rows

    @torch.library.custom_op("arke::sample_tokens", mutates_args=())
    def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                      min_p: float = 0.0, temperature_rows: Optional[torch.Tensor] = None, top_k_rows: Optional[torch.Tensor] = None,
                      top_p_rows: Optional[torch.Tensor] = None, min_p_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        return ops.sample_tokens(logits, u, either(temperature_rows, temperature), either(top_k_rows, top_k), either(top_p_rows, top_p),
                                 either(min_p_rows, min_p))

    @sample_tokens.register_fake
    def _(logits, u, *args, **kwargs):
        return logits.new_empty((logits.shape[0],), dtype=torch.int64)

    @torch.library.custom_op("arke::sample_tokens_logprob", mutates_args=())
    def sample_tokens_logprob(logits: torch.Tensor, u: torch.Tensor, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                              min_p: float = 0.0, temperature_rows: Optional[torch.Tensor] = None,
                              top_k_rows: Optional[torch.Tensor] = None, top_p_rows: Optional[torch.Tensor] = None,
                              min_p_rows: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
        return ops.sample_tokens(logits, u, either(temperature_rows, temperature), either(top_k_rows, top_k), either(top_p_rows, top_p),
                                 either(min_p_rows, min_p), return_logprob=True)

    @sample_tokens_logprob.register_fake
    def _(logits, u, *args, **kwargs):
        return logits.new_empty((logits.shape[0],), dtype=torch.int64), logits.new_empty((logits.shape[0],), dtype=torch.float32)

    _REGISTERED = True
    return True
