"""Public op wrappers with the reference's names, arguments and error behaviour.

Mirrors the public section of vllm_gguf_plugin/ops.py:181-208: `ggml_dequantize`,
`ggml_mul_mat_vec_a8` and `ggml_mul_mat_a8` forward to `torch.ops._C_gguf.*`.  Unlike the reference
there is no Triton fallback behind them: if the `_C_gguf` extension cannot be loaded the import fails.

Importing this module loads `kaillm_b200/_C_gguf.so`, which registers the six op schemas of the
reference's extension (vllm_gguf_plugin/csrc/torch_bindings.cpp:22-41) under the same namespace, so
code that calls `torch.ops._C_gguf.ggml_*` directly works unchanged.
"""
from __future__ import annotations

import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
EXT_PATH = os.path.join(_HERE, "_C_gguf.so")

# GGML type ids served by the CUDA kernels (gguf-reader/gguf/constants.py:5763-5799)
SUPPORTED_QUANT_TYPES = frozenset({2, 3, 6, 7, 8, 10, 11, 12, 13, 14, 20, 21, 23})
GEMM_QUANT_TYPES = frozenset({2, 3, 6, 7, 8, 10, 11, 12, 13, 14})


def _load_extension() -> None:
    if hasattr(torch.ops, "_C_gguf") and hasattr(torch.ops._C_gguf, "ggml_mul_mat_vec_a8"):
        return
    if not os.path.exists(EXT_PATH):
        raise ImportError(
            f"{EXT_PATH} is missing: build it with `python -m kaillm_b200._build` "
            "(the GGUF ops have no Triton or CPU fallback)")
    torch.ops.load_library(EXT_PATH)


_load_extension()


def ggml_dequantize(W: torch.Tensor, quant_type: int, m: int, n: int, dtype: torch.dtype | None) -> torch.Tensor:
    return torch.ops._C_gguf.ggml_dequantize(W, quant_type, m, n, dtype)


def ggml_mul_mat_vec_a8(W: torch.Tensor, X: torch.Tensor, quant_type: int, row: int) -> torch.Tensor:
    return torch.ops._C_gguf.ggml_mul_mat_vec_a8(W, X, quant_type, row)


def ggml_mul_mat_a8(W: torch.Tensor, X: torch.Tensor, quant_type: int, row: int) -> torch.Tensor:
    return torch.ops._C_gguf.ggml_mul_mat_a8(W, X, quant_type, row)


def ggml_dequant_mul_mat(W: torch.Tensor, X: torch.Tensor, quant_type: int, row: int) -> torch.Tensor:
    """X @ ggml_dequantize(W).T, fused where the kernel covers the call (no gradient: see linear.fused_mul_mat_gguf)."""
    return torch.ops._C_gguf.ggml_dequant_mul_mat(W, X, quant_type, row)


def ggml_dequantize_rows(W: torch.Tensor, ids: torch.Tensor, quant_type: int, k: int, dtype: torch.dtype, f32_math: bool) -> torch.Tensor:
    """Rows `ids` of the table W, dequantized (kq_dequantize_rows): [*ids.shape, k]."""
    return torch.ops._C_gguf.ggml_dequantize_rows(W, ids, quant_type, k, dtype, f32_math)


def ggml_mul_mat_merged(Ws: list[torch.Tensor], X: torch.Tensor, quant_types: list[int], mmq: list[int]) -> torch.Tensor:
    """Several projections of the same activations, quantized once: [m, sum of rows] (no gradient)."""
    return torch.ops._C_gguf.ggml_mul_mat_merged(Ws, X, quant_types, mmq)


def ggml_moe_a8(X: torch.Tensor, W: torch.Tensor, sorted_token_ids: torch.Tensor, expert_ids: torch.Tensor,
                num_tokens_post_padded: torch.Tensor, quant_type: int, row: int, top_k: int, tokens: int) -> torch.Tensor:
    """vllm_gguf_plugin/ops.py:211-246."""
    return torch.ops._C_gguf.ggml_moe_a8(X, W, sorted_token_ids, expert_ids, num_tokens_post_padded, quant_type, row, top_k,
                                         tokens)


def ggml_moe_a8_vec(X: torch.Tensor, W: torch.Tensor, topk_ids: torch.Tensor, top_k: int, quant_type: int, row: int,
                    tokens: int) -> torch.Tensor:
    """vllm_gguf_plugin/ops.py:249-278."""
    return torch.ops._C_gguf.ggml_moe_a8_vec(X, W, topk_ids, top_k, quant_type, row, tokens)


def ggml_moe_get_block_size(quant_type: int) -> int:
    """vllm_gguf_plugin/ops.py:281-284."""
    return torch.ops._C_gguf.ggml_moe_get_block_size(quant_type)


def fused_moe_swiglu(X: torch.Tensor, W1: torch.Tensor, W2: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor,
                     quant_type: int, quant_type2: int, block: bool) -> torch.Tensor:
    """The whole SiLU feed-forward of `linear.fused_moe_gguf` as one call (no gradient); `block`: expert-sorted branch."""
    return torch.ops._C_gguf.fused_moe_swiglu(X, W1, W2, topk_weights, topk_ids, quant_type, quant_type2, block)


def _direct(name: str):
    if not hasattr(torch.ops._C_gguf, name):       # the namespace is another library's, with the reference's operators only
        def missing(*args):
            raise ImportError(f"torch.ops._C_gguf was registered by another library, which has no {name}")

        return missing
    from . import _C_gguf

    return _C_gguf.direct(name, getattr(torch.ops._C_gguf, name).default)


# The operators that a decode step calls in every layer, for `attention` and `linear`: positional arguments only; plain calls go past the
# dispatcher, everything else to the overload in torch.ops (a dispatched call takes 2 us longer)
QK_NORM_ROPE = _direct("qk_norm_rope")
QK_NORM_ROPE_STORE = _direct("qk_norm_rope_store")
PAGED_ATTENTION = _direct("paged_attention")
PLAN_PAGES = _direct("plan_pages")
MOE_ROUTE = _direct("moe_route")


def qk_norm_rope(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, num_heads: int, num_kv_heads: int,
                 q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float, interleaved: bool,
                 factor: float) -> tuple[torch.Tensor, torch.Tensor]:
    """`attention.qk_norm_rope` (no gradient)."""
    return QK_NORM_ROPE(qkv, positions, inv_freq, num_heads, num_kv_heads, q_weight, k_weight, eps, interleaved, factor)


def qk_norm_rope_store(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, num_heads: int, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, slots: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                       eps: float, interleaved: bool, factor: float) -> torch.Tensor:
    """`attention.qk_norm_rope_store` (no gradient)."""
    return QK_NORM_ROPE_STORE(qkv, positions, inv_freq, num_heads, k_cache, v_cache, slots, q_weight, k_weight, eps, interleaved, factor)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    scale: float, window: int, softcap: float, lse: bool) -> tuple[torch.Tensor, torch.Tensor | None]:
    """`attention.paged_attention` (no gradient): the output and, if asked for, the log of the sum of exponentials (else None)."""
    return PAGED_ATTENTION(q, k_cache, v_cache, block_table, seq_lens, scale, window, softcap, lse)


def plan_pages(block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor, taken: torch.Tensor,
               page_size: int, num_tokens: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """`attention.plan_pages`."""
    return PLAN_PAGES(block_table, seq_lens, new_lens, free_pages, taken, page_size, num_tokens)


def moe_route(logits: torch.Tensor, top_k: int, sigmoid: bool, bias: torch.Tensor | None, groups: int, top_groups: int, renormalize: bool,
              scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """`linear.route_experts` (no gradient): weights and ids."""
    return MOE_ROUTE(logits, top_k, sigmoid, bias, groups, top_groups, renormalize, scale)
