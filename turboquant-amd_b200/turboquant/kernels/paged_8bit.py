"""Paged KV cache in 8 bits: e4m3 codes with one power-of-two scale per 16 tokens and head, and the attention that reads it.

For the layers that the packed 2- to 4-bit cache leaves out (TurboQuantConfig.should_compress protects the first and last ones), and for
whatever needs several query tokens over cached context: prompt chunks and speculated tokens.  The reference keeps such
layers in the engine's own cache (turboquant/integration/vllm_backend.py:237-289) and serves extends from it
(turboquant/integration/tq_fp4_backend.py:555-601).

The cache is uint8 [num_blocks, num_kv_heads, block_size / 16 * page_bytes], like the packed one.  A page holds 16 tokens of one head:
K codes [16, D], V codes [16, D], the fp32 scales of K and V, 24 unused bytes.  A value is code * scale.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from turboquant.kernels import _native
from turboquant.kernels.paged_layout import PAGE_TOKENS


def page_bytes_8bit(head_dim: int = 128) -> int:
    rc = _native.lib().tq_cache8_page_bytes(head_dim)
    if rc < 0:
        raise ValueError("the 8-bit cache is built for head_dim 64 and 128")
    return rc


def cache_shape_8bit(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int = 128) -> tuple[int, int, int]:
    if block_size < PAGE_TOKENS or block_size % PAGE_TOKENS:
        raise ValueError("block_size must be a multiple of 16")
    return (num_blocks, num_kv_heads, block_size // PAGE_TOKENS * page_bytes_8bit(head_dim))


def allocate_cache_8bit(num_blocks: int, block_size: int, num_kv_heads: int, device, head_dim: int = 128) -> torch.Tensor:
    return torch.zeros(cache_shape_8bit(num_blocks, block_size, num_kv_heads, head_dim), dtype=torch.uint8, device=device)


def codes_and_scales(cache: torch.Tensor, block_size: int, head_dim: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """Views of a cache: e4m3 codes [num_blocks, heads, block_size / 16, 2, 16, D] and fp32 scales [num_blocks, heads,
    block_size / 16, 2], K and V in the fourth dimension."""
    blocks, heads, row = cache.shape
    page, values = page_bytes_8bit(head_dim), 2 * PAGE_TOKENS * head_dim
    if block_size % PAGE_TOKENS or row != block_size // PAGE_TOKENS * page:
        raise ValueError(f"cache row of {row} bytes does not match block_size {block_size} and head_dim {head_dim}")
    pages = cache.view(blocks, heads, block_size // PAGE_TOKENS, page)
    codes = pages[..., :values].unflatten(-1, (2, PAGE_TOKENS, head_dim)).view(torch.float8_e4m3fn)
    return codes, pages[..., values:values + 8].view(torch.float32)


def quantize_and_scatter(key: torch.Tensor, value: torch.Tensor, cache: torch.Tensor, slot_mapping: torch.Tensor,
                         block_size: int) -> None:
    """Write key / value [T, Hkv, D] (fp16, bf16 or fp32; D 64 or 128) at slot_mapping [T] into the 8-bit cache.

    Slot s lands in block s // block_size at offset s % block_size; negative slots are skipped, ones beyond the cache are skipped
    and set STATUS_BAD_SLOT.  A page's scale is the smallest power of two that fits its values into +-448; a page that a
    call begins takes it from the call's rows, one that is continued keeps the larger one and has its older codes rescaled
    when it grows.  Infinities saturate, NaN stays NaN, neither counts for the scale.  Rows of one page stand next to
    one another in ascending order; of a page that a call names in two places, or with a slot twice, the content is unspecified.
    """
    if not torch.compiler.is_compiling() and _native.host().quantize8(key, value, cache, slot_mapping, block_size):
        return
    if slot_mapping.dtype != torch.int64:
        slot_mapping = slot_mapping.to(torch.int64)
    torch.ops.tq_b200.quantize8_paged(key, value, cache, slot_mapping.contiguous(), int(block_size))


def paged_attention_8bit(q: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                         block_size: int, sm_scale: Optional[float] = None, query_start_loc: Optional[torch.Tensor] = None,
                         max_query_len: int = 1, max_seq_len: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [T, Hq, D] (fp16 or bf16) over the 8-bit cache; returns [T, Hq, D].

    Without query_start_loc row i is the only query of sequence i.  With it (int32 [num_seqs + 1], ascending) rows
    query_start_loc[i] .. query_start_loc[i + 1] are the last tokens of sequence i, causal among themselves: row j of n sees
    the first seq_lens[i] - n + j + 1 tokens, and max_query_len is at least the largest n (rows beyond it are left out and
    set STATUS_TOO_LONG; the others are served as if they were all).  The tokens themselves are in the cache already.  Rows that
    see nothing become zeros; rows that are left out or that no sequence has - before the first one, behind the last one - become
    zeros too, or are left as they were when `out` is given.
    max_seq_len: the longest sequence of the step when the host knows it; launch and workspace are sized for it.
    sm_scale defaults to 1 / sqrt(D).  Query head h reads KV head h // (Hq // Hkv).
    """
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[-1])
    if not torch.compiler.is_compiling():
        res = _native.host().attend8(q, cache, block_tables, seq_lens, query_start_loc, out, sm_scale, block_size, max_query_len,
                                     max_seq_len)
        if res is not None:
            return res
    if block_tables.dtype != torch.int32:
        block_tables = block_tables.to(torch.int32)
    if seq_lens.dtype != torch.int32:
        seq_lens = seq_lens.to(torch.int32)
    if query_start_loc is not None:
        query_start_loc = query_start_loc.to(torch.int32).contiguous()
    if out is None:
        return torch.ops.tq_b200.attend8_paged(q.contiguous(), cache, block_tables, seq_lens.contiguous(), query_start_loc,
                                               float(sm_scale), int(block_size), int(max_query_len), int(max_seq_len))
    if torch.is_grad_enabled() and (q.requires_grad or out.requires_grad):
        raise RuntimeError("paged_attention_8bit(out=...) has no autograd")
    _native._attend8_impl(out, q.contiguous(), cache, block_tables, seq_lens.contiguous(), query_start_loc, sm_scale, block_size,
                          max_query_len, max_seq_len, zero_rest=False)
    return out
