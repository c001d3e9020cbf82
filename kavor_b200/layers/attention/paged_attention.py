"""Paged-KV attention layer (drop-in for kavor/layers/attention/flash_attention_kvcache.py).

``store_kvcache`` and ``Attention`` keep the reference's signatures and
behaviour; the KV write, the varlen/paged prefill attention and the paged
decode attention are the sm_100a kernels of ``libkavor_b200.so``.
"""
from __future__ import annotations

import torch
from torch import nn

from kavor_b200 import _kernels as K
from kavor_b200.utils.context import get_context


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slot_mapping: torch.Tensor) -> None:
    """Write key/value [N, Hkv, hd] rows into the paged cache at slot_mapping
    (flash_attention_kvcache.py:37-46); -1 slots are skipped."""
    K.store_kvcache(key, value, k_cache, v_cache, slot_mapping)


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """``store_kvcache`` into a cache of 8-bit values: every key/value row [128]
    is held as e4m3 values with one power-of-two scale. The caches are
    ``float8_e4m3fn`` [num_blocks, block_size, Hkv, 128], the scales
    ``float8_e8m0fnu`` [num_blocks, Hkv, block_size]; -1 slots are skipped, the
    others must be distinct. The scale is the smallest power of two (at least
    2^-100) that brings the row's largest finite magnitude to at most 448;
    values round to nearest even, infinities to the row's +-448."""
    K.store_kvcache_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)


def load_kvcache_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                     block_tables: torch.Tensor, cu_seqlens_k: torch.Tensor, total_k: int,
                     k_out: torch.Tensor | None = None,
                     v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Read whole sequences back from an 8-bit cache: (k, v) bf16 [total_k, Hkv,
    128], sequence b at rows cu_seqlens_k[b]..cu_seqlens_k[b+1], exactly the
    held values (a held 2^128, from values within 1/32 of the largest bf16
    value, as infinity). ``total_k`` is the row count of the outputs; rows from
    cu_seqlens_k[-1] on are left as they are."""
    return K.load_kvcache_fp8(k_cache, v_cache, k_scale, v_scale, block_tables, cu_seqlens_k, total_k, k_out, v_out)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                   context_lens: torch.Tensor, cu_seqlens_q: torch.Tensor, max_seqlen_q: int, scale: float,
                   tree_mask: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a tree of drafted tokens per sequence over the paged cache.

    Sequence b has ``context_lens[b]`` tokens in the cache, the last T_b =
    cu_seqlens_q[b+1] - cu_seqlens_q[b] of them its drafted nodes (already
    stored); q [total_q, Hq, 128] holds one row per node. Node i sees every
    token before the draft and the nodes whose bits are set in its row of
    ``tree_mask`` (int32 [total_q, words], bit j % 32 of word j // 32 for node
    j; ``build_tree_mask`` makes it from parents); without a mask, nodes 0..i.
    One node per sequence is decode. ``max_seqlen_q`` is at least the largest
    T_b. With ``k_scale``/``v_scale`` the caches are 8-bit
    (``store_kvcache_fp8``). A node that sees nothing gives zeros; what unseen
    nodes hold has no influence. Sums are fp32; the softmax's weights are rounded
    to bf16 before they meet V, as in the decode attention, or, over an 8-bit cache
    with at most 32 query rows (nodes x Hq / Hkv) a kv head, to halves scaled to the
    row's largest contribution. |V| up to 2^90. Returns [total_q, Hq, 128]; rows from
    cu_seqlens_q[-1] on are not written."""
    return K.tree_attention(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, max_seqlen_q, scale,
                            tree_mask, k_scale, v_scale, out)


def build_tree_mask(parents: list[list[int]], words: int | None = None) -> torch.Tensor:
    """The ``tree_mask`` (int32 [total nodes, words], on the CPU) of drafted trees:
    ``parents[b][i]`` is the node of sequence b that node i continues (an earlier
    one), or -1 when it continues the context. A node sees itself and its
    ancestors. ``words`` defaults to what the largest tree needs."""
    need = max((len(p) + 31) // 32 for p in parents) if parents else 0
    words = max(need, 1) if words is None else words
    if words < need:
        raise ValueError(f"a tree of more than {32 * words} nodes does not fit {words} mask words")
    rows = []
    for b, tree in enumerate(parents):
        seen: list[int] = []
        for i, p in enumerate(tree):
            if not -1 <= p < i:
                raise ValueError(f"node {i} of sequence {b} has parent {p}: a parent is an earlier node or -1")
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        rows.extend([bits >> (32 * w) & 0xFFFFFFFF for w in range(words)] for bits in seen)
    return torch.tensor(rows, dtype=torch.int64).reshape(-1, words).to(torch.int32)


class Attention(nn.Module):
    """flash_attention_kvcache.py:49-84.

    ``k_cache[slot]`` / ``v_cache[slot]`` are [num_blocks, block_size, Hkv, hd]
    views into the page pool, bound by the cache pool. ``forward`` writes the
    step's K/V (unless ``kv_stored``: the fused Qwen3 prologue already wrote
    them) and returns [T, Hq, hd] for prefill or [B, Hq, hd] for decode.
    """

    def __init__(self, num_heads: int, head_dim: int, scale: float, num_kv_heads: int, num_kv_slots: int = 1):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.num_kv_slots = num_kv_slots
        self.k_cache = [torch.tensor([]) for _ in range(num_kv_slots)]
        self.v_cache = [torch.tensor([]) for _ in range(num_kv_slots)]

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slot: int = 0,
                kv_stored: bool = False) -> torch.Tensor:
        ctx = get_context()
        k_cache, v_cache = self.k_cache[slot], self.v_cache[slot]
        has_cache = k_cache.numel() > 0 and v_cache.numel() > 0
        if has_cache and not kv_stored:
            store_kvcache(k, v, k_cache, v_cache, ctx.slot_mapping)
        if ctx.is_prefill:
            if ctx.block_tables is not None:  # prefix cache: keys come from the pages
                return K.prefill_attention(q, k_cache, v_cache, ctx.cu_seqlens_q, ctx.cu_seqlens_k,
                                           ctx.max_seqlen_q, self.scale, block_tables=ctx.block_tables)
            return K.prefill_attention(q, k, v, ctx.cu_seqlens_q, ctx.cu_seqlens_k, ctx.max_seqlen_q, self.scale)
        return K.paged_decode_attention(q, k_cache, v_cache, ctx.block_tables, ctx.context_lens, self.scale)
