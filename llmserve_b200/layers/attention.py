"""Attention layer over the paged KV pool (``llmserve/layers/attention.py:60-133`` of the reference).

The QK RMSNorm, RoPE and the K/V store into the pool run as one kernel; then prefill (varlen
paged) or decode (split-KV) attention reads the pool.  In tree-verify mode the nodes' K/V are not
stored: they are captured in ``tree_k``/``tree_v`` and attended with the ancestor mask, and the
accepted path is committed afterwards by ``ops.kv.commit_tree_kv``.  A pool of 4-bit pages
(``kv_int4.Int4Pages``) takes the same steps through the operators of ``ops.kv_int4``; there the nodes of
a tree are quantised before they are attended, as decode would store them, and kept in that form.
"""
import torch
from torch import nn

from llmserve_b200.ops import attention as attn_ops
from llmserve_b200.ops import kv_int4
from llmserve_b200.ops import rope as rope_ops
from llmserve_b200.utils.context import get_context


class Attention(nn.Module):

    def __init__(self, num_heads: int, head_dim: int, scale: float, num_kv_heads: int):
        super().__init__()
        self.num_heads, self.head_dim, self.scale, self.num_kv_heads = num_heads, head_dim, scale, num_kv_heads
        self.k_cache = self.v_cache = torch.tensor([])
        self.tree_k = self.tree_v = torch.tensor([])

    def forward(self, qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                q_norm_w: torch.Tensor | None, k_norm_w: torch.Tensor | None, eps: float) -> torch.Tensor:
        ctx = get_context()
        T = positions.shape[0]
        if isinstance(self.k_cache, kv_int4.Int4Pages):
            forward = self._forward_int4 if ctx.tree_attention_mask is None else self._forward_tree_int4
            return forward(qkv, positions, cos_sin, q_norm_w, k_norm_w, eps, ctx).reshape(T, -1)
        if ctx.tree_attention_mask is not None:
            q, k, v = rope_ops.qkv_norm_rope_store(qkv, positions, cos_sin, q_norm_w, k_norm_w, eps,
                                                   None, None, None, self.num_heads, self.num_kv_heads,
                                                   self.head_dim)
            self.tree_k, self.tree_v = k.contiguous(), v.contiguous()
            o = attn_ops.tree_attention(q, self.k_cache, self.v_cache, ctx.tree_block_table,
                                        ctx.tree_prefix_len, self.tree_k, self.tree_v,
                                        ctx.tree_attention_mask, self.scale, ctx.tree_mask_bits)
            return o.reshape(T, -1)
        q, _, _ = rope_ops.qkv_norm_rope_store(qkv, positions, cos_sin, q_norm_w, k_norm_w, eps,
                                               self.k_cache, self.v_cache, ctx.slot_mapping,
                                               self.num_heads, self.num_kv_heads, self.head_dim)
        if ctx.is_prefill and ctx.uniform_q and q.is_cuda and attn_ops.verify_fits_decode_kernel(
                ctx.uniform_q, self.num_heads, self.num_kv_heads, self.k_cache.shape[2], self.head_dim):
            o = attn_ops.verify_attention(q, self.k_cache, self.v_cache, ctx.block_tables, ctx.seqlens_k, self.scale,
                                          ctx.uniform_q, ctx.decode_workspace)
        elif ctx.is_prefill:
            o = attn_ops.prefill_attention(q, self.k_cache, self.v_cache, ctx.cu_seqlens_q, ctx.seqlens_k,
                                           ctx.block_tables, self.scale, ctx.max_seqlen_q)
        else:
            o = attn_ops.decode_attention(q, self.k_cache, self.v_cache, ctx.block_tables, ctx.context_lens,
                                          self.scale, ctx.decode_workspace)
        return o.reshape(T, -1)

    def _forward_int4(self, qkv, positions, cos_sin, q_norm_w, k_norm_w, eps, ctx) -> torch.Tensor:
        q = kv_int4.qkv_norm_rope_store_int4(qkv, positions, cos_sin, q_norm_w, k_norm_w, eps, self.k_cache,
                                             self.v_cache, ctx.slot_mapping, self.num_heads, self.num_kv_heads,
                                             self.head_dim)
        if ctx.is_prefill and ctx.uniform_q:
            return kv_int4.verify_attention_int4(q, self.k_cache, self.v_cache, ctx.block_tables, ctx.seqlens_k,
                                                 self.scale, ctx.uniform_q, ctx.decode_workspace)
        if ctx.is_prefill:
            return kv_int4.prefill_attention_int4(q, self.k_cache, self.v_cache, ctx.cu_seqlens_q, ctx.seqlens_k,
                                                  ctx.block_tables, self.scale, ctx.max_seqlen_q)
        return kv_int4.decode_attention_int4(q, self.k_cache, self.v_cache, ctx.block_tables, ctx.context_lens,
                                             self.scale, ctx.decode_workspace)

    def _forward_tree_int4(self, qkv, positions, cos_sin, q_norm_w, k_norm_w, eps, ctx) -> torch.Tensor:
        # scratch pages of one block: the kernel that quantises a decoded token's K/V quantises the nodes'.  A node
        # whose position is outside the angle table is skipped: it reads as zeros, since V that nobody sees has to be finite
        T = positions.shape[0]
        pages = kv_int4.Int4Pages.scratch_pair((1, self.num_kv_heads, -(-T // 16) * 16, self.head_dim), qkv.device)
        slots = ctx.slot_mapping             # node i in row i
        if slots is None:
            slots = torch.arange(T, dtype=torch.int32, device=qkv.device)
        q = kv_int4.qkv_norm_rope_store_int4(qkv, positions, cos_sin, q_norm_w, k_norm_w, eps, *pages, slots,
                                             self.num_heads, self.num_kv_heads, self.head_dim)
        self.tree_k, self.tree_v = (p.rows(T) for p in pages)
        k, v = kv_int4.load_kvcache_int4(*pages, slots)
        return kv_int4.tree_attention_int4(q, self.k_cache, self.v_cache, ctx.tree_block_table, ctx.tree_prefix_len,
                                           k, v, ctx.tree_attention_mask, self.scale, ctx.tree_mask_bits)
