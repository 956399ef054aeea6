"""A paged KV cache held in 4 bits: the store, the read-back and the attention that reads it.

``Int4Pages`` is one pool (K or V): codes ``uint8 [blocks, kv_heads, block_size, head_dim / 2]``, dim
``2i`` in the low nibble, and scale words ``int16 [blocks, kv_heads, block_size, head_dim / 64]``.
Every token, KV head and group of 64 dims has its own range, widened to hold zero.  A word is the
bfloat16 pattern of the group's scale ``s`` with the four low mantissa bits replaced by the zero code
``z``; a code ``c`` stands for ``s * (c - z)``, which is exact in bfloat16.  4.25 bits per element.

* ``store_kvcache_int4``        -- quantise K/V rows into the pages by flat slot (``slot < 0`` skips;
  the slots of one call are distinct).
* ``load_kvcache_int4``         -- the rows at given slots as bfloat16 (``slot < 0`` gives zeros).
* ``qkv_norm_rope_store_int4``  -- one step's projection: QK-norm, RoPE, query out, K/V into the pages.
* ``decode_attention_int4``     -- one query per sequence; ``verify_attention_int4``: ``nq`` of them.
* ``tree_attention_int4``       -- EAGLE3 tree verify on a 4-bit prefix.
* ``commit_tree_kv_int4``       -- copy accepted tree nodes, quantised when they were verified, into the pools.
* ``prefill_attention_int4``    -- ragged causal chunks, on a cached prefix or without.

On CUDA a slot or block id outside the pool is skipped (its keys are not seen) and recorded for
``check_status``.  A query that sees no key gives zeros.  Stored values stay below 2^127 in magnitude, V
that attention reads below 2^100 (weights reach 2^8 before they are divided by their sum), queries below 2^125.
"""
import torch

from llmserve_b200.ops import attention as attn_ops
from llmserve_b200.ops._ext import C, status
from llmserve_b200.ops.norm import rms_norm_ref
from llmserve_b200.ops.rope import apply_rope_ref

GROUP = 64


class Int4Pages:
    """One 4-bit pool; a leading layer dimension is indexed away with ``pages[layer]``."""
    __slots__ = ("codes", "words")

    def __init__(self, codes: torch.Tensor, words: torch.Tensor):
        self.codes, self.words = codes, words

    @classmethod
    def zeros(cls, shape, device) -> "Int4Pages":
        """Empty pages for logical rows ``[..., blocks, kv_heads, block_size, head_dim]``."""
        *lead, hd = shape
        if hd not in (64, 128) or lead[-1] % 16:
            raise ValueError("4-bit pages need head_dim 64 or 128 and a block_size that is a multiple of 16")
        return cls(torch.zeros(*lead, hd // 2, dtype=torch.uint8, device=device),
                   torch.zeros(*lead, hd // GROUP, dtype=torch.int16, device=device))

    @classmethod
    def scratch_pair(cls, shape, device) -> tuple["Int4Pages", "Int4Pages"]:
        """K and V pages whose rows read as zeros until they are stored (scale 0; the codes hold anything)."""
        *lead, hd = shape
        pair = cls(torch.empty(2, *lead, hd // 2, dtype=torch.uint8, device=device),
                   torch.zeros(2, *lead, hd // GROUP, dtype=torch.int16, device=device))
        return pair[0], pair[1]

    @property
    def shape(self) -> tuple:
        return (*self.codes.shape[:-1], 2 * self.codes.shape[-1])

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.words.numel()

    def numel(self) -> int:
        return 2 * self.codes.numel()

    def __getitem__(self, layer) -> "Int4Pages":
        return Int4Pages(self.codes[layer], self.words[layer])

    def rows(self, n: int) -> "Int4Pages":
        """The first ``n`` rows of a pool of one block, as logical rows ``[n, kv_heads, head_dim]``."""
        return Int4Pages(self.codes[0, :, :n].transpose(0, 1), self.words[0, :, :n].transpose(0, 1))


def _check_pages(k_pages, v_pages, nkv=None, hd=None):
    for name, p in (("K", k_pages), ("V", v_pages)):
        if not isinstance(p, Int4Pages):
            raise ValueError(f"{name} pages must be Int4Pages")
        c, w = p.codes, p.words
        if c.dtype != torch.uint8 or w.dtype != torch.int16 or c.dim() != 4 or w.dim() != 4:
            raise ValueError(f"{name} pages must be 4-dimensional uint8 codes and int16 scale words")
        if p.shape[3] not in (64, 128) or w.shape != (*c.shape[:3], p.shape[3] // GROUP) or c.shape[2] % 16:
            raise ValueError(f"{name} pages: head_dim 64 or 128, block_size a multiple of 16, one word per 64 dims")
    if k_pages.shape != v_pages.shape:
        raise ValueError("K and V pages differ in shape")
    if nkv is not None and (k_pages.shape[1] != nkv or k_pages.shape[3] != hd):
        raise ValueError("head layout does not match the pages")


def _check_query(q, k_pages, v_pages, scale):
    _check_pages(k_pages, v_pages)
    if q.dim() != 3 or q.shape[2] != k_pages.shape[3] or q.shape[1] < 1 or q.shape[1] % k_pages.shape[1]:
        raise ValueError("query heads do not match the pages")
    if not 0 < scale < float("inf"):
        raise ValueError("scale must be positive")


# ---- fp32 restatement (the CPU path) -----------------------------------------------------------
def quantise_int4_ref(x: torch.Tensor):
    """Rows ``[..., head_dim]`` -> (codes, words) of the page format, computed in fp32."""
    g = x.float().unflatten(-1, (-1, GROUP))
    mx, mn = g.amax(-1).clamp(min=0), g.amin(-1).clamp(max=0)
    r = (mx * 0.5 - mn * 0.5) / torch.full_like(mx, 7.5)
    finite = torch.isfinite(r)
    bits = (torch.where(finite, r, torch.ones_like(r)).view(torch.int32) + 0xFFFFF) & 0x7FF00000
    live = finite & (r >= 2.0 ** -126)
    s = torch.where(live, bits.view(torch.float32), torch.ones_like(r))
    z = torch.where(live, torch.round(-mn / s), torch.zeros_like(r))
    c = torch.where(live[..., None], torch.round(g / s[..., None]) + z[..., None], torch.zeros_like(g))
    c = c.clamp(0, 15).flatten(-2).to(torch.uint8)
    words = torch.where(live, (bits >> 16) | z.int(), torch.where(finite, 0, 0x7FC0).int())
    return c[..., 0::2] | (c[..., 1::2] << 4), words.to(torch.int16)


def dequantise_int4_ref(codes: torch.Tensor, words: torch.Tensor) -> torch.Tensor:
    """What the pages stand for, fp32 ``[..., head_dim]``."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    w = words.int()
    s = ((w & 0x7FF0) << 16).view(torch.float32)
    return ((c - (w & 15).float()[..., None]) * s[..., None]).flatten(-2)


def store_kv_int4_ref(k, v, k_pages, v_pages, slot_mapping):
    bs = k_pages.shape[2]
    slots = slot_mapping.long()
    keep = slots >= 0
    blk, off = slots[keep] // bs, slots[keep] % bs
    for x, p in ((k, k_pages), (v, v_pages)):
        p.codes[blk, :, off], p.words[blk, :, off] = quantise_int4_ref(x[keep])


def load_kv_int4_ref(k_pages, v_pages, slot_mapping, dtype=torch.bfloat16):
    bs = k_pages.shape[2]
    slots = slot_mapping.long()
    at = slots.clamp(min=0)
    out = []
    for p in (k_pages, v_pages):
        x = dequantise_int4_ref(p.codes[at // bs, :, at % bs], p.words[at // bs, :, at % bs])
        x[slots < 0] = 0
        out.append(x.to(dtype))
    return tuple(out)


def commit_tree_kv_int4_ref(tree_k, tree_v, k_pages, v_pages, node_indices, slot_mapping):
    bs = k_pages.shape[3]
    for node, slot in zip(node_indices.tolist(), slot_mapping.tolist()):
        if slot < 0:
            continue
        for x, p in ((tree_k, k_pages), (tree_v, v_pages)):
            p.codes[:, slot // bs, :, slot % bs] = x.codes[:, node]
            p.words[:, slot // bs, :, slot % bs] = x.words[:, node]


def attention_int4_ref(q, k_pages, v_pages, cu_seqlens_q, seqlens_k, block_tables, scale):
    """Row ``j`` of a chunk of ``q_len`` sees keys ``< k_len - q_len + j + 1``."""
    out = torch.zeros_like(q)
    bs = k_pages.shape[2]
    cu, lens = cu_seqlens_q.tolist(), seqlens_k.tolist()
    for i, k_len in enumerate(lens):
        lo, hi = cu[i], cu[i + 1]
        k_len = min(k_len, block_tables.shape[1] * bs)
        if hi == lo or k_len <= 0:
            continue
        ids = block_tables[i, :-(-k_len // bs)].long()
        k, v = (dequantise_int4_ref(p.codes[ids], p.words[ids]).transpose(1, 2).flatten(0, 1)[:k_len]
                for p in (k_pages, v_pages))
        last = torch.arange(lens[i] - (hi - lo), lens[i], device=q.device).unsqueeze(1)
        mask = torch.arange(k_len, device=q.device).unsqueeze(0) <= last
        # a group of V that holds NaN reaches the rows that see its key, not those that give it no weight
        nan = v.isnan()
        o = attn_ops._attend(q[lo:hi], k, v.masked_fill(nan, 0), scale, mask)
        if nan.any():
            seen = (mask.float() @ nan.flatten(1).float()).view(-1, *nan.shape[1:]) > 0
            o = o.masked_fill(seen.repeat_interleave(q.shape[1] // k.shape[1], 1), float("nan"))
        out[lo:hi] = torch.where(mask.any(1)[:, None, None], o, torch.zeros_like(o))
    return out


# ---- public entry points -----------------------------------------------------------------------
def store_kvcache_int4(k, v, k_pages: Int4Pages, v_pages: Int4Pages, slot_mapping):
    """Quantise ``k`` / ``v`` ``[T, kv_heads, head_dim]`` (rows may be strided) into the pages at
    ``slot_mapping`` int32 [T]."""
    if not k.is_cuda:
        _check_pages(k_pages, v_pages, k.shape[1], k.shape[2])
        return store_kv_int4_ref(k, v, k_pages, v_pages, slot_mapping)
    C().store_kvcache_int4(k, v, k_pages.codes, k_pages.words, v_pages.codes, v_pages.words, slot_mapping,
                           status(k.device))


def load_kvcache_int4(k_pages: Int4Pages, v_pages: Int4Pages, slot_mapping):
    """``(k, v)`` rows ``[T, kv_heads, head_dim]`` at ``slot_mapping`` int32 [T]; bfloat16, exactly the
    values the pages hold."""
    codes = k_pages.codes
    if not codes.is_cuda:
        _check_pages(k_pages, v_pages)
        return load_kv_int4_ref(k_pages, v_pages, slot_mapping)
    return C().load_kvcache_int4(codes, k_pages.words, v_pages.codes, v_pages.words, slot_mapping, status(codes.device))


_NO_WEIGHT = {}


def _no_weight(device):
    t = _NO_WEIGHT.get(device)
    if t is None:
        t = _NO_WEIGHT[device] = torch.empty(0, dtype=torch.bfloat16, device=device)
    return t


def qkv_norm_rope_store_int4(qkv, positions, cos_sin, q_norm_w, k_norm_w, eps, k_pages: Int4Pages, v_pages: Int4Pages,
                             slot_mapping, num_heads, num_kv_heads, head_dim):
    """Split ``qkv [T, (nh + 2 nkv) * hd]`` (or fp32 split-K planes ``[S, T, ..]``, summed here), normalise
    (with weights given) and rotate q and k, store k and v into the pages; returns the rotated query
    ``[T, nh, hd]``.  Everything up to the one rounding of the query and the quantisation is fp32."""
    if not qkv.is_cuda:
        _check_pages(k_pages, v_pages, num_kv_heads, head_dim)
        x = qkv.float().sum(0) if qkv.dim() == 3 else qkv.float()
        q, k, v = x.unflatten(-1, (-1, head_dim)).split((num_heads, num_kv_heads, num_kv_heads), 1)
        if q_norm_w is not None:
            q, k = rms_norm_ref(q, q_norm_w.float(), eps), rms_norm_ref(k, k_norm_w.float(), eps)
        q, k = apply_rope_ref(q, positions, cos_sin), apply_rope_ref(k, positions, cos_sin)
        store_kv_int4_ref(k, v, k_pages, v_pages, slot_mapping)
        return q if qkv.dim() == 3 else q.to(qkv.dtype)
    if num_kv_heads != k_pages.codes.shape[1] or head_dim != 2 * k_pages.codes.shape[3]:
        raise ValueError("head layout does not match the pages")
    d = qkv.device
    q = torch.empty(qkv.shape[-2], num_heads, head_dim, dtype=torch.bfloat16, device=d)
    C().qkv_rope_int4(q, qkv.contiguous(), positions, cos_sin, q_norm_w if q_norm_w is not None else _no_weight(d),
                      k_norm_w if k_norm_w is not None else _no_weight(d), eps, k_pages.codes, k_pages.words,
                      v_pages.codes, v_pages.words, slot_mapping, num_heads, status(d))
    return q


def verify_attention_int4(q, k_pages: Int4Pages, v_pages: Int4Pages, block_tables, seqlens_k, scale, nq: int,
                          workspace=None):
    """Causal attention of ``nq`` consecutive new tokens per sequence (``q [B * nq, nh, hd]``, sequence
    b's at positions ``seqlens_k[b] - nq ..``).  ``workspace``: a ``DecodeWorkspace`` for at least
    ``B * nq`` rows and the keys that the block tables can address, which calls (and captured graphs) on
    one stream may share; calls that can overlap need one each.  Without one the call makes its own."""
    if nq < 1 or q.shape[0] != seqlens_k.shape[0] * nq:
        raise ValueError("q must hold nq >= 1 rows per sequence")
    if not q.is_cuda:
        _check_query(q, k_pages, v_pages, scale)
        cu = torch.arange(0, q.shape[0] + 1, nq, dtype=torch.int32)
        return attention_int4_ref(q, k_pages, v_pages, cu, seqlens_k, block_tables, scale)
    rows, nh, hd = q.shape
    cap = block_tables.shape[-1] * k_pages.codes.shape[2]
    if workspace is None or workspace.max_batch < rows or workspace.max_splits * 128 < cap:
        workspace = attn_ops.DecodeWorkspace(rows, nh, hd, cap, q.device)
    q = q.contiguous()
    out = torch.empty_like(q)
    C().decode_attention_int4(out, q, k_pages.codes, k_pages.words, v_pages.codes, v_pages.words, nq,
                              seqlens_k, block_tables, scale, workspace.partial_out, workspace.partial_ml,
                              workspace.counters, workspace.max_splits, status(q.device))
    return out


def decode_attention_int4(q, k_pages: Int4Pages, v_pages: Int4Pages, block_tables, context_lens, scale,
                          workspace=None):
    """One query token per sequence: ``q [B, nh, hd]`` against ``context_lens`` int32 [B] keys."""
    return verify_attention_int4(q, k_pages, v_pages, block_tables, context_lens, scale, 1, workspace)


def tree_attention_int4(q, k_pages: Int4Pages, v_pages: Int4Pages, block_table, prefix_len, tree_k, tree_v, tree_mask,
                        scale, mask_bits=None):
    """Tree verify on a 4-bit prefix: the sequence's pages are read back once (exact in bfloat16) and
    ``ops.attention.tree_attention`` runs on the copy.  ``tree_k`` / ``tree_v`` are attended as they are
    given: a node stands for the token that decode would write and read back, so its rows have to be
    what pages hold of them (``qkv_norm_rope_store_int4`` into scratch pages, then ``load_kvcache_int4``)."""
    bs = k_pages.shape[2]
    prefix_len = min(prefix_len, block_table.shape[0] * bs)      # a context ends at its table
    ids = block_table[:max(1, -(-prefix_len // bs))]
    if not q.is_cuda:
        ids = ids.long()
        k, v = (dequantise_int4_ref(p.codes[ids], p.words[ids]).to(q.dtype) for p in (k_pages, v_pages))
        table = torch.arange(ids.shape[0], dtype=torch.int32)
    else:
        ids = ids.to(torch.int32).contiguous() if ids.shape[0] else torch.full((1,), -1, dtype=torch.int32, device=q.device)
        k, v, table = C().load_pages_int4(k_pages.codes, k_pages.words, v_pages.codes, v_pages.words, ids)
    return attn_ops.tree_attention(q.contiguous(), k, v, table, prefix_len, tree_k, tree_v, tree_mask, scale, mask_bits)


def commit_tree_kv_int4(tree_k: Int4Pages, tree_v: Int4Pages, k_pages: Int4Pages, v_pages: Int4Pages, node_indices,
                        slot_mapping):
    """Copy rows ``node_indices`` int32 [m] of every layer's tree nodes (``[layers, nodes, kv_heads, head_dim]``)
    into the pools ``[layers, blocks, kv_heads, block_size, head_dim]`` at ``slot_mapping`` int32 [m]: codes
    and words as they are, so that an accepted node reads back as it was attended."""
    for x in (tree_k, tree_v, k_pages, v_pages):
        if not isinstance(x, Int4Pages):
            raise ValueError("tree K/V and pools must be Int4Pages")
    t, p = tree_k.shape, k_pages.shape
    if len(t) != 4 or tree_v.shape != t:
        raise ValueError("tree K/V must be [layers, nodes, kv_heads, head_dim]")
    if len(p) != 5 or v_pages.shape != p:
        raise ValueError("target K/V pages must be [layers, blocks, kv_heads, block_size, head_dim]")
    if (t[0], t[2], t[3]) != (p[0], p[2], p[4]):
        raise ValueError("tree K/V and target pages differ in layers or heads")
    if node_indices.ndim != 1 or node_indices.shape != slot_mapping.shape:
        raise ValueError("selected nodes and slots must have matching one-dimensional shapes")
    if not k_pages.codes.is_cuda:
        return commit_tree_kv_int4_ref(tree_k, tree_v, k_pages, v_pages, node_indices, slot_mapping)
    C().commit_tree_kv_int4(tree_k.codes.contiguous(), tree_k.words.contiguous(), tree_v.codes.contiguous(),
                            tree_v.words.contiguous(), k_pages.codes, k_pages.words, v_pages.codes, v_pages.words,
                            node_indices, slot_mapping, status(k_pages.codes.device))


def prefill_attention_int4(q, k_pages: Int4Pages, v_pages: Int4Pages, cu_seqlens_q, seqlens_k, block_tables, scale,
                           max_seqlen_q: int):
    """Varlen causal attention of packed query rows ``[T, nh, hd]``; row ``j`` of a chunk of ``q_len``
    sees keys ``< seqlens_k - q_len + j + 1``.  ``max_seqlen_q`` is at least the longest chunk: of a
    longer one, rows are left unwritten, as are the rows behind the last sequence."""
    if not q.is_cuda:
        _check_query(q, k_pages, v_pages, scale)
        return attention_int4_ref(q, k_pages, v_pages, cu_seqlens_q, seqlens_k, block_tables, scale)
    q = q.contiguous()
    out = torch.empty_like(q)
    C().prefill_attention_int4(out, q, k_pages.codes, k_pages.words, v_pages.codes, v_pages.words,
                               cu_seqlens_q, seqlens_k, block_tables, scale, max_seqlen_q, status(q.device))
    return out
