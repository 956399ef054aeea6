"""Measured cases of the operators that serve from a KV cache held in 4 bits.

Operators: ``store`` (K/V rows into 4-bit pages and back), ``rope_store`` (QK-norm, RoPE and the
4-bit store of one step's projection), ``decode`` (one or a few queries per sequence against the
pages), ``prefill`` (ragged causal chunks against the pages) and ``maps`` (a step's positions, slots
and block tables from request lengths).

Pages: codes ``uint8 [blocks, kv_heads, block_size, head_dim / 2]`` (dim ``2i`` in the low nibble)
and scale words ``int16 [blocks, kv_heads, block_size, head_dim / 64]``.  A word is the bfloat16
pattern of the group's scale with the low four bits holding the zero code; a code ``c`` stands for
``scale * (c - zero)``.
"""
import math
import random

import numpy as np
import torch

own = False

GROUP = 64
EPS = 1e-6
DEV = "cuda"
# (query heads, kv heads, head dim): grouped 4, 2, 5, 8, 7, 1 to a kv head, and tensor-parallel shards
HEADS = [(32, 8, 128), (16, 8, 128), (40, 8, 128), (64, 8, 128), (28, 4, 128), (14, 2, 64), (8, 1, 128),
         (4, 1, 128), (32, 8, 64), (12, 12, 64), (4, 2, 64)]
BLOCKS = [16, 32, 48, 64, 128, 256]


# ---- cases -------------------------------------------------------------------------------------
def listed():
    h = {"nh": 32, "nkv": 8, "hd": 128, "bs": 256}
    return [
        # rows of one decode step of 64 requests, scattered over the pool
        {"name": "store step 64", "op": "store", **h, "rows": 64},
        # a full prefill budget of 16384 tokens
        {"name": "store prompt 16384", "op": "store", **h, "rows": 16384},
        # the decode step's QKV projection arrives as fp32 split-K planes
        {"name": "rope store step 64", "op": "rope_store", **h, "rows": 64, "planes": 4, "qknorm": True},
        # a long prompt's projection, bf16, ragged count
        {"name": "rope store prompt 8191", "op": "rope_store", **h, "rows": 8191, "planes": 0, "qknorm": True},
        # one request, short context: latency
        {"name": "decode 1x513", "op": "decode", **h, "batch": 1, "lo": 513, "hi": 513, "nq": 1, "pick": 1},
        # the serving benchmark's batch: 64 requests between 256 and 512 tokens
        {"name": "decode 64x512", "op": "decode", **h, "batch": 64, "lo": 256, "hi": 512, "nq": 1, "pick": 2},
        # long ragged contexts, from nearly nothing to 32768 tokens
        {"name": "decode 32x32768", "op": "decode", **h, "batch": 32, "lo": 1, "hi": 32768, "nq": 1, "pick": 3},
        # a verify step: the last token and three drafts of every request
        {"name": "verify 64x4", "op": "decode", **h, "batch": 64, "lo": 200, "hi": 2048, "nq": 4, "pick": 4},
        # one prompt of 4096 tokens
        {"name": "prefill 4096", "op": "prefill", **h, "batch": 1, "q_lo": 4096, "q_hi": 4096, "p_lo": 0, "p_hi": 0,
         "pick": 5},
        # chunked prefill next to decodes: ragged chunks on cached prefixes, small heads, small blocks
        {"name": "prefill chunks", "op": "prefill", "nh": 14, "nkv": 2, "hd": 64, "bs": 32, "batch": 9, "q_lo": 1,
         "q_hi": 700, "p_lo": 0, "p_hi": 6000, "pick": 6},
        # a decode step's maps at the engine's largest batch
        {"name": "maps step 512", "op": "maps", "bs": 256, "batch": 512, "q_lo": 1, "q_hi": 1, "p_lo": 1, "p_hi": 4000,
         "pick": 7},
        # a prefill step's maps: 37 ragged prompts
        {"name": "maps prompts 37", "op": "maps", "bs": 16, "batch": 37, "q_lo": 1, "q_hi": 880, "p_lo": 0,
         "p_hi": 2000, "pick": 8},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["store", "rope_store", "decode", "decode", "prefill", "prefill", "maps"])
    nh, nkv, hd = rng.choice(HEADS)
    case = {"op": op, "nh": nh, "nkv": nkv, "hd": hd, "bs": rng.choice(BLOCKS)}
    if op == "store":
        return {**case, "rows": _log(rng, 1, 16384 * 8 // max(nkv, 8))}
    if op == "rope_store":
        planes = rng.choice([0, 0, 1, 2, 4, 8])
        return {**case, "rows": _log(rng, 1, 256 if planes else 8191 * 48 // max(nh + 2 * nkv, 48)), "planes": planes,
                "qknorm": rng.random() < 0.7}
    pick = rng.randrange(1 << 30)
    if op == "decode":
        nq = rng.choice([1, 1, 1, 2, 4])
        batch = _log(rng, 1, 256)
        hi = _log(rng, 2 * nq, max(2 * nq, min(32768, 4000000 // (batch * max(nkv, 4)))))
        return {**case, "batch": batch, "lo": rng.choice([0, nq, hi // 2, hi]) if nq == 1 else rng.choice([nq, hi]),
                "hi": hi, "nq": nq, "pick": pick}
    if op == "prefill":
        batch = _log(rng, 1, 12)
        # the plain form pads to the longest chunk and key count: keep that product within a 4096-token prompt's
        q_hi = _log(rng, 2, 4096 if batch == 1 else 1024)
        p_hi = rng.choice([0, _log(rng, 1, 16384)])
        while batch * nh * q_hi * (q_hi + p_hi) > 32 * 4096 * 4096:
            q_hi, p_hi = max(2, q_hi * 2 // 3), p_hi * 2 // 3
        return {**case, "batch": batch, "q_lo": rng.choice([1, q_hi]), "q_hi": q_hi, "p_lo": 0, "p_hi": p_hi, "pick": pick}
    batch = _log(rng, 1, 512)
    q_hi = rng.choice([1, _log(rng, 1, max(1, 16384 // batch))])
    return {"op": op, "bs": case["bs"], "batch": batch, "q_lo": 1, "q_hi": q_hi, "p_lo": 0, "p_hi": _log(rng, 1, 4000),
            "pick": pick}


def _lengths(case):
    """(new tokens, cached tokens before them) of each request."""
    r = random.Random(case["pick"])
    if case["op"] == "decode":
        k = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
        return [case["nq"]] * case["batch"], [n - case["nq"] for n in k]
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    return q, [r.randint(case["p_lo"], case["p_hi"]) for _ in q]


def work(case):
    op = case["op"]
    if op == "maps":
        q, p = _lengths(case)
        blocks = [-(-(a + b) // case["bs"]) for a, b in zip(q, p)]
        n = len(q)
        return {"bytes": 8 * n + 4 * sum(blocks) + 12 * sum(q) + 4 * n * max(blocks) + 12 * n + 4, "flops": 0}
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    row = 2 * nkv * (hd // 2 + 2 * (hd // GROUP))          # one token's K and V in the pages
    if op == "store":
        t = case["rows"]
        return {"bytes": t * (2 * (2 * nkv * hd * 2) + 2 * row + 8), "flops": 0}
    if op == "rope_store":
        t, wide = case["rows"], (nh + 2 * nkv) * hd
        return {"bytes": t * (wide * (4 * case["planes"] or 2) + 4 * hd + 2 * nh * hd + 2 * row + 2 * nkv * hd * 2 + 16),
                "flops": 0}
    q, p = _lengths(case)
    seen = sum(a * b + a * (a + 1) // 2 for a, b in zip(q, p)) if op == "prefill" or case["nq"] > 1 else sum(
        a + b for a, b in zip(q, p))
    keys = sum(a + b for a, b in zip(q, p))
    return {"bytes": keys * row + 4 * sum(q) * nh * hd + 4 * sum(-(-(a + b) // case["bs"]) for a, b in zip(q, p)),
            "flops": 4 * nh * hd * seen}


# ---- inputs ------------------------------------------------------------------------------------
def _quantise(x):
    """fp32 [..., hd] -> codes, scale words: the group's range widened to hold zero, the scale rounded
    up to four significant bits, everything in 32 bits."""
    g = x.unflatten(-1, (-1, GROUP))
    mx, mn = g.amax(-1).clamp(min=0), g.amin(-1).clamp(max=0)
    r = (mx * 0.5 - mn * 0.5) / torch.full_like(mx, 7.5)      # a true division: whole quotients stay whole
    bits = (r.view(torch.int32) + 0xFFFFF) & 0x7FF00000
    bits = torch.where(r < 2.0 ** -126, torch.zeros_like(bits), bits)
    s = bits.view(torch.float32)
    safe = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.where(s > 0, torch.round(-mn / safe), torch.zeros_like(s))
    c = torch.where(s[..., None] > 0, torch.round(g / safe[..., None]) + z[..., None], torch.zeros_like(g))
    bad = ~torch.isfinite(r)
    words = torch.where(bad, torch.full_like(bits, 0x7FC0), (bits >> 16) | z.nan_to_num().int())
    c = torch.where(bad[..., None], torch.zeros_like(c), c).clamp(0, 15).flatten(-2).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), words.to(torch.int16)


def _values(codes, words):
    """What the pages stand for, fp32 [..., hd]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    w = words.int()
    scale = ((w & 0x7FF0) << 16).view(torch.float32)
    return ((c - (w & 15).float()[..., None]) * scale[..., None]).flatten(-2)


def _pool(case, blocks, g):
    """A pool in use: every row holds a token's K and V, keys with a few strong channels."""
    shape = (blocks, case["nkv"], case["bs"], case["hd"])
    strong = 1 + 3 * (torch.rand(case["hd"], device=DEV, generator=g) > 0.95)
    kc, kw = _quantise(torch.randn(shape, device=DEV, generator=g) * strong)
    vc, vw = _quantise(torch.randn(shape, device=DEV, generator=g) * 0.5)
    return {"k_codes": kc, "k_words": kw, "v_codes": vc, "v_words": vw}


def _empty_pool(case, blocks):
    shape = (blocks, case["nkv"], case["bs"])
    return {a + b: torch.zeros(*shape, n, dtype=t, device=DEV) for a in ("k_", "v_") for b, n, t in
            (("codes", case["hd"] // 2, torch.uint8), ("words", case["hd"] // GROUP, torch.int16))}


def _tables(blocks, g):
    """A block table whose pages are scattered over the pool, zero padded."""
    total, width = sum(blocks), max(1, max(blocks))
    ids = torch.randperm(max(total, 1), device=DEV, generator=g).int()
    t = torch.zeros(len(blocks), width, dtype=torch.int32, device=DEV)
    keep = torch.arange(width, device=DEV) < torch.tensor(blocks, device=DEV)[:, None]
    t[keep] = ids[:total]
    return t, ids[:total], max(total, 1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)
    op, s = case["op"], {"case": dict(case)}
    if op in ("store", "rope_store"):
        t, bs = case["rows"], case["bs"]
        blocks = -(-t // bs) + 2
        s |= _empty_pool(case, blocks)
        s["slots"] = torch.randperm(blocks * bs, device=DEV, generator=g)[:t].int()
        if op == "store":
            s["k"] = (torch.randn(t, case["nkv"], case["hd"], device=DEV, generator=g) * 2).bfloat16()
            s["v"] = torch.randn(t, case["nkv"], case["hd"], device=DEV, generator=g).bfloat16()
            return s
        wide, hd = (case["nh"] + 2 * case["nkv"]) * case["hd"], case["hd"]
        if case["planes"]:
            s["qkv"] = torch.randn(case["planes"], t, wide, device=DEV, generator=g)
        else:
            s["qkv"] = torch.randn(t, wide, device=DEV, generator=g).bfloat16()
        s["positions"] = torch.randperm(max(t, 8192), device=DEV, generator=g)[:t]
        inv = 1.0 / (1e6 ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd))
        angle = torch.arange(max(t, 8192), device=DEV, dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat((angle.cos(), angle.sin()), -1).float()
        s["qw"] = s["kw"] = None
        if case["qknorm"]:
            s["qw"] = (1 + 0.3 * torch.randn(hd, device=DEV, generator=g)).bfloat16()
            s["kw"] = (1 + 0.3 * torch.randn(hd, device=DEV, generator=g)).bfloat16()
        return s
    q, p = _lengths(case)
    lens = [a + b for a, b in zip(q, p)]
    blocks = [-(-max(n, 0) // case["bs"]) for n in lens]
    s["q_lens"] = torch.tensor(q, dtype=torch.int32, device=DEV)
    s["k_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["tables"], s["ids"], total = _tables(blocks, g)
    s["rows"], s["width"], s["max_q"] = sum(q), s["tables"].shape[1], max(q)
    if op != "maps":
        s |= _pool(case, total, g)
        s["q"] = (torch.randn(sum(q), case["nh"], case["hd"], device=DEV, generator=g) * 1.5).bfloat16()
        s["cu_q"] = torch.tensor([0] + list(np.cumsum(q)), dtype=torch.int32, device=DEV)
    return s


# ---- one pass ----------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from llmserve_b200.ops import attention, kv_int4, step_maps
    case = s["case"]
    op = case["op"]
    if op == "maps":
        m = step_maps.build_step_maps(s["q_lens"], s["k_lens"], s["ids"], case["bs"], s["rows"], s["width"])
        return {"cu": m.cu_seqlens_q, "positions": m.positions, "slots": m.slot_mapping, "tables": m.block_tables,
                "last": m.last_token_indices}
    if "pages" not in s:          # a program binds its pools (and decode scratch) once
        s["pages"] = (kv_int4.Int4Pages(s["k_codes"], s["k_words"]), kv_int4.Int4Pages(s["v_codes"], s["v_words"]))
        if op == "decode":
            s["workspace"] = attention.DecodeWorkspace(s["q"].shape[0], case["nh"], case["hd"],
                                                       s["tables"].shape[1] * case["bs"], DEV)
    kp, vp = s["pages"]
    if op == "store":
        kv_int4.store_kvcache_int4(s["k"], s["v"], kp, vp, s["slots"])
        return kv_int4.load_kvcache_int4(kp, vp, s["slots"])
    if op == "rope_store":
        q = kv_int4.qkv_norm_rope_store_int4(s["qkv"], s["positions"], s["cos_sin"], s["qw"], s["kw"], EPS, kp, vp,
                                             s["slots"], case["nh"], case["nkv"], case["hd"])
        return (q, *kv_int4.load_kvcache_int4(kp, vp, s["slots"]))
    scale = case["hd"] ** -0.5
    if op == "prefill":
        return kv_int4.prefill_attention_int4(s["q"], kp, vp, s["cu_q"], s["k_lens"], s["tables"], scale, s["max_q"])
    if case["nq"] > 1:
        return kv_int4.verify_attention_int4(s["q"], kp, vp, s["tables"], s["k_lens"], scale, case["nq"], s["workspace"])
    return kv_int4.decode_attention_int4(s["q"], kp, vp, s["tables"], s["k_lens"], scale, s["workspace"])


def _write(s, kind, x):
    """Quantise rows into the pages at the slots; the rows as the pages now hold them."""
    bs = s["case"]["bs"]
    at = s["slots"].long()
    blk, off = at // bs, at % bs
    codes, words = _quantise(x)
    s[kind + "_codes"][blk, :, off] = codes
    s[kind + "_words"][blk, :, off] = words
    return _values(s[kind + "_codes"][blk, :, off], s[kind + "_words"][blk, :, off]).bfloat16()


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "store":
        return _write(s, "k", s["k"].float()), _write(s, "v", s["v"].float())
    if op == "rope_store":
        nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
        x = s["qkv"].sum(0) if case["planes"] else s["qkv"].float()
        q, k, v = x.unflatten(-1, (-1, hd)).split((nh, nkv, nkv), 1)
        cos, sin = s["cos_sin"][s["positions"]][:, None].chunk(2, -1)
        q = _rotate(_normed(q, s["qw"]), cos, sin).bfloat16()
        return q, _write(s, "k", _rotate(_normed(k, s["kw"]), cos, sin)), _write(s, "v", v)
    if op == "maps":
        return _plain_maps(s)
    return _plain_attention(s)


def _plain_maps(s):
    bs, q, k, width = s["case"]["bs"], s["q_lens"].long(), s["k_lens"].long(), s["width"]
    n = q.shape[0]
    cu = torch.cat((q.new_zeros(1), q.cumsum(0)))
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), q, output_size=s["rows"])
    pos = torch.arange(s["rows"], device=DEV) - cu[seq] + (k - q)[seq]
    blocks = (k + bs - 1) // bs
    first = blocks.cumsum(0) - blocks
    col = torch.arange(width, device=DEV)
    at = (first[:, None] + col).clamp(max=max(s["ids"].shape[0] - 1, 0))
    tables = torch.where(col < blocks[:, None], s["ids"][at], 0).int()
    slots = tables[seq, pos // bs].long() * bs + pos % bs
    return {"cu": cu.int(), "positions": pos, "slots": slots.int(), "tables": tables, "last": cu[1:] - 1}


def _plain_attention(s):
    """Chunks and keys padded to the longest of the batch; a row that sees no key gives zeros."""
    case = s["case"]
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    q_lens, k_lens, mq = s["q_lens"].long(), s["k_lens"].long(), s["max_q"]
    n, group = q_lens.shape[0], nh // nkv
    tables = s["tables"].long()
    k = _values(s["k_codes"][tables], s["k_words"][tables]).transpose(1, 2).flatten(2, 3)      # [n, nkv, keys, hd]
    v = _values(s["v_codes"][tables], s["v_words"][tables]).transpose(1, 2).flatten(2, 3)
    j = torch.arange(mq, device=DEV)
    live = j < q_lens[:, None]
    at = (s["cu_q"][:-1].long()[:, None] + j).clamp(max=s["rows"] - 1)
    q = s["q"][at].float().unflatten(2, (nkv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)     # [n, nkv, group * mq, hd]
    a = torch.matmul(q, k.transpose(2, 3)).unflatten(2, (group, mq)).mul_(hd ** -0.5)
    last = (k_lens - q_lens)[:, None] + j                                                       # key seen last by row j
    hidden = torch.arange(k.shape[2], device=DEV) > last[..., None]
    hidden |= (torch.arange(k.shape[2], device=DEV) >= k_lens[:, None])[:, None]
    a.masked_fill_(hidden[:, None, None], -math.inf)
    a = a.sub_(a.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    a = a.div_(a.sum(-1, keepdim=True).clamp(min=1e-30)).flatten(2, 3)
    o = torch.matmul(a, v).unflatten(2, (group, mq)).permute(0, 3, 1, 2, 4).flatten(2, 3)      # [n, mq, nh, hd]
    return o[live].bfloat16()


# ---- the definition in 64 bits -----------------------------------------------------------------
def _store64(x):
    """Values that rows ``x`` (float64 [..., hd]) have in the pages."""
    y = torch.zeros_like(x)
    for g in range(x.shape[-1] // GROUP):
        part = x[..., g * GROUP:(g + 1) * GROUP]
        low, high = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
        low, high = torch.minimum(low, torch.zeros_like(low)), torch.maximum(high, torch.zeros_like(high))
        m, e = torch.frexp((high - low) / 15)
        scale = torch.ldexp(torch.ceil(m * 16) / 16, e)
        fine = high > low
        scale = torch.where(fine, scale, torch.ones_like(scale))
        zero = torch.round(-low / scale)
        code = torch.minimum(torch.round(part / scale) + zero, torch.full_like(part, 15))
        y[..., g * GROUP:(g + 1) * GROUP] = torch.where(fine, scale * (code - zero), torch.zeros_like(part))
    return y


def _page_rows64(s, kind, i, n):
    """The first n rows of request i, float64 [n, nkv, hd]."""
    bs = s["case"]["bs"]
    pages = s["tables"][i, :-(-n // bs)].long()
    c, w = s[kind + "_codes"][pages], s[kind + "_words"][pages].to(torch.int64)
    out = torch.empty(*c.shape[:-1], 2 * c.shape[-1], dtype=torch.float64, device=DEV)
    out[..., 0::2], out[..., 1::2] = (c % 16).double(), (c // 16).double()
    w = w.repeat_interleave(GROUP, -1)
    mantissa, exponent = ((w >> 4) % 8).double() / 8 + 1, (w >> 7) % 256
    scale = torch.where(exponent > 0, torch.ldexp(mantissa, exponent - 127), torch.zeros_like(mantissa))
    out = (out - (w % 16).double()) * scale
    return out.transpose(1, 2).reshape(-1, out.shape[1], out.shape[3])[:n]


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "maps":
        return None
    if op == "store":
        return _store64(s["k"].double()), _store64(s["v"].double())
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if op == "rope_store":
        x = s["qkv"].double()
        x = (x.sum(0) if case["planes"] else x).reshape(case["rows"], nh + 2 * nkv, hd)
        table = s["cos_sin"].double()[s["positions"]]
        turn = torch.complex(table[:, :hd // 2], table[:, hd // 2:])[:, None]

        def turned(y, w):
            if w is not None:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / hd + EPS) * w.double()
            y = torch.complex(y[..., :hd // 2], y[..., hd // 2:]) * turn
            return torch.cat((y.real, y.imag), -1)

        return turned(x[:, :nh], s["qw"]), _store64(turned(x[:, nh:nh + nkv], s["kw"])), _store64(x[:, nh + nkv:])
    q_lens, p = _lengths(case)
    out = torch.zeros(sum(q_lens), nh, hd, dtype=torch.float64, device=DEV)
    at = 0
    for i, (n, before) in enumerate(zip(q_lens, p)):
        if n + before > 0:
            k, v = _page_rows64(s, "k", i, n + before), _page_rows64(s, "v", i, n + before)
            sees = torch.arange(n + before, device=DEV)[None] <= torch.arange(before, before + n, device=DEV)[:, None]
            for h in range(nh):
                a = s["q"][at:at + n, h].double() @ k[:, h // (nh // nkv)].T / math.sqrt(hd)
                a = torch.softmax(a.masked_fill(~sees, -math.inf), -1)
                out[at:at + n, h] = a @ v[:, h // (nh // nkv)]
        at += n
    return out
