"""4-bit KV cache kernels against the format's 64-bit definition."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from llmserve_b200.ops import kv_int4, rope, step_maps  # noqa: E402
from llmserve_b200.ops._ext import C, check_status  # noqa: E402
from llmserve_b200.ops.attention import DecodeWorkspace  # noqa: E402
from llmserve_b200.ops.kv_int4 import Int4Pages  # noqa: E402
from tests import int4_oracle as oracle  # noqa: E402

DEV = "cuda"


@pytest.fixture(autouse=True)
def _status():
    C()
    yield
    check_status(torch.device(DEV))


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _pages(shape):
    return Int4Pages.zeros(shape, DEV)


def _dequantised(x):
    c, s, z = oracle.quantise(x.double().cpu().numpy())
    return torch.from_numpy((c - np.repeat(z, 64, -1)) * np.repeat(s, 64, -1))


# ---- store and load ----------------------------------------------------------------------------
@pytest.mark.parametrize("T,nkv,hd,bs", [(1, 1, 64, 16), (7, 3, 128, 48), (300, 8, 128, 256), (33, 2, 64, 32)])
def test_store_and_load_hold_the_definitions_codes(T, nkv, hd, bs):
    g = torch.Generator().manual_seed(T + hd)
    x = torch.randn(2, T, nkv, hd, generator=g).bfloat16()
    x[0, 0, 0] = 0
    x[1, 0, 0] = x[1, 0, 0].abs() + 3
    x[:, -1] *= 1e-20
    k, v = x.to(DEV)
    blocks = -(-T // bs) + 1
    kp, vp = _pages((blocks, nkv, bs, hd)), _pages((blocks, nkv, bs, hd))
    slots = torch.randperm(blocks * bs, generator=g)[:T].int()
    if T > 3:
        slots[3] = -1
    kv_int4.store_kvcache_int4(k, v, kp, vp, slots.to(DEV))
    at = slots.long().clamp(min=0)
    for x, p in ((k, kp), (v, vp)):
        want = oracle.quantise(x.double().cpu().numpy())
        got = oracle.unpack(p.codes.cpu()[at // bs, :, at % bs], p.words.cpu()[at // bs, :, at % bs])
        keep = (slots >= 0).numpy()
        for a, b in zip(got, want):
            assert np.array_equal(a[keep], b[keep])
    assert int(kp.words.ne(0).any(-1).sum()) == int(((slots >= 0).sum() * nkv) - (1 if T > 0 else 0))   # the zero row
    for x, y in zip((k, v), kv_int4.load_kvcache_int4(kp, vp, slots.to(DEV))):
        want = _dequantised(x)
        want[slots < 0] = 0
        assert torch.equal(y.double().cpu(), want)


def test_exact_ties_and_every_quotient_round_like_a_division():
    """Every bf16 mantissa against every scale mantissa: 8 scales x codes that lie on and around the
    half-way points."""
    rows = []
    for s8 in range(8, 16):
        s = s8 / 8.0
        body = torch.arange(-62, 62) / 124.0 * 7.5 * s
        half = (torch.arange(-7, 7) + 0.5) * s
        for part in (half, body[:62], body[62:]):
            row = torch.zeros(64)
            row[:part.shape[0]] = part
            row[62], row[63] = 7.5 * s, -7.5 * s
            rows.append(row)
    x = torch.stack(rows).bfloat16().unsqueeze(1)
    T = x.shape[0]
    kp, vp = _pages((2, 1, 16, 64)), _pages((2, 1, 16, 64))
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    kv_int4.store_kvcache_int4(x.to(DEV), -x.to(DEV), kp, vp, slots)
    for y, p in ((x, kp), (-x, vp)):
        c, s, z = oracle.unpack(p.codes.transpose(1, 2).reshape(32, 1, 32)[:T], p.words.transpose(1, 2).reshape(32, 1, 1)[:T])
        want = oracle.quantise(y.double().numpy())
        assert np.array_equal(s, want[1]) and np.array_equal(z, want[2]) and np.array_equal(c, want[0])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_group_that_is_not_finite_reads_back_as_nan(bad):
    x = torch.randn(3, 2, 128, device=DEV).bfloat16()
    x[1, 1, 100] = bad
    kp, vp = _pages((1, 2, 16, 128)), _pages((1, 2, 16, 128))
    slots = _i32(0, 1, 2)
    kv_int4.store_kvcache_int4(x, x, kp, vp, slots)
    k, _ = kv_int4.load_kvcache_int4(kp, vp, slots)
    nan = torch.zeros_like(x, dtype=torch.bool)
    nan[1, 1, 64:] = True
    assert torch.equal(k.isnan(), nan)


def test_store_takes_strided_rows_and_skips_slots_outside_the_pool():
    wide = torch.randn(6, 5 * 64, device=DEV).bfloat16()
    k, v = wide[:, :128].unflatten(1, (2, 64)), wide[:, 129:257].unflatten(1, (2, 64))   # v is not 16-byte aligned
    kp, vp = _pages((2, 2, 16, 64)), _pages((2, 2, 16, 64))
    slots = _i32(31, 0, 5, 6, 7, 8)
    kv_int4.store_kvcache_int4(k, v, kp, vp, slots)
    for x, y in zip((k, v), kv_int4.load_kvcache_int4(kp, vp, slots)):
        assert torch.equal(y.double().cpu(), _dequantised(x))
    before = kp.codes.clone()
    kv_int4.store_kvcache_int4(k[:1] * 2, v[:1], kp, vp, _i32(32))
    with pytest.raises(RuntimeError, match="out-of-range"):
        check_status(torch.device(DEV))
    k2, _ = kv_int4.load_kvcache_int4(kp, vp, _i32(32))
    with pytest.raises(RuntimeError, match="out-of-range"):
        check_status(torch.device(DEV))
    assert torch.equal(before, kp.codes) and k2.eq(0).all()


# ---- fused norm, rotation and store ------------------------------------------------------------
@pytest.mark.parametrize("T,nh,nkv,hd,planes,norm", [(1, 4, 2, 64, 0, True), (37, 32, 8, 128, 0, True),
                                                      (5, 6, 1, 128, 0, False), (64, 32, 8, 128, 3, True),
                                                      (3, 14, 2, 64, 8, False)])
def test_rope_store_matches_the_definition(T, nh, nkv, hd, planes, norm):
    g = torch.Generator().manual_seed(T * nh)
    wide = (nh + 2 * nkv) * hd
    qkv = torch.randn(planes, T, wide, generator=g) if planes else torch.randn(T, wide, generator=g).bfloat16()
    pos = torch.randint(0, 500, (T,), generator=g)
    cs = rope.build_cos_sin_cache(hd, 500, 1e4)
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g)).bfloat16() for _ in range(2)) if norm else (None, None)
    bs = 16
    blocks = -(-T // bs)
    kp, vp = _pages((blocks, nkv, bs, hd)), _pages((blocks, nkv, bs, hd))
    slots = torch.randperm(blocks * bs, generator=g)[:T].int().to(DEV)
    dev = lambda x: x if x is None else x.to(DEV)  # noqa: E731
    q = kv_int4.qkv_norm_rope_store_int4(dev(qkv), dev(pos), dev(cs), dev(qw), dev(kw), 1e-6, kp, vp, slots, nh, nkv, hd)
    k, v = kv_int4.load_kvcache_int4(kp, vp, slots)
    x = qkv.double().sum(0) if planes else qkv.double()
    q64, k64, v64 = x.reshape(T, -1, hd).split((nh, nkv, nkv), 1)

    def turned(y, w):
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.double()
        c, s = cs.double()[pos][:, None].chunk(2, -1)
        a, b = y.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    want = turned(q64, qw)
    # one bfloat16 rounding; a rotated value is a difference of two terms, so fp32 adds 2^-21 of the row
    assert ((q.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * want.abs().amax(-1, keepdim=True)).all()
    for y, got, p in ((turned(k64, kw), k, kp), (v64, v, vp)):
        c, s, z = oracle.quantise(y.numpy())
        step = torch.from_numpy(np.repeat(s, 64, -1))
        want = torch.from_numpy((c - np.repeat(z, 64, -1)) * np.repeat(s, 64, -1))
        off = (got.double().cpu() - want).abs()
        # fp32 noise of 2^-20 moves a value over a border between codes once in 2^16 values or so
        assert (off <= 1.2 * step).all() and int((off > 1e-3 * step).sum()) <= 2


def test_rope_store_skips_positions_and_slots_outside_their_tables():
    qkv = torch.randn(3, 6 * 64, device=DEV).bfloat16()
    kp, vp = _pages((1, 1, 16, 64)), _pages((1, 1, 16, 64))
    cs = rope.build_cos_sin_cache(64, 8, 1e4).to(DEV)
    pos = torch.tensor([1, 8, 2], device=DEV)
    q = kv_int4.qkv_norm_rope_store_int4(qkv, pos, cs, None, None, 1e-6, kp, vp, _i32(4, 5, -1), 4, 1, 64)
    with pytest.raises(RuntimeError, match="out-of-range"):
        check_status(torch.device(DEV))
    assert q[1].eq(0).all() and q[0].ne(0).any() and q[2].ne(0).any()
    assert kp.words[0, 0, :, 0].ne(0).nonzero().flatten().tolist() == [4]


# ---- attention ---------------------------------------------------------------------------------
def _case(B, nh, nkv, hd, bs, q_lens, k_lens, seed, spare=1):
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-max(n, 0) // bs) for n in k_lens]
    width = max(1, max(blocks))
    nblk = sum(blocks) + spare
    kp = oracle.random_pages(nblk, nkv, bs, hd, seed + 1)
    vp = oracle.random_pages(nblk, nkv, bs, hd, seed + 2)
    ids = torch.randperm(nblk, generator=g).int()
    tables = torch.zeros(B, width, dtype=torch.int32)
    at = 0
    for i, n in enumerate(blocks):
        tables[i, :n] = ids[at:at + n]
        at += n
    # what lies behind a context in its last page: NaN scales
    for i, n in enumerate(k_lens):
        if n > 0 and n % bs:
            for p in (kp, vp):
                p[1][tables[i, n // bs], :, n % bs:] = 0x7FC0
    q = torch.randn(sum(q_lens), nh, hd, generator=g).bfloat16()
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    return q, kp, vp, cu, tables


def _on(p):
    return Int4Pages(p[0].to(DEV), p[1].to(DEV))


def _assert_close(got, want, mag):
    off = (got.double().cpu() - want).abs()
    tol = oracle.attention_tolerance(want, mag)
    assert torch.isfinite(got.float()).all()
    assert (off <= tol).all(), f"{(off / tol).max().item():.3f} of the tolerance"


HEADS = [(32, 8, 128), (14, 2, 64), (4, 4, 64), (8, 1, 128), (10, 2, 128), (24, 1, 64)]


@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("bs", [16, 48, 256])
def test_decode(nh, nkv, hd, bs):
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 127, 129, 700]
    q, kp, vp, cu, tables = _case(len(lens), nh, nkv, hd, bs, [1] * len(lens), lens, nh + bs)
    want, mag = oracle.attention(q, kp, vp, cu, lens, tables, hd ** -0.5)
    ws = DecodeWorkspace(len(lens), nh, hd, tables.shape[1] * bs, DEV)
    for w in (ws, None, ws):
        out = kv_int4.decode_attention_int4(q.to(DEV), _on(kp), _on(vp), tables.to(DEV), _i32(*lens), hd ** -0.5, w)
        _assert_close(out, want, mag)
        assert out[1].eq(0).all()
    assert int(ws.counters.abs().sum()) == 0


@pytest.mark.parametrize("B,length", [(1, 20000), (2, 9001), (150, 200)])
def test_decode_long_and_many(B, length):
    lens = [length - 3 * i if length > 1000 else 1 + (i * 37) % length for i in range(B)]
    q, kp, vp, cu, tables = _case(B, 8, 2, 128, 64, [1] * B, lens, B)
    want, mag = oracle.attention(q, kp, vp, cu, lens, tables, 0.088)
    out = kv_int4.decode_attention_int4(q.to(DEV), _on(kp), _on(vp), tables.to(DEV), _i32(*lens), 0.088)
    _assert_close(out, want, mag)


@pytest.mark.parametrize("nq", [2, 3, 4, 7])
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_verify(nq, nh, nkv, hd):
    lens = [nq, nq + 1, 64, 130, 515, 1, 0]         # the last two hold fewer keys than new tokens
    q, kp, vp, cu, tables = _case(len(lens), nh, nkv, hd, 32, [nq] * len(lens), lens, nq)
    want, mag = oracle.attention(q, kp, vp, cu, lens, tables, hd ** -0.5)
    out = kv_int4.verify_attention_int4(q.to(DEV), _on(kp), _on(vp), tables.to(DEV), _i32(*lens), hd ** -0.5, nq)
    _assert_close(out, want, mag)


@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("bs", [16, 48, 256])
def test_prefill(nh, nkv, hd, bs):
    q_lens, k_lens = [1, 130, 0, 33, 64, 5], [300, 130, 40, 65, 1000, 5]
    q, kp, vp, cu, tables = _case(len(q_lens), nh, nkv, hd, bs, q_lens, k_lens, nh * bs)
    want, mag = oracle.attention(q, kp, vp, cu, k_lens, tables, hd ** -0.5)
    out = kv_int4.prefill_attention_int4(q.to(DEV), _on(kp), _on(vp), _i32(*cu), _i32(*k_lens), tables.to(DEV),
                                         hd ** -0.5, max(q_lens))
    _assert_close(out, want, mag)


def test_prefill_long_chunk_and_rows_without_keys():
    q_lens, k_lens = [700, 9], [1500, 4]            # the second chunk's first five rows see nothing
    q, kp, vp, cu, tables = _case(2, 8, 2, 128, 64, q_lens, k_lens, 3)
    want, mag = oracle.attention(q, kp, vp, cu, k_lens, tables, 0.09)
    out = kv_int4.prefill_attention_int4(q.to(DEV), _on(kp), _on(vp), _i32(*cu), _i32(*k_lens), tables.to(DEV), 0.09, 700)
    _assert_close(out, want, mag)
    assert out[700:705].eq(0).all()


@pytest.mark.parametrize("kind", ["prefill", "verify"])
def test_a_nan_token_reaches_only_the_rows_that_see_it(kind):
    """Token 40 of 64 holds NaN in the second group of its V: rows before it are untouched, rows from it on
    are NaN in that group's dims of that KV head's queries and right elsewhere."""
    n, new = 64, 64 if kind == "prefill" else 30
    q, kp, vp, cu, tables = _case(1, 4, 2, 128, 16, [new], [n], 21)
    at = tables[0, 40 // 16], 1, 40 % 16
    whole = vp[1][at].clone()
    vp[1][at][1] = 0x7FC0
    args = (q.to(DEV), _on(kp), _on(vp))
    if kind == "prefill":
        out = kv_int4.prefill_attention_int4(*args, _i32(*cu), _i32(n), tables.to(DEV), 0.09, new)
    else:
        out = kv_int4.verify_attention_int4(*args, tables.to(DEV), _i32(n), 0.09, new)
    vp[1][at] = whole
    want, mag = oracle.attention(q, kp, vp, cu, [n], tables, 0.09)
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[40 - (n - new):, 2:, 64:] = True
    assert torch.equal(out.isnan(), nan)
    keep = ~nan.cpu()
    assert ((out.double().cpu() - want).abs() <= oracle.attention_tolerance(want, mag))[keep].all()


def test_prefill_of_many_ragged_sequences():
    q_lens = [(i * 7) % 5 for i in range(300)]
    q_lens[150] = 400
    k_lens = [n + (i * 13) % 40 for i, n in enumerate(q_lens)]
    q, kp, vp, cu, tables = _case(300, 8, 1, 64, 16, q_lens, k_lens, 2)
    want, mag = oracle.attention(q, kp, vp, cu, k_lens, tables, 0.125)
    out = kv_int4.prefill_attention_int4(q.to(DEV), _on(kp), _on(vp), _i32(*cu), _i32(*k_lens), tables.to(DEV), 0.125, 400)
    _assert_close(out, want, mag)


def test_strong_scores_and_extreme_scales():
    """Scores in the hundreds (one key takes all), V scales from 1e-30 to 1e30."""
    q, kp, vp, cu, tables = _case(3, 8, 2, 128, 16, [1, 1, 1], [40, 300, 77], 9)
    q = q * 30
    for i, s in enumerate((1e-30, 1.0, 1e30)):
        ids = tables[i, :-(-[40, 300, 77][i] // 16)].long()
        vp[1][ids] = oracle.random_pages(len(ids), 2, 16, 128, i, scale=s)[1]
    want, mag = oracle.attention(q, kp, vp, cu, [40, 300, 77], tables, 1.0)
    out = kv_int4.decode_attention_int4(q.to(DEV), _on(kp), _on(vp), tables.to(DEV), _i32(40, 300, 77), 1.0)
    off = (out.double().cpu() - want).abs()
    # a score is a sum of 128 products in fp32: at most 12 partial sums one after another, each off by
    # 2^-23 of the magnitudes added, so off by e = 12 * 2^-23 * sum |q k|.  A weight exp(s) is then off by
    # a factor within exp(+-e), the sum it is divided by too: 2 e of the magnitudes averaged
    k = oracle.values(*kp).abs()
    most = max((q[i].double().abs().view(2, 4, 128) @ k[tables[i, :-(-n // 16)].long()].transpose(0, 1).flatten(1, 2)
                .transpose(1, 2)).amax().item() for i, n in enumerate((40, 300, 77)))
    tol = oracle.attention_tolerance(want, mag) + 2 * 12 * 2.0 ** -23 * most * mag
    assert (off <= tol).all(), f"{(off / tol).max().item():.3f} of the tolerance"


def test_block_ids_outside_the_pool_are_not_seen_and_long_contexts_end_at_their_table():
    lens, bs = [100, 150, 400, 30], 64
    q, kp, vp, cu, tables = _case(4, 8, 2, 128, bs, [1] * 4, lens, 5)
    tables[1, 1] = kp[0].shape[0] + 7
    tables[3, 0] = -2
    tables = tables[:, :3].contiguous()
    lens_t = _i32(*lens)
    want, mag = oracle.attention(q, kp, vp, cu, lens, tables, 0.088)
    out = kv_int4.decode_attention_int4(q.to(DEV), _on(kp), _on(vp), tables.to(DEV), lens_t, 0.088)
    with pytest.raises(RuntimeError, match="out-of-range"):
        check_status(torch.device(DEV))
    _assert_close(out, want, mag)
    assert out[3].eq(0).all()
    out = kv_int4.prefill_attention_int4(q.to(DEV), _on(kp), _on(vp), _i32(*cu), lens_t, tables.to(DEV), 0.088, 1)
    with pytest.raises(RuntimeError, match="out-of-range"):
        check_status(torch.device(DEV))
    _assert_close(out, want, mag)


def test_offsets_past_32_bits():
    """Pools of 2.4 GB of codes each: the last blocks lie more than 2^31 bytes from the first."""
    nkv, bs, hd, blocks = 8, 16, 128, 290000
    n = 75
    q, kp, vp, cu, tables = _case(1, 16, nkv, hd, bs, [9], [n], 31, spare=0)
    small = kp[0].shape[0]
    big = [_pages((blocks, nkv, bs, hd)) for _ in range(2)]
    for p, b in zip((kp, vp), big):
        b.codes[blocks - small:], b.words[blocks - small:] = p[0].to(DEV), p[1].to(DEV)
    far = (tables + blocks - small).to(DEV)
    want, mag = oracle.attention(q, kp, vp, cu, [n], tables, 0.09)
    _assert_close(kv_int4.prefill_attention_int4(q.to(DEV), *big, _i32(*cu), _i32(n), far, 0.09, 9), want, mag)
    _assert_close(kv_int4.verify_attention_int4(q.to(DEV), *big, far, _i32(n), 0.09, 9), want, mag)
    x = torch.randn(2, nkv, hd, device=DEV).bfloat16()
    slots = _i32(blocks * bs - 1, 3)
    kv_int4.store_kvcache_int4(x, -x, *big, slots)
    k, v = kv_int4.load_kvcache_int4(*big, slots)
    assert torch.equal(k.double().cpu(), _dequantised(x)) and torch.equal(v.double().cpu(), _dequantised(-x))
    qkv = torch.randn(2, 18 * hd, device=DEV).bfloat16()
    kv_int4.qkv_norm_rope_store_int4(qkv, torch.zeros(2, dtype=torch.long, device=DEV),
                                     rope.build_cos_sin_cache(hd, 4, 1e4).to(DEV), None, None, 1e-6, *big, slots, 2, nkv, hd)
    v = kv_int4.load_kvcache_int4(*big, slots)[1]
    assert torch.equal(v.double().cpu(), _dequantised(qkv[:, 10 * hd:].reshape(2, nkv, hd)))


def test_two_streams_with_a_workspace_each():
    lens = [900, 33, 4000]
    q, kp, vp, cu, tables = _case(3, 8, 2, 128, 64, [1] * 3, lens, 12)
    want, mag = oracle.attention(q, kp, vp, cu, lens, tables, 0.09)
    qd, k, v, t, n = q.to(DEV), _on(kp), _on(vp), tables.to(DEV), _i32(*lens)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    spaces = [DecodeWorkspace(3, 8, 128, tables.shape[1] * 64, DEV) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, w in zip(streams, spaces):
            with torch.cuda.stream(stream):
                outs.append(kv_int4.decode_attention_int4(qd, k, v, t, n, 0.09, w))
    torch.cuda.synchronize()
    _assert_close(outs[0], want, mag)
    # pieces are merged in their order: the same bits every time
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_captured_decode_replays_on_new_lengths_and_side_streams():
    lens = [300, 0, 17, 512]
    q, kp, vp, cu, tables = _case(4, 8, 2, 128, 64, [1] * 4, [512] * 4, 8)
    qd, k, v, t = q.to(DEV), _on(kp), _on(vp), tables.to(DEV)
    n = _i32(1, 1, 1, 1)
    ws = DecodeWorkspace(4, 8, 128, 512, DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv_int4.decode_attention_int4(qd, k, v, t, n, 0.088, ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = kv_int4.decode_attention_int4(qd, k, v, t, n, 0.088, ws)
        for L in (lens, [1, 2, 3, 4], lens):
            n.copy_(_i32(*L))
            graph.replay()
            want, mag = oracle.attention(q, kp, vp, cu, L, tables, 0.088)
            side.synchronize()
            _assert_close(out, want, mag)


# ---- step maps ---------------------------------------------------------------------------------
@pytest.mark.parametrize("B,bs,hi", [(1, 16, 1), (3, 256, 700), (513, 48, 9), (2000, 16, 40)])
def test_step_maps_equal_the_host_form(B, bs, hi):
    g = torch.Generator().manual_seed(B)
    q = torch.randint(0, hi + 1, (B,), generator=g).int()
    k = (q + torch.randint(0, 300, (B,), generator=g)).int()
    blocks = (k + bs - 1) // bs
    ids = torch.randperm(int(blocks.sum()) + 5, generator=g).int()
    T, width = int(q.sum()) + 3, max(1, int(blocks.max()) - (B > 500))
    want = step_maps.build_step_maps(q, k, ids, bs, T, width)
    got = step_maps.build_step_maps(q.to(DEV), k.to(DEV), ids.to(DEV), bs, T, width)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b)


def test_step_maps_record_lengths_that_contradict():
    for q, k, ids, T in (((3, 2), (2, 9), (0, 1, 2), 5), ((4,), (4,), (0,), 3), ((1,), (40,), (0, 1), 1),
                         ((2 ** 30, 2 ** 30, 2 ** 30, 1), (2 ** 30,) * 3 + (1,), (0,), 4)):
        m = step_maps.build_step_maps(_i32(*q), _i32(*k), _i32(*ids), 16, T, 4)
        with pytest.raises(RuntimeError, match="out-of-range"):
            check_status(torch.device(DEV))
        assert int(m.slot_mapping.max()) < len(ids) * 16
    with pytest.raises(RuntimeError, match="8192"):
        step_maps.build_step_maps(torch.zeros(8193, dtype=torch.int32, device=DEV),
                                  torch.zeros(8193, dtype=torch.int32, device=DEV), _i32(0), 16, 1, 1)
    assert step_maps.build_step_maps(_i32(), _i32(), _i32(), 16, 2, 1).slot_mapping.tolist() == [-1, -1]


# ---- refusals ----------------------------------------------------------------------------------
def test_refusals():
    x = torch.randn(2, 2, 64, device=DEV).bfloat16()
    kp, vp = _pages((2, 2, 16, 64)), _pages((2, 2, 16, 64))
    s, t = _i32(0, 1), _i32(0, 1).view(2, 1)
    for k, p, slots in ((x.float(), kp, s), (x, kp, s.long()), (x, kp, _i32(0)), (x, kp, s.cpu()),
                        (x, _pages((2, 2, 16, 128)), s), (x, Int4Pages(kp.codes[:, :, ::2], kp.words[:, :, ::2]), s),
                        (x, Int4Pages(kp.codes, kp.words[:1]), s), (x, Int4Pages(kp.codes.cpu(), kp.words.cpu()), s)):
        with pytest.raises(RuntimeError, match="llmserve_b200"):
            kv_int4.store_kvcache_int4(k, x, p, vp, slots)
    for q, tables, lens in ((x.half(), t, s), (x[:, :1], t, s), (x, t.view(-1), s), (x, t, s.long()), (x, t[:1], s)):
        with pytest.raises(RuntimeError, match="llmserve_b200"):
            kv_int4.decode_attention_int4(q, kp, vp, tables, lens, 1.0)
    with pytest.raises(RuntimeError, match="cu_seqlens_q"):
        kv_int4.prefill_attention_int4(x, kp, vp, s, s, t, 1.0, 1)
    with pytest.raises(RuntimeError, match="width"):
        kv_int4.qkv_norm_rope_store_int4(x.view(2, 128), torch.zeros(2, dtype=torch.long, device=DEV),
                                         torch.zeros(4, 64, device=DEV), None, None, 1e-6, kp, vp, s, 2, 2, 64)
