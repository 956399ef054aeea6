"""4-bit KV cache kernels where a block has more than one piece of work: shares of several chunks that cross KV heads
and sequences (decode), several heads to a lane group (norm, rotation and store)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from llmserve_b200.ops import attention, kv_int4, rope  # noqa: E402
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


def _case(lens, nh, nkv, hd, bs, nq, seed):
    """Contexts in scattered blocks, NaN scales behind each of them."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // bs) for n in lens]
    kp, vp = (oracle.random_pages(sum(blocks), nkv, bs, hd, seed + i) for i in (1, 2))
    ids = torch.randperm(sum(blocks), generator=g).int().split(blocks)
    tables = torch.zeros(len(lens), max(blocks), dtype=torch.int32)
    for i, n in enumerate(lens):
        tables[i, :blocks[i]] = ids[i]
        if n % bs:
            for p in (kp, vp):
                p[1][ids[i][-1].item(), :, n % bs:] = 0x7FC0
    return torch.randn(len(lens) * nq, nh, hd, generator=g).bfloat16(), kp, vp, tables


def _ragged(batch, hi, seed):
    """Lengths over the whole range, with runs of empty contexts inside and at both ends."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, hi + 1, (batch,), generator=g).tolist()
    for i in (0, 1, 7, 8, 9, 20, batch - 1):
        lens[i] = 0
    return lens


@pytest.mark.parametrize("lens,nh,nkv,hd,nq", [
    (_ragged(48, 2000, 1), 16, 4, 128, 1),
    (_ragged(48, 2000, 2), 16, 4, 64, 1),
    (_ragged(48, 2000, 3), 16, 4, 128, 4),              # two row tiles: 296 blocks
    (_ragged(48, 2000, 4), 8, 4, 64, 4),
    (_ragged(100, 300, 5), 8, 8, 64, 1),                # more (sequence, head) pairs than blocks
    ([3000, 0, 0, 1700, 5, 2500], 24, 1, 128, 7),       # 21 row tiles: 28 blocks
    ([9000] + [1] * 30 + [0] * 3 + [6000], 8, 2, 64, 1),
])
def test_decode_shares_of_several_chunks(lens, nh, nkv, hd, nq):
    bs = 48
    tiles = -(-nq * nh // nkv // 8)
    chunks = [-(-n // 128) for n in lens]
    blocks = min(148 * 4 // tiles, len(lens) * nkv * -(-max(lens) // 128))
    # what this is about: some block's share holds more than one chunk
    assert sum(chunks) * nkv > blocks or len(lens) * nkv > blocks or max(chunks) > 8
    q, kp, vp, tables = _case(lens, nh, nkv, hd, bs, nq, nh + hd + nq)
    scale = hd ** -0.5
    want, mag = oracle.attention(q, kp, vp, list(range(0, len(q) + 1, nq)), lens, tables, scale)
    ws = DecodeWorkspace(len(q), nh, hd, tables.shape[1] * bs, DEV)
    args = (q.to(DEV), Int4Pages(*(x.to(DEV) for x in kp)), Int4Pages(*(x.to(DEV) for x in vp)), tables.to(DEV), _i32(*lens), scale)
    outs = [kv_int4.verify_attention_int4(*args, nq, ws) for _ in range(2)]
    assert torch.isfinite(outs[0].float()).all()
    off, tol = (outs[0].double().cpu() - want).abs(), oracle.attention_tolerance(want, mag)
    assert (off <= tol).all(), f"{(off / tol).max().item():.3f} of the tolerance"
    assert torch.equal(*outs)                           # pieces are merged in their order
    assert int(ws.counters.abs().sum()) == 0


def test_one_workspace_serves_4_bit_and_bf16_decode_by_turns():
    """A draft's bf16 pool and the target's 4-bit pages share the runner's workspace."""
    lens, nh, nkv, hd, bs = [2000, 0, 300, 5000], 8, 2, 128, 64
    q, kp, vp, tables = _case(lens, nh, nkv, hd, bs, 1, 3)
    for p in (kp, vp):
        p[1][p[1] == 0x7FC0] = 0                        # the bf16 kernels read whole pages
    want, mag = oracle.attention(q, kp, vp, list(range(5)), lens, tables, 0.09)
    k, v = (oracle.values(*p).bfloat16().to(DEV) for p in (kp, vp))
    args = (tables.to(DEV), _i32(*lens), 0.09, DecodeWorkspace(4, nh, hd, tables.shape[1] * bs, DEV))
    pages = [Int4Pages(*(x.to(DEV) for x in p)) for p in (kp, vp)]
    for _ in range(3):
        packed = kv_int4.decode_attention_int4(q.to(DEV), *pages, *args)
        plain = attention.decode_attention(q.to(DEV), k, v, *args)
        for out in (packed, plain):
            keep = [0, 2, 3]
            off, tol = (out.double().cpu() - want).abs(), oracle.attention_tolerance(want, mag)
            assert (off <= tol)[keep].all()
    assert int(args[3].counters.abs().sum()) == 0


# heads to a lane group: 2 (18 heads, the last group ragged), 2 (36 heads over 5 groups of 8), 6, 2 of fp32 planes
@pytest.mark.parametrize("T,nh,nkv,hd,planes,steps", [(2400, 14, 2, 64, 0, 2), (1200, 28, 4, 128, 0, 2), (2400, 32, 8, 128, 0, 6),
                                                      (1200, 28, 4, 128, 2, 2)])
def test_rope_store_of_several_heads_a_lane_group(T, nh, nkv, hd, planes, steps):
    chunks = -(-(nh + 2 * nkv) // (128 // (hd // 8)))
    assert max(1, min(chunks, T * chunks // (148 * 16))) == steps
    g = torch.Generator().manual_seed(T + nh)
    wide = (nh + 2 * nkv) * hd
    qkv = torch.randn(planes, T, wide, generator=g) if planes else torch.randn(T, wide, generator=g).bfloat16()
    pos = torch.randint(0, 500, (T,), generator=g)
    cs = rope.build_cos_sin_cache(hd, 500, 1e4)
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g)).bfloat16() for _ in range(2))
    bs = 16
    kp, vp = (Int4Pages.zeros((T // bs + 1, nkv, bs, hd), DEV) for _ in range(2))
    slots = torch.randperm((T // bs + 1) * bs, generator=g)[:T].int().to(DEV)
    q = kv_int4.qkv_norm_rope_store_int4(qkv.to(DEV), pos.to(DEV), cs.to(DEV), qw.to(DEV), kw.to(DEV), 1e-6, kp, vp, slots, nh, nkv,
                                         hd)
    k, v = kv_int4.load_kvcache_int4(kp, vp, slots)
    x = qkv.double().sum(0) if planes else qkv.double()
    q64, k64, v64 = x.reshape(T, -1, hd).split((nh, nkv, nkv), 1)

    def turned(y, w):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.double()
        c, s = cs.double()[pos][:, None].chunk(2, -1)
        a, b = y.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    want = turned(q64, qw)
    # one bfloat16 rounding; a rotated value is a difference of two terms, so fp32 adds 2^-21 of the row
    assert ((q.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * want.abs().amax(-1, keepdim=True)).all()
    for y, got, exact in ((turned(k64, kw), k, False), (v64, v, not planes)):
        c, s, z = oracle.quantise(y.numpy())
        step = torch.from_numpy(np.repeat(s, 64, -1))
        want = torch.from_numpy((c - np.repeat(z, 64, -1)) * np.repeat(s, 64, -1))
        off = (got.double().cpu() - want).abs()
        # fp32 noise of 2^-20 of the largest value (7.5 steps or more away from zero) moves a value over a border between codes
        # once in 2^16 values, and a range over a border between scales (16 of them in a factor of two) once in 2^15
        # groups of 64; either way both results lie within half a step of the value.  Four times those counts, and two groups
        n = off.numel()
        assert (off <= 1.2 * step).all()
        assert int((off > 1e-3 * step).sum()) <= (0 if exact else 4 * n * (2.0 ** -16 + 2.0 ** -15) + 128)
