"""4-bit KV cache kernels on the calls that their documentation allows beside the ordinary ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from llmserve_b200.ops import kv_int4, step_maps  # noqa: E402
from llmserve_b200.ops._ext import C, check_status  # noqa: E402
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


def _on(p):
    return Int4Pages(p[0].to(DEV), p[1].to(DEV))


def _assert_close(got, want, mag):
    off = (got.double().cpu() - want).abs()
    tol = oracle.attention_tolerance(want, mag)
    assert torch.isfinite(got.float()).all()
    assert (off <= tol).all(), f"{(off / tol).max().item():.3f} of the tolerance"


def test_queries_in_any_order_of_strides():
    """A transposed [heads, rows, head_dim] query is dense but not contiguous; a slice of a wider row is neither."""
    nh, nkv, hd, bs = 8, 2, 64, 16
    kp, vp = (oracle.random_pages(6, nkv, bs, hd, s) for s in (1, 2))
    tables, lens = torch.tensor([[3, 1, 5], [0, 2, 4]], dtype=torch.int32), [41, 30]
    g = torch.Generator().manual_seed(4)
    dense = torch.randn(nh, 4, hd, generator=g).bfloat16().to(DEV).transpose(0, 1)
    wide = torch.randn(4, nh + 2, hd + 64, generator=g).bfloat16().to(DEV)[:, 1:nh + 1, :hd]
    for q in (dense, wide):
        assert not q.is_contiguous()
        args = (q, _on(kp), _on(vp))
        want, mag = oracle.attention(q, kp, vp, [0, 2, 4], lens, tables, 0.125)
        _assert_close(kv_int4.verify_attention_int4(*args, tables.to(DEV), _i32(*lens), 0.125, 2), want, mag)
        _assert_close(kv_int4.prefill_attention_int4(*args, _i32(0, 2, 4), _i32(*lens), tables.to(DEV), 0.125, 2), want, mag)
        want, mag = oracle.attention(q[:2], kp, vp, [0, 1, 2], lens, tables, 0.125)
        _assert_close(kv_int4.decode_attention_int4(q[:2], *args[1:], tables.to(DEV), _i32(*lens), 0.125), want, mag)
        # a tree of two nodes that see themselves, one after the other
        tk, tv = (torch.randn(2, nkv, hd, generator=g).bfloat16().to(DEV) for _ in range(2))
        mask = torch.tril(torch.ones(2, 2, dtype=torch.bool, device=DEV))
        tree = [kv_int4.tree_attention_int4(x, *args[1:], tables[0].to(DEV), 41, tk, tv, mask, 0.125)
                for x in (q[:2], q[:2].contiguous())]
        assert torch.equal(*tree) and tree[0].is_contiguous()


def _recorded():
    with pytest.raises(RuntimeError, match="out-of-range"):
        check_status(torch.device(DEV))


def test_step_maps_after_a_contradicting_request():
    """Requests before it are mapped; from it on none is, so that no token lands in another request's block."""
    for q, k in ((3, 1), (-1, 4), (9, 9)):          # more new tokens than keys, a negative length, more than all rows
        m = step_maps.build_step_maps(_i32(2, q, 2), _i32(18, k, 2), _i32(4, 5, 6, 7), 16, 8, 3)
        _recorded()
        assert m.cu_seqlens_q.tolist() == [0, 2, 2, 2]
        assert m.slot_mapping.tolist() == [5 * 16, 5 * 16 + 1] + [-1] * 6
        assert m.positions.tolist() == [16, 17] + [0] * 6
        assert m.block_tables.tolist() == [[4, 5, 0], [0, 0, 0], [0, 0, 0]]


def test_step_maps_of_lengths_whose_sums_pass_32_bits():
    # blocks: 2 (2^31 - 1) wraps to -2, which no id list is too short for
    m = step_maps.build_step_maps(_i32(1, 1), _i32(2 ** 31 - 1, 2 ** 31 - 1), _i32(0, 1), 1, 2, 1)
    _recorded()
    assert m.slot_mapping.tolist() == [-1, -1] and m.cu_seqlens_q.tolist() == [0, 1, 2]
    # new tokens: 8192 * 2^18 = 2^31
    n, t = 8192, 2 ** 18
    lens = torch.full((n,), t, dtype=torch.int32, device=DEV)
    ids = torch.arange(n, dtype=torch.int32, device=DEV)
    m = step_maps.build_step_maps(lens, lens, ids, t, t, 1)
    _recorded()
    assert m.cu_seqlens_q.tolist() == [0] + [t] * n and m.last_token_indices.tolist() == [t - 1] * n
    assert torch.equal(m.slot_mapping, torch.arange(t, dtype=torch.int32, device=DEV))
    assert torch.equal(m.block_tables.flatten(), ids)


def test_prefill_takes_row_tables_that_leave_the_query():
    """Cumulative lengths below zero, past the rows, out of order: rows of the query are worked on, nothing else."""
    nh, nkv, hd, bs = 4, 2, 64, 16
    kp, vp = (oracle.random_pages(4, nkv, bs, hd, s) for s in (1, 2))
    q = torch.randn(5, nh, hd, generator=torch.Generator().manual_seed(7)).bfloat16()
    tables = torch.tensor([[3, 1], [0, 2], [1, 0]], dtype=torch.int32)
    args = (q.to(DEV), _on(kp), _on(vp))
    low = -2 ** 31
    for given, seen in (((low, 2, 2, low), (0, 2, 2, 2)), ((0, 2, 2 ** 31 - 1, 5), (0, 2, 5, 5)), ((low, low, low, low), (0, 0, 0, 0)),
                        ((0, 2, 5, low), (0, 2, 5, 5))):
        out = kv_int4.prefill_attention_int4(*args, _i32(*given), _i32(20, 30, 9), tables.to(DEV), 0.125, 5)
        want, mag = oracle.attention(q, kp, vp, seen, [20, 30, 9], tables, 0.125)
        n = seen[-1]
        _assert_close(out[:n], want[:n], mag[:n])


def test_a_chunk_longer_than_stated_costs_no_other_sequence_its_rows():
    nh, nkv, hd, bs = 64, 2, 64, 16                       # 32 heads a KV head: four queries a tile, eight a block
    q_lens, k_lens = [90, 3, 7], [90, 20, 7]
    kp, vp = (oracle.random_pages(9, nkv, bs, hd, s) for s in (1, 2))
    tables = torch.tensor([[3, 1, 8, 0, 5, 2], [4, 6, 0, 0, 0, 0], [7, 0, 0, 0, 0, 0]], dtype=torch.int32)
    q = torch.randn(100, nh, hd, generator=torch.Generator().manual_seed(7)).bfloat16()
    out = kv_int4.prefill_attention_int4(q.to(DEV), _on(kp), _on(vp), _i32(0, 90, 93, 100), _i32(*k_lens), tables.to(DEV), 0.125, 7)
    want, mag = oracle.attention(q, kp, vp, [0, 90, 93, 100], k_lens, tables, 0.125)
    _assert_close(out[90:], want[90:], mag[90:])
    _assert_close(out[:7], want[:7], mag[:7])


@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), float("inf"), 1e-46, 1e39])
def test_scales_that_float32_does_not_hold_are_refused(scale):
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    p = Int4Pages.zeros((1, 2, 16, 64), DEV)
    t, n = _i32(0).view(1, 1), _i32(1)
    with pytest.raises(RuntimeError, match="scale"):
        kv_int4.decode_attention_int4(q, p, p, t, n, scale)
    with pytest.raises(RuntimeError, match="scale"):
        kv_int4.prefill_attention_int4(q, p, p, _i32(0, 1), n, t, scale, 1)


def _nan_key_case():
    """Token 40 of 64 holds NaN in the first group of its K."""
    kp, vp = (oracle.random_pages(5, 2, 16, 128, s) for s in (1, 2))
    tables = torch.tensor([[3, 1, 4, 0]], dtype=torch.int32)
    q = torch.randn(64, 4, 128, generator=torch.Generator().manual_seed(6)).bfloat16()
    want, mag = oracle.attention(q, kp, vp, [0, 64], [64], tables, 0.09)
    kp[1][4, 1, 8, 0] = 0x7FC0
    nan = torch.zeros_like(q, dtype=torch.bool)
    nan[40:, 2:] = True
    return q, kp, vp, tables, want, mag, nan


@pytest.mark.parametrize("new", [64, 30])
def test_a_nan_key_breaks_only_the_rows_that_see_it(new):
    q, kp, vp, tables, want, mag, nan = _nan_key_case()
    q, want, mag, nan = (x[64 - new:] for x in (q, want, mag, nan))
    args = (q.to(DEV), _on(kp), _on(vp))
    for out in (kv_int4.prefill_attention_int4(*args, _i32(0, new), _i32(64), tables.to(DEV), 0.09, new),
                kv_int4.verify_attention_int4(*args, tables.to(DEV), _i32(64), 0.09, new)):
        out = out.cpu()
        assert torch.equal(out.isnan(), nan)
        assert ((out.double() - want).abs() <= oracle.attention_tolerance(want, mag))[~nan].all()


def test_captured_prefill_replays_on_new_lengths_and_tables():
    nh, nkv, hd, bs, T = 8, 2, 64, 16, 200
    kp, vp = (oracle.random_pages(20, nkv, bs, hd, s) for s in (1, 2))
    q = torch.randn(T, nh, hd, generator=torch.Generator().manual_seed(1)).bfloat16()
    args, cu, lens, tables = (q.to(DEV), _on(kp), _on(vp)), _i32(0, 0, 0, 0), _i32(0, 0, 0), torch.zeros(3, 14, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv_int4.prefill_attention_int4(*args, cu, lens, tables, 0.125, T)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = kv_int4.prefill_attention_int4(*args, cu, lens, tables, 0.125, T)
        for seed, (q_lens, k_lens) in enumerate((((130, 1, 69), (200, 90, 69)), ((0, 200, 0), (5, 220, 0)), ((1, 1, 1), (1, 2, 224)))):
            table = torch.randint(0, 20, (3, 14), generator=torch.Generator().manual_seed(seed)).int()
            ends = [0, q_lens[0], q_lens[0] + q_lens[1], sum(q_lens)]
            cu.copy_(_i32(*ends)), lens.copy_(_i32(*k_lens)), tables.copy_(table)
            graph.replay()
            side.synchronize()
            want, mag = oracle.attention(q, kp, vp, ends, k_lens, table, 0.125)
            _assert_close(out[:ends[-1]], want[:ends[-1]], mag[:ends[-1]])
