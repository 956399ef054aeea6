"""Tree verify on 4-bit pages on the GPU: nodes as decode stores them, and their commit."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from llmserve_b200.layers.attention import Attention  # noqa: E402
from llmserve_b200.ops import kv_int4, rope  # noqa: E402
from llmserve_b200.ops._ext import C, check_status  # noqa: E402
from llmserve_b200.ops.kv_int4 import Int4Pages  # noqa: E402
from llmserve_b200.speculative.tree import build_fixed_tree_topology  # noqa: E402
from llmserve_b200.speculative.tree_kv import TreeKVCacheManager  # noqa: E402
from llmserve_b200.utils.context import reset_context, set_context  # noqa: E402
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


@pytest.mark.parametrize("nkv,hd,bs", [(3, 64, 16), (8, 128, 48), (1, 128, 256)])
def test_commit_copies_the_chosen_rows_of_every_layer(nkv, hd, bs):
    L, blocks, n = 3, 2, 11
    tk, tv = (_on(oracle.random_pages(L, n, nkv, hd, s)) for s in (1, 2))
    # rows of a step's scratch pages are strided
    tk = Int4Pages(tk.codes.transpose(1, 2).contiguous().transpose(1, 2), tk.words.transpose(1, 2).contiguous().transpose(1, 2))
    cpu = [oracle.random_pages(L * blocks, nkv, bs, hd, s) for s in (3, 4)]
    k, v = (Int4Pages(*(x.to(DEV).view(L, blocks, nkv, bs, -1) for x in p)) for p in cpu)
    want = [Int4Pages(*(x.clone().view(L, blocks, nkv, bs, -1) for x in p)) for p in cpu]
    nodes, slots = _i32(10, 0, 4, 5), _i32(bs + 1, 2, -1, 2 * bs - 1)
    kv_int4.commit_tree_kv_int4(tk, tv, k, v, nodes, slots)
    kv_int4.commit_tree_kv_int4_ref(*(Int4Pages(x.codes.cpu(), x.words.cpu()) for x in (tk, tv)), *want, nodes.cpu(), slots.cpu())
    for a, b in zip((k, v), want):
        assert torch.equal(a.codes.cpu(), b.codes) and torch.equal(a.words.cpu(), b.words)
    for bad in ((_i32(n), _i32(0)), (_i32(-1), _i32(0)), (_i32(0), _i32(2 * bs))):
        kv_int4.commit_tree_kv_int4(tk, tv, k, v, *bad)
        with pytest.raises(RuntimeError, match="out-of-range"):
            check_status(torch.device(DEV))
    for a, b in zip((k, v), want):
        assert torch.equal(a.codes.cpu(), b.codes) and torch.equal(a.words.cpu(), b.words)
    for bad in ((nodes.long(), slots), (nodes, slots.cpu()), (nodes[:2], slots)):
        with pytest.raises((RuntimeError, ValueError)):
            kv_int4.commit_tree_kv_int4(tk, tv, k, v, *bad)


@pytest.mark.parametrize("planes", [0, 3])
@pytest.mark.parametrize("nh,nkv,hd,bs,prefix,nodes", [(8, 2, 128, 32, 77, 6), (14, 2, 64, 16, 300, 10), (4, 4, 128, 64, 5, 10)])
def test_nodes_are_attended_and_committed_as_decode_stores_them(nh, nkv, hd, bs, prefix, nodes, planes):
    topo = build_fixed_tree_topology(nodes)
    n = len(topo.parents)
    g = torch.Generator().manual_seed(prefix)
    pools = [oracle.random_pages(-(-(prefix + 4) // bs) + 1, nkv, bs, hd, s) for s in (1, 2)]
    table = torch.randperm(pools[0][0].shape[0], generator=g)[:-(-(prefix + 4) // bs)].int()
    wide = (nh + 2 * nkv) * hd
    qkv = torch.randn(planes, n, wide, generator=g) if planes else torch.randn(n, wide, generator=g).bfloat16()
    qkv = qkv.to(DEV)
    norm = [(1 + 0.2 * torch.randn(hd, generator=g)).bfloat16().to(DEV) for _ in range(2)]
    cos_sin = rope.build_cos_sin_cache(hd, 512, 1e4).to(DEV)
    positions = torch.tensor([prefix + d for d in topo.depths], device=DEV)
    layer = Attention(nh, hd, hd ** -0.5, nkv)
    tree = [Int4Pages(p.codes[None].clone(), p.words[None].clone()) for p in map(_on, pools)]
    layer.k_cache, layer.v_cache = (p[0] for p in tree)
    set_context(True, tree_attention_mask=topo.attention_mask(DEV), tree_prefix_len=prefix, tree_block_table=table.to(DEV))
    got = layer(qkv, positions, cos_sin, *norm, 1e-6).view(n, nh, hd)
    reset_context()

    # every node as one decoded token: its row of the projection through the decode path's store
    scratch = [Int4Pages.zeros((n, nkv, 16, hd), DEV) for _ in range(2)]
    q = kv_int4.qkv_norm_rope_store_int4(qkv, positions, cos_sin, *norm, 1e-6, *scratch,
                                         torch.arange(n, dtype=torch.int32, device=DEV) * 16, nh, nkv, hd)
    for node in range(n):
        # prefix and ancestors in the pages, the way decode would have left them
        path = topo.ancestors_and_self(node)
        kp, vp = ((c.clone(), w.clone()) for c, w in pools)
        for j, a in enumerate(sorted(path, key=lambda x: topo.depths[x])):
            at = table[(prefix + j) // bs], slice(None), (prefix + j) % bs
            for p, s in ((kp, scratch[0]), (vp, scratch[1])):
                p[0][at], p[1][at] = s.codes[a, :, 0].cpu(), s.words[a, :, 0].cpu()
        keys = prefix + len(path)
        want, mag = oracle.attention(q[node:node + 1], kp, vp, [0, 1], [keys], table[None], hd ** -0.5)
        off = (got[node:node + 1].double().cpu() - want).abs()
        assert (off <= oracle.attention_tolerance(want, mag)).all()

    leaf = max(range(n), key=lambda x: topo.depths[x])
    path = sorted(topo.ancestors_and_self(leaf), key=lambda x: topo.depths[x])
    slots = torch.tensor([int(table[(prefix + j) // bs]) * bs + (prefix + j) % bs for j in range(len(path))],
                         dtype=torch.int32, device=DEV)
    TreeKVCacheManager([layer], k_cache=tree[0], v_cache=tree[1]).commit(path, slots)
    for p, s in zip(tree, scratch):
        for j, a in enumerate(path):
            at = 0, int(slots[j]) // bs, slice(None), int(slots[j]) % bs
            assert torch.equal(p.codes[at], s.codes[a, :, 0]) and torch.equal(p.words[at], s.words[a, :, 0])


def _tree_case(nh, nkv, hd, bs, prefix, n, seed):
    """(inputs of the operator without the table, 64-bit result for a table of block ids)."""
    g = torch.Generator().manual_seed(seed)
    kp, vp = (oracle.random_pages(6, nkv, bs, hd, s) for s in (1, 2))
    q, tk, tv = (torch.randn(n, h, hd, generator=g).bfloat16() for h in (nh, nkv, nkv))
    mask = torch.tril(torch.ones(n, n, dtype=torch.bool))

    def want(table):
        ok = ((table >= 0) & (table < 6)).repeat_interleave(bs)[:prefix]
        rows = [oracle.values(*p)[table.clamp(0, 5).long()].transpose(1, 2).reshape(-1, nkv, hd)[:prefix][ok] for p in (kp, vp)]
        k, v = (torch.cat((a, b.double())) for a, b in zip(rows, (tk, tv)))
        sees = torch.cat((torch.ones(n, int(ok.sum()), dtype=torch.bool), mask), 1)
        out, mag = torch.zeros(2, n, nh, hd, dtype=torch.float64)
        for h in range(nh):
            a = torch.softmax((q[:, h].double() @ k[:, h // (nh // nkv)].T * hd ** -0.5).masked_fill(~sees, -torch.inf), -1)
            out[:, h], mag[:, h] = a @ v[:, h // (nh // nkv)], a @ v[:, h // (nh // nkv)].abs()
        return out, mag

    return (q.to(DEV), _on(kp), _on(vp)), (tk.to(DEV), tv.to(DEV), mask.to(DEV), hd ** -0.5), want


@pytest.mark.parametrize("nh,nkv,hd,bs", [(8, 2, 128, 32), (14, 2, 64, 48)])         # tensor-core and CUDA-core kernel
def test_blocks_outside_the_pool_are_not_seen_by_a_tree(nh, nkv, hd, bs):
    prefix = 5 * bs - 3
    left, right, want = _tree_case(nh, nkv, hd, bs, prefix, 6, 8)
    # the last but one: id * block_size passes 2^32 and would wrap to a slot of the pool in 32 bits
    for bad in (-1, 6, 2 ** 32 // bs + 1, -2 ** 31):
        table = torch.tensor([4, 1, bad, 0, 3], dtype=torch.int32)
        out = kv_int4.tree_attention_int4(*left, table.to(DEV), prefix, *right)
        with pytest.raises(RuntimeError, match="out-of-range"):
            check_status(torch.device(DEV))
        ref, mag = want(table)
        assert ((out.double().cpu() - ref).abs() <= oracle.attention_tolerance(ref, mag)).all()


@pytest.mark.parametrize("prefix,blocks", [(0, 0), (0, 2), (1, 1), (64, 2), (200, 3)])
def test_tree_prefix_ends_at_its_table(prefix, blocks):
    bs = 32
    left, right, want = _tree_case(8, 2, 128, bs, min(prefix, blocks * bs), 10, prefix)
    table = torch.tensor([5, 2, 0][:blocks], dtype=torch.int32)
    out = kv_int4.tree_attention_int4(*left, table.to(DEV), prefix, *right)
    ref, mag = want(table)
    assert ((out.double().cpu() - ref).abs() <= oracle.attention_tolerance(ref, mag)).all()


def test_prefix_copies_of_ever_new_sizes_keep_no_more_than_a_bounded_set():
    """Two tensor maps a size: 2200 sizes pass the bound of 4096."""
    from llmserve_b200.ops._ext import raw_module
    left, right, want = _tree_case(4, 2, 64, 16, 33, 6, 5)
    table = torch.tensor([5, 2, 0], dtype=torch.int32)
    ref, mag = want(table)
    long = torch.zeros(2200, dtype=torch.int32, device=DEV)
    for n in range(1, 2200):
        kv_int4.tree_attention_int4(*left, long, 16 * n, *right)
        assert raw_module().kv_pool_map_count() <= 4096
    out = kv_int4.tree_attention_int4(*left, table.to(DEV), 33, *right)
    assert ((out.double().cpu() - ref).abs() <= oracle.attention_tolerance(ref, mag)).all()


def test_nodes_past_the_last_position_leave_the_others_as_they_are():
    """The deepest nodes of a tree at the end of the model's positions are skipped and recorded; scratch memory that
    held NaN patterns before must not reach the nodes above them."""
    nh, nkv, hd, bs, prefix = 8, 2, 64, 16, 37
    topo = build_fixed_tree_topology(10)
    n = len(topo.parents)
    g = torch.Generator().manual_seed(2)
    layer = Attention(nh, hd, hd ** -0.5, nkv)
    layer.k_cache, layer.v_cache = (_on(oracle.random_pages(3, nkv, bs, hd, s)) for s in (1, 2))
    qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g).bfloat16().to(DEV)
    positions = torch.tensor([prefix + d for d in topo.depths], device=DEV)
    weight = torch.ones(hd, dtype=torch.bfloat16, device=DEV)
    cos_sin = rope.build_cos_sin_cache(hd, 512, 1e4).to(DEV)
    set_context(True, tree_attention_mask=topo.attention_mask(DEV), tree_prefix_len=prefix, tree_block_table=_i32(2, 0, 1))
    want = layer(qkv, positions, cos_sin, weight, weight, 1e-6)
    last = prefix + max(topo.depths)
    short = cos_sin[:last].contiguous()
    for _ in range(3):
        junk = [torch.full((size,), 255, dtype=torch.uint8, device=DEV) for size in (512, 1024, 1088, 2048, 2176, 4096, 1 << 20) * 8]
        del junk
        got = layer(qkv, positions, short, weight, weight, 1e-6)
        with pytest.raises(RuntimeError, match="out-of-range"):
            check_status(torch.device(DEV))
        keep = positions < last
        assert torch.equal(got[keep], want[keep])
    reset_context()
