"""Tree verify on 4-bit pages, CPU path: the same tokens as plain decode, the same codes after the commit."""
import pytest
import torch

from llmserve_b200 import LLM, SamplingParams
from llmserve_b200.engine.model_runner import GreedySampler
from llmserve_b200.layers.attention import Attention
from llmserve_b200.models.synthetic import TINY, write_eagle3_checkpoint, write_qwen3_checkpoint
from llmserve_b200.ops import kv_int4, rope
from llmserve_b200.ops.kv_int4 import Int4Pages
from llmserve_b200.speculative.tree_kv import TreeKVCacheManager
from llmserve_b200.utils.context import reset_context, set_context
from tests import int4_oracle as oracle


def _run(path, prompts, **kw):
    llm = LLM(path, device="cpu", enforce_eager=True, kvcache_block_size=16, max_model_len=256, num_kvcache_blocks=64,
              kv_cache_dtype="int4", **kw)
    llm.model_runner.sampler = GreedySampler()
    params = SamplingParams(max_tokens=32, ignore_eos=True)
    out = [llm.generate([p], params, use_tqdm=False)[0]["token_ids"] for p in prompts]
    llm.exit()
    return out


def test_tree_speculation_serves_the_tokens_of_plain_decode(tmp_path):
    target = write_qwen3_checkpoint(str(tmp_path / "target"), TINY, seed=0)
    draft = write_eagle3_checkpoint(str(tmp_path / "draft"), TINY, draft_vocab=512, seed=0)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1024, (int(n),), generator=g).tolist() for n in torch.randint(8, 65, (24,), generator=g)]
    plain = _run(target, prompts)
    for nodes in (6, 10):
        assert _run(target, prompts, speculative_model=draft, speculative_tree_nodes=nodes) == plain


def test_nodes_are_attended_and_committed_as_decode_stores_them():
    """Three nodes in a row after a prefix of 17 keys against three decoded tokens at the same places."""
    nh, nkv, hd, bs, prefix, n = 4, 2, 64, 16, 17, 3
    g = torch.Generator().manual_seed(3)
    layer = Attention(nh, hd, hd ** -0.5, nkv)
    pools = [oracle.random_pages(3, nkv, bs, hd, s) for s in (1, 2)]
    cos_sin, table = rope.build_cos_sin_cache(hd, 64, 1e4), torch.tensor([2, 0], dtype=torch.int32)
    qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g)
    positions = torch.arange(prefix, prefix + n)
    slots = (table[positions // bs] * bs + positions % bs).int()
    weight = torch.ones(hd)

    def pages():
        return [Int4Pages(c[None].clone(), w[None].clone()) for c, w in pools]

    decoded, tree = pages(), pages()
    layer.k_cache, layer.v_cache = (p[0] for p in decoded)
    want = []
    for j in range(n):
        set_context(False, slot_mapping=slots[j:j + 1], context_lens=torch.tensor([prefix + j + 1], dtype=torch.int32),
                    block_tables=table[None])
        want.append(layer(qkv[j:j + 1], positions[j:j + 1], cos_sin, weight, weight, 1e-6))
    layer.k_cache, layer.v_cache = (p[0] for p in tree)
    set_context(True, tree_attention_mask=torch.tril(torch.ones(n, n, dtype=torch.bool)), tree_prefix_len=prefix,
                tree_block_table=table)
    got = layer(qkv, positions, cos_sin, weight, weight, 1e-6)
    reset_context()
    # fp32 sums of 20 weights and values in another order
    assert (got - torch.cat(want)).abs().max() <= 1e-5
    TreeKVCacheManager([layer], k_cache=tree[0], v_cache=tree[1]).commit([0, 1, 2], slots)
    for a, b in zip(decoded, tree):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.words, b.words)
    assert layer.tree_k.numel() == 0 and layer.tree_v.numel() == 0


def test_commit_copies_the_chosen_rows_of_every_layer():
    tk, tv = (Int4Pages(*oracle.random_pages(2, 5, 3, 64, s)) for s in (1, 2))       # [layers, nodes, kv_heads, hd]
    k, v = (Int4Pages(*(x.reshape(2, 4, 3, 16, -1) for x in oracle.random_pages(8, 3, 16, 64, s))) for s in (3, 4))
    before = [Int4Pages(p.codes.clone(), p.words.clone()) for p in (k, v)]
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    kv_int4.commit_tree_kv_int4(tk, tv, k, v, i(4, 0, 2), i(17, -1, 63))
    for x, p, old in ((tk, k, before[0]), (tv, v, before[1])):
        for a, b, rows in ((p.codes, old.codes, x.codes), (p.words, old.words, x.words)):
            b[:, 1, :, 1], b[:, 3, :, 15] = rows[:, 4], rows[:, 2]
            assert torch.equal(a, b)


def test_commit_refusals():
    rows = lambda *s: Int4Pages(torch.zeros(*s[:-1], s[-1] // 2, dtype=torch.uint8),  # noqa: E731
                                torch.zeros(*s[:-1], s[-1] // 64, dtype=torch.int16))
    t, p = rows(2, 5, 3, 64), Int4Pages.zeros((2, 4, 3, 16, 64), "cpu")
    i = torch.zeros(1, dtype=torch.int32)
    for tk, tv, k, v, nodes, slots in ((t.codes, t, p, p, i, i), (t, rows(2, 4, 3, 64), p, p, i, i), (t[0], t[0], p, p, i, i),
                                       (t, t, p[0], p[0], i, i), (t, t, p, Int4Pages.zeros((2, 5, 3, 16, 64), "cpu"), i, i),
                                       (rows(1, 5, 3, 64), rows(1, 5, 3, 64), p, p, i, i),
                                       (rows(2, 5, 2, 64), rows(2, 5, 2, 64), p, p, i, i), (t, t, p, p, i, i[:0]),
                                       (t, t, p, p, i[None], i[None])):
        with pytest.raises(ValueError):
            kv_int4.commit_tree_kv_int4(tk, tv, k, v, nodes, slots)
    layer = Attention(4, 64, 1.0, 3)
    layer.tree_k = layer.tree_v = torch.zeros(5, 3, 64)
    with pytest.raises(ValueError, match="4-bit pages"):
        TreeKVCacheManager([layer], k_cache=p, v_cache=p).commit([0], i)
    assert layer.tree_k.numel() == 0
