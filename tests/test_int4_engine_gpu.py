"""The engine with its KV cache in 4-bit pages, on one B200."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ckpts(tmp_path_factory):
    from llmserve_b200.models.synthetic import TINY, write_eagle3_checkpoint, write_qwen3_checkpoint
    d = tmp_path_factory.mktemp("int4")
    cfg = dict(TINY, torch_dtype="bfloat16", num_hidden_layers=4)
    return (write_qwen3_checkpoint(str(d / "target"), cfg, seed=2),
            write_eagle3_checkpoint(str(d / "draft"), cfg, draft_vocab=512, seed=2))


def _prompts(lens, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1024, (n,), generator=g).tolist() for n in lens]


def _run(path, prompts, max_tokens, sampler, **kw):
    from llmserve_b200 import LLM, SamplingParams
    kw = {"enforce_eager": False, "max_num_batched_tokens": 2048, **kw}
    llm = LLM(path, max_model_len=512, max_num_seqs=16, kvcache_block_size=16, gpu_memory_utilization=0.3,
              num_kvcache_blocks=256, kv_cache_dtype="int4", **kw)
    llm.model_runner.sampler = sampler
    out = [o["token_ids"] for o in llm.generate(prompts, SamplingParams(max_tokens=max_tokens, ignore_eos=True),
                                                use_tqdm=False)]
    llm.exit()
    return out


@pytest.mark.timeout(600)
def test_logits_follow_the_fp32_engine_on_the_same_pages(ckpts):
    """Prefill (33 to 200 tokens: every kernel's tile edges) and 12 decode steps against the CPU fp32
    engine with 4-bit pages, teacher-forced.  bfloat16 against fp32 stays below 3%.  Codes add to that:
    activations that reach K and V are about 1% of their deviation s off.  A step is the range of 64
    normals, some 4.8 s, over 15, rounded up by 6% on average: 0.34 s.  A share 0.8 * 0.01 / 0.34 = 2.4%
    of the codes moves by a step, an error of sqrt(0.024) * 0.34 = 5.3% of K and V: 8.3% in all."""
    from tests.support import RecordingSampler, compare_logits
    target, _ = ckpts
    prompts = _prompts((33, 7, 200, 129))
    rec = RecordingSampler()
    _run(target, prompts, 13, rec)
    ref = RecordingSampler(forced=rec.tokens)
    _run(target, prompts, 13, ref, device="cpu", enforce_eager=True)
    worst, checked = compare_logits(rec.logits, ref.logits, 8.3e-2)
    # rows whose top two are further apart than that error decide; a random model has some, not most
    assert checked > 0, (worst, checked)


@pytest.mark.timeout(600)
def test_graphs_and_eager_steps_agree(ckpts):
    from llmserve_b200.engine.model_runner import GreedySampler
    target, _ = ckpts
    prompts = _prompts((40, 17, 300, 64, 1))
    graphed = _run(target, prompts, 30, GreedySampler())
    assert graphed == _run(target, prompts, 30, GreedySampler(), enforce_eager=True)


@pytest.mark.timeout(900)
def test_speculation_runs_on_the_pages(ckpts):
    from llmserve_b200.engine.model_runner import GreedySampler
    target, draft = ckpts
    prompts = _prompts((40, 17, 80))
    kw = dict(speculative_model=draft, speculative_gamma=3)
    eager = _run(target, prompts, 30, GreedySampler(), **kw)
    graphed = _run(target, prompts, 30, GreedySampler(), speculative_cuda_graphs=True, **kw)
    assert eager == graphed and all(len(t) == 30 for t in eager)
    tree = _run(target, prompts[:1], 20, GreedySampler(), speculative_model=draft, speculative_tree_nodes=10)
    assert len(tree[0]) == 20


def test_tree_attention_on_a_4_bit_prefix():
    from llmserve_b200.ops import attention, kv_int4
    from llmserve_b200.ops.kv_int4 import Int4Pages
    from tests import int4_oracle as oracle
    nh, nkv, hd, bs, prefix, n = 8, 2, 128, 32, 77, 6
    kp, vp = (oracle.random_pages(6, nkv, bs, hd, s) for s in (1, 2))
    g = torch.Generator().manual_seed(4)
    q, tk, tv = (torch.randn(n, h, hd, generator=g).bfloat16().cuda() for h in (nh, nkv, nkv))
    table = torch.tensor([4, 0, 3], dtype=torch.int32, device="cuda")
    mask = torch.tril(torch.ones(n, n, dtype=torch.bool, device="cuda"))
    k, v = (Int4Pages(c.cuda(), w.cuda()) for c, w in (kp, vp))
    out = kv_int4.tree_attention_int4(q, k, v, table, prefix, tk, tv, mask, hd ** -0.5)
    pools = [oracle.values(*p).float() for p in (kp, vp)]
    ref = attention.tree_attention_ref(q.cpu().float(), *pools, table.cpu(), prefix, tk.cpu().float(), tv.cpu().float(),
                                       mask.cpu(), hd ** -0.5)
    assert ((out.float().cpu() - ref).norm() / ref.norm()).item() < 1e-2
