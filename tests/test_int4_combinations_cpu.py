"""4-bit pages with the engine's other features, on the CPU fp32 path: tensor parallelism, AutoAWQ weights, prefix cache."""
import socket

import pytest
import torch

from llmserve_b200 import LLM, SamplingParams
from llmserve_b200.engine.model_runner import GreedySampler
from llmserve_b200.models.synthetic import TINY, write_awq_checkpoint, write_eagle3_checkpoint, write_qwen3_checkpoint
from tests.support import RecordingSampler, compare_logits


def _port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _prompts(lens, seed=11):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1024, (n,), generator=g).tolist() for n in lens]


def _run(path, prompts, sampler, max_tokens=12, **kw):
    llm = LLM(path, device="cpu", enforce_eager=True, num_kvcache_blocks=64, kvcache_block_size=16, max_model_len=256,
              kv_cache_dtype="int4", comm_timeout_s=60, distributed_init_method=f"tcp://127.0.0.1:{_port()}", **kw)
    llm.model_runner.sampler = sampler
    out = [o["token_ids"] for o in llm.generate(prompts, SamplingParams(max_tokens=max_tokens, ignore_eos=True), use_tqdm=False)]
    llm.exit()
    return out


@pytest.fixture(scope="module")
def ckpts(tmp_path_factory):
    d = tmp_path_factory.mktemp("int4")
    return (write_qwen3_checkpoint(str(d / "t"), TINY, seed=1), write_eagle3_checkpoint(str(d / "d"), TINY, draft_vocab=512, seed=1),
            write_awq_checkpoint(str(d / "awq"), TINY, seed=3))


def test_two_ranks_hold_their_heads_pages(ckpts):
    """Sums over ranks in another order move activations by some 1e-6 and a code over a border once in 1e5 values or so;
    a code moves one value of one key by a step, a third of a deviation: 1e-2 of the logits is far above, and any
    mixed-up head or page far beyond."""
    prompts = _prompts((9, 33, 17, 50))
    one = RecordingSampler()
    _run(ckpts[0], prompts, one)
    two = RecordingSampler(forced=one.tokens)
    _run(ckpts[0], prompts, two, tensor_parallel_size=2)
    _, checked = compare_logits(two.logits, one.logits, 1e-2)
    assert checked > 0


def test_awq_weights_on_4_bit_pages(ckpts):
    """A quantised target with chain and tree speculation serves its own plain decode's tokens."""
    prompts = _prompts((21, 8, 40))
    plain = _run(ckpts[2], prompts, GreedySampler())
    assert _run(ckpts[2], prompts, GreedySampler(), speculative_model=ckpts[1]) == plain
    for p, want in zip(prompts, plain):
        assert _run(ckpts[2], [p], GreedySampler(), speculative_model=ckpts[1], speculative_tree_nodes=10) == [want]


def test_a_cached_prefix_is_read_from_the_pages(ckpts):
    """Two prompts share 48 tokens: served one after the other by one engine, the second finds them in the pages."""
    shared = _prompts((48,))[0]
    prompts = [shared + p for p in _prompts((7, 12), seed=2)]
    alone = [_run(ckpts[0], [p], GreedySampler())[0] for p in prompts]
    llm = LLM(ckpts[0], device="cpu", enforce_eager=True, num_kvcache_blocks=64, kvcache_block_size=16, max_model_len=256,
              kv_cache_dtype="int4")
    llm.model_runner.sampler = GreedySampler()
    params = SamplingParams(max_tokens=12, ignore_eos=True)
    assert [llm.generate([p], params, use_tqdm=False)[0]["token_ids"] for p in prompts] == alone
    llm.exit()
