"""The engine with its KV cache in 4-bit pages, on the CPU fp32 path."""
import os

import pytest
import torch

from llmserve_b200 import LLM, SamplingParams
from llmserve_b200.config import Config
from llmserve_b200.engine.model_runner import GreedySampler
from llmserve_b200.models.synthetic import TINY, write_config_only, write_eagle3_checkpoint, write_qwen3_checkpoint


@pytest.fixture(scope="module")
def ckpts(tmp_path_factory):
    d = tmp_path_factory.mktemp("ckpt")
    return (write_qwen3_checkpoint(str(d / "target"), TINY, seed=0),
            write_eagle3_checkpoint(str(d / "draft"), TINY, draft_vocab=512, seed=0))


def _run(path, prompts, max_tokens=16, **kw):
    llm = LLM(path, device="cpu", enforce_eager=True, kvcache_block_size=16, max_model_len=256, num_kvcache_blocks=64,
              kv_cache_dtype="int4", **kw)
    llm.model_runner.sampler = GreedySampler()
    out = llm.generate(prompts, SamplingParams(max_tokens=max_tokens, ignore_eos=True), use_tqdm=False)
    memory = llm.model_runner.get_memory_metrics()
    llm.exit()
    return [o["token_ids"] for o in out], memory


def _prompts(n, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1024, (int(k),), generator=g).tolist() for k in torch.randint(8, 65, (n,), generator=g)]


def test_every_path_of_the_engine_serves_the_same_tokens(ckpts):
    target, draft = ckpts
    prompts = _prompts(4, 1)
    plain, memory = _run(target, prompts)
    # 4.25 bits per element: K and V, 2 layers, 64 blocks of 16 tokens, 2 heads of 64
    assert memory["kv_cache_bytes"] == 2 * 2 * 64 * 16 * 2 * (32 + 2)
    chunked, _ = _run(target, prompts, enable_chunked_prefill=True, max_num_batched_tokens=24)
    chain, _ = _run(target, prompts, speculative_model=draft, speculative_gamma=3)
    assert plain == chunked == chain
    tree, _ = _run(target, prompts[:1], speculative_model=draft, speculative_tree_nodes=6)
    assert tree[0] == plain[0]


def test_config_refuses_what_the_pages_do_not_hold(tmp_path):
    path = write_config_only(str(tmp_path / "m"), dict(TINY, head_dim=96))
    with pytest.raises(ValueError, match="head_dim"):
        Config(path, kv_cache_dtype="int4", device="cpu")
    path = write_config_only(str(tmp_path / "n"), dict(TINY, torch_dtype="float16"))
    with pytest.raises(ValueError, match="bfloat16"):
        Config(path, kv_cache_dtype="int4")
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        Config(path, kv_cache_dtype="fp8")
    with pytest.raises(ValueError, match="disaggregation"):
        Config(path, kv_cache_dtype="int4", device="cpu", pd_disaggregation=True, pd_prefill_devices=(0,),
               pd_decode_devices=(1,))
    assert os.path.isdir(path) and Config(path, device="cpu").kv_cache_dtype == "auto"
