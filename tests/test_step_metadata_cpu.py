"""Metadata of prefill and eager decode steps as the GPU path builds it, with the maps' CPU form."""
from types import SimpleNamespace

import pytest
import torch

from llmserve_b200.engine.model_runner import ModelRunner
from llmserve_b200.engine.sequence import Sequence
from llmserve_b200.utils.context import get_context, reset_context


@pytest.fixture
def runner():
    r = object.__new__(ModelRunner)
    r.is_cuda, r.device, r.block_size, r.h2d_bytes, r.decode_workspace = True, torch.device("cpu"), 16, 0, None
    r.config = SimpleNamespace(debug_bounds_checks=False, num_kvcache_blocks=16)
    yield r
    reset_context()


def _seq(n, blocks, scheduled=0):
    s = Sequence(list(range(n)))
    s.block_table, s.num_scheduled_tokens = list(blocks), scheduled
    return s


@pytest.mark.parametrize("blocks", [[5], []])
def test_a_sequence_without_blocks_for_its_tokens_is_refused(runner, blocks):
    with pytest.raises(IndexError, match="holds"):
        runner.prepare_decode([_seq(17, blocks)])
    with pytest.raises(IndexError, match="holds"):
        runner.prepare_prefill([_seq(40, [1, 2, 3], 40), _seq(17, blocks, 17)])
