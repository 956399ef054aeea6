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


def test_a_prefill_step_carries_every_field_of_the_host_form(runner):
    """A prompt, a chunk after 20 cached tokens, and a decode of a mixed step."""
    seqs = [_seq(33, [7, 2, 9], 33), _seq(40, [1, 0, 4], 15), _seq(18, [3, 5])]
    seqs[1].num_cached_tokens = 20
    got, want = [], []
    for out, runner.is_cuda in ((got, True), (want, False)):
        ids, positions = runner.prepare_prefill(seqs, [seqs[2]])
        c = get_context()
        out += [ids, positions, c.cu_seqlens_q, c.cu_seqlens_k, c.slot_mapping, c.block_tables, c.seqlens_k, c.last_token_indices,
                torch.tensor([c.max_seqlen_q, c.max_seqlen_k])]
    assert want[3].tolist() == [0, 33, 68, 86]
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_a_decode_step_carries_every_field_of_the_host_form(runner):
    seqs = [_seq(17, [7, 2]), _seq(1, [4]), _seq(32, [1, 0])]
    got, want = [], []
    for out, runner.is_cuda in ((got, True), (want, False)):
        ids, positions = runner.prepare_decode(seqs)
        c = get_context()
        out += [ids, positions, c.slot_mapping, c.context_lens, c.block_tables]
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a, b)
