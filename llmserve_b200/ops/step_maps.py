"""A step's addressing tensors built on the GPU from request lengths.

``build_step_maps`` takes each request's new tokens and total keys and the block ids of all requests
back to back, and returns what the attention and store kernels of the step read: cumulative query
lengths, the position and pool slot of every new token, zero-padded block tables and the last row of
each request.  The host sends ``8 * B + 4 * blocks`` bytes instead of the filled tensors.
"""
from typing import NamedTuple

import torch

from llmserve_b200.ops._ext import C, status


MAX_REQUESTS = 8192      # one block's shared memory holds their prefix sums


class StepMaps(NamedTuple):
    cu_seqlens_q: torch.Tensor         # int32 [B + 1]
    positions: torch.Tensor            # int64 [num_tokens]
    slot_mapping: torch.Tensor         # int32 [num_tokens]
    block_tables: torch.Tensor         # int32 [B, table_width]
    last_token_indices: torch.Tensor   # int64 [B]


def _check(q_lens, k_lens, block_ids, block_size, num_tokens, table_width):
    for name, t in (("q_lens", q_lens), ("k_lens", k_lens), ("block_ids", block_ids)):
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous one-dimensional int32")
    if q_lens.shape != k_lens.shape:
        raise ValueError("q_lens and k_lens differ in length")
    if block_size < 1 or num_tokens < 0 or table_width < 0:
        raise ValueError("block_size must be positive, num_tokens and table_width not negative")


def build_step_maps_ref(q_lens, k_lens, block_ids, block_size, num_tokens, table_width) -> StepMaps:
    q, k, ids = q_lens.tolist(), k_lens.tolist(), block_ids.tolist()
    if any(n < 0 or m < n for n, m in zip(q, k)):
        raise ValueError("a request has a negative length or more new tokens than keys")
    if sum(q) > num_tokens or sum(-(-n // block_size) for n in k) > len(ids):
        raise ValueError("the requests need more tokens or block ids than were given")
    cu, pos, slots, last, at = [0], [], [], [], 0
    tables = torch.zeros(len(q), table_width, dtype=torch.int32)
    for i, (n, m) in enumerate(zip(q, k)):
        mine = ids[at:at + -(-m // block_size)]
        at += len(mine)
        tables[i, :min(len(mine), table_width)] = torch.tensor(mine[:table_width], dtype=torch.int32)
        pos += range(m - n, m)
        slots += [mine[p // block_size] * block_size + p % block_size for p in range(m - n, m)]
        cu.append(cu[-1] + n)
        last.append(max(0, cu[-1] - 1))
    pad = num_tokens - len(pos)
    return StepMaps(torch.tensor(cu, dtype=torch.int32), torch.tensor(pos + [0] * pad, dtype=torch.int64),
                    torch.tensor(slots + [-1] * pad, dtype=torch.int32), tables, torch.tensor(last, dtype=torch.int64))


def build_step_maps(q_lens: torch.Tensor, k_lens: torch.Tensor, block_ids: torch.Tensor, block_size: int,
                    num_tokens: int, table_width: int) -> StepMaps:
    """``q_lens`` / ``k_lens`` int32 [B]: new tokens and keys after the step of each request (at most
    8192 requests); ``block_ids`` int32: ``ceil(k_len / block_size)`` ids per request, back to back.
    ``num_tokens`` is the number of rows to fill: rows past the sum of ``q_lens`` get position 0 and
    slot -1 (padding of a captured step).  A table row holds its first ``table_width`` ids.  The last
    row of a request without new tokens is the one before its place (0 for the first).  On CUDA,
    lengths that contradict one another (or the ids and rows given) are recorded as an out-of-range
    index for ``check_status``: from the first request with a negative length, more new tokens than keys
    or more of them than ``num_tokens`` on, requests count as empty (their rows get slot -1), and a row whose block id
    is not given gets slot -1."""
    if not q_lens.is_cuda:
        _check(q_lens, k_lens, block_ids, block_size, num_tokens, table_width)
        return build_step_maps_ref(q_lens, k_lens, block_ids, block_size, num_tokens, table_width)
    return StepMaps(*C().step_maps(q_lens, k_lens, block_ids, block_size, num_tokens, table_width, status(q_lens.device)))
