"""4-bit KV cache on the CPU path: the calls beside the ordinary ones."""
import math

import pytest
import torch

from llmserve_b200.ops import kv_int4
from llmserve_b200.ops.kv_int4 import Int4Pages
from tests import int4_oracle as oracle


@pytest.mark.parametrize("dtype,message", [("fp8", "must be 'auto' or 'int4'"), ("int4", "disaggregation")])
def test_disaggregated_engine_names_what_it_refuses(dtype, message):
    from llmserve_b200.engine.pd_engine import PDEngine
    with pytest.raises(ValueError, match=message):
        PDEngine("nowhere", kv_cache_dtype=dtype)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_broken_token_reaches_only_the_rows_that_see_it(which, bad):
    """Token 9 of 20 is not finite in its second group: the rows before it keep their results."""
    hd, nh, nkv, bs, n = 128, 4, 2, 16, 20
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(n, nkv, hd, generator=g) for _ in range(2))
    q = torch.randn(n, nh, hd, generator=g)
    cu, lens, table = (torch.tensor(x, dtype=torch.int32) for x in ([0, n], [n], [[1, 0]]))
    slots = torch.arange(16, 16 + n, dtype=torch.int32) % 32
    outs = []
    for broken in (False, True):
        if broken:
            (k if which == "k" else v)[9, 1, 100] = bad
        kp, vp = (Int4Pages.zeros((2, nkv, bs, hd), "cpu") for _ in range(2))
        kv_int4.store_kvcache_int4(k, v, kp, vp, slots)
        outs.append(kv_int4.prefill_attention_int4(q, kp, vp, cu, lens, table, 0.1, n))
    nan = torch.zeros_like(q, dtype=torch.bool)
    nan[9:, 2:, 0 if which == "k" else 64:] = True       # a broken key breaks the whole row, a broken value its group
    assert torch.equal(outs[1].isnan(), nan)
    assert torch.allclose(outs[1][~nan], outs[0][~nan], rtol=0, atol=1e-6)
