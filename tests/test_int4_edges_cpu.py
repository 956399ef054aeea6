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
