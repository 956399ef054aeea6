"""4-bit KV cache on the CPU path: format, store and load, attention, step maps, refusals."""
import math

import numpy as np
import pytest
import torch

from llmserve_b200.ops import kv_int4, step_maps
from llmserve_b200.ops.kv_int4 import Int4Pages
from tests import int4_oracle as oracle


def _rows(t, nkv, hd, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(t, nkv, hd, generator=g).bfloat16()


@pytest.mark.parametrize("hd", [64, 128])
def test_codes_and_words_follow_the_definition(hd):
    x = _rows(97, 3, hd)
    x[3] = 0                                     # an empty range
    x[4] = x[4].abs() + 1                        # one sign: the range is widened to zero
    x[5] = -x[5].abs()
    x[6, :, 0] = 1e30                            # one channel far above the others
    x[7] *= 1e-30
    codes, words = kv_int4.quantise_int4_ref(x)
    c, s, z = oracle.quantise(x.double().numpy())
    c2, s2, z2 = oracle.unpack(codes, words)
    assert np.array_equal(s, s2) and np.array_equal(z, z2) and np.array_equal(c, c2)


def test_values_are_exact_in_bfloat16_and_near_the_input():
    x = _rows(64, 2, 128, seed=3)
    codes, words = kv_int4.quantise_int4_ref(x)
    y = kv_int4.dequantise_int4_ref(codes, words)
    assert torch.equal(y, y.bfloat16().float())
    # half a step, and half a step more where both ends of the range rounded outward
    step = torch.from_numpy(np.repeat(oracle.unpack(codes, words)[1], 64, -1))
    assert ((y.double() - x.double()).abs() <= step * (1 + 1e-6)).all()
    inner = torch.from_numpy(oracle.unpack(codes, words)[0]) < 15
    assert ((y.double() - x.double()).abs() <= 0.5 * step * (1 + 1e-6))[inner].all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_group_that_is_not_finite_reads_back_as_nan(bad):
    x = _rows(2, 1, 128)
    x[0, 0, 70] = bad
    y = kv_int4.dequantise_int4_ref(*kv_int4.quantise_int4_ref(x))
    assert y[0, 0, 64:].isnan().all() and torch.isfinite(y[0, 0, :64]).all() and torch.isfinite(y[1]).all()


def test_store_and_load_by_slot():
    k, v = _rows(5, 2, 64, 1), _rows(5, 2, 64, 2)
    kp, vp = (Int4Pages.zeros((3, 2, 16, 64), "cpu") for _ in range(2))
    slots = torch.tensor([0, 47, -1, 17, 16], dtype=torch.int32)
    kv_int4.store_kvcache_int4(k, v, kp, vp, slots)
    k2, v2 = kv_int4.load_kvcache_int4(kp, vp, slots)
    for x, y in ((k, k2), (v, v2)):
        c, s, z = oracle.quantise(x.double().numpy())
        want = torch.from_numpy((c - np.repeat(z, 64, -1)) * np.repeat(s, 64, -1))
        want[2] = 0
        assert torch.equal(y.double(), want)
    assert kp.words.count_nonzero() == 4 * 2      # nothing else was touched


def test_prefill_and_decode_against_the_oracle():
    hd, nh, nkv, bs = 64, 4, 2, 16
    kp, vp = (oracle.random_pages(12, nkv, bs, hd, s) for s in (1, 2))
    cu, lens = [0, 3, 3, 8], [40, 0, 5]
    tables = torch.tensor([[5, 2, 9], [0, 0, 0], [7, 0, 0]], dtype=torch.int32)
    q = torch.randn(8, nh, hd, generator=torch.Generator().manual_seed(5))
    out = kv_int4.prefill_attention_int4(q, Int4Pages(*kp), Int4Pages(*vp), torch.tensor(cu, dtype=torch.int32),
                                         torch.tensor(lens, dtype=torch.int32), tables, 0.125, 5)
    want, mag = oracle.attention(q, kp, vp, cu, lens, tables, 0.125)
    assert ((out.double() - want).abs() <= 1e-5 * (1 + mag)).all()
    one = kv_int4.decode_attention_int4(q[:3], Int4Pages(*kp), Int4Pages(*vp), tables,
                                        torch.tensor(lens, dtype=torch.int32), 0.125)
    want, mag = oracle.attention(q[:3], kp, vp, [0, 1, 2, 3], lens, tables, 0.125)
    assert ((one.double() - want).abs() <= 1e-5 * (1 + mag)).all() and one[1].eq(0).all()


def test_step_maps():
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    m = step_maps.build_step_maps(i(2, 0, 1, 3), i(2, 0, 17, 33), i(4, 7, 1, 9, 3, 8), 16, 8, 4)
    assert m.cu_seqlens_q.tolist() == [0, 2, 2, 3, 6]
    assert m.positions.tolist() == [0, 1, 16, 30, 31, 32, 0, 0]
    assert m.slot_mapping.tolist() == [64, 65, 16, 3 * 16 + 14, 3 * 16 + 15, 8 * 16, -1, -1]
    assert m.block_tables.tolist() == [[4, 0, 0, 0], [0, 0, 0, 0], [7, 1, 0, 0], [9, 3, 8, 0]]
    assert m.last_token_indices.tolist() == [1, 1, 2, 5]


def test_refusals():
    k = _rows(2, 2, 64)
    kp, vp = (Int4Pages.zeros((1, 2, 16, 64), "cpu") for _ in range(2))
    s = torch.zeros(2, dtype=torch.int32)
    for shape in ((1, 2, 16, 96), (1, 2, 24, 64)):
        with pytest.raises(ValueError):
            Int4Pages.zeros(shape, "cpu")
    with pytest.raises(ValueError, match="head layout"):
        kv_int4.store_kvcache_int4(_rows(2, 3, 64), k, kp, vp, s)
    with pytest.raises(ValueError, match="differ in shape"):
        kv_int4.store_kvcache_int4(k, k, kp, Int4Pages.zeros((2, 2, 16, 64), "cpu"), s)
    with pytest.raises(ValueError, match="Int4Pages"):
        kv_int4.store_kvcache_int4(k, k, kp.codes, vp, s)
    with pytest.raises(ValueError, match="nq"):
        kv_int4.verify_attention_int4(_rows(5, 2, 64), kp, vp, s[None], s[:2], 1.0, 2)
    for q, scale in ((_rows(2, 3, 64), 1.0), (_rows(2, 2, 128), 1.0), (_rows(2, 2, 64), 0.0)):
        with pytest.raises(ValueError):
            kv_int4.decode_attention_int4(q, kp, vp, s[:, None], s, scale)
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    for q, n, ids, rows in ((i(3), i(2), i(0), 3), (i(-1), i(2), i(0), 3), (i(2), i(2), i(0), 1), (i(2), i(17), i(0), 2)):
        with pytest.raises(ValueError):
            step_maps.build_step_maps(q, n, ids, 16, rows, 1)
    with pytest.raises(ValueError, match="int32"):
        step_maps.build_step_maps(i(1).long(), i(1), i(0), 16, 1, 1)
    with pytest.raises(ValueError, match="differ in length"):
        step_maps.build_step_maps(i(1, 1), i(1), i(0), 16, 1, 1)
