"""What the attention block's entry points refuse before any device is needed, and the oracle's buckets."""
import ctypes
import math

import numpy as np
import pytest

from aikit_amd import enchip
from block_oracle import bucket_of


def test_null_context():
    lib, out = enchip.load(), ctypes.c_uint64()
    assert lib.enchip_head_norm_rope_rows_dev(None, 0, 0, None, 8, None, 8, 1, 1, 1, 0, 8, None, None, 1e-6, None, 0, None) == enchip.ERR_ARG
    assert lib.enchip_relpos_create(None, None, 8, 1, 20, ctypes.byref(out)) == enchip.ERR_ARG
    assert lib.enchip_relpos_create_map(None, None, 8, 1, None, 0, ctypes.byref(out)) == enchip.ERR_ARG
    assert lib.enchip_relpos_release(None, 1) == enchip.ERR_ARG
    assert lib.enchip_attention_bias_dev(None, 0, None, 32, None, 32, None, 32, None, 32, None, 1, 1, 1, 1, 32, 1.0, None) == enchip.ERR_ARG
    assert lib.enchip_pool_mean_l2_spans_dev(None, None, 8, 1, None, 1, 8, None, 8, None) == enchip.ERR_ARG
    assert lib.enchip_adapters_create(None, 8, 8, 1, 1, ctypes.byref(out)) == enchip.ERR_ARG
    assert lib.enchip_adapters_set(None, 1, 0, None, None, 1.0) == enchip.ERR_ARG
    assert lib.enchip_adapters_release(None, 1) == enchip.ERR_ARG
    assert lib.enchip_adapters_add_dev(None, 1, None, 8, 1, None, None, 8, None, 8, None) == enchip.ERR_ARG
    assert lib.enchip_w8a8_linear_adapters_dev(None, 1, 1, None, 1, None, None, 0, None, None) == enchip.ERR_ARG


def test_python_shape_checks():
    c = enchip.Context.__new__(enchip.Context)  # no device: the checks come first
    c._h, c._lib = None, enchip.load()
    f = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    s = enchip.Adapters(1, 64, 32, 4, 2)
    for A, B in ((f(4, 63), f(32, 4)), (f(4, 64), f(31, 4)), (f(4, 64), f(32, 3)), (f(5, 64), f(32, 5)), (f(0, 64), f(32, 0)), (f(64), f(32, 4))):
        with pytest.raises(ValueError):
            c.set_adapter(s, 0, A, B)
    with pytest.raises(ValueError):
        c.relpos(f(8), 20)
    for m in (np.zeros(4, np.int32), np.zeros((3, 3), np.int32), np.zeros(0, np.int32)):
        with pytest.raises(ValueError):
            c.relpos_from_map(f(8, 2), m)


def test_which_models_take_the_biased_attention():
    from aikit_amd.bert_dev import DeviceBert

    m = DeviceBert.__new__(DeviceBert)
    for hd in (16, 32, 64, 128):
        m.relpos, m.H, m.KV, m.hd, m.fused = None, 4, 4, hd, False
        assert not m.bias_attention() and not m.fused_attention(64)  # as without spans, bias and shared heads
        assert m.bias_attention(np.zeros((1, 2)))
        m.KV = 2
        assert m.bias_attention()
        m.KV, m.relpos = 4, enchip.RelPos(1, 4)
        assert m.bias_attention()


def test_buckets_by_whole_numbers_are_those_of_the_logarithm():
    for buckets, reach in ((32, 128), (16, 64), (64, 1000), (8, 5), (4, 2)):
        half, e = buckets // 2, buckets // 4
        d = np.arange(-2 * reach, 2 * reach + 1)
        for x, b in zip(d, bucket_of(d, buckets, reach)):
            n = abs(int(x))
            k = n if n < e else min(half - 1, e + math.floor(math.log(n / e) / math.log(reach / e) * (half - e) + 1e-9))
            assert b == k + (half if x > 0 else 0), (buckets, reach, x)
