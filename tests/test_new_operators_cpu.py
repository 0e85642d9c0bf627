"""What the rotary, 4-bit and gated entry points refuse before any device is needed."""
import ctypes

import numpy as np
import pytest

from aikit_amd import enchip


def test_null_context():
    lib, out = enchip.load(), ctypes.c_uint64()
    assert lib.enchip_rope_create(None, 8, 1e4, 0, 1.0, 0, ctypes.byref(out)) == enchip.ERR_ARG
    assert lib.enchip_rope_create_freqs(None, None, 4, 1.0, ctypes.byref(out)) == enchip.ERR_ARG
    assert lib.enchip_rope_release(None, 1) == enchip.ERR_ARG
    assert lib.enchip_rope_rows_dev(None, 1, 0, None, 8, None, 8, 1, 1, 1, 8, None, 0, None) == enchip.ERR_ARG
    assert lib.enchip_weight4_register(None, None, None, 1, 32, 32, ctypes.byref(out)) == enchip.ERR_ARG
    assert lib.enchip_weight4_release(None, 1) == enchip.ERR_ARG
    assert lib.enchip_weight4_shape(None, 1, None, None, None) == enchip.ERR_ARG
    assert lib.enchip_matmul_bt_q4(None, 1, None, 1, None) == enchip.ERR_ARG
    assert lib.enchip_matmul_bt_q4_dev(None, 1, None, 32, 1, None, 1, None) == enchip.ERR_ARG
    for call in (lib.enchip_gated_q8, lib.enchip_gated_q4, lib.enchip_w8a8_gated):
        assert call(None, 1, 1, None, 1, None, None, 3, None) == enchip.ERR_ARG
    for call in (lib.enchip_gated_q8_dev, lib.enchip_gated_q4_dev):
        assert call(None, 1, 1, None, 32, 1, None, None, 3, None, 1, None) == enchip.ERR_ARG
    assert lib.enchip_w8a8_gated_dev(None, 1, 1, None, 1, None, None, 3, None, None) == enchip.ERR_ARG


def test_python_shape_checks():
    c = enchip.Context.__new__(enchip.Context)  # no device: the checks come first
    c._h, c._lib = None, enchip.load()
    w4, w8 = enchip.Weight4(1, 40, 100, 32), enchip.Weight(1, 40, 100)
    f = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    with pytest.raises(ValueError):
        c.register_weight4(np.zeros((4, 50), np.uint8), np.zeros((4, 3), np.float16), 100, 32)
    with pytest.raises(ValueError):
        c.register_weight4(np.zeros((4, 49), np.uint8), np.zeros((4, 4), np.float16), 100, 32)
    with pytest.raises(ValueError):
        c.register_weight4(np.zeros(50, np.uint8), np.zeros((4, 4), np.float16), 100, 32)
    with pytest.raises(ValueError):
        c.rope_from_freqs(np.zeros((2, 2)))
    for call, w in ((c.gated_q8, w8), (c.gated_q4, w4), (c.w8a8_gated, w8)):
        with pytest.raises(ValueError):
            call(w, w, f(2, 99))
        with pytest.raises(ValueError):
            call(w, w, f(100))
        with pytest.raises(ValueError):
            call(w, w, f(2, 100), bias_gate=f(39))
    with pytest.raises(ValueError):
        c.matmul_bt_q4(w4, f(2, 99))
