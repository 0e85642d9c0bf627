"""What DeviceBert refuses before it calls the library."""
from types import SimpleNamespace

import pytest

from aikit_amd.bert_dev import DeviceBert


class Tensor:
    """The attributes of a device tensor that the checks read."""

    def __init__(self, *shape, dtype="f32", device="cuda", contiguous=True):
        self.shape, self.dtype, self.device, self._c = shape, dtype, SimpleNamespace(type=device), contiguous

    def is_contiguous(self):
        return self._c

    def data_ptr(self):
        raise AssertionError("read before it was checked")


def model():
    m = DeviceBert.__new__(DeviceBert)
    m.torch, m.D, m.ctx = SimpleNamespace(float32="f32", int32="i32"), 64, None
    m.forward = lambda *a, **k: pytest.fail("the layers ran")
    return m


@pytest.mark.parametrize("spans", [None, 5])
def test_embed_refuses_outputs_that_do_not_hold_the_rows(spans):
    m, S = model(), 2
    sp = None if spans is None else Tensor(spans, 2, dtype="i32")
    n = S if spans is None else spans
    for bad in (Tensor(n - 1, 64), Tensor(n, 63), Tensor(n, 65), Tensor(n * 64), Tensor(n, 64, contiguous=False), Tensor(n, 64, dtype="f16"),
                Tensor(n, 64, device="cpu"), Tensor(1, n, 64)):
        with pytest.raises(ValueError, match="pooled"):
            m.embed(Tensor(20, 64), S, 10, bad, spans=sp)


def test_forward_refuses_hidden_rows_that_are_not_f32_on_the_device():
    m = model()
    del m.forward
    m.H = m.KV = 2
    m.hd, m.W = 32, 192
    for bad in (Tensor(19, 64), Tensor(21, 64), Tensor(20, 64, dtype="f64"), Tensor(20, 64, device="cpu"), Tensor(20, 64, contiguous=False)):
        with pytest.raises(ValueError, match="h must"):
            m.forward(bad, 2, 10)


@pytest.mark.parametrize("n", [0, 1, 65535, 65536, 200000])
def test_any_number_of_spans_is_pooled(n):
    m, calls = model(), []
    m.forward, m.mark = (lambda *a, **k: None), None
    m.ctx = SimpleNamespace(pool_mean_l2_spans_dev=lambda *a: calls.append(a))
    at = {}
    for name, t in (("h", Tensor(20, 64)), ("spans", Tensor(n, 2, dtype="i32")), ("pooled", Tensor(n, 64))):
        at[name] = t
        t.data_ptr = lambda base=len(at) << 40: base
    m.embed(at["h"], 2, 10, at["pooled"], 7, spans=at["spans"])
    done = 0
    for h, ldh, rows, spans, k, D, out, ldo, stream in calls:
        assert (h, ldh, rows, D, ldo, stream) == (1 << 40, 64, 20, 64, 64, 7) and 1 <= k <= 65535
        assert spans == (2 << 40) + 8 * done and out == (3 << 40) + 4 * 64 * done
        done += k
    assert done == n
