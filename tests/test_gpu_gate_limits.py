"""The GELU gate at infinities and NaN, on every gated kernel: x Phi(x) as the formula has it (NaN for NaN, +inf
for +inf, -inf times 0 is NaN), and its neighbours untouched."""
import numpy as np
import pytest

from test_gpu_gated import Pair
from weight_only_oracle import act64, act_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["q8", "q4", "w8a8"])
@pytest.mark.parametrize("M", [1, 4, 33, 300, 1500, 5000])
def test_gelu_gate_of_non_finite_values(ctx, form, M):
    x = np.random.default_rng(9).uniform(-12, 12, size=400).astype(np.float32)
    x[[3, 64, 399]], x[[4, 65, 130]], x[[5, 66, 255]] = np.nan, np.inf, -np.inf
    with Pair(ctx, form, np.random.default_rng(2), len(x), 64) as p:
        p.b = [x, np.full(len(x), 0.5, np.float32)]
        print(f"[case] gate limits {form} M={M}", flush=True)
        got = p.run(np.zeros((M, 64), np.float32), "gelu").astype(np.float64)
    fin = np.isfinite(x)
    assert np.isnan(got[:, np.isnan(x) | np.isneginf(x)]).all()
    assert (got[:, np.isposinf(x)] == np.inf).all()
    want = 0.5 * act64("gelu", x[fin].astype(np.float64))
    assert np.all(np.abs(got[:, fin] - want) <= 0.5 * act_bound("gelu", x[fin].astype(np.float64)) + 1e-37)
