"""Fragment-major codes of rows of any length and alignment: those of the row-major quantizer, in the
fragment order, bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def codes(ctx, a, off, ldq):
    """(row-major codes, scales, codes read back from the fragment order, its scales)"""
    import torch

    M, K = a.shape
    buf = torch.full((M * K + 8,), 9.0, device="cuda")
    da = buf[off:off + M * K]
    da.copy_(torch.from_numpy(a).reshape(-1))
    rb = (M + 31) // 32
    q = torch.full((M, ldq), 77, dtype=torch.int8, device="cuda")
    f = torch.full((rb * 32 * ldq,), 77, dtype=torch.int8, device="cuda")
    s, t = torch.full((M,), -1.0, device="cuda"), torch.full((M + 1,), -1.0, device="cuda")
    torch.cuda.synchronize()
    ctx.quant_rows_dev(da.data_ptr(), M, K, q.data_ptr(), s.data_ptr(), ldq=ldq)
    ctx.quant_rows_frag_dev(da.data_ptr(), M, K, f.data_ptr(), ldq, t.data_ptr())
    torch.cuda.synchronize()
    assert float(t[M]) == -1.0
    # [block][ldq / 32][half][row][16] -> [row][k]
    rows = f.cpu().numpy().reshape(rb, ldq // 32, 2, 32, 16).transpose(0, 3, 1, 2, 4).reshape(rb * 32, ldq)
    assert np.all(rows[M:] == 77)  # rows behind the last are left as they were
    return q.cpu().numpy(), s.cpu().numpy(), rows[:M], t[:M].cpu().numpy()


@pytest.mark.parametrize("M", [1, 5, 33, 130])
@pytest.mark.parametrize("K,off,extra", [(1, 0, 0), (33, 0, 0), (63, 1, 64), (1000, 1, 0), (1001, 0, 0), (2047, 0, 0), (2048, 3, 0),
                                         (2049, 0, 0), (4096, 1, 0), (4097, 0, 0), (4100, 0, 0), (8191, 0, 64), (8192, 0, 0),
                                         (8192, 2, 0), (8193, 0, 0), (8196, 0, 0), (20001, 0, 0), (20000, 0, 128)])
def test_any_length(ctx, M, K, off, extra):
    print(f"[case] quant_rows_frag M={M} K={K} off={off}", flush=True)
    g = np.random.default_rng(K + M)
    a = (g.standard_normal((M, K)) * 10.0 ** g.integers(-3, 4, size=(M, 1))).astype(np.float32)
    a[M // 2] = 0
    if M > 4:
        a[0, K // 2], a[1, 0], a[2, K - 1], a[3] = np.nan, np.inf, -np.inf, 1e-42
    q, s, f, t = codes(ctx, a, off, (K + 63) // 64 * 64 + extra)
    assert np.array_equal(s, t) and np.array_equal(q[:, :K], f[:, :K])
    assert not f[:, K:].any()
