"""GPU tests of attention over chunks at the borders of its plan, against the definition in 64 bits; tolerances as in
tests/test_gpu_chunks.py."""
import pytest
import torch

import qauntrunner_amd as qr
from tests.chunkutil import TORCH, attend64, randn, row_errors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,act,D,heads,kv_heads", [("f16", "f16", 64, 32, 8), ("bf16", "f32", 64, 32, 8), ("f16", "f32", 64, 32, 8),
                                                       ("f32", "f32", 64, 32, 8), ("bf16", "bf16", 96, 32, 8)])
def test_more_scores_than_are_kept(gpu, dtype, act, D, heads, kv_heads):
    """Chunks of few rows whose weights come from kept scores up to 256 MB of them, from scores computed again beyond."""
    n, rows, length = 24, 8, 16384  # 16.8 MB of scores each
    k, v = (randn(s, length, kv_heads, D, dtype=dtype) for s in (1, 2))
    with qr.PagedKvCache(1, heads, kv_heads, D, length, dtype, n) as kv:
        for s in range(n):
            kv.AppendRangeDev(0, 0, k.view(length, -1), v.view(length, -1), dtype, seq_id=s)
        q = randn(3, n * rows, heads, D, dtype=act, scale=1.5)
        out, w = torch.empty_like(q), torch.zeros(n, kv_heads, length, device="cuda")
        kv.AttentionChunksDev(0, list(range(n)), [length - rows] * n, [rows] * n, q, out, D ** -0.5, weights=w)
        tol = torch.finfo(TORCH[act]).eps if act != "f32" else 2.0 ** -16 if dtype == "f32" else 2.0 ** -15
        for s in (0, 15, 16, n - 1):
            want, size, ww = attend64(q[s * rows:(s + 1) * rows], k, v, length - rows, D ** -0.5, heads, kv_heads)
            e = row_errors(out[s * rows:(s + 1) * rows], want, size)
            assert e <= tol, f"out of {s}: {e:.3g}"
            e = row_errors(w[s], ww)
            assert e <= (2.0 ** -16 if dtype == "f32" else 2.0 ** -15), f"weights of {s}: {e:.3g}"
