"""GPU tests of NaN and infinite values in long contexts: which rows show them, and that they cost no more than a look at
the values."""
import math
import time

import pytest
import torch

import qauntrunner_amd as qr
from tests.chunkutil import TORCH, attend64, randn, row_errors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,act", [("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("n", [1, 12, 25, 70])
def test_a_nan_in_every_dim_takes_no_longer(gpu, dtype, act, n):
    """One early value that is NaN in all its dims, 64 sequences of 8192 positions whose keys are not split: the call takes
    its milliseconds (walking the keys for each dim by itself took 60 to 120)."""
    heads, kv_heads, D, length, seqs = 32, 8, 128, 8192, 64
    k, v = (randn(s, length, kv_heads, D, dtype=dtype) for s in (1, 2))
    with qr.PagedKvCache(1, heads, kv_heads, D, length, dtype, seqs) as kv:
        for s in range(seqs):
            kv.AppendRangeDev(0, 0, k.view(length, -1), v.view(length, -1), dtype, seq_id=s)
        q = randn(3, seqs * n, heads, D, dtype=act)
        out, again = torch.empty_like(q), torch.empty_like(q)
        call = lambda o: kv.AttentionChunksDev(0, list(range(seqs)), [length - n] * seqs, [n] * seqs, q, o, D ** -0.5)  # noqa: E731
        call(out)
        v[5, 2] = float("nan")
        kv.AppendRangeDev(0, 5, k[5:6].reshape(1, -1), v[5:6].reshape(1, -1), dtype, seq_id=3)
        torch.cuda.synchronize()
        t = time.perf_counter()
        call(again)
        torch.cuda.synchronize()
        t = time.perf_counter() - t
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[3 * n:4 * n, 8:12] = True
        assert again[hit].isnan().all() and torch.equal(again[~hit], out[~hit])
        assert t < 0.04, f"{1e3 * t:.1f} ms"
