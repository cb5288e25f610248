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


@pytest.mark.parametrize("dtype,act,D", [("bf16", "bf16", 128), ("f16", "f16", 64), ("f16", "f32", 128), ("bf16", "f32", 64), ("f32", "f32", 64),
                                         ("f32", "f32", 128), ("f32", "bf16", 96), ("bf16", "bf16", 96), ("f16", "f32", 256), ("f32", "f32", 80),
                                         ("bf16", "bf16", 20)])
@pytest.mark.parametrize("n", [1, 12, 25, 70])
@pytest.mark.parametrize("seqs", [1, 64])  # the keys split over many workgroups, and not
@pytest.mark.parametrize("at", [3, 2100])  # before and behind the keys of large weight
def test_infinite_values_of_little_weight(gpu, dtype, act, D, n, seqs, at):
    """A weight of e^-190 is zero in 32 bits, but none in the formula: a row that sees an infinite V shows that infinity
    whatever its weight, and NaN where it sees both or a NaN.  The others' sums: tolerances as in tests/test_gpu_chunks.py."""
    heads, kv_heads, length = 8, 2, 2500
    if D in (80, 20) and seqs > 1:
        seqs = 8
    k, v = (randn(s, length, kv_heads, D, dtype="f32") for s in (1, 2))
    k[:, :, 0] = 0
    k[max(at - 200, 0):at + 200, :, 0] = -(190 * math.sqrt(D) / 8)  # against queries of 8 there; whole parts of split keys
    inf = math.inf
    v[at, 0, 1], v[at, 0, 3], v[at, 1, D - 1], v[at, 1, 2] = inf, -inf, inf, math.nan
    v[at + 40, :, 3] = inf
    k, v = k.to(TORCH[dtype]), v.to(TORCH[dtype])
    q = randn(3, seqs * n, heads, D, dtype="f32")
    q[:, :, 0] = 8
    q = q.to(TORCH[act])
    out = torch.empty_like(q)
    with qr.PagedKvCache(1, heads, kv_heads, D, length, dtype, seqs) as kv:
        for s in range(seqs):
            kv.AppendRangeDev(0, 0, k.view(length, -1), v.view(length, -1), dtype, seq_id=s)
        kv.AttentionChunksDev(0, list(range(seqs)), [length - n] * seqs, [n] * seqs, q, out, D ** -0.5)
    for s in (0, seqs - 1):
        got = out[s * n:(s + 1) * n].double()
        assert (got[:, :4, 1] == inf).all() and got[:, :4, 3].isnan().all()
        assert (got[:, 4:, D - 1] == inf).all() and got[:, 4:, 2].isnan().all() and (got[:, 4:, 3] == inf).all()
        want, size, _ = attend64(q[s * n:(s + 1) * n], k, torch.where(v.isfinite(), v, 0), length - n, D ** -0.5, heads, kv_heads)
        for x in (got, want):
            for h, d in ((slice(0, 4), 1), (slice(0, 4), 3), (slice(4, 8), D - 1), (slice(4, 8), 2), (slice(4, 8), 3)):
                x[:, h, d] = 0
        tol = torch.finfo(TORCH[act]).eps if act != "f32" else 2.0 ** -16 if dtype == "f32" else 2.0 ** -15
        e = row_errors(got, want, size)
        assert e <= tol, f"out: {e:.3g}"
