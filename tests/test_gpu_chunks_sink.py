"""GPU tests of attention over chunks where one key takes nearly all of a row's weight and holds no value: the output is
what the many small weights leave, at every kernel's number of rows, against the definition in 64 bits.

The small weights are 2^-15 to 2^-23 of the largest.  Tolerances, relative to a row's norm, as for weights of like size: each
weight is rounded relative to itself, not to the largest.
  16-bit queries: the weights and the output are each rounded to the type, half a step each: eps.
  fp32 queries over an fp16 cache: two parts of a weight keep 2^-18 of the smallest here (the second part's last bit is 2^-24
    where the largest weight is 2^15 or so), and the score of the large key, 16 nats or so, is off by a few 2^-24 of itself:
    2^-15, as for other rows.
  weights: the scores' part alone, 2^-15.
"""
import math

import pytest
import torch

import qauntrunner_amd as qr
from tests.chunkutil import TORCH, attend64, randn, row_errors

pytestmark = pytest.mark.gpu

HEADS, KV, SEQS = 32, 8, 64  # as many sequences as leave no chunk's keys split


def sink_rows(D, dtype, length, logit):
    """K and V [length, KV, D]; position 0 scores `logit` nats (with the queries of sink_queries and scale D^-1/2), the
    others around 0."""
    k, v = randn(3, length, KV, D, dtype="f32"), 8 + randn(4, length, KV, D, dtype="f32")
    k[:, :, 0] = 0
    k[0] = 0
    k[0, :, 0] = logit * math.sqrt(D) / 8
    v[0] = 0
    return k.to(TORCH[dtype]), v.to(TORCH[dtype])


def sink_queries(seed, rows, D, act):
    q = randn(seed, rows, HEADS, D, dtype="f32")
    q[:, :, 0] = 8
    return q.to(TORCH[act])


@pytest.mark.parametrize("dtype,act", [("f16", "f16"), ("f16", "f32"), ("f16", "bf16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 8, 12, 25, 70])
@pytest.mark.parametrize("mass", [0.9, 0.999])
def test_small_weights_beside_a_large_one(gpu, dtype, act, D, n, mass):
    length = 2048
    # the others' weights have mean e^(1/2)
    k, v = sink_rows(D, dtype, length, math.log(length * mass / (1 - mass)) + 0.5)
    with qr.PagedKvCache(1, HEADS, KV, D, length, dtype, SEQS) as kv:
        for s in range(SEQS):
            kv.AppendRangeDev(0, 0, k.view(length, -1), v.view(length, -1), dtype, seq_id=s)
        q = sink_queries(n, SEQS * n, D, act)
        out, w = torch.empty_like(q), torch.zeros(SEQS, KV, length, device="cuda")
        kv.AttentionChunksDev(0, list(range(SEQS)), [length - n] * SEQS, [n] * SEQS, q, out, D ** -0.5, weights=w)
        tol = torch.finfo(TORCH[act]).eps if act != "f32" else 2.0 ** -15
        for s in (0, SEQS - 1):
            want, size, ww = attend64(q[s * n:(s + 1) * n], k, v, length - n, D ** -0.5, HEADS, KV)
            assert float(ww[:, 0].min()) > 0.8 * mass * n * HEADS / KV
            e = row_errors(out[s * n:(s + 1) * n], want, size)
            assert e <= tol, f"out: {e:.3g}"
            e = row_errors(w[s, :, 1:], ww[:, 1:])
            assert e <= 2.0 ** -15, f"weights: {e:.3g}"


@pytest.mark.parametrize("dtype,act", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("n", [1, 12, 70])
@pytest.mark.parametrize("top", [2.0 ** 20, 2.0 ** 24, 2.0 ** 26, -(2.0 ** 24)])
def test_scores_whose_steps_are_whole_units(gpu, dtype, act, n, top):
    """Scores so large that a step of theirs is up to 8: the largest is ahead of the others by thousands, so that a row is
    the value of its key (weights and output rounded: eps, or 2^-15)."""
    D, length, at = 64, 600, 333
    k, v = (randn(s, length, KV, D, dtype="f32") for s in (5, 6))
    k[:, :, 0] = 1 - torch.rand(length, KV, device="cuda").round() / 64  # at least 2^14 below it
    k[:, :, 0] -= 1 / 64
    k[at, :, 0] = 1
    if top < 0:
        k[:, :, 0] = 2 - k[:, :, 0]  # the least far from zero
    k, v = k.to(TORCH[dtype]), v.to(TORCH[dtype])
    with qr.PagedKvCache(1, HEADS, KV, D, length, dtype, 1) as kv:
        kv.AppendRangeDev(0, 0, k.view(length, -1), v.view(length, -1), dtype)
        q = torch.zeros(n, HEADS, D, device="cuda")
        q[:, :, 0] = math.copysign(2.0 ** 12, top)
        q = q.to(TORCH[act])
        out = torch.empty_like(q)
        kv.AttentionChunksDev(0, [0], [length - n], [n], q, out, abs(top) * math.log(2) / 2 ** 12)
        want = v[at].repeat_interleave(HEADS // KV, 0).expand(n, -1, -1)
        e = row_errors(out, want)
        assert e <= (torch.finfo(TORCH[act]).eps if act != "f32" else 2.0 ** -15), f"out: {e:.3g}"
