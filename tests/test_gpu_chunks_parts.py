"""Attention over chunks with fp32 queries over bf16 caches in the MFMA page layout keeps 24 bits of queries and weights
(three parts of bf16 each), against the definition in 64 bits.

Tolerances.
Queries.  A score is 3 D / 16 accumulations (24 at head_dim 128), each off by at most a step, 2^-23 of the sum, of random
  sign: sqrt(3 D / 16) 2^-23 |s| ln 2 of a weight for a score of s log2 units, independently from key to key, so that a row
  is off by as much of its size (chunkutil.attend64), where s is the score at which the size's terms p_t^2 lie: scores of
  standard deviation a = 1.5 nats give e^(2 s) e^(-s^2 / 2 a^2), whose mean is 2 a^2 = 4.5 nats = 6.5 log2 units: 2.6e-6 at
  head_dim 128, 1.9e-6 at 64.  (At first s was taken as the scores' own size, 2.2 log2 units, which is where the keys lie, not
  the weights; rows reached 1.95e-6 where that gives 0.9e-6.)  Weights summed over n rows: that / sqrt(n), and 2^-23 for the
  sum itself.
Weights.  Where each score is one exact product, what is left are the exponent's rounding, 2^-24 of up to 8 log2 units where
  the weights lie, the exponential's (2^-23) and the sums' (2^-23): 2^-24 8 ln 2 + 2^-22 = 5.7e-7, and twice that for a row
  among hundreds: 2^-20 rounded down.
Two parts of either leave more, which the first test shows on the CPU.
"""
import math

import pytest
import torch

import qauntrunner_amd as qr
from tests.chunkutil import attend64, randn, row_errors

WEIGHTS = 2.0 ** -20


def tol(D):
    return math.sqrt(3 * D / 16) * 2.0 ** -23 * 2 * 1.5 ** 2  # (nats: without the two factors of ln 2)


def wtol(D, n):
    return tol(D) / math.sqrt(n) + 2.0 ** -23


def kept(x, parts):
    """What `parts` parts of bf16 keep of fp32 values."""
    left = x.clone()
    for _ in range(parts):
        left -= left.to(torch.bfloat16).float()
    return x - left


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [20, 40])
def test_two_parts_would_be_seen(D, n):
    g = torch.Generator()
    g.manual_seed(D + n)
    length = 3000
    k, v = (torch.randn(length, D, generator=g).to(torch.bfloat16).double() for _ in range(2))
    q = 1.5 * torch.randn(n, D, generator=g)

    def attend(q, weights):
        s = (q.double() @ k.t()) * D ** -0.5
        e = torch.exp(s - s.max(1, keepdim=True).values)
        p = e / e.sum(1, keepdim=True)
        if weights:
            p = kept(e.float(), weights).double() / e.float().double().sum(1, keepdim=True)
        return p @ v, p

    want, p = attend(q, 0)
    size = (p.square() @ v.square().sum(1)).sqrt()
    for parts, over in ((2, True), (3, False)):
        out, w = attend(kept(q, parts), 0)
        assert (row_errors(out, want, size) > tol(D)) == over
        assert (row_errors(w.sum(0), p.sum(0)) > wtol(D, n)) == over
        assert (row_errors(attend(q, parts)[0], want, size) > WEIGHTS) == over


def run(n, length, D, k, v, q):
    out, w = torch.empty_like(q), torch.zeros(2, 8, length, device="cuda")
    with qr.PagedKvCache(1, 8, 8, D, length, "bf16", 2) as kv:
        for s in range(2):
            kv.AppendRangeDev(0, 0, k.view(length, -1), v.view(length, -1), "bf16", seq_id=s)
        kv.AttentionChunksDev(0, [0, 1], [length - n] * 2, [n] * 2, q, out, D ** -0.5, weights=w)
    for s in range(2):
        yield out[s * n:(s + 1) * n], w[s], attend64(q[s * n:(s + 1) * n], k, v, length - n, D ** -0.5, 8, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 20, 32, 40, 64, 100, 128, 300])
@pytest.mark.parametrize("length", [700, 3000])
def test_fp32_queries_over_bf16(gpu, D, n, length):
    k, v = (randn(s, length, 8, D, dtype="bf16") for s in (1, 2))
    for got, w, (want, size, ww) in run(n, length, D, k, v, randn(3, 2 * n, 8, D, scale=1.5)):
        e = row_errors(got, want, size)
        assert e <= tol(D), f"out: {e:.3g}"
        e = row_errors(w, ww)
        assert e <= wtol(D, n), f"weights: {e:.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 20, 32, 40, 64, 100, 128, 300])
@pytest.mark.parametrize("length", [700, 3000])
def test_weights_of_exact_scores(gpu, D, n, length):
    k, v = (randn(s, length, 8, D, dtype="bf16") for s in (1, 2))
    q = torch.zeros(2 * n, 8, D, device="cuda")
    q[:, :, 5] = 1.5 * math.sqrt(D) * torch.linspace(0.75, 1.25, 2 * n, device="cuda")[:, None]
    for got, w, (want, size, ww) in run(n, length, D, k, v, q.to(torch.bfloat16).float()):
        e = row_errors(got, want, size)
        assert e <= WEIGHTS, f"out: {e:.3g}"
