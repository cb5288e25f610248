"""GPU tests of causal attention over chunks of several sequences with the weight of each cached position
(qr_kv_attention_chunks_dev), against the definition in 64 bits.

Tolerances, per row (one query head's output; one kv head's weights), 2-norm relative to the row's (an output row: to
its size where that is more, chunkutil.attend64), from the arithmetic:
  fp32 queries, fp32 cache: products and sums in fp32.  A score of D products of which |s| <= 8 or so is off by a few
    2^-24 sqrt(D) |s| < 2^-17 for D <= 512; a weight by as much relatively: 2^-16.
  fp32 queries, 16-bit cache: q and the softmax weights may enter as two parts of the cache's type, which keeps 2^-17
    (bf16) of each: another 8 x 2^-17 for a score, 2^-17 for a weight: 2^-13 bounds a row, where the parts' errors of
    all D products would have to agree; they do not: 2^-15.
  16-bit queries: the softmax weights and the output are each rounded to the type, half a step (eps / 2) each: eps.
  weights: the scores' part alone, 2^-15 (2^-16 for fp32 caches).
"""
import math

import pytest
import torch

import qauntrunner_amd as qr
from tests.chunkutil import TORCH, attend64, filled, randn, row_errors

pytestmark = pytest.mark.gpu


def tol(dtype, act):
    if act != "f32":
        return torch.finfo(TORCH[act]).eps
    return 2.0 ** -16 if dtype == "f32" else 2.0 ** -15


def wtol(dtype):
    return 2.0 ** -16 if dtype == "f32" else 2.0 ** -15


def run(kv, rows, chunks, heads, kv_heads, D, dtype, act, weights=True, scale=None, seed=7, qscale=1.5, check=True):
    """chunks: (sequence, pos0, rows).  Returns (out, weights, expected out, expected weights)."""
    scale = 1 / math.sqrt(D) if scale is None else scale
    total = sum(c[2] for c in chunks)
    q = randn(seed, total, heads, D, dtype=act, scale=qscale)
    out = torch.full((total, heads * D), 7.0, dtype=TORCH[act], device="cuda")
    w = randn(seed + 1, kv.MaxBatch, kv_heads, kv.MaxSeq).abs() * 1e-3 if weights else None
    before = w.clone() if weights else None
    kv.AttentionChunksDev(0, [c[0] for c in chunks], [c[1] for c in chunks], [c[2] for c in chunks], q, out, scale,
                          weights=w)
    want, ww = torch.empty(total, heads, D, dtype=torch.float64, device="cuda"), before.double() if weights else None
    size = torch.empty(total, heads, dtype=torch.float64, device="cuda")
    at = 0
    for s, p, n in chunks:
        if n:
            want[at:at + n], size[at:at + n], x = attend64(q[at:at + n], *rows[s], p, scale, heads, kv_heads)
            if weights:
                ww[s, :, :p + n] += x
        at += n
    got = out.view(total, heads, D)
    if check:
        e = row_errors(got, want, size)
        assert e <= tol(dtype, act), f"out: {e:.3g}"
        if weights:
            e = row_errors(w - before, ww - before.double())
            # the sum is rounded at the size of what was there: 2^-24 of it
            assert e <= wtol(dtype) + 2.0 ** -20, f"weights: {e:.3g}"
            untouched = torch.ones_like(w, dtype=torch.bool)
            for s, p, n in chunks:
                if n:
                    untouched[s, :, :p + n] = False
            assert torch.equal(w[untouched], before[untouched])
    return got, w, want, ww


CHUNKS = {
    "decode": [(0, 0, 1), (1, 300, 1), (2, 255, 1), (3, 256, 1), (4, 1000, 1)],
    "ragged": [(4, 900, 101), (0, 0, 1), (1, 255, 3), (2, 200, 0), (3, 0, 257)],
    "verify": [(0, 0, 8), (4, 990, 9), (2, 250, 7), (1, 100, 2)],
}
LENGTHS = [8, 301, 257, 257, 1001]
SHAPES = [(8, 2, 64), (8, 8, 128), (28, 4, 128), (24, 8, 64), (16, 1, 128), (64, 1, 64), (4, 2, 96), (5, 2, 64),
          (3, 3, 40), (6, 2, 256), (7, 1, 20), (2, 1, 512), (2, 2, 1), (72, 1, 64)]


@pytest.mark.parametrize("name", list(CHUNKS))
@pytest.mark.parametrize("heads,kv_heads,D", SHAPES)
@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
def test_shapes(gpu, dtype, act, heads, kv_heads, D, name):
    kv, rows = filled(heads, kv_heads, D, dtype, LENGTHS)
    with kv:
        run(kv, rows, CHUNKS[name], heads, kv_heads, D, dtype, act)


@pytest.mark.parametrize("dtype,act", [("f32", "bf16"), ("f32", "f16"), ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("D", [64, 80])
def test_mixed_types(gpu, dtype, act, D):
    kv, rows = filled(8, 2, D, dtype, LENGTHS)
    with kv:
        run(kv, rows, CHUNKS["ragged"], 8, 2, D, dtype, act)


@pytest.mark.parametrize("dtype,act,heads,kv_heads,D", [("f32", "f32", 8, 2, 64), ("bf16", "bf16", 32, 8, 128), ("f16", "f32", 28, 4, 128),
                                                       ("bf16", "f32", 16, 16, 64), ("f32", "f32", 24, 8, 96)])
@pytest.mark.parametrize("weights", [False, True])
def test_long_contexts_are_split(gpu, dtype, act, heads, kv_heads, D, weights):
    lengths = [9000, 1, 4097, 700]
    kv, rows = filled(heads, kv_heads, D, dtype, lengths)
    with kv:
        run(kv, rows, [(0, 8999, 1), (1, 0, 1), (2, 4090, 7), (3, 690, 1)], heads, kv_heads, D, dtype, act, weights)


@pytest.mark.parametrize("dtype,act,heads,kv_heads,D", [("bf16", "bf16", 32, 8, 128), ("f16", "f16", 8, 2, 64), ("f32", "f32", 8, 4, 128),
                                                       ("bf16", "f32", 24, 8, 128)])
@pytest.mark.parametrize("weights", [False, True])
def test_prompts(gpu, dtype, act, heads, kv_heads, D, weights):
    lengths = [1200, 515, 130]
    kv, rows = filled(heads, kv_heads, D, dtype, lengths)
    with kv:
        run(kv, rows, [(0, 400, 800), (1, 0, 515), (2, 129, 1)], heads, kv_heads, D, dtype, act, weights)


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("heads,kv_heads", [(12, 3), (10, 5), (24, 12), (14, 14), (16, 16), (2, 1), (63, 9)])
def test_kv_heads_over_the_xcds(gpu, dtype, act, heads, kv_heads):
    """Kernels of many rows deal the kv heads of a launch to eight parts of the GPU: counts that divide and that do not."""
    kv, rows = filled(heads, kv_heads, 64, dtype, [700, 300, 40])
    with kv:
        run(kv, rows, [(1, 1, 299), (0, 290, 410), (2, 0, 40)], heads, kv_heads, 64, dtype, act)


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
def test_two_graphs_of_one_cache(gpu, dtype, act):
    """Graphs of a small and a large call share the handle's workspace, which grew between their captures."""
    lengths = [900, 600, 33]
    kv, rows = filled(8, 2, 128, dtype, lengths)
    calls = [([0, 1, 2], [899, 599, 32], [1, 1, 1]), ([0, 2, 1], [300, 0, 0], [600, 33, 600])]
    with kv:
        graphs, ins, outs, ws = [], [], [], []
        for ids, p, n in calls:
            q = randn(len(graphs), sum(n), 8 * 128, dtype=act)
            out, w = torch.zeros_like(q), torch.zeros(3, 2, 900, device="cuda")
            kv.AttentionChunksDev(0, ids, p, n, q, out, 0.1, weights=w)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                kv.AttentionChunksDev(0, ids, p, n, q, out, 0.1, weights=w)
            for l, x in zip((graphs, ins, outs, ws), (g, q, out, w)):
                l.append(x)
        for turn in range(3):
            for i in (0, 1, 1, 0):
                ins[i].copy_(randn(10 + turn, *ins[i].shape, dtype=act))
                outs[i].zero_()
                ws[i].zero_()
                graphs[i].replay()
            for i, (ids, p, n) in enumerate(calls):
                out, w = torch.zeros_like(outs[i]), torch.zeros_like(ws[i])
                kv.AttentionChunksDev(0, ids, p, n, ins[i], out, 0.1, weights=w)
                assert torch.equal(out, outs[i]) and torch.equal(w, ws[i])


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16")])
def test_more_chunks_than_one_launch_takes(gpu, dtype, act):
    n = 131
    lengths = [1 + (37 * i) % 300 for i in range(n)]
    kv, rows = filled(8, 2, 64, dtype, lengths)
    with kv:
        chunks = [(i, 0 if i % 3 else lengths[i] - 1, lengths[i] if i % 3 else 1) for i in range(n)]
        run(kv, rows, [c if c[0] % 7 else (c[0], 0, 0) for c in chunks], 8, 2, 64, dtype, act)


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("D", [128, 48])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, dtype, act, D):
    """NaN and infinities behind a row's position, in the same tile and page, leave it as it was; a NaN V reaches
    the rows that see it, and only those."""
    heads, kv_heads = 8, 2
    lengths = [300, 40]
    kv, rows = filled(heads, kv_heads, D, dtype, lengths, max_seq=512)
    with kv:
        chunks = [(0, 250, 6), (1, 30, 3)]
        clean, wc, _, _ = run(kv, rows, chunks, heads, kv_heads, D, dtype, act)
        for s, at in ((0, 256), (1, 33)):
            for bad in (float("nan"), float("inf")):
                k = torch.full((44 if s == 0 else 7, kv_heads * D), bad, dtype=TORCH[dtype], device="cuda")
                kv.AppendRangeDev(0, at, k, k, dtype, seq_id=s)
                got, w, _, _ = run(kv, rows, chunks, heads, kv_heads, D, dtype, act)
                assert torch.equal(got, clean) and torch.equal(w, wc)
        v = rows[0][1][253:254].clone()
        v[0, 0, 5] = float("nan")
        v[0, 1, 7] = float("inf")
        kv.AppendRangeDev(0, 253, rows[0][0][253:254].reshape(1, -1), v.reshape(1, -1), dtype, seq_id=0)
        got, w, _, _ = run(kv, rows, chunks, heads, kv_heads, D, dtype, act, check=False)
        # rows 0..2 of chunk 0 sit before position 253
        same = torch.ones_like(got, dtype=torch.bool)
        same[3:6, 0:4, 5] = False
        same[3:6, 4:8, 7] = False
        tight = tol(dtype, act)
        assert torch.allclose(got[same].double(), clean[same].double(), rtol=tight, atol=tight)
        assert torch.isnan(got[3:6, 0:4, 5]).all() and torch.isinf(got[3:6, 4:8, 7]).all()
        assert torch.equal(w, wc)


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [6, 12, 20, 33, 150])
def test_special_rows_in_a_chunk(gpu, dtype, act, D, n):
    """A NaN or infinite key or value inside a chunk (of every number of rows that has a kernel) and what lies behind it:
    rows before it give what they give without, rows that see it show it."""
    heads, kv_heads, p0 = 8, 2, 210
    end = p0 + n
    kv, rows = filled(heads, kv_heads, D, dtype, [end], max_seq=512)
    tight = tol(dtype, act)
    with kv:
        chunks = [(0, p0, n)]
        clean, wc, _, _ = run(kv, rows, chunks, heads, kv_heads, D, dtype, act)
        k0, v0 = rows[0]
        behind = torch.full((512 - end, kv_heads * D), float("nan"), dtype=TORCH[dtype], device="cuda")
        kv.AppendRangeDev(0, end, behind, behind, dtype, seq_id=0)
        at = n // 2  # the row whose own position is the special one
        for bad in (float("nan"), float("inf"), -float("inf")):
            v = v0[p0 + at:p0 + at + 1].clone()
            v[0, 1, D - 3] = bad
            kv.AppendRangeDev(0, p0 + at, k0[p0 + at:p0 + at + 1].reshape(1, -1), v.reshape(1, -1), dtype, seq_id=0)
            got, w, _, _ = run(kv, rows, chunks, heads, kv_heads, D, dtype, act, check=False)
            same = torch.ones_like(got, dtype=torch.bool)
            same[at:, 4:, D - 3] = False
            assert torch.allclose(got[same].double(), clean[same].double(), rtol=tight, atol=tight)
            shown = got[at:, 4:, D - 3]
            assert (shown.isnan() if bad != bad else shown == bad).all()
            assert torch.equal(w, wc)
        k = k0[p0 + at:p0 + at + 1].clone()
        k[0, 0, 2] = float("nan")
        kv.AppendRangeDev(0, p0 + at, k.reshape(1, -1), v0[p0 + at:p0 + at + 1].reshape(1, -1), dtype, seq_id=0)
        got, w, _, _ = run(kv, rows, chunks, heads, kv_heads, D, dtype, act, check=False)
        assert torch.allclose(got[:at].double(), clean[:at].double(), rtol=tight, atol=tight)
        assert torch.allclose(got[:, 4:].double(), clean[:, 4:].double(), rtol=tight, atol=tight)
        assert got[at:, :4].isnan().all()
        assert torch.equal(w[0, 1], wc[0, 1]) and w[0, 0, p0 + at].isnan()


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("scale", [0.0, -0.125, 0.5])
def test_scales(gpu, dtype, act, scale):
    kv, rows = filled(8, 2, 64, dtype, LENGTHS)
    with kv:
        run(kv, rows, CHUNKS["ragged"], 8, 2, 64, dtype, act, scale=scale, qscale=0.5)


@pytest.mark.parametrize("dtype,D", [("f16", 64), ("f16", 128), ("f32", 64), ("bf16", 64)])
def test_large_queries_and_values(gpu, dtype, D):
    """Queries past fp16's range over an fp16 cache, values near the top of the cache's range."""
    kv, rows = filled(8, 2, D, dtype, [300, 40])
    with kv:
        run(kv, rows, [(0, 200, 100), (1, 39, 1)], 8, 2, D, dtype, "f32", qscale=1e5, scale=1e-5 / math.sqrt(D))
        big = 6e4 if dtype == "f16" else 1e37
        for s, n in ((0, 300), (1, 40)):
            v = (rows[s][1].float().sign() * big).to(TORCH[dtype])
            kv.AppendRangeDev(0, 0, rows[s][0].reshape(n, -1), v.reshape(n, -1), dtype, seq_id=s)
            rows[s] = (rows[s][0], v)
        run(kv, rows, [(0, 200, 100), (1, 39, 1)], 8, 2, D, dtype, "f32")


@pytest.mark.parametrize("dtype,act,D", [("f32", "f32", 64), ("bf16", "bf16", 128), ("f16", "f32", 64), ("bf16", "bf16", 96)])
def test_two_runs_are_equal_and_orders_of_chunks_do_not_matter(gpu, dtype, act, D):
    kv, rows = filled(8, 2, D, dtype, [2000, 1001, 300])
    with kv:
        chunks = [(0, 1900, 100), (1, 1000, 1), (2, 0, 300)]
        a, wa, _, _ = run(kv, rows, chunks, 8, 2, D, dtype, act)
        b, wb, _, _ = run(kv, rows, chunks, 8, 2, D, dtype, act)
        assert torch.equal(a, b) and torch.equal(wa, wb)
        run(kv, rows, chunks[::-1], 8, 2, D, dtype, act)


def test_the_same_sequence_twice_without_weights(gpu):
    kv, rows = filled(8, 2, 64, "bf16", [400])
    with kv:
        run(kv, rows, [(0, 399, 1), (0, 0, 64), (0, 399, 1)], 8, 2, 64, "bf16", "bf16", weights=False)
        q = randn(3, 2, 512, dtype="bf16")
        w = torch.zeros(1, 2, 400, device="cuda")
        with pytest.raises(qr.QrInvalidArgument, match="two entries"):
            kv.AttentionChunksDev(0, [0, 0], [3, 4], [1, 1], q, torch.empty_like(q), 1.0, weights=w)
        # a chunk without rows takes no part
        kv.AttentionChunksDev(0, [0, 0], [3, 4], [1, 0], q[:1].contiguous(), torch.empty_like(q[:1]), 1.0, weights=w)


@pytest.mark.parametrize("dtype,act,D", [("bf16", "bf16", 128), ("f16", "f32", 64), ("f32", "f32", 128), ("f32", "bf16", 64), ("f32", "f32", 40),
                                         ("bf16", "f32", 96)])
def test_tensors_off_vector_alignment(gpu, dtype, act, D):
    """q, out and weights whose addresses are aligned to their element only give what aligned ones give."""
    kv, rows = filled(8, 2, D, dtype, [700, 300, 130, 9])
    chunks = ([0, 1, 2, 3], [400, 299, 110, 0], [300, 1, 20, 9])
    n = sum(chunks[2])
    with kv:
        q = randn(3, n, 8 * D, dtype=act)
        out, w = torch.zeros_like(q), torch.zeros(4, 2, 700, device="cuda")
        kv.AttentionChunksDev(0, *chunks, q, out, D ** -0.5, weights=w)
        for off in (1, 2):
            def moved(x):
                y = torch.full((x.numel() + 8,), 5.0, dtype=x.dtype, device="cuda")
                y[off:off + x.numel()] = x.flatten()
                return y, y[off:off + x.numel()].view_as(x)
            (_, q1), (oe, o1), (we, w1) = moved(q), moved(torch.zeros_like(q)), moved(torch.zeros_like(w))
            kv.AttentionChunksDev(0, *chunks, q1, o1, D ** -0.5, weights=w1)
            assert torch.equal(o1, out) and torch.equal(w1, w)
            for e, x in ((oe, out), (we, w)):
                assert (e[:off] == 5).all() and (e[off + x.numel():] == 5).all()


def test_nothing_to_do(gpu):
    kv, _ = filled(8, 2, 64, "f32", [4, 4])
    with kv:
        q = torch.empty(0, 512, device="cuda")
        kv.AttentionChunksDev(0, [], [], [], q, q.clone(), 1.0)
        kv.AttentionChunksDev(0, [0, 1], [3, 900], [0, 0], q, q.clone(), 1.0)


@pytest.mark.parametrize("dtype,act,D", [("f32", "f32", 64), ("bf16", "bf16", 128)])
def test_on_another_stream_and_layer(gpu, dtype, act, D):
    kv, rows = filled(8, 2, D, dtype, [700, 90], layers=3, layer=2)
    with kv:
        q = randn(5, 41, 8 * D, dtype=act)
        want = torch.empty_like(q)
        kv.AttentionChunksDev(2, [0, 1], [660, 89], [40, 1], q, want, 0.1)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        for explicit in (False, True):
            out = torch.zeros_like(q)
            torch.cuda.synchronize()
            if explicit:
                kv.AttentionChunksDev(2, [0, 1], [660, 89], [40, 1], q, out, 0.1, stream=side)
            else:
                with torch.cuda.stream(side):
                    kv.AttentionChunksDev(2, [0, 1], [660, 89], [40, 1], q, out, 0.1)
            side.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize("dtype,act,D", [("f32", "f32", 64), ("bf16", "bf16", 128), ("f16", "f32", 128)])
def test_captured_and_replayed(gpu, dtype, act, D):
    """A captured call with weights, replayed between eager calls on the same cache: every replay equals the eager
    call on the inputs of its time."""
    kv, rows = filled(8, 2, D, dtype, [1500, 90, 300])
    with kv:
        args = (0, [0, 1, 2], [1490, 89, 0], [10, 1, 300])
        q = randn(5, 311, 8 * D, dtype=act)
        out, w = torch.zeros_like(q), torch.zeros(3, 2, 1500, device="cuda")
        kv.AttentionChunksDev(*args, q, out, 0.1, weights=w)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv.AttentionChunksDev(*args, q, out, 0.1, weights=w)
        for k in range(4):
            q.copy_(randn(20 + k, 311, 8 * D, dtype=act))
            w.fill_(0.25 * k)
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            got, gw = out.clone(), w.clone()
            w.fill_(0.25 * k)
            kv.AttentionChunksDev(*args, q, out, 0.1, weights=w)
            torch.cuda.synchronize()
            assert torch.equal(got, out) and torch.equal(gw, w)


def test_refusals(gpu):
    kv, _ = filled(8, 2, 64, "f32", [300, 20], max_seq=512)
    with kv:
        q = torch.zeros(2, 512, device="cuda")
        out = torch.empty_like(q)
        call = lambda ids, pos, n, q=q, out=out, layer=0, scale=1.0, **kw: kv.AttentionChunksDev(layer, ids, pos, n, q, out, scale, **kw)  # noqa: E731
        with pytest.raises(qr.QrNotResident):
            call([1], [255], [2])
        with pytest.raises(qr.QrOutOfRange):
            call([0], [511], [2])
        with pytest.raises(qr.QrOutOfRange):
            call([0], [-1], [2])
        with pytest.raises(qr.QrInvalidArgument):
            call([2], [0], [2])
        with pytest.raises(qr.QrInvalidArgument):
            call([0], [0], [2], layer=1)
        with pytest.raises(qr.QrInvalidArgument):
            call([0], [0], [2], scale=float("nan"))
        for bad in (dict(q=q.double()), dict(q=q[:1]), dict(q=q.cpu()), dict(out=out.half()), dict(out=q), dict(q=q.t()),
                    dict(weights=torch.zeros(2, 2, 300, device="cuda")), dict(weights=torch.zeros(2, 2, 512, device="cuda").half())):
            with pytest.raises(ValueError):
                call([0], [0], [2], **bad)
        with pytest.raises(ValueError):
            call([0, 1], [0], [2])
        with pytest.raises(ValueError):
            call([0], [0.5], [2])
        with pytest.raises(ValueError):
            call([0], [1 << 40], [2])
        with pytest.raises(ValueError):
            call([0, 1], [0, 0], [3, -1])
