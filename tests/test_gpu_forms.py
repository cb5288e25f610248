"""GPU tests of attention in its other forms and behind shared prefixes (qr_kv_attention_forms_dev), against the definition
in 64 bits.

Tolerances, per row (one query head's output), 2-norm relative to the row's norm, or to its size where that is more
(chunkutil.attend64), from the arithmetic, as for attention over chunks (tests/test_gpu_chunks.py):
  16-bit queries: the softmax weights and the output are each rounded to the type, half a step each: eps.
  fp32 queries: scores, weights and sums in 32 bits, or in parts that keep as many: 2^-16 (fp32 caches), 2^-15 (others).
  caps: cap tanh(z / cap) of |z| up to about cap is off by a few steps of 32 bits of cap: 2^-22 x 50 < 2^-16 for caps up to 50, a
    weight by as much relatively: with fp32 queries 2^-16 more.
  slopes: slope x distance up to 2^14 at 2^-24 of itself: 2^-10 of a nat, but then the weight is e^-(2^13) of the nearest; what
    still weighs (less than 16 nats away) is off by 2^-20 each: 2^-18 more, inside the bounds above.
"""
import math

import pytest
import torch

import qauntrunner_amd as qr
from tests.chunkutil import TORCH, randn, row_errors
from tests.formutil import e4m3_values, filled_as, forms64

pytestmark = pytest.mark.gpu


def tol(dtype, act, cap):
    if act != "f32":
        return torch.finfo(TORCH[act]).eps
    return (2.0**-16 if dtype == "f32" else 2.0**-15) + (2.0**-16 if cap else 0)


def slopes_of(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")


def expected(rows, chunks, q, scale, heads, kv_heads, D, first=None, full=None, prefix=None, **form):
    """chunks: (sequence, pos0, rows); prefix: (sequence, length) of each chunk or None."""
    want = torch.zeros(q.shape[0], heads, D, dtype=torch.float64, device="cuda")
    size = torch.zeros(q.shape[0], heads, dtype=torch.float64, device="cuda")
    at = 0
    for i, (s, p, n) in enumerate(chunks):
        if n:
            ps, pl = prefix[i] if prefix else (0, 0)
            fu = full[i] if full else 0
            end = max(p + n, fu - pl)
            k, v = (torch.cat([rows[ps][j][:pl], rows[s][j][:end]]) for j in (0, 1))
            want[at:at + n], size[at:at + n] = forms64(q[at:at + n], k, v, pl + p, scale, heads, kv_heads, first=first[i] if first else 0,
                                                       full=fu, **form)
        at += n
    return want, size


def run(kv, rows, chunks, dtype, act, cap=0.0, slopes=False, window=0, first=None, full=None, prefix=None, scale=None, seed=7, qscale=1.5):
    heads, kv_heads, D = kv.Heads, kv.KvHeads, kv.HeadDim
    scale = 1 / math.sqrt(D) if scale is None else scale
    total = sum(c[2] for c in chunks)
    q = randn(seed, total, heads, D, dtype=act, scale=qscale)
    out = torch.full((total, heads * D), 7.0, dtype=TORCH[act], device="cuda")
    sl = slopes_of(heads) if slopes else None
    kv.AttentionFormsDev(0, [c[0] for c in chunks], [c[1] for c in chunks], [c[2] for c in chunks], q, out, scale, cap=cap, slopes=sl,
                         window=window, first=first, full=full, prefix_ids=[x[0] for x in prefix] if prefix else None,
                         prefix_len=[x[1] for x in prefix] if prefix else None)
    want, size = expected(rows, chunks, q, scale, heads, kv_heads, D, first, full, prefix, cap=cap, slopes=sl, window=window)
    got = out.view(total, heads, D)
    assert torch.isfinite(got).all()
    e = row_errors(got, want, size)
    assert e <= tol(dtype, act, cap), f"{e:.3g}"
    # rows that see nothing are zeros
    assert not got[(size == 0) & (want == 0).all(-1)].any()
    return got, want


CHUNKS = {
    "decode": [(0, 0, 1), (1, 300, 1), (2, 255, 1), (3, 256, 1), (4, 1000, 1)],
    "ragged": [(4, 900, 101), (0, 0, 1), (1, 255, 3), (2, 200, 0), (3, 0, 257)],
    "verify": [(0, 0, 8), (4, 990, 9), (2, 250, 7), (1, 100, 2)],
}
LENGTHS = [8, 301, 257, 257, 1001]
SHAPES = [(8, 2, 64), (8, 8, 128), (28, 4, 128), (24, 8, 64), (16, 1, 128), (64, 1, 64), (4, 2, 96), (5, 2, 64), (3, 3, 40), (7, 1, 20),
          (2, 1, 512), (2, 2, 1), (72, 1, 64)]
TYPES = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("e4m3", "bf16"), ("e4m3", "f16"), ("e4m3", "f32"), ("bf16", "f32"), ("f16", "f32")]
FORMS = {
    "plain": {},
    "cap": dict(cap=3.0),
    "slopes": dict(slopes=True),
    "window": dict(window=100),
    "all": dict(cap=20.0, slopes=True, window=130),
}


@pytest.mark.parametrize("name", list(CHUNKS))
@pytest.mark.parametrize("heads,kv_heads,D", SHAPES)
@pytest.mark.parametrize("dtype,act", TYPES)
def test_shapes(gpu, dtype, act, heads, kv_heads, D, name):
    kv, rows = filled_as(heads, kv_heads, D, dtype, LENGTHS)
    with kv:
        for form in ("plain", "all"):
            run(kv, rows, CHUNKS[name], dtype, act, **FORMS[form])


@pytest.mark.parametrize("name", list(CHUNKS))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype,act,heads,kv_heads,D", [("f32", "f32", 8, 2, 64), ("bf16", "bf16", 32, 8, 128), ("f16", "f16", 28, 4, 64),
                                                        ("e4m3", "bf16", 32, 8, 128), ("e4m3", "f32", 8, 2, 64), ("bf16", "f32", 6, 3, 24)])
def test_masks(gpu, dtype, act, heads, kv_heads, D, form, name):
    """Documents and prefixes of each chunk, rows that see nothing among them."""
    kv, rows = filled_as(heads, kv_heads, D, dtype, LENGTHS)
    chunks = CHUNKS[name]
    with kv:
        first = [min(i * 83, c[1] + c[2] // 2) if i != 1 else c[1] + c[2] for i, c in enumerate(chunks)]  # chunk 1 sees nothing
        run(kv, rows, chunks, dtype, act, first=first, **FORMS[form])
        full = [min(c[1] + c[2] + 5 * (i % 2), LENGTHS[c[0]]) if i % 3 else c[1] // 2 for i, c in enumerate(chunks)]
        run(kv, rows, chunks, dtype, act, full=full, **FORMS[form])
        run(kv, rows, chunks, dtype, act, full=full, first=[x // 2 for x in full], **FORMS[form])


PREFIXES = [300, 1, 257, 1000]


@pytest.mark.parametrize("name", list(CHUNKS))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype,act,heads,kv_heads,D", [("f32", "f32", 8, 2, 64), ("bf16", "bf16", 32, 8, 128), ("f16", "f16", 28, 4, 64),
                                                        ("e4m3", "bf16", 64, 8, 128), ("e4m3", "f32", 8, 2, 64), ("f16", "f32", 16, 4, 128),
                                                        ("bf16", "bf16", 6, 4, 48)])
def test_shared_prefixes(gpu, dtype, act, heads, kv_heads, D, form, name):
    """Runs of chunks with one prefix, chunks with another or none between, whole and part of the prefix's sequence."""
    kv, rows = filled_as(heads, kv_heads, D, dtype, LENGTHS + PREFIXES)
    chunks = CHUNKS[name]
    with kv:
        for lens in ([(5, 300)] * 5, [(8, 1000), (8, 1000), (0, 0), (8, 1000), (7, 200)], [(8, 999), (8, 998), (6, 1), (7, 257), (7, 257)]):
            prefix = lens[:len(chunks)]
            run(kv, rows, chunks, dtype, act, prefix=prefix, **FORMS[form])
        prefix = [(8, 1000)] * len(chunks)
        run(kv, rows, chunks, dtype, act, prefix=prefix, first=[0, 500, 1000, 1100, 3000][:len(chunks)],
            full=[1000 + c[1] + c[2] for c in chunks], **FORMS[form])


@pytest.mark.parametrize("dtype,act,heads,kv_heads,D", [("f32", "f32", 8, 2, 64), ("bf16", "bf16", 32, 8, 128), ("e4m3", "bf16", 32, 8, 128),
                                                        ("f16", "f32", 28, 4, 128), ("e4m3", "f32", 24, 8, 128)])
@pytest.mark.parametrize("form", ["plain", "all", "window"])
def test_long_contexts_are_split(gpu, dtype, act, heads, kv_heads, D, form):
    kv, rows = filled_as(heads, kv_heads, D, dtype, [9000, 1, 4097, 700, 6001])
    chunks = [(0, 8999, 1), (1, 0, 1), (2, 4090, 7), (3, 690, 1)]
    with kv:
        run(kv, rows, chunks, dtype, act, **FORMS[form])
        run(kv, rows, chunks, dtype, act, prefix=[(4, 6001)] * 4, **FORMS[form])


@pytest.mark.parametrize("dtype,act,heads,kv_heads,D", [("bf16", "bf16", 32, 8, 128), ("f16", "f16", 8, 2, 64), ("f32", "f32", 8, 4, 128),
                                                        ("e4m3", "bf16", 28, 4, 128), ("bf16", "f32", 24, 8, 128), ("e4m3", "f16", 16, 16, 64)])
@pytest.mark.parametrize("form", list(FORMS))
def test_prompts(gpu, dtype, act, heads, kv_heads, D, form):
    kv, rows = filled_as(heads, kv_heads, D, dtype, [1200, 515, 130])
    with kv:
        run(kv, rows, [(0, 400, 800), (1, 0, 515), (2, 129, 1)], dtype, act, **FORMS[form])
        run(kv, rows, [(0, 400, 800), (1, 0, 515), (2, 129, 1)], dtype, act, prefix=[(2, 130), (2, 130), (0, 0)], full=[900, 200, 0],
            **FORMS[form])


@pytest.mark.parametrize("dtype,act", TYPES)
@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("n", [1, 9, 70])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_what_no_row_sees_does_not_matter(gpu, odd, n, D, dtype, act):
    """NaN and infinities at positions in front of a document, past a window and behind a row, in the tiles that rows see part
    of; a value of the row's own documents beside them."""
    if dtype == "f16" and odd == math.inf:
        pass  # an infinity is a number of the type
    length, first = 600, 293

    def edit(i, k, v):
        if i == 0:
            for t in (0, 17, 100, 255, 256, 291, 292):
                k[t], v[t] = odd, -odd

    kv, rows = filled_as(8, 2, D, dtype, [length, 40], edit=edit)
    clean = [(k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)) for k, v in rows]
    with kv:
        run(kv, clean, [(0, 400, n), (1, 3, 1)], dtype, act, first=[first, 0])
        run(kv, clean, [(0, 400, n)], dtype, act, window=400 - first + 1 if n == 1 else 100)
        # rows of one chunk of which the early ones see the odd values: the late ones do not
        pos, m, w = 292 - 20, 60, 25
        q = randn(3, m, 8, D, dtype=act)
        out = torch.empty(m, 8 * D, dtype=TORCH[act], device="cuda")
        kv.AttentionFormsDev(0, [0], [pos], [m], q, out, D**-0.5, window=w)
        want, size = forms64(q, clean[0][0][:pos + m], clean[0][1][:pos + m], pos, D**-0.5, 8, 2, window=w)
        blind = torch.tensor([all(not (pos + j - w < t <= pos + j) for t in (255, 256, 291, 292)) for j in range(m)], device="cuda")
        assert blind.any() and not blind.all()
        e = row_errors(out.view(m, 8, D)[blind], want[blind], size[blind])
        assert e <= tol(dtype, act, 0), f"{e:.3g}"
        # ... and a prefix's odd values stay with the rows that see them
        run(kv, clean, [(1, 3, 1), (1, 0, 30)], dtype, act, prefix=[(0, 400)] * 2, first=[first, 300])


@pytest.mark.parametrize("dtype,act", TYPES)
@pytest.mark.parametrize("n", [1, 8, 70])
def test_scales_and_large_scores(gpu, dtype, act, n):
    """Scale zero (the mean of the values), negative scales, scores far beyond the cap."""
    kv, rows = filled_as(8, 2, 64, dtype, [500])
    with kv:
        for scale in (0.0, -0.125, 2.0):
            run(kv, rows, [(0, 400, n)], dtype, act, scale=scale, cap=20.0 if scale == 2.0 else 0.0, qscale=0.5 if act == "f32" else 1.0)
        run(kv, rows, [(0, 400, n)], dtype, act, scale=0.0, cap=10.0, slopes=True)


@pytest.mark.parametrize("dtype", ["e4m3"])
@pytest.mark.parametrize("act", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("n", [1, 40])
def test_rows_of_very_different_scale(gpu, dtype, act, n):
    """K and V rows from 2^-20 to 2^10: every position has its own exponents."""
    def edit(i, k, v):
        by = (2.0 ** (torch.arange(k.shape[0]) * 7 % 31 - 20)).to(k.dtype).cuda()[:, None, None]
        k.mul_(by * 2.0**-10)
        v.mul_(by)

    kv, rows = filled_as(8, 2, 128, dtype, [700], edit=edit)
    with kv:
        run(kv, rows, [(0, 600, n)], dtype, act)


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("e4m3", "bf16"), ("f16", "f32")])
def test_equal_to_the_chunk_call(gpu, dtype, act):
    """With nothing set the call is attention over chunks, null form included."""
    kv, rows = filled_as(8, 2, 128, dtype, LENGTHS)
    chunks = CHUNKS["ragged"]
    with kv:
        got, _ = run(kv, rows, chunks, dtype, act)
        q = randn(7, sum(c[2] for c in chunks), 8, 128, dtype=act, scale=1.5)
        out = torch.empty(q.shape[0], 8 * 128, dtype=TORCH[act], device="cuda")
        kv.AttentionChunksDev(0, [c[0] for c in chunks], [c[1] for c in chunks], [c[2] for c in chunks], q, out, 128**-0.5)
        assert row_errors(out.view_as(got), got.double()) <= 2 * tol(dtype, act, 0)


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("e4m3", "bf16")])
def test_many_chunks_and_one_sequence_in_several(gpu, dtype, act):
    """More chunks than one launch takes; packed documents of one sequence as chunks of their own."""
    kv, rows = filled_as(8, 2, 64, dtype, [900, 300])
    docs = [0, 100, 130, 131, 400, 899]
    with kv:
        chunks = [(0, a, b - a) for a, b in zip(docs, docs[1:] + [900])]
        run(kv, rows, chunks, dtype, act, first=docs)
        many = [(i % 2, (i * 13) % 250, 1 + i % 3) for i in range(150)]
        run(kv, rows, many, dtype, act, prefix=[(0, 600)] * 150, window=700)


@pytest.mark.parametrize("dtype,act,heads,kv_heads,D", [("f32", "f32", 8, 2, 64), ("bf16", "bf16", 32, 8, 128), ("e4m3", "bf16", 32, 8, 128),
                                                        ("f16", "f16", 6, 3, 40)])
def test_two_graphs_of_one_cache(gpu, dtype, act, heads, kv_heads, D):
    """Graphs of a small and a large call share the handle's workspace, which grew between their captures; eager calls run
    between their replays."""
    kv, rows = filled_as(heads, kv_heads, D, dtype, [3000, 600, 2000])
    calls = [([(1, 599, 1)], [(2, 700)]), ([(0, 2900, 100), (1, 500, 100)], [(2, 2000), (2, 2000)])]
    with kv:
        graphs = []
        for chunks, prefix in calls:
            total = sum(c[2] for c in chunks)
            q = randn(total, total, heads, D, dtype=act)
            out = torch.empty(total, heads * D, dtype=TORCH[act], device="cuda")

            def call():
                kv.AttentionFormsDev(0, [c[0] for c in chunks], [c[1] for c in chunks], [c[2] for c in chunks], q, out, D**-0.5, cap=30.0,
                                     window=2500, prefix_ids=[x[0] for x in prefix], prefix_len=[x[1] for x in prefix])

            call()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call()
            graphs.append((g, q, out, chunks, prefix))
        for i in range(4):
            for g, q, out, chunks, prefix in graphs:
                q.copy_(randn(50 + i, *q.shape, dtype=act))
                g.replay()
                torch.cuda.synchronize()
                want, size = expected(rows, chunks, q, D**-0.5, heads, kv_heads, D, prefix=prefix, cap=30.0, window=2500)
                e = row_errors(out.view_as(want), want, size)
                assert e <= tol(dtype, act, 30.0), f"{e:.3g}"
                run(kv, rows, [(0, 2000, 3)], dtype, act)


@pytest.mark.parametrize("dtype,act", TYPES)
@pytest.mark.parametrize("cap", [0.001, 1.0, 30.0, 1e6])
@pytest.mark.parametrize("n", [1, 40, 150])
def test_caps_of_every_size(gpu, dtype, act, cap, n):
    """Scores far below the cap, about it and far beyond, with a mask in the first tile.  (A cap of 0.001 leaves nearly even
    weights, one of a million none but the scores' own.)"""
    kv, rows = filled_as(8, 2, 64, dtype, [400])
    with kv:
        run(kv, rows, [(0, 230, n)], dtype, act, cap=cap, first=[7])


@pytest.mark.parametrize("dtype,act,D", [("f32", "f32", 64), ("f32", "bf16", 128), ("f16", "f16", 128), ("bf16", "bf16", 64), ("e4m3", "bf16", 128),
                                         ("e4m3", "f16", 64), ("bf16", "f32", 24)])
def test_rows_off_vector_alignment_and_another_stream(gpu, dtype, act, D):
    """q and out one element behind a vector boundary, on a stream that is not the current one; the values around out stay."""
    heads, n = 8, 50
    kv, rows = filled_as(heads, 2, D, dtype, [300, 90])
    width = n * heads * D
    q = torch.zeros(width + 8, dtype=TORCH[act], device="cuda")[1:width + 1].view(n, heads * D)
    q.copy_(randn(3, n, heads * D, dtype=act))
    whole = torch.full((width + 8,), 7.0, dtype=TORCH[act], device="cuda")
    out = whole[1:width + 1].view(n, heads * D)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with kv:
        kv.AttentionFormsDev(0, [0, 1, 0], [200, 60, 299], [19, 30, 1], q, out, D**-0.5, window=120, prefix_ids=[1] * 3, prefix_len=[33] * 3, stream=s)
        s.synchronize()
        want, size = expected(rows, [(0, 200, 19), (1, 60, 30), (0, 299, 1)], q.view(n, heads, D), D**-0.5, heads, 2, D, prefix=[(1, 33)] * 3, window=120)
        assert row_errors(out.view(n, heads, D), want, size) <= tol(dtype, act, 0)
        assert (whole[:1] == 7).all() and (whole[width + 1:] == 7).all()


@pytest.mark.parametrize("dtype,act", [("bf16", "bf16"), ("e4m3", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("n", [1, 5, 20, 70])
def test_positions_far_behind_a_long_prefix(gpu, dtype, act, n):
    """Slopes and windows over positions past 2^16, of which the prefix holds most: distances are whole numbers of 32 bits."""
    kv, rows = filled_as(8, 2, 64, dtype, [100, 70000])
    with kv:
        run(kv, rows, [(0, 100 - n, n)] * 2, dtype, act, prefix=[(1, 70000)] * 2, slopes=True)
        run(kv, rows, [(0, 100 - n, n)] * 2, dtype, act, prefix=[(1, 70000)] * 2, window=300, first=[0, 69990])
        run(kv, rows, [(1, 69999 - n, n), (0, 0, n)], dtype, act, prefix=[(1, 500), (1, 69999)], cap=30.0)


@pytest.mark.parametrize("dtype,act", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("e4m3", "bf16"), ("e4m3", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("n", [1, 12, 40])
@pytest.mark.parametrize("mass", [0.9, 0.999])
def test_small_weights_beside_a_large_one(gpu, dtype, act, n, mass):
    """One key takes nearly all of a row's weight and holds no value: the output is what the many small weights leave (2^-15 to
    2^-23 of the largest).  Each weight is rounded relative to itself, so the tolerances are those of the other rows."""
    from tests.test_gpu_chunks_sink import sink_queries, sink_rows

    length, heads, kv_heads, D = 2048, 32, 8, 64
    k, v = sink_rows(D, "bf16" if dtype == "e4m3" else dtype, length, math.log(length * mass / (1 - mass)) + 0.5)
    with qr.PagedKvCache(1, heads, kv_heads, D, length, dtype) as kv:
        kv.AppendNormRopeDev(0, [0], [0], [length], None, k.view(length, -1), v.view(length, -1), None, None, None, 1e-6, 1e4, rotary_dim=0)
        if dtype == "e4m3":
            k, v = e4m3_values(k), e4m3_values(v)
        q = sink_queries(5, n, D, act)
        out = torch.empty(n, heads * D, dtype=TORCH[act], device="cuda")
        kv.AttentionFormsDev(0, [0], [length - n], [n], q, out, D**-0.5)
        want, size = forms64(q.view(n, heads, D), k, v, length - n, D**-0.5, heads, kv_heads)
        e = row_errors(out.view(n, heads, D), want, size)
        assert e <= tol(dtype, act, 0), f"{e:.3g}"


def test_a_serving_step(gpu):
    """The calls as they are used: a prompt's prefix enters an 8-bit cache once, sequences behind it append and attend, each
    position rotated by where it stands behind the prefix; the same as sequences that hold the prefix themselves."""
    heads, kv_heads, D, plen, theta = 8, 2, 64, 300, 1e4
    width = (heads + 2 * kv_heads) * D
    prompt = randn(1, plen, width, dtype="bf16")
    qn, kn = (1 + 0.1 * randn(i, D) for i in (2, 3))
    cut = [heads * D, kv_heads * D, kv_heads * D]

    def append(kv, ids, pos, n, rows, rope):
        q, k, v = rows.split(cut, 1)
        out = torch.empty(sum(n), heads * D, dtype=torch.bfloat16, device="cuda")
        kv.AppendNormRopeDev(0, ids, pos, n, q, k, v, out, qn, kn, 1e-6, theta, rope_pos0=rope)
        return out

    with qr.PagedKvCache(1, heads, kv_heads, D, 512, "e4m3", 4) as shared, qr.PagedKvCache(1, heads, kv_heads, D, 512, "e4m3", 3) as whole:
        append(shared, [3], [0], [plen], prompt, [0])
        for i in range(3):
            append(whole, [i], [0], [plen], prompt, [0])
        at = [0, 0, 0]
        for step, n in enumerate([[40, 1, 7], [1, 1, 1], [3, 0, 5], [1, 1, 1]]):
            new = randn(10 + step, sum(n), width, dtype="bf16")
            q = append(shared, [0, 1, 2], at, n, new, [plen + a for a in at])
            q2 = append(whole, [0, 1, 2], [plen + a for a in at], n, new, None)
            assert torch.equal(q, q2)
            a, b = torch.empty_like(q), torch.empty_like(q)
            shared.AttentionFormsDev(0, [0, 1, 2], at, n, q, a, D**-0.5, cap=30.0, prefix_ids=[3] * 3, prefix_len=[plen] * 3)
            whole.AttentionFormsDev(0, [0, 1, 2], [plen + x for x in at], n, q, b, D**-0.5, cap=30.0)
            # two roundings of the output, two of the weights: each eps / 2
            assert row_errors(a.view(-1, heads, D), b.view(-1, heads, D)) <= 2 * torch.finfo(torch.bfloat16).eps
            at = [x + y for x, y in zip(at, n)]


def test_refusals(gpu):
    kv, _ = filled_as(8, 2, 64, "bf16", [300, 40])
    q = torch.zeros(2, 512, device="cuda")
    out = torch.empty_like(q)
    slopes = torch.zeros(8, device="cuda")

    def call(rows=(2,), pos=(10,), ids=(0,), q=q, out=out, scale=1.0, **k):
        kv.AttentionFormsDev(0, list(ids), list(pos), list(rows), q, out, scale, **k)

    with kv:
        call()
        call(rows=[0], q=q[:0], out=out[:0])
        kv.AttentionFormsDev(0, [], [], [], q[:0], out[:0], 1.0, first=[])
        for bad in (dict(cap=-1.0), dict(cap=math.nan), dict(cap=math.inf), dict(cap=1e-4), dict(cap=2e6), dict(window=-1), dict(first=[-1]), dict(full=[-5]), dict(scale=math.nan),
                    dict(prefix_ids=[2], prefix_len=[5]), dict(prefix_ids=[1], prefix_len=[-1]), dict(ids=[2])):
            with pytest.raises(qr.QrInvalidArgument):
                call(**bad)
        for bad in (dict(prefix_ids=[1], prefix_len=[301]), dict(full=[301]), dict(pos=[299]), dict(prefix_ids=[1], prefix_len=[40], full=[341])):
            with pytest.raises(qr.QrOutOfRange):
                call(**bad)
        for bad in (dict(prefix_ids=[1], prefix_len=[257]), dict(ids=[1], pos=[1], full=[257])):
            with pytest.raises(qr.QrNotResident):
                call(**bad)
        for bad in (dict(slopes=slopes[:4]), dict(slopes=slopes.half()), dict(slopes=slopes.cpu()), dict(first=[0, 0]), dict(full=[1.5]),
                    dict(prefix_ids=[1]), dict(out=q), dict(q=q.double()), dict(out=out.half()), dict(q=q[:1]),
                    dict(slopes=out.view(-1)[:8])):
            with pytest.raises(ValueError):
                call(**bad)


@pytest.mark.parametrize("dtype,act,D", [("bf16", "bf16", 128), ("f16", "f16", 64), ("f16", "f32", 128), ("bf16", "f32", 64), ("f32", "f32", 64),
                                         ("f32", "f32", 128), ("f32", "bf16", 96), ("bf16", "bf16", 20)])
@pytest.mark.parametrize("n", [1, 12, 25, 70])
@pytest.mark.parametrize("seqs", [1, 24])  # the keys split over many workgroups, and not
@pytest.mark.parametrize("at", [3, 2100])  # before and behind the keys of large weight
@pytest.mark.parametrize("form", ["plain", "cap", "prefix"])
def test_infinite_values_of_little_weight(gpu, form, dtype, act, D, n, seqs, at):
    """A weight of e^-190 is zero in 32 bits, but none in the formula: a row that sees an infinite V shows that infinity
    whatever its weight (a cap of 1e5 leaves the scores as they are to 1e-6 of them), and NaN where it sees both or a NaN."""
    heads, kv_heads, length = 8, 2, 2500
    if D == 20 and seqs > 1:
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
    front = 2200 if form == "prefix" else 0
    own = length - front
    with qr.PagedKvCache(1, heads, kv_heads, D, length, dtype, seqs + 1) as kv:
        if front:
            kv.AppendRangeDev(0, 0, k[:front].reshape(front, -1), v[:front].reshape(front, -1), dtype, seq_id=seqs)
        for s in range(seqs):
            kv.AppendRangeDev(0, 0, k[front:].reshape(own, -1), v[front:].reshape(own, -1), dtype, seq_id=s)
        more = dict(prefix_ids=[seqs] * seqs, prefix_len=[front] * seqs) if front else dict(cap=1e5) if form == "cap" else {}
        kv.AttentionFormsDev(0, list(range(seqs)), [own - n] * seqs, [n] * seqs, q, out, D**-0.5, **more)
    for s in (0, seqs - 1):
        got = out[s * n:(s + 1) * n].double()
        assert (got[:, :4, 1] == inf).all() and got[:, :4, 3].isnan().all()
        assert (got[:, 4:, D - 1] == inf).all() and got[:, 4:, 2].isnan().all() and (got[:, 4:, 3] == inf).all()
        want, size = forms64(q[s * n:(s + 1) * n], k, torch.where(v.isfinite(), v, 0), length - n, D**-0.5, heads, kv_heads, cap=more.get("cap", 0.0))
        for x in (got, want):
            for h, d in ((slice(0, 4), 1), (slice(0, 4), 3), (slice(4, 8), D - 1), (slice(4, 8), 2), (slice(4, 8), 3)):
                x[:, h, d] = 0
        e = row_errors(got, want, size)
        assert e <= tol(dtype, act, more.get("cap", 0.0)), f"out: {e:.3g}"


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_slopes_over_far_positions(gpu, dtype):
    """Distances of rows past position 2^24, where fp32 has no odd numbers, are exact: the slope's differences between
    neighbouring keys are the formula's."""
    heads, kv_heads, D, base, n = 2, 1, 64, 2**24 + 129, 40
    with qr.PagedKvCache(1, heads, kv_heads, D, 2**24 + 512, dtype, 1) as kv:
        k, v = (randn(s, n, kv_heads, D, dtype=dtype) for s in (1, 2))
        kv.AppendNormRopeDev(0, [0], [base], [n], None, k.view(n, -1), v.view(n, -1), None, None, None, 1e-6, 1e4, rotary_dim=0)
        for m in (1, n):
            q = randn(3, m, heads, D, dtype=dtype)
            out = torch.empty_like(q)
            slopes = torch.tensor([2.0, 0.5], device="cuda")
            kv.AttentionFormsDev(0, [0], [base + n - m], [m], q, out, D**-0.5, slopes=slopes, first=[base])
            want, size = forms64(q, k, v, n - m, D**-0.5, heads, kv_heads, slopes=slopes)
            e = row_errors(out, want, size)
            assert e <= tol(dtype, dtype, 0), f"{e:.3g}"


@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 96), (28, 4, 96), (8, 2, 256), (16, 1, 256), (3, 3, 256), (5, 2, 256), (40, 2, 96)])
@pytest.mark.parametrize("dtype,act", TYPES)
def test_wide_and_odd_heads(gpu, dtype, act, heads, kv_heads, D):
    """Head sizes whose rows lie in order in the page: every form, single tokens, blocks of several row tiles, a prefix."""
    kv, rows = filled_as(heads, kv_heads, D, dtype, LENGTHS)
    with kv:
        for name in CHUNKS:
            for form in FORMS:
                run(kv, rows, CHUNKS[name], dtype, act, **FORMS[form])
        run(kv, rows, [(0, 7, 1), (1, 300, 1), (2, 255, 2)], dtype, act, prefix=[(4, 777)] * 3, window=600, cap=20.0)
        run(kv, rows, [(4, 900, 101), (3, 100, 3)], dtype, act, prefix=[(1, 257), (0, 0)], first=[300, 101], full=[1200, 0], slopes=True)


@pytest.mark.parametrize("D", [96, 256])
@pytest.mark.parametrize("dtype,act", TYPES)
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_what_no_row_sees_does_not_matter_in_wide_heads(gpu, odd, dtype, act, D):
    def edit(i, k, v):
        for t in (0, 100, 255, 256, 291, 292):
            k[t], v[t] = odd, -odd

    kv, rows = filled_as(8, 2, D, dtype, [600], edit=edit)
    clean = [(k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)) for k, v in rows]
    with kv:
        for n in (1, 9, 70):
            run(kv, clean, [(0, 400, n)], dtype, act, first=[293])
            run(kv, clean, [(0, 400, n)], dtype, act, window=108 if n == 1 else 50)
