"""GPU tests of attention in its other forms at head sizes, head counts and lengths beside those of test_gpu_forms.py, against the
definition in 64 bits (tolerances there)."""
import ctypes
import math

import pytest
import torch

from qauntrunner_amd import _lib
from tests.chunkutil import TORCH, randn, row_errors
from tests.formutil import filled_as
from tests.test_gpu_forms import CHUNKS, FORMS, LENGTHS, TYPES, expected, run, slopes_of, tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("heads,kv_heads,D", [(3, 3, 1), (5, 1, 3), (3, 1, 33), (7, 7, 5)])
def test_odd_numbers_of_odd_partials(gpu, dtype, act, heads, kv_heads, D):
    """The keys split into as many parts as leave an odd number of values in front of the parts' sums."""
    kv, rows = filled_as(heads, kv_heads, D, dtype, [5000, 1001, 20000])
    with kv:
        for chunks in ([(0, 4999, 1)], [(0, 4997, 3)], [(2, 19999, 1)], [(0, 4998, 1), (1, 998, 3)]):
            run(kv, rows, chunks, dtype, act)
            run(kv, rows, chunks, dtype, act, prefix=[(1, 333)] * len(chunks), **FORMS["all"])


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("e4m3", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 96), (16, 1, 256), (6, 2, 160), (4, 2, 192), (5, 2, 96)])
@pytest.mark.parametrize("form", ["plain", "all", "window"])
def test_long_contexts_of_wide_heads(gpu, dtype, act, heads, kv_heads, D, form):
    kv, rows = filled_as(heads, kv_heads, D, dtype, [9000, 1, 4097, 700, 3001])
    chunks = [(0, 8999, 1), (1, 0, 1), (2, 4090, 7), (3, 660, 40)]
    with kv:
        run(kv, rows, chunks, dtype, act, **FORMS[form])
        run(kv, rows, chunks, dtype, act, prefix=[(4, 3001)] * 4, **FORMS[form])


@pytest.mark.parametrize("dtype,act", TYPES)
@pytest.mark.parametrize("heads,kv_heads,D", [(6, 2, 160), (8, 8, 192), (7, 3, 192)])
def test_head_sizes_of_the_plain_kernel(gpu, dtype, act, heads, kv_heads, D):
    kv, rows = filled_as(heads, kv_heads, D, dtype, LENGTHS)
    with kv:
        for name in CHUNKS:
            for form in ("plain", "all"):
                run(kv, rows, CHUNKS[name], dtype, act, **FORMS[form])


@pytest.mark.parametrize("dtype,act", TYPES)
@pytest.mark.parametrize("D", [96, 256, 160])
@pytest.mark.parametrize("cap", [0.001, 1.0, 30.0, 1e6])
def test_caps_of_every_size_in_wide_heads(gpu, dtype, act, D, cap):
    kv, rows = filled_as(8, 2, D, dtype, [400])
    with kv:
        for n in (1, 40, 150):
            run(kv, rows, [(0, 230, n)], dtype, act, cap=cap, first=[7])


@pytest.mark.parametrize("dtype,act,heads,kv_heads,D,big", [("bf16", "bf16", 8, 2, 96, 100), ("e4m3", "bf16", 8, 2, 256, 100), ("f32", "f32", 16, 1, 96, 100),
                                                            ("f16", "f32", 6, 2, 160, 100), ("bf16", "bf16", 64, 8, 128, 1100)])
def test_graphs_of_wide_heads_and_of_several_launches(gpu, dtype, act, heads, kv_heads, D, big):
    """Two graphs that share the handle's workspace, replayed with eager calls between; the slopes change between replays.  (2200 rows
    of 64 heads of 128 behind a prefix are two launches.)"""
    kv, rows = filled_as(heads, kv_heads, D, dtype, [3000, 1200, 700])
    calls = [([(1, 599, 1)], [(2, 700)]), ([(0, 2900 - big, big), (1, 1200 - big, big)], [(2, 700), (2, 700)])]
    with kv:
        graphs = []
        for chunks, prefix in calls:
            total = sum(c[2] for c in chunks)
            q, slopes = randn(total, total, heads, D, dtype=act), slopes_of(heads)
            out = torch.empty(total, heads * D, dtype=TORCH[act], device="cuda")

            def call():
                kv.AttentionFormsDev(0, [c[0] for c in chunks], [c[1] for c in chunks], [c[2] for c in chunks], q, out, D**-0.5, cap=30.0, slopes=slopes,
                                     window=2500, prefix_ids=[x[0] for x in prefix], prefix_len=[x[1] for x in prefix])

            call()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call()
            graphs.append((g, q, slopes, out, chunks, prefix))
        for i in range(4):
            for g, q, slopes, out, chunks, prefix in graphs:
                q.copy_(randn(50 + i, *q.shape, dtype=act))
                slopes.copy_(slopes_of(heads) * 2.0**-i)
                g.replay()
                torch.cuda.synchronize()
                want, size = expected(rows, chunks, q, D**-0.5, heads, kv_heads, D, prefix=prefix, cap=30.0, window=2500, slopes=slopes)
                e = row_errors(out.view_as(want), want, size)
                assert e <= tol(dtype, act, 30.0), f"{e:.3g}"
                run(kv, rows, [(0, 1800, 3)], dtype, act)


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 128), (28, 4, 64), (4, 2, 96), (5, 2, 40)])
@pytest.mark.parametrize("name", list(CHUNKS))
def test_chunk_call_on_8_bits(gpu, name, heads, kv_heads, D, act):
    """AttentionChunksDev on an 8-bit cache against the definition."""
    kv, rows = filled_as(heads, kv_heads, D, "e4m3", LENGTHS)
    chunks = CHUNKS[name]
    q = randn(7, sum(c[2] for c in chunks), heads, D, dtype=act, scale=1.5)
    out = torch.full((q.shape[0], heads * D), 7.0, dtype=TORCH[act], device="cuda")
    with kv:
        kv.AttentionChunksDev(0, [c[0] for c in chunks], [c[1] for c in chunks], [c[2] for c in chunks], q, out, D**-0.5)
        want, size = expected(rows, chunks, q, D**-0.5, heads, kv_heads, D)
        e = row_errors(out.view_as(want), want, size)
        assert e <= tol("e4m3", act, 0), f"{e:.3g}"


@pytest.mark.parametrize("dtype,act", TYPES)
def test_no_form_at_the_c_entry(gpu, dtype, act):
    """A null form is plain causal attention."""
    heads, kv_heads, D, n = 8, 2, 128, 60
    kv, rows = filled_as(heads, kv_heads, D, dtype, [300])
    q = randn(7, n, heads, D, dtype=act)
    out = torch.full((n, heads * D), 7.0, dtype=TORCH[act], device="cuda")
    one = lambda x: (ctypes.c_int * 1)(x)  # noqa: E731
    with kv:
        _lib.check(kv._lib.qr_kv_attention_forms_dev(kv._h, 1, one(0), 0, one(240), one(n), q.data_ptr(), _lib.DTYPES[act], out.data_ptr(), D**-0.5, None,
                                                     torch.cuda.current_stream().cuda_stream))
        want, size = expected(rows, [(0, 240, n)], q, D**-0.5, heads, kv_heads, D)
        assert row_errors(out.view_as(want), want, size) <= tol(dtype, act, 0)


@pytest.mark.parametrize("dtype,act", TYPES)
@pytest.mark.parametrize("D", [64, 128, 96, 40])
@pytest.mark.parametrize("n", [1, 12, 40, 150])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_queries_that_are_no_numbers_stay_with_their_rows(gpu, odd, n, D, dtype, act):
    """The row itself is the formula's: no number, or finite where a cap makes its infinite scores so (no number there where queries
    enter in parts)."""
    parts = dtype != "f32" and D in (64, 128) and act != ("f16" if dtype == "f16" else "bf16")
    heads = 8
    kv, rows = filled_as(heads, 2, D, dtype, [700, 300])
    q = randn(3, n, heads, D, dtype=act)
    q[n // 2, 1, 3] = odd
    others = torch.ones(n, heads, dtype=torch.bool, device="cuda")
    others[n // 2, 1] = False
    with kv:
        for form in (dict(), dict(cap=30.0), dict(window=90, slopes=slopes_of(heads)), dict(prefix=[(1, 300)])):
            out = torch.empty(n, heads, D, dtype=TORCH[act], device="cuda")
            prefix = form.pop("prefix", None)
            more = dict(prefix_ids=[1], prefix_len=[300]) if prefix else {}
            kv.AttentionFormsDev(0, [0], [700 - n], [n], q, out, D**-0.5, **form, **more)
            want, size = expected(rows, [(0, 700 - n, n)], q, D**-0.5, heads, 2, D, prefix=prefix, **form)
            # the row itself, from all that it sees
            k, v = (torch.cat([rows[1][j][:300 if prefix else 0], rows[0][j][:700 - n + n // 2 + 1]])[-form.get("window", 0):, 0].double() for j in (0, 1))
            z = D**-0.5 * (q[n // 2, 1].double() @ k.t().contiguous())
            z = 30 * torch.tanh(z / 30) if "cap" in form else z
            if "slopes" in form:
                z = z - form["slopes"][1] * torch.arange(len(k) - 1, -1, -1, device="cuda")
            w = torch.softmax(z, 0)
            row, its = out[n // 2, 1].double(), w @ v
            size_of = (w.square() @ v.square().sum(1)).sqrt()
            if parts and odd == math.inf and "cap" in form:
                its = row * math.nan
            assert row.isnan().all() if its.isnan().any() else (row - its).norm() <= tol(dtype, act, 30) * torch.maximum(its.norm(), size_of), form
            e = row_errors(out[others], want[others], size[others])
            assert e <= tol(dtype, act, form.get("cap", 0)), f"{form}: {e:.3g}"


@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("D", [64, 128, 96, 40])
@pytest.mark.parametrize("n", [1, 12, 40, 150])
@pytest.mark.parametrize("cap", [0.0, 30.0, 1e3])
def test_infinite_keys(gpu, cap, n, D, dtype, act):
    """A key with an infinite value scores an infinity of the query's sign there: none of the weight, or all of it, which is no number
    (infinity less itself); plus or minus the cap with one."""
    heads = 8

    def edit(i, k, v):
        k[520, :, 3] = math.inf

    kv, rows = filled_as(heads, 2, D, dtype, [700], edit=edit)
    q = randn(3, n, heads, D, dtype=act)
    with kv:
        out = torch.empty(n, heads, D, dtype=TORCH[act], device="cuda")
        kv.AttentionFormsDev(0, [0], [700 - n], [n], q, out, D**-0.5, cap=cap)
    want, size = expected(rows, [(0, 700 - n, n)], q, D**-0.5, heads, 2, D, cap=cap)
    none = (q[:, :, 3] > 0) & (cap == 0)
    assert out[none].isnan().all() and not out[~none].isnan().any()
    assert row_errors(out[~none], want[~none], size[~none]) <= tol(dtype, act, cap)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("kv_heads,D", [(1, 1), (3, 33), (8, 128), (2, 96), (1, 512), (5, 64), (2, 256)])
def test_rows_read_as_every_type(gpu, dtype, kv_heads, D):
    """Several chunks, from inside a page and over its end, of every cache as every type: the value rounded once."""
    lengths = [300, 1, 700]
    kv, rows = filled_as(kv_heads, kv_heads, D, dtype, lengths)
    chunks = [(2, 250, 300), (0, 299, 1), (1, 0, 0), (2, 0, 3), (1, 0, 1), (0, 5, 252)]
    want = [torch.cat([rows[s][j][p:p + n] for s, p, n in chunks]) for j in (0, 1)]
    total = sum(c[2] for c in chunks)
    with kv:
        for act in ("f32", "f16", "bf16"):
            got = [torch.full((total + 1, kv.KvDim), 7.0, dtype=TORCH[act], device="cuda") for _ in (0, 1)]
            kv.ReadAsDev(0, [c[0] for c in chunks], [c[1] for c in chunks], [c[2] for c in chunks], *(x[:total] for x in got))
            for x, w in zip(got, want):
                assert torch.equal(x[:total].view_as(w), w.float().to(TORCH[act])) and (x[total] == 7).all()
