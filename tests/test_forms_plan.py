"""Host-side plans of attention in its other forms (CPU only): the workspace's bound and its layout, and what is launched."""
import ctypes
import os

import pytest

from qauntrunner_amd import _lib
from tests.hosthip import run
from tests.test_chunks_plan import BATCH, MB, Geom

_i, _sz = ctypes.c_int, ctypes.c_size_t


class Chunk(ctypes.Structure):  # FormChunk
    _fields_ = [(f, _i) for f in ("pt_off", "pre_off", "pre_len", "pos0", "rows", "row0", "first", "full")]


class Args(ctypes.Structure):  # FormsArgs
    _fields_ = [("c", Chunk * BATCH), ("n", _i), ("rows", _i), ("pool", ctypes.c_void_p), ("page_table", ctypes.c_void_p), ("geom", Geom),
                ("dtype", _i), ("act", _i), ("heads", _i), ("q", ctypes.c_void_p), ("out", ctypes.c_void_p), ("scale", ctypes.c_float),
                ("cap", ctypes.c_float), ("slopes", ctypes.c_void_p), ("window", _i)]


class Rows(ctypes.Structure):  # FormRows
    _fields_ = [(f, _i) for f in ("row0", "rows", "p0", "first", "full", "parts")] + [("slot0", ctypes.c_longlong)]


class Item(ctypes.Structure):  # FormItem
    _fields_ = [(f, _i) for f in ("pt_off", "c0", "nc", "row0", "rows", "base", "keys", "unit0", "blocks", "splits", "per", "part0", "kind")]


class Plan(ctypes.Structure):  # FormsPlan
    _fields_ = [("it", Item * (2 * BATCH)), ("us", ctypes.c_float * (2 * BATCH)), ("n", _i), ("c", Rows * BATCH), ("part_ml", _sz),
                ("workspace_bytes", _sz), ("merge", ctypes.c_bool)]


DTYPES = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 16}


def plan(dtype, heads, kv_heads, D, chunks, act=2, window=0, cap=0.0):
    """chunks: (pos0, rows, prefix length, first visible position, prefix)"""
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    f = ctypes.CDLL(_lib.LIB_PATH)._ZN2qr10plan_formsERKNS_9FormsArgsE
    f.restype, f.argtypes = Plan, [ctypes.POINTER(Args)]
    a = Args()
    tiles = dtype != "f32" and D in (64, 128)
    a.geom.planes, a.geom.kv_heads, a.geom.head_dim, a.geom.mfma = 2, kv_heads, D, tiles | (2 if dtype == "e4m3" else 0)
    a.dtype, a.act, a.heads, a.n, a.window, a.cap, a.scale = DTYPES[dtype], act, heads, len(chunks), window, cap, 1.0
    for i, (pos0, rows, pre, first, of) in enumerate(chunks):
        c = a.c[i]
        c.pt_off, c.pre_off, c.pre_len, c.pos0, c.rows, c.row0, c.first = i, 1000 + of, pre, pos0, rows, a.rows, first
        a.rows += rows
    return f(ctypes.byref(a))


BOUND = """
FORMS = lambda kv, n, rows, pre, D: L.qr_kv_attention_forms_dev(kv._h, n, ints(*range(n)), 0, ints(*[0] * n), ints(*[rows] * n), ROWS, 2, ROWS, 1.0,
    ctypes.byref(_lib.AttnForm(0.0, None, 0, None, None, ctypes.cast(ints(*[n] * n), ctypes.c_void_p), ctypes.cast(ints(*[pre] * n), ctypes.c_void_p))), None)
for dtype, heads, kv_heads, D, n, rows, pre in (("bf16", 32, 8, 128, 64, 1000, 2048), ("e4m3", 64, 8, 128, 64, 500, 300), ("bf16", 64, 8, 128, 1, 16384, 5),
                                                ("f32", 28, 4, 128, 3, 5001, 1), ("bf16", 5, 2, 40, 7, 9000, 700), ("e4m3", 32, 8, 128, 64, 8, 65536)):
    kv = PagedKvCache(1, heads, kv_heads, D, max(rows, pre), dtype, n + 1)
    assert append(kv, list(range(n + 1)), [0] * (n + 1), [rows] * n + [pre]) == 0, L.qr_last_error()
    before = live.value
    assert FORMS(kv, n, rows, pre, D) == 0, L.qr_last_error()
    # (a buffer grows by doubling, so a launch that needs more than the last may leave up to twice what it needs)
    assert live.value - before <= 2 * (256 << 20), (dtype, heads, D, n, rows, (live.value - before) / 2**20)
    kv.close()
"""


def test_rows_behind_a_prefix_run_in_a_bounded_workspace(tmp_path):
    """Two partials of every row behind a prefix pass any bound with the rows of a call: more launches then."""
    run(tmp_path, BOUND)


def test_rows_that_see_no_prefix_are_not_counted(tmp_path):
    """Behind a window they leave no second partial: one launch, as without a prefix (a merge beside it where keys are split)."""
    run(tmp_path, """
kv = PagedKvCache(1, 64, 8, 128, 4096, "bf16", 5)
assert append(kv, list(range(5)), [0] * 5, [4096] * 5) == 0, L.qr_last_error()
def launched(window, pre, n=4, rows=1000):
    before = launches.value
    form = _lib.AttnForm(0.0, None, window, None, None, ctypes.cast(ints(*[4] * n), ctypes.c_void_p), ctypes.cast(ints(*[pre] * n), ctypes.c_void_p))
    assert L.qr_kv_attention_forms_dev(kv._h, n, ints(*range(n)), 0, ints(*[3000] * n), ints(*[rows] * n), ROWS, 2, ROWS, 1.0, ctypes.byref(form), None) == 0
    return launches.value - before
assert launched(3001, 2048) == launched(3001, 0) <= 2
assert launched(3002, 2048) == 4  # the first rows see the prefix's last position: two launches and their merges
""")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("heads,kv_heads,D", [(32, 8, 128), (64, 8, 64), (28, 4, 128), (16, 1, 256), (5, 2, 40)])
def test_partials_of_a_launch_are_bounded(dtype, heads, kv_heads, D):
    """As many rows behind prefixes as a launch takes, long contexts of chunks without one, and both."""
    most = 128 * MB // (2 * (4 * D + 8) * heads)
    for n in (1, 7, 64):
        for lens in ((100, 1), (16384, 2000), (1000000, 5)):
            chunks = [(lens[1], most // n, lens[0], 0, i % 2) for i in range(n)]
            assert plan(dtype, heads, kv_heads, D, chunks).workspace_bytes <= 256 * MB
            assert plan(dtype, heads, kv_heads, D, chunks[:n // 2] + [(lens[0], 16, 0, 0, 0)] * (n - n // 2)).workspace_bytes <= 256 * MB
    assert plan(dtype, 200000, 1, 512, [(0, 1, 5, 0, 0)]).workspace_bytes == 2 * 200000 * (4 * 512 + 8)  # (one row's own)


def test_the_partials_sums_are_aligned():
    """(maximum, sum) pairs stand behind partials of D floats each: aligned for any number of them and any head size."""
    odd = 0
    for heads, kv_heads, D in ((3, 3, 1), (5, 1, 3), (3, 1, 33), (7, 7, 5), (32, 8, 128)):
        for keys in (100, 1000, 5000, 20000, 100000):
            for rows in (1, 2, 3):
                p = plan("f32", heads, kv_heads, D, [(keys, rows, 0, 0, 0)], act=0)
                parts = rows * heads * p.c[0].parts if p.merge else 0
                odd += parts * D % 2
                assert p.part_ml % 16 == 0 and p.part_ml >= parts * D * 4, (heads, D, keys, rows, p.part_ml)
                assert p.workspace_bytes == p.part_ml + 8 * parts
    assert odd


def test_positions_past_2_30_are_refused(tmp_path):
    """Slots are counted in 32 bits up to the tile behind the last one, so both attention calls of an 8-bit cache end at 2^30 (seen
    before whether the position is there)."""
    run(tmp_path, """
kv = PagedKvCache(1, 1, 1, 1, 2**31 - 1, "e4m3", 1)
assert append(kv, [0], [0], [1]) == 0, L.qr_last_error()
before = launches.value
for p, n in ((2**30, 1), (2**31 - 2, 1), (2**30 - 5, 6)):
    assert attend(kv, [0], [p], [n], weights=False) == _lib.QR_ERR_OUT_OF_RANGE, (p, L.qr_last_error())
    assert L.qr_kv_attention_forms_dev(kv._h, 1, ints(0), 0, ints(p), ints(n), ROWS, 0, ROWS, 1.0, None, None) == _lib.QR_ERR_OUT_OF_RANGE
full = _lib.AttnForm(0.0, None, 0, None, ctypes.cast(ints(2**30 + 1), ctypes.c_void_p), None, None)
assert L.qr_kv_attention_forms_dev(kv._h, 1, ints(0), 0, ints(0), ints(1), ROWS, 0, ROWS, 1.0, ctypes.byref(full), None) == _lib.QR_ERR_OUT_OF_RANGE
assert attend(kv, [0], [2**30 - 5], [5], weights=False) == _lib.QR_ERR_NOT_RESIDENT
assert attend(kv, [0], [2**30], [0], weights=False) == 0 and launches.value == before
assert attend(kv, [0], [0], [1], weights=False) == 0, L.qr_last_error()
""")


def test_a_prefix_that_no_row_sees_takes_no_part():
    """Windows and first positions behind the whole prefix: the chunk has its own keys alone, and writes its output without partials
    where these are one part.  Chunks that see it share it beside others that do not."""
    far, near = (2000, 5, 2048, 0, 0), (100, 5, 2048, 0, 0)
    p = plan("bf16", 32, 8, 128, [far] * 3, window=500)
    assert p.n == 3 and [p.it[i].nc for i in range(3)] == [1] * 3 and [p.it[i].base for i in range(3)] == [2048] * 3
    assert [p.c[i].p0 for i in range(3)] == [4048] * 3
    lone = plan("bf16", 32, 8, 128, [(30, 5, 64, 64, 0)])
    assert lone.n == 1 and lone.c[0].parts == 1 and not lone.merge and lone.workspace_bytes == 0
    p = plan("bf16", 32, 8, 128, [near, far, near, near], window=500)
    assert [(p.it[i].c0, p.it[i].nc, p.it[i].base) for i in range(p.n)] == [(0, 1, 0), (2, 2, 0)] + [(i, 1, 2048) for i in range(4)]
    # the first row of a chunk sees the prefix's last position; one further, none does
    assert plan("bf16", 32, 8, 128, [(499, 9, 2048, 0, 0)], window=501).n == 2 and plan("bf16", 32, 8, 128, [(499, 9, 2048, 0, 0)], window=500).n == 1
    assert plan("bf16", 32, 8, 128, [(0, 1, 300, 299, 0)]).n == 2 and plan("bf16", 32, 8, 128, [(0, 1, 300, 300, 0)]).n == 1
