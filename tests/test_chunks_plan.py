"""Host-side plans of attention over chunks of several sequences: the workspace stays bounded (CPU only)."""
import ctypes
import os

import pytest

from qauntrunner_amd import _lib
from tests.hosthip import run

BATCH = 64
MB = 1 << 20


class Geom(ctypes.Structure):  # PageGeom
    _fields_ = [("planes", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int), ("mfma", ctypes.c_int)]


class Item(ctypes.Structure):  # ChunkItem
    _fields_ = [(f, ctypes.c_int) for f in ("pt_off", "seq", "pos0", "rows", "row0", "unit0", "blocks", "splits", "slot0", "per", "parts")] + \
               [("score0", ctypes.c_longlong)]


class Args(ctypes.Structure):  # ChunksArgs
    _fields_ = [("it", Item * BATCH), ("n", ctypes.c_int), ("rows", ctypes.c_int), ("pool", ctypes.c_void_p), ("page_table", ctypes.c_void_p),
                ("geom", Geom), ("dtype", ctypes.c_int), ("act", ctypes.c_int), ("heads", ctypes.c_int), ("q", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("weights", ctypes.c_void_p), ("max_seq", ctypes.c_int), ("scale", ctypes.c_float)]


class PlanItem(ctypes.Structure):  # ChunkPlanItem
    _fields_ = [(f, ctypes.c_int) for f in ("kind", "blocks", "splits", "per")] + [("slot0", ctypes.c_longlong)] + \
               [(f, ctypes.c_int) for f in ("wkind", "wblocks", "wper", "wparts")] + [("wslot0", ctypes.c_longlong), ("score0", ctypes.c_longlong)]


class Plan(ctypes.Structure):  # ChunksPlan
    _fields_ = [("it", PlanItem * BATCH), ("wmerge", ctypes.c_bool)] + \
               [(f, ctypes.c_size_t) for f in ("part_ml", "row_ml", "row_scale", "scores", "wpart", "workspace_bytes")]


def plan(dtype, act, heads, kv_heads, D, chunks, weights=True):
    """chunks: (pos0, rows)"""
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    f = ctypes.CDLL(_lib.LIB_PATH)._ZN2qr11plan_chunksERKNS_10ChunksArgsE
    f.restype, f.argtypes = Plan, [ctypes.POINTER(Args)]
    a = Args()
    a.geom.planes, a.geom.kv_heads, a.geom.head_dim, a.geom.mfma = 2, kv_heads, D, dtype != 0 and D in (64, 128)
    a.dtype, a.act, a.heads, a.n = dtype, act, heads, len(chunks)
    a.weights = 256 if weights else None
    for i, (p, n) in enumerate(chunks):
        a.it[i].pos0, a.it[i].rows, a.it[i].row0 = p, n, a.rows
        a.rows += n
    return f(ctypes.byref(a))


SHAPES = [(8, 2, 64), (32, 8, 128), (28, 4, 128), (64, 8, 128), (24, 8, 96), (16, 16, 256), (16, 1, 64)]


@pytest.mark.parametrize("dtype,act", [(0, 0), (1, 1), (2, 2), (1, 0), (2, 0)])
@pytest.mark.parametrize("heads,kv_heads,D", SHAPES)
def test_kept_scores_are_bounded(dtype, act, heads, kv_heads, D):
    """Whatever the chunks' rows and lengths: at most 256 MB of scores, in whole runs of the chunks that keep them."""
    for n in (1, 16, 64):
        for rows in (1, 2, 8, 32):
            for pos0 in (0, 4000, 32767 - rows, 131072, 1000000):
                p = plan(dtype, act, heads, kv_heads, D, [(pos0, rows)] * n)
                at = 0
                for i in range(n):
                    if p.it[i].score0 >= 0:
                        assert p.it[i].score0 == at
                        at += rows * heads * (pos0 + rows + 7 & ~7)
                assert at * 4 <= 256 * MB
                assert p.wpart - p.scores >= at * 4


def test_a_decode_batch_keeps_its_scores():
    """A full launch of single tokens of 32 heads up to 32768 positions."""
    p = plan(1, 1, 32, 8, 128, [(32767, 1)] * 64)
    assert all(x.score0 >= 0 for x in p.it)


def test_long_batches_run_in_a_bounded_workspace(tmp_path):
    out = run(tmp_path, """
n = 64
kv = PagedKvCache(1, 32, 8, 64, 16384, "f16", n)
assert append(kv, range(n), [0] * n, [16384] * n) == 0
before = live.value
assert attend(kv, range(n), [16384 - 8] * n, [8] * n) == 0
print((live.value - before) >> 20)
""")
    assert int(out) < 512
