"""CPU tests of 8-bit caches and of attention in its other forms: what is refused before the library or the GPU is reached,
null handles and arguments at the C entries, and the host code on host memory (tests/hosthip.py)."""
import ctypes

import pytest
import torch

import qauntrunner_amd as qr
from qauntrunner_amd import _lib
from tests.hosthip import run
from tests.test_chunk_calls import NULL, kv, rows  # noqa: F401


def test_null_handles():
    L = _lib.load()
    bad = _lib.QR_ERR_INVALID_ARGUMENT
    assert L.qr_kv_attention_forms_dev(NULL, 0, NULL, 0, NULL, NULL, NULL, 0, NULL, 1.0, NULL, NULL) == bad
    assert b"null" in L.qr_last_error()
    assert L.qr_kv_read_as_dev(NULL, 0, NULL, 0, NULL, NULL, 0, NULL, NULL, NULL) == bad


def test_lists_must_agree(kv):  # noqa: F811
    q, out = rows(2, 64), rows(2, 64)
    for bad in (dict(first=[0]), dict(full=[0, 0, 0]), dict(prefix_ids=[0], prefix_len=[1, 1]), dict(prefix_ids=[0, 0]), dict(prefix_len=[0, 0]),
                dict(first=[0.5, 0]), dict(full=[1 << 40, 0])):
        with pytest.raises(ValueError):
            kv.AttentionFormsDev(0, [0, 1], [0, 0], [1, 1], q, out, 1.0, **bad)


def test_tensors_are_checked(kv):  # noqa: F811
    good = dict(q=rows(2, 64), out=rows(2, 64))
    for bad in (dict(q=rows(1, 64)), dict(out=rows(2, 32)), dict(out=rows(2, 64, torch.float16)), dict(q=rows(2, 64, dev=1)),
                dict(q=rows(2, 64, torch.float64)), dict(slopes=rows(1, 3)), dict(slopes=rows(1, 4, torch.float16)), dict(slopes=torch.zeros(4)),
                dict(out=good["q"])):
        with pytest.raises(ValueError):
            kv.AttentionFormsDev(0, [0, 1], [0, 0], [1, 1], scale=1.0, **{**good, **bad})
    for k, v in ((rows(2, 32), rows(2, 32, torch.float16)), (rows(1, 32), rows(2, 32)), (rows(2, 32, torch.float64),) * 2):
        with pytest.raises(ValueError):
            kv.ReadAsDev(0, [0, 1], [0, 0], [1, 1], k, v)


def test_an_8_bit_cache_is_read_as_values(kv):  # noqa: F811
    kv.KvDtype = _lib.DTYPE_E4M3
    with pytest.raises(ValueError, match="ReadAsDev"):
        kv.ReadDev(0, [0], [0], [1], rows(1, 32), rows(1, 32))


HEAD = """
kv = PagedKvCache(2, 8, 2, 64, 600, "e4m3", 3)
def forms(seqs=(0,), pos0=(0,), rows=(1,), q=ROWS, out=ROWS, act=_lib.DTYPE_F32, scale=1.0, layer=0, **f):
    arrays = {k: ints(*f[k]) if k in f else None for k in ("first", "full", "prefix_ids", "prefix_len")}
    form = _lib.AttnForm(f.get("cap", 0.0), f.get("slopes"), f.get("window", 0), *(ctypes.cast(a, ctypes.c_void_p) if a else None for a in arrays.values()))
    return L.qr_kv_attention_forms_dev(kv._h, len(seqs), ints(*seqs), layer, ints(*pos0), ints(*rows), q, act, out, scale, ctypes.byref(form), None)
BAD, RANGE, ABSENT = _lib.QR_ERR_INVALID_ARGUMENT, _lib.QR_ERR_OUT_OF_RANGE, _lib.QR_ERR_NOT_RESIDENT
inf, nan = float("inf"), float("nan")
"""


def test_refusals_at_the_c_entry(tmp_path):
    run(tmp_path, HEAD + """
assert append(kv, [0, 1], [0, 0], [300, 40]) == 0, L.qr_last_error()
before = launches.value
assert forms(scale=nan) == BAD and forms(act=16) == BAD and forms(act=7) == BAD and forms(cap=-1.0) == BAD and forms(cap=inf) == BAD and forms(cap=1e-4) == BAD and forms(cap=2e6) == BAD
assert forms(window=-1) == BAD and forms(first=[-1]) == BAD and forms(full=[-1]) == BAD and forms(layer=2) == BAD and forms(seqs=[3]) == BAD
assert forms(rows=[-1]) == BAD and forms(q=None) == BAD and forms(out=None) == BAD and forms(q=ROWS + 2) == BAD and forms(slopes=ROWS + 2) == BAD
assert forms(prefix_ids=[3], prefix_len=[1]) == BAD and forms(prefix_ids=[1], prefix_len=[-1]) == BAD
assert forms(prefix_ids=[1]) == BAD and forms(prefix_len=[1]) == BAD
assert forms(pos0=[600]) == RANGE and forms(pos0=[599], rows=[2]) == RANGE and forms(full=[601]) == RANGE
assert forms(prefix_ids=[1], prefix_len=[601]) == RANGE and forms(prefix_ids=[1], prefix_len=[40], full=[641]) == RANGE
assert forms(pos0=[512]) == ABSENT and forms(seqs=[2]) == ABSENT and forms(layer=1) == ABSENT and forms(seqs=[1], full=[257]) == ABSENT
assert forms(prefix_ids=[1], prefix_len=[257]) == ABSENT and forms(prefix_ids=[2], prefix_len=[1]) == ABSENT
assert launches.value == before
# chunks without rows take no part
assert forms(rows=[0], q=None, out=None, first=[-5], prefix_ids=[9], prefix_len=[-1]) == 0 and launches.value == before
assert L.qr_kv_attention_forms_dev(kv._h, 0, None, 0, None, None, None, 0, None, 1.0, None, None) == 0 and launches.value == before
assert forms() == 0 and forms(prefix_ids=[1], prefix_len=[256], full=[512], first=[1 << 30], window=5, cap=3.0, slopes=ROWS) == 0, L.qr_last_error()
assert L.qr_kv_attention_forms_dev(kv._h, 1, ints(0), 0, ints(0), ints(1), ROWS, 0, ROWS, 1.0, None, None) == 0
assert launches.value > before
""")


def test_an_8_bit_cache_refuses_the_other_calls(tmp_path):
    run(tmp_path, HEAD + """
assert append(kv, [0], [0], [300]) == 0, L.qr_last_error()
before = launches.value
i, r, h = ints(0), ROWS, kv._h
one = ints(1)
for status in (
    L.qr_kv_append(h, 0, 0, 0, r, 128, r, 128), L.qr_kv_append_range(h, 0, 0, 0, 1, r, r, 0), L.qr_kv_append_range_dev(h, 0, 0, 0, 1, r, r, 0, None),
    L.qr_kv_append_rope(h, 0, 0, 0, r, r, r, 1e4), L.qr_kv_append_rope_dev(h, 0, 0, 0, 1, r, r, r, 1e4, None),
    L.qr_kv_append_rope_step_dev(h, 0, 0, r, r, r, r, 1e4, None), L.qr_kv_append_rope_chunk_step_dev(h, 0, 0, 1, r, r, r, r, 1e4, None),
    L.qr_kv_attention(h, 0, 0, 0, r, r, 1.0), L.qr_kv_attention_batch(h, 1, i, 0, i, r, r, 1.0), L.qr_kv_attention_dev(h, 1, i, 0, i, r, r, 1.0, None),
    L.qr_kv_attention_dev_noalloc(h, 1, i, 0, i, r, r, 1.0, None), L.qr_kv_attention_step_dev(h, 1, i, 0, r, r, r, 1.0, None),
    L.qr_kv_attention_chunk(h, 0, 0, 0, 1, r, 0, r, 1.0), L.qr_kv_attention_chunk_dev(h, 0, 0, 0, 1, r, 0, r, 1.0, None),
    L.qr_kv_attention_chunk_step_dev(h, 0, 0, 1, r, r, 0, r, 1.0, None), L.qr_kv_attention_chunks_dev(h, 1, i, 0, i, one, r, 0, r, r, 1.0, None),
    L.qr_kv_evict_dev(h, 1, i, 0, one, 1, 1, 1, r, r, r, None), L.qr_kv_read(h, 0, 0, 0, 1, r, r), L.qr_kv_read_dev(h, 1, i, 0, i, one, r, r, None),
    L.qr_kv_decode_plan(h, 1, i, 0, i, one, one)):
    assert status == BAD and b"8-bit" in L.qr_last_error(), (status, L.qr_last_error())
assert launches.value == before
assert L.qr_kv_read_as_dev(h, 1, i, 0, i, one, 16, r, r, None) == BAD and L.qr_kv_read_as_dev(h, 1, i, 0, i, ints(301 + 300), 0, r, r, None) == RANGE
assert L.qr_kv_read_as_dev(h, 1, i, 0, ints(512), one, 0, r, r, None) == ABSENT and L.qr_kv_read_as_dev(h, 1, i, 0, i, one, 0, None, r, None) == BAD
assert L.qr_kv_read_as_dev(h, 1, i, 0, i, one, 1, r + 1, r, None) == BAD
assert launches.value == before
assert L.qr_kv_read_as_dev(h, 1, i, 0, i, one, 2, r, r, None) == 0 and L.qr_kv_attention_chunks_dev(h, 1, i, 0, i, one, r, 0, r, None, 1.0, None) == 0
assert launches.value > before
assert kv.BytesPerToken == 2 * 2 * 2 * 65 and kv.BytesUsed == 2 * 256 * 2 * 2 * 65
kv.Truncate(5); kv.Reset()
assert kv.SeqLen == 0
""")


def test_the_workspace_stays_in_bounds(tmp_path):
    """However many rows and keys: the parts' sums take up to 256 MB of a launch, or one part for each row."""
    run(tmp_path, """
kv = PagedKvCache(1, 64, 8, 128, 65536, "e4m3", 64)
assert append(kv, list(range(64)), [0] * 64, [65536] * 64) == 0, L.qr_last_error()
before = live.value
form = _lib.AttnForm(0.0, None, 0, None, None, ctypes.cast(ints(*[0] * 64), ctypes.c_void_p), ctypes.cast(ints(*[65536] * 64), ctypes.c_void_p))
for rows in (1, 8, 100, 500):
    assert L.qr_kv_attention_forms_dev(kv._h, 64, ints(*range(64)), 0, ints(*[65536 - rows] * 64), ints(*[rows] * 64), ROWS, 0, ROWS, 1.0, ctypes.byref(form), None) == 0
    two = 64 * rows * 64 * 2 * (128 * 4 + 8)  # two lists of keys, one part each
    assert live.value - before <= 2 * max(2 * (256 << 20) + two, two) + 4096, (rows, live.value - before)
""")
