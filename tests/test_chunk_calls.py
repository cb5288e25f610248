"""CPU tests of the calls over chunks of several sequences: what is refused before the library or the GPU is reached,
and null handles at the C entries."""
import ctypes

import numpy as np
import pytest
import torch

import qauntrunner_amd as qr
from qauntrunner_amd import _lib
from qauntrunner_amd.caches import _ints, _overlap, _strided, _whole

NULL = ctypes.c_void_p()


class OnGpu:
    """A CPU tensor that says it is on GPU `dev`."""

    is_cuda = True

    def __init__(self, t, dev=0):
        self.t, self.dev = t, dev
        self.dtype, self.shape = t.dtype, t.shape

    def get_device(self):
        return self.dev

    def __getattr__(self, name):
        return getattr(self.t, name)


class Refuses:
    """A library that is not to be reached."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


@pytest.fixture
def kv():
    c = object.__new__(qr.PagedKvCache)
    c._lib, c._h, c._device = Refuses(), NULL, 0
    c.Layers, c.Heads, c.KvHeads, c.HeadDim, c.MaxSeq, c.MaxBatch = 1, 4, 2, 16, 64, 3
    c.KvDim, c.KvDtype = 32, _lib.DTYPE_F32
    yield c
    c._h = None


def rows(n, width, dtype=torch.float32, dev=0):
    return OnGpu(torch.zeros(n, width, dtype=dtype), dev)


def test_null_handles():
    L = _lib.load()
    bad = _lib.QR_ERR_INVALID_ARGUMENT
    assert L.qr_kv_append_norm_rope_dev(NULL, 0, NULL, 0, NULL, NULL, NULL, NULL, 0, NULL, 0, NULL, 0, 0, NULL, NULL, NULL, 1e-6,
                                        1e4, 0, NULL) == bad
    assert b"null" in L.qr_last_error()
    assert L.qr_kv_attention_chunks_dev(NULL, 0, NULL, 0, NULL, NULL, NULL, 0, NULL, NULL, 1.0, NULL) == bad
    assert L.qr_kv_evict_dev(NULL, 0, NULL, 0, NULL, 1, 0, 0, NULL, NULL, NULL, NULL) == bad
    assert L.qr_kv_read_dev(NULL, 0, NULL, 0, NULL, NULL, NULL, NULL, NULL) == bad
    out = ctypes.c_int(-5)
    assert L.qr_kv_device(NULL, ctypes.byref(out)) == bad and out.value == -5


@pytest.mark.parametrize("x", [[1.5], ["1"], [None], [2 ** 31], [-2 ** 31 - 1], np.zeros((2, 2), int), np.zeros(2), torch.zeros(2),
                               np.array([2 ** 31]), np.array([2 ** 32 + 1], np.uint64)])
def test_lists_that_are_not_whole_numbers(x):
    with pytest.raises(ValueError):
        _ints(x, "x")


@pytest.mark.parametrize("x", [[1, 2], (1, 2), np.array([1, 2]), np.array([1, 2], np.uint8), torch.tensor([1, 2]), range(1, 3)])
def test_lists_of_whole_numbers(x):
    assert list(_ints(x, "x")) == [1, 2]


def test_rows_and_their_extent():
    fused = torch.zeros(5, 48)
    part, stride = _strided(OnGpu(fused[:, 8:24]), 5, 16, _lib.DTYPE_F32, 0, "q")
    assert part == (fused.data_ptr() + 32, fused.data_ptr() + 32 + 4 * (4 * 48 + 16)) and stride == 48
    assert _strided(OnGpu(fused[:1, 8:24]), 1, 16, _lib.DTYPE_F32, 0, "q")[1] == 16
    for bad in (fused[:, :17], fused[:4, :16], fused[:, ::3], fused[:, :16].double(), fused[:1, :16].expand(5, 16)):
        with pytest.raises(ValueError):
            _strided(OnGpu(bad), 5, 16, _lib.DTYPE_F32, 0, "q")
    for bad in (fused[:, 8:24], fused.half(), fused[:4], fused.t()):
        with pytest.raises(ValueError):
            _whole(OnGpu(bad), 240, _lib.DTYPE_F32, 0, "out")
    a, b = _whole(OnGpu(fused[:2]), 96, _lib.DTYPE_F32, 0, "a"), _whole(OnGpu(fused[2:]), 144, _lib.DTYPE_F32, 0, "b")
    assert not _overlap(a, b) and _overlap(a, _whole(OnGpu(fused), 240, _lib.DTYPE_F32, 0, "c"))


def test_refused_append(kv):
    def go(ids=(0, 1), pos=(0, 5), n=(2, 1), q=rows(3, 64), k=rows(3, 32), v=rows(3, 32), out=rows(3, 64), qn=None, kn=None, **kw):
        kv.AppendNormRopeDev(0, list(ids), list(pos), list(n), q, k, v, out, qn, kn, 1e-6, 1e4, **kw)

    both = rows(3, 64)
    for kw in (dict(pos=(0,)), dict(n=(3, -1)), dict(n=(2, 2)), dict(q=None), dict(out=None), dict(q=rows(3, 63)), dict(k=rows(3, 31)),
               dict(v=rows(2, 32)), dict(q=rows(3, 64, torch.float16)), dict(v=rows(3, 32, torch.bfloat16)), dict(k=rows(3, 32, torch.int32)),
               dict(out=rows(3, 64, torch.float16)), dict(out=rows(2, 64)), dict(q=torch.zeros(3, 64)), dict(k=rows(3, 32, dev=1)),
               dict(k=OnGpu(both.t[:, :32]), out=both), dict(v=OnGpu(both.t[:, 32:]), out=both), dict(qn=rows(1, 15)), dict(kn=rows(1, 17)),
               dict(qn=rows(1, 16, torch.float16)), dict(rope_pos0=[1]), dict(rope_pos0=[0.5, 1])):
        with pytest.raises(ValueError):
            go(**kw)
    with pytest.raises(AssertionError, match="qr_kv_append_norm_rope_dev"):
        go(q=both, out=both, stream=0)


def test_refused_attention(kv):
    w = OnGpu(torch.zeros(3, 2, 64))
    q = rows(3, 64)

    def go(ids=(0, 1), pos=(0, 5), n=(2, 1), q=q, out=rows(3, 64), weights=w, **kw):
        kv.AttentionChunksDev(0, list(ids), list(pos), list(n), q, out, 1.0, weights=weights, **kw)

    for kw in (dict(ids=(0,)), dict(n=(1, 1)), dict(out=q), dict(out=rows(3, 64, torch.float16)), dict(q=OnGpu(torch.zeros(3, 128)[:, :64])),
               dict(weights=OnGpu(torch.zeros(3, 2, 63))), dict(weights=OnGpu(torch.zeros(3, 2, 64).half())), dict(weights=torch.zeros(3, 2, 64)),
               dict(out=OnGpu(w.t.view(-1)[:192].view(3, 64))), dict(out=rows(3, 64, dev=1))):
        with pytest.raises(ValueError):
            go(**kw)
    with pytest.raises(AssertionError, match="qr_kv_attention_chunks_dev"):
        go(stream=0)


def test_refused_eviction(kv):
    w = OnGpu(torch.zeros(3, 2, 64))

    def go(ids=(0,), ln=(60,), budget=(1, 2, 3), weights=w, kept=OnGpu(torch.zeros(1, 2, 6, dtype=torch.int32)), **kw):
        kv.EvictDev(0, list(ids), list(ln), *budget, weights, kept, **kw)

    wide = torch.zeros(4, 2, 64)
    for kw in (dict(ln=(60, 3)), dict(budget=(-1, 4, 3)), dict(budget=(1, 2, 4)), dict(weights=rows(3, 64)),
               dict(kept=OnGpu(torch.zeros(1, 2, 6))), dict(kept=OnGpu(torch.zeros(2, 1, 6, 2, dtype=torch.int32)[..., 0])),
               dict(kept=OnGpu(w.t.view(torch.int32).view(-1)[:12])), dict(weights=OnGpu(wide[:3]), kept_weights=OnGpu(wide[1:])),
               dict(kept_weights=rows(3, 64)), dict(kept=torch.zeros(1, 2, 6, dtype=torch.int32))):
        with pytest.raises(ValueError):
            go(**kw)
    with pytest.raises(AssertionError, match="qr_kv_evict_dev"):
        go(kept_weights=w, stream=0)


def test_refused_read(kv):
    k = rows(3, 32)
    for a, b in ((k, k), (k, rows(2, 32)), (rows(3, 32, torch.float16), k), (rows(3, 32, dev=1), k), (torch.zeros(3, 32), k)):
        with pytest.raises(ValueError):
            kv.ReadDev(0, [0], [0], [3], a, b)
    with pytest.raises(AssertionError, match="qr_kv_read_dev"):
        kv.ReadDev(0, [0], [0], [3], k, rows(3, 32), stream=0)
