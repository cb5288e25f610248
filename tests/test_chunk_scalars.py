"""CPU tests: whole numbers that the calls over chunks of several sequences take one at a time (layer, window, dims, budgets) reach the
library as they are or are refused; none is wrapped to 32 bits, and no cap becomes the zero that stands for none."""
import sys

import pytest
import torch

from tests.test_chunk_calls import kv, rows  # noqa: F401

WRONG = [2**32, 2**32 + 5, -(2**32) + 1, 2**31, -(2**31) - 1, sys.maxsize, 1.5, "1", None]


class Reached(Exception):
    pass


class Library:
    """Records what a call passes."""

    def __getattr__(self, name):
        def call(*a):
            raise Reached(a)

        return call


def call(kv, name, layer=0, **more):  # noqa: F811
    one = ([0], [0], [1])
    q, o, k, v = rows(1, 64), rows(1, 64), rows(1, 32), rows(1, 32)
    stream = type("", (), {"cuda_stream": 0})()
    if name == "append":
        kv.AppendNormRopeDev(layer, *one, None, k, v, None, None, None, 1e-6, 1e4, stream=stream, **more)
    elif name == "chunks":
        kv.AttentionChunksDev(layer, *one, q, o, 1.0, stream=stream)
    elif name == "forms":
        kv.AttentionFormsDev(layer, *one, q, o, 1.0, stream=stream, **more)
    elif name == "evict":
        w = rows(kv.MaxBatch * kv.KvHeads, kv.MaxSeq)
        more = {"first": 1, "heavy": 1, "recent": 1, **more}
        kept = rows(1, kv.KvHeads * 3, torch.int32)
        kv.EvictDev(layer, [0], [1], weights=w, kept=kept, stream=stream, **more)
    else:
        getattr(kv, name)(layer, *one, k, v, stream=stream)


@pytest.mark.parametrize("name", ["append", "chunks", "forms", "evict", "ReadDev", "ReadAsDev"])
def test_layers(kv, name):  # noqa: F811
    for x in WRONG:
        with pytest.raises(ValueError, match="layer"):
            call(kv, name, layer=x)
    kv._lib = Library()
    with pytest.raises(Reached) as e:
        call(kv, name, layer=2**31 - 1)
    assert 2**31 - 1 in e.value.args[0]


def test_windows(kv):  # noqa: F811
    """2^32 + 5 is no window of 5 positions, and the largest integer no negative one."""
    for x in WRONG:
        with pytest.raises(ValueError, match="window"):
            call(kv, "forms", window=x)


def test_rotary_dims(kv):  # noqa: F811
    for x in WRONG[:-1]:  # (None: the head size)
        with pytest.raises(ValueError, match="rotary_dim"):
            call(kv, "append", rotary_dim=x)


@pytest.mark.parametrize("what", ["first", "heavy", "recent"])
def test_budgets(kv, what):  # noqa: F811
    for x in WRONG:
        with pytest.raises(ValueError):
            call(kv, "evict", **{what: x})


def test_a_cap_too_small_for_32_bits_is_no_missing_cap(kv):  # noqa: F811
    for x in (1e-50, -1e-50, 1e-46):
        with pytest.raises(ValueError, match="cap"):
            call(kv, "forms", cap=x)
    kv._lib = Library()
    for x in (0.0, -0.0, 0, 30.0, 1e-3):
        with pytest.raises(Reached):
            call(kv, "forms", cap=x)
