"""GPU tests of rows behind shared prefixes: calls of more rows than one launch takes, against the definition in 64 bits
(tolerances: test_gpu_forms.py)."""
import pytest

from tests.formutil import filled_as
from tests.test_gpu_forms import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,act", [("bf16", "bf16"), ("e4m3", "bf16"), ("f32", "f32")])
def test_more_rows_than_a_launch_takes(gpu, dtype, act):
    """64 heads of 128: 2016 rows behind prefixes fill a launch's partials, so that chunks are cut, also inside a block of rows."""
    kv, rows = filled_as(64, 8, 128, dtype, [901, 1303, 7, 700, 300, 65])
    chunks = [(0, 0, 901), (1, 3, 1300), (2, 6, 1), (3, 100, 600)]
    with kv:
        run(kv, rows, chunks, dtype, act, prefix=[(4, 300), (4, 300), (0, 0), (5, 65)])
        run(kv, rows, chunks, dtype, act, prefix=[(4, 300), (4, 300), (4, 300), (5, 65)], window=500, first=[0, 250, 3, 64], full=[1150, 0, 0, 700], cap=30.0)


@pytest.mark.parametrize("dtype,act,heads,kv_heads,D", [("bf16", "bf16", 32, 8, 128), ("e4m3", "f16", 8, 2, 64), ("f32", "f32", 28, 4, 96), ("f16", "f16", 6, 4, 40)])
def test_prefixes_that_few_rows_see(gpu, dtype, act, heads, kv_heads, D):
    """Windows and first positions that hide the whole prefix from some chunks, from all, and from a chunk's late rows."""
    kv, rows = filled_as(heads, kv_heads, D, dtype, [900, 40, 130, 512])
    chunks = [(0, 700, 150), (1, 0, 40), (2, 129, 1), (1, 39, 1)]
    with kv:
        for window in (0, 1, 30, 100, 130, 200, 600):
            run(kv, rows, chunks, dtype, act, prefix=[(3, 512)] * 4, window=window)
            run(kv, rows, chunks, dtype, act, prefix=[(3, 512)] * 4, window=window, first=[511, 512, 0, 551], full=[0, 530, 0, 0])
