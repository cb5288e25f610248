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
