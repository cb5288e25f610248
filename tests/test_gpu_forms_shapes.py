"""GPU tests of attention in its other forms at head sizes, head counts and lengths beside those of test_gpu_forms.py, against the
definition in 64 bits (tolerances there)."""
import pytest

from tests.formutil import filled_as
from tests.test_gpu_forms import FORMS, run

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
