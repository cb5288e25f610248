"""Host-side memory of the calls over chunks of several sequences, without a GPU (tests/hosthip.py): how the pool and the
workspace grow."""
from tests.hosthip import run


def test_the_pool_grows_by_what_fits(tmp_path):
    """An append whose pool cannot double takes the pages it needs, as the other appends do."""
    out = run(tmp_path, """
kv = PagedKvCache(1, 1, 1, 64, 256 * 64, "f32", 2)
page = 2 * 256 * 64 * 4
assert append(kv, [0], [0], [256 * 16]) == 0
assert launches.value > 0
budget.value = live.value + 20 * page  # 17 pages fit beside the old ones, 32 do not
assert append(kv, [0, 1], [256 * 16, 0], [1, 0]) == 0, L.qr_last_error()
print("pages", (live.value - budget.value) // page + 20)
budget.value = live.value + 10 * page
assert append(kv, [1], [0], [1]) == _lib.QR_ERR_OUT_OF_MEMORY
budget.value = live.value + 18 * page
assert append(kv, [1], [0], [1]) == 0, L.qr_last_error()
""")
    assert out.split() == ["pages", "1"]
