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


def test_the_workspace_grows_by_doubling(tmp_path):
    """A decode loop with weights, whose workspace grows with the sequences: few allocations, each a wait for the GPU, and
    what a captured graph keeps alive stays within twice the largest."""
    out = run(tmp_path, """
n = 16
kv = PagedKvCache(1, 32, 8, 128, 4096, "f16", n)
seqs = list(range(n))
assert append(kv, seqs, [0] * n, [4096] * n) == 0
before, allocations, waits = live.value, mallocs.value, syncs.value
for captured in (0, 1):
    capturing.value = captured
    assert attend(kv, seqs, [0] * n, [1] * n) == 0, L.qr_last_error()
capturing.value = 0
for p in range(1, 4096):
    assert attend(kv, seqs, [p] * n, [1] * n) == 0, L.qr_last_error()
need = 4 * n * 32 * 4096  # a score per row, head and position, beside which the partials are small
print(mallocs.value - allocations, syncs.value - waits, (live.value - before) / need)
""")
    allocations, waits, held = map(float, out.split())
    assert allocations <= 20 and waits <= 40 and held <= 6, out


def test_the_workspace_takes_what_it_needs_where_it_cannot_double(tmp_path):
    out = run(tmp_path, """
kv = PagedKvCache(1, 32, 8, 128, 65536, "f16", 16)
seqs = list(range(16))
assert append(kv, seqs, [0] * 16, [65536] * 16) == 0
before = live.value
assert attend(kv, seqs, [9999] * 16, [1] * 16) == 0
small = live.value - before
budget.value = live.value + small // 4  # room for a quarter more once the old one is given back
assert attend(kv, seqs, [10999] * 16, [1] * 16) == 0, L.qr_last_error()
print((live.value - before) / small)
assert attend(kv, seqs, [39999] * 16, [1] * 16) == _lib.QR_ERR_OUT_OF_MEMORY
assert attend(kv, seqs, [9999] * 16, [1] * 16) == 0, L.qr_last_error()
""")
    assert 1.0 < float(out) < 1.25


def test_a_refused_allocation_does_not_fail_the_next_call(tmp_path):
    """The runtime keeps a failed call's error until it is asked for; the launch checks of a later call must not find it."""
    run(tmp_path, """
kv = PagedKvCache(1, 8, 2, 64, 65536, "f32", 8)
seqs = list(range(8))
assert append(kv, seqs, [0] * 8, [4096] * 8) == 0
budget.value = live.value
assert append(kv, [0], [4096], [65536 - 4096]) == _lib.QR_ERR_OUT_OF_MEMORY  # the pool
assert append(kv, [0], [0], [1]) == 0, L.qr_last_error()
assert attend(kv, seqs, [4095] * 8, [1] * 8) == _lib.QR_ERR_OUT_OF_MEMORY  # the workspace
assert append(kv, [0], [0], [1]) == 0, L.qr_last_error()
""")


def test_a_refused_weight_does_not_fail_the_next_call(tmp_path):
    run(tmp_path, """
kv = PagedKvCache(1, 8, 2, 64, 4096, "f32", 1)
assert append(kv, [0], [0], [16]) == 0
budget.value = live.value
w = ctypes.c_void_p()
assert L.qr_weight_create(ctypes.byref(w), _lib.FORMATS["F32"], 4, 256, rows_memory) == _lib.QR_ERR_OUT_OF_MEMORY
assert append(kv, [0], [0], [16]) == 0, L.qr_last_error()
""")
