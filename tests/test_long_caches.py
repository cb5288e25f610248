"""CPU tests of caches whose positions reach the end of 32 bits, on host memory (tests/hosthip.py)."""
from tests.hosthip import run


def test_caches_of_every_length(tmp_path):
    """The number of pages of max_seq positions is counted without passing 32 bits."""
    run(tmp_path, """
mla = ctypes.c_void_p()
for n in (1, 256, 257, 2**31 - 257, 2**31 - 256, 2**31 - 255, 2**31 - 1):
    for dtype in ("f32", "e4m3"):
        kv = PagedKvCache(1, 1, 1, 1, n, dtype, 1)
        assert append(kv, [0], [0], [1]) == 0 and kv.SeqLen == 1, L.qr_last_error()
        assert append(kv, [0], [n], [1]) == _lib.QR_ERR_OUT_OF_RANGE
        kv.close()
    assert L.qr_mla_create(ctypes.byref(mla), 1, 16, 0, n, 0) == 0, L.qr_last_error()
    assert L.qr_mla_destroy(mla) == 0
""")
