"""Runs a piece of Python in a process of its own whose libqr_attn sits on host memory (tests/host_hip.c) instead of a GPU."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HEAD = """
import ctypes, sys
sys.path.insert(0, {root!r})
hip = ctypes.CDLL({hip!r}, ctypes.RTLD_GLOBAL)  # found before the runtime that the library names
from qauntrunner_amd import _lib
from qauntrunner_amd.caches import PagedKvCache
L = _lib.load()
def counter(name):
    return ctypes.c_longlong.in_dll(hip, "hh_" + name)
live, budget, mallocs, syncs, launches = map(counter, ("live", "budget", "mallocs", "syncs", "launches"))
capturing = ctypes.c_int.in_dll(hip, "hh_capturing")
def ints(*x):
    return (ctypes.c_int * len(x))(*x)
rows_memory = ctypes.create_string_buffer(1 << 12)  # stands for any rows: no kernel reads them
ROWS = (ctypes.addressof(rows_memory) + 255) & ~255
def append(kv, seqs, pos0, rows, layer=0):
    w = kv.KvDim
    return L.qr_kv_append_norm_rope_dev(kv._h, len(seqs), ints(*seqs), layer, ints(*pos0), ints(*rows), None, None, 0, ROWS, w, ROWS, w,
                                        _lib.DTYPE_F32, None, None, None, 1e-6, 1e4, 0, None)
def attend(kv, seqs, pos0, rows, weights=True, act=_lib.DTYPE_F32):
    return L.qr_kv_attention_chunks_dev(kv._h, len(seqs), ints(*seqs), 0, ints(*pos0), ints(*rows), ROWS, act, ROWS,
                                        ROWS if weights else None, 1.0, None)
"""


def run(tmp_path, code):
    """The process's output; it must end well."""
    if not shutil.which("gcc"):
        pytest.skip("needs gcc")
    hip = os.path.join(str(tmp_path), "libhosthip.so")
    subprocess.run(["gcc", "-O1", "-w", "-shared", "-fPIC", "-o", hip, os.path.join(ROOT, "tests", "host_hip.c")], check=True)
    env = {k: v for k, v in os.environ.items() if k != "QR_ATTN_LIB"}
    p = subprocess.run([sys.executable, "-c", HEAD.format(root=ROOT, hip=hip) + code], capture_output=True, text=True, timeout=120, env=env)
    assert p.returncode == 0, (p.returncode, p.stdout[-2000:], p.stderr[-4000:])
    return p.stdout
