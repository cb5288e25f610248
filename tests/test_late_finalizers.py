"""CPU test: handles that outlive the package's modules at the end of a process are finalized without a word."""
import subprocess
import sys

from tests.hosthip import ROOT

CODE = """
import sys
sys.path.insert(0, {root!r})
from qauntrunner_amd import _lib, caches, store, weights
kinds = (caches.PagedKvCache, caches.MlaLatentCache, store.ModelStore, weights.Weight)
left = [object.__new__(c) for c in kinds]
_lib.finalizing = None  # as a module that has been torn down
del left
print("done")
"""


def test_finalizers_after_the_modules(tmp_path):
    p = subprocess.run([sys.executable, "-c", CODE.format(root=ROOT)], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.split() == ["done"] and p.stderr == "", p.stderr
