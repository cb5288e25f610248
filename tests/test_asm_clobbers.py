"""CPU test: inline assembly that writes m0 says so, since the compiler may keep an index of its own there."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qauntrunner_amd", "csrc")


def test_m0_is_named_where_assembly_writes_it():
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        with open(path) as f:
            for block in re.findall(r"\basm\b(?: volatile)?\s*\((.*?)\);", f.read(), re.S):
                if re.search(r"\bs_\w+ m0\b", block):
                    found += 1
                    assert '"m0"' in block.rsplit(":", 1)[1], (os.path.basename(path), block)
    assert found
