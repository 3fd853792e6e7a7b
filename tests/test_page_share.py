"""How the attention over pages shares out its list of (sequence, head, page) units, checked on the host up to the longest
list that a call may have, 2^31 - 1 units: every unit in one share."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "native", "page_share_check.cpp")
OUT = os.path.join(HERE, "..", "innerq_amd", "_build", "page_share_check")


def test_every_unit_is_in_one_share():
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-std=c++20", "-O1", SRC, "-o", OUT], check=True,
                   capture_output=True)
    totals = [0, 1, 3, 4, 5, 511, 512, 513, 2047, 2048, 2049, 4200, 100003, 10 ** 9, 2139095039, 2 ** 31 - 513, 2 ** 31 - 512,
              2 ** 31 - 511, 2 ** 31 - 257, 2 ** 31 - 256, 2 ** 31 - 2, 2 ** 31 - 1]
    cases = [(t, g) for t in totals for g in (1, 7, 256, 512)]
    r = subprocess.run([OUT], input="".join(f"{t} {g}\n" for t, g in cases), capture_output=True, text=True, check=True)
    lines = r.stdout.split("\n")[:-1]
    assert len(lines) == len(cases)
    bad = [(c, line) for c, line in zip(cases, lines) if line != "ok"]
    assert not bad, bad[:5]
