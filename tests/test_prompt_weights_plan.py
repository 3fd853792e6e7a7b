"""Which launches weigh a prompt's keys (iq_prompt_weights.h), checked on the host."""
import os
import random
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "native", "prompt_weights_check.cpp")
OUT = os.path.join(HERE, "..", "innerq_amd", "_build", "prompt_weights_check")
FEW = 256  # rows (times heads) that a workgroup of the few-rows launch holds


@pytest.fixture(scope="module")
def plan():
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-std=c++20", "-O1", SRC, "-o", OUT], check=True,
                   capture_output=True)

    def run(cases):
        """(few, steps, shares, rows of a chunk) of each (S, N, Nk, Hq, H)."""
        r = subprocess.run([OUT], input="".join("%d %d %d %d %d\n" % c for c in cases), capture_output=True, text=True, check=True)
        out = [tuple(map(int, line.split())) for line in r.stdout.splitlines()]
        assert len(out) == len(cases)
        return out

    return run


def test_uneven_rows_are_shared(plan):
    """The host knows the sum of the rows, not whose they are.  The few-rows launch walks over a sequence's rows FEW at a time
    in one workgroup, so it is taken only where all of them in one sequence would be 4 turns at most."""
    rng = random.Random(1)
    cases = [(64, 4096, 512000, 32, 8), (64, 63 + 4000, 64 * 8000, 32, 8), (16, 1024, 128000, 32, 8), (4, 256, 64256, 32, 8)]
    for _ in range(3000):
        S, H, r = rng.randrange(1, 300), rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 3, 4, 8])
        N = int(2 ** rng.uniform(0, 15))
        cases.append((S, N, int(2 ** rng.uniform(0, 22)), r * H, H))
    found = plan(cases)
    for (S, N, Nk, Hq, H), (few, steps, shares, chunk) in zip(cases, found):
        assert not few or N * Hq // H <= 4 * FEW, (S, N, Nk, Hq, H)
        assert not few or shares == 1
        assert 256 <= chunk <= 2048 and 1 <= shares <= 16
    assert [f[0] for f in found[:4]] == [0, 0, 0, 1] and sum(f[0] for f in found) > 50
