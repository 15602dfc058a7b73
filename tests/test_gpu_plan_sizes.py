"""GPU: plans whose lengths just fit the shared memory that a kernel may use
without asking for more. Each in a process of its own: a larger plan before it
would have raised the limit."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

CODE = """
import sys
sys.path[:0] = [%r, %r]
import numpy as np
import test_gpu_attn as ta
n = %d
rng = np.random.default_rng(n)
past, new = rng.integers(0, 40, n), rng.integers(0, 3, n)
table = np.full((n, 3), -1)
for s in range(n):
    table[s, :-(-past[s] // 16)] = 3 * s + np.arange(-(-past[s] // 16))
args = (past, new, 16, 5 * n, np.arange(3 * n, 5 * n), 0, table, int(new.sum()) + 5)
for alias in (False, True):
    for a, b in zip(ta.run_plan(*args, alias=alias), ta.plan_reference(*args)):
        assert np.array_equal(a, b)
"""


@pytest.mark.parametrize("n_seq", [4074, 4075, 4085, 4096, 4097])
def test_plan_at_the_shared_memory_limit(gpu, n_seq):
    r = subprocess.run([sys.executable, "-c", CODE % (os.path.join(os.path.dirname(HERE), "moe.cc_b200"), HERE, n_seq)],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-800:]
