"""Graphs as deep as a long run of calls: built, differentiated and let go of. A
release that goes down a chain by nested destructors runs out of stack (at some
70 000 nodes of 8 MB), which ends the process: each case is a process of its own."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

HEAD = """
import sys
sys.path.insert(0, {root!r})
import numpy as np
import oracle
from ormi_amd import Tensor, causal_conv, linear_recurrence
oracle.load()
N = 150_000
def z(*s, grad=False): return Tensor(np.zeros(s, np.float32), "cpu", requires_grad=grad)
"""
CASES = {
    "states of recurrences": """
g, x, state = z(1, 1, 1), z(1, 1, 1), None
for _ in range(N): state = linear_recurrence(g, x, state)[1]
del state
""",
    "states with gradients": """
g, x, state = z(1, 1, 1, grad=True), z(1, 1, 1), z(1, 1)
for _ in range(N): state = linear_recurrence(g, x, state)[1]
del g, x, state
""",
    "inputs kept by convolutions": """
w, x, kept = z(1, 2), z(1, 1, 1), None
for _ in range(N): kept = causal_conv(x, w, None, kept)[1]
del kept
""",
    "sums": """
a, total = z(4), z(4)
for _ in range(N): total = total + a
del total
""",
    "trees shared at every level": """
a = z(4)
for _ in range(N): a = a * a
del a
""",
    "gradients let go of by the graph": """
a = z(4, grad=True)
total = a
for _ in range(N): total = total + a
total = total.sum()
total.backward()
total.zero_grad_graph()
a.zero_grad()
del total, a
""",
    "gradients let go of leaf by leaf": """
a = z(4, grad=True)
b = a
for _ in range(N): b = b * a
b.sum().backward()
b.zero_grad_graph()
grad = a.grad
del a, b, grad
""",
}


@pytest.mark.parametrize("name", CASES)
def test_release_of_a_long_chain(name):
    run = subprocess.run([sys.executable, "-c", HEAD.format(root=str(ROOT)) + CASES[name] + "print('released', flush=True)"],
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.endswith("released\n"), (run.returncode, run.stderr[-500:])
