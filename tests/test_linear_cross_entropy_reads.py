"""Bounds of every load of the weights in the cross entropy of hidden states, on the CPU
(tests/cpp/test_linear_cross_entropy_reads.cpp)."""
from __future__ import annotations

import subprocess

from tests.test_cpp_host import _binary


def test_no_load_leaves_the_weights():
    r = subprocess.run([_binary("test_linear_cross_entropy_reads")], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
    assert " 0 failures" in r.stdout
