"""The paged cache's kernels on buffers fenced by unmapped pages (tests/guard/run_guarded_kv.py), each case in a child process."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "guard"))
from run_guarded_kv import CASES  # noqa: E402

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not os.path.exists(os.path.join(HERE, "guard", "libwtguard.so")),
                                 reason="tests/guard/libwtguard.so was not built (__graft_entry__.build() reports why)")]


@pytest.mark.parametrize("mode", ["end", "start"])
@pytest.mark.parametrize("case", CASES)
def test_fenced_buffers(case, mode):
    p = subprocess.run([sys.executable, os.path.join(HERE, "guard", "run_guarded_kv.py"), case, mode], cwd=os.path.dirname(HERE), capture_output=True,
                       text=True, timeout=100)
    assert p.returncode == 0, f"{case}/{mode}: exit {p.returncode}\n{p.stdout[-1500:]}\n{p.stderr[-3000:]}"
    assert f"guarded {case}/{mode}: ok" in p.stdout
