"""Refusals and empty calls of the paged cache, its attention and the logits' rules, on the CPU over a HIP runtime that
records (tests/fake_hip.cpp)."""
import subprocess
import sys
import os

import pytest

import paged_host_cases
from test_host import fake  # noqa: F401 (the fixture that builds the runtime)

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("case", [f.__name__ for f in paged_host_cases.CASES])
def test_paged_host(fake, case):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.join(HERE, "paged_host_cases.py"), fake, case], capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout[-2000:] + r.stderr[-4000:]
