"""Refusals and empty calls of the operators of drafts and beams, on the CPU over a HIP runtime that records
(tests/fake_hip.cpp)."""
import os
import subprocess
import sys

import pytest

import drafts_host_cases
from test_host import fake  # noqa: F401 (the fixture that builds the runtime)

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("case", [f.__name__ for f in drafts_host_cases.CASES])
def test_drafts_host(fake, case):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.join(HERE, "drafts_host_cases.py"), fake, case], capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout[-2000:] + r.stderr[-4000:]
