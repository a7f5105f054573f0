"""The library's first calls in a process may be captured ones, where the
headers ask for no eager call before (tests/harness/first_call_in_capture.py,
in a process of its own)."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.gpu
def test_first_calls_of_a_process_in_a_capture(gpu):
    print("\n[case] first calls of a process in a capture", flush=True)
    r = subprocess.run([sys.executable, os.path.join(HERE, "harness", "first_call_in_capture.py")], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.split()[-1:] == ["ok"], r.stdout + r.stderr
