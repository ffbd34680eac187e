"""What is left of a call whose bounded waits ran out."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_calls_that_give_up_return_and_leave_rows_right_or_alone():
    """In a process of its own, with a library whose attention gives up after 1 to 512 looks at a barrier, by CTA."""
    subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "flash-llm_b200", "csrc"), "impatient"], check=True)
    run = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "attention_give_up.py")], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "FLASHLLM_LIBRARY": os.path.join(ROOT, "build", "libSpMM_API_impatient.so"),
                              "PYTHONPATH": ROOT})
    assert run.returncode == 0, run.stdout + run.stderr
    assert "gave up" in run.stdout
