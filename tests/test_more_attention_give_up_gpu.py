"""What is left of a call through a window or over a cache of 4 bits whose bounded waits ran out, and first calls that are captured."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_calls_that_give_up_return_and_leave_rows_right_or_alone():
    """In a process of its own, with a library whose attention gives up after 1 to 512 looks at a barrier, by CTA."""
    subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "flash-llm_b200", "csrc"), "impatient"], check=True)
    run = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "more_attention_give_up.py")], capture_output=True, text=True,
                         timeout=300, env={**os.environ, "FLASHLLM_LIBRARY": os.path.join(ROOT, "build", "libSpMM_API_impatient.so"),
                                           "PYTHONPATH": ROOT})
    assert run.returncode == 0, run.stdout + run.stderr
    assert run.stdout.count("gave up") == 2


SCRIPT = """
import torch
import flash_llm_b200.torch_op
from four_bit_cache import FourBitBatch
from paged_cache import Batch
ops = torch.ops.flashllm
frequencies = torch.rand(64, dtype=torch.float64, device="cuda")
norm = torch.rand(128, device="cuda").half()
for kind in (Batch, FourBitBatch):
    for counts in ([1, 1], [40, 9]):
        b, other = (kind([60, 200], counts, 8, 2, 128, 32, seed=1) for _ in range(2))
        qkv = torch.randn((b.rows, 12 * 128), device="cuda").to(torch.float16)

        def step(batch):
            if kind is Batch:
                q = ops.norm_rotary_append(qkv, *batch.arrays, norm, norm, 1e-6, frequencies)
                return q, ops.window_attention(q, *batch.arrays, 50, 2)
            q = ops.four_bit_append(qkv, *batch.arrays, norm, norm, 1e-6, frequencies)
            return q, ops.four_bit_attention(q, *batch.arrays), *ops.four_bit_read(*batch.arrays, b.rows)

        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(b)
        graph.replay()
        want = step(other)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        for x, y in ((b.k_cache, other.k_cache), (b.v_cache, other.v_cache)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
print("replayed")
"""


def test_the_first_calls_of_a_process_can_be_captured(lib):
    run = subprocess.run([sys.executable, "-c", SCRIPT], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "PYTHONPATH": os.pathsep.join((ROOT, os.path.join(ROOT, "tests")))})
    assert run.returncode == 0 and "replayed" in run.stdout, run.stdout + run.stderr
