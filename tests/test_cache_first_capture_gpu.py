"""The cache operators' first calls of a process, captured."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch
import flash_llm_b200.torch_op
from paged_cache import Batch, random_tree
ops = torch.ops.flashllm
b = Batch([60, 200], [16, 9], 8, 2, 128, 32, seed=1)
other = Batch([60, 200], [16, 9], 8, 2, 128, 32, seed=1)
qkv = torch.randn((b.rows, 12 * 128), device="cuda").to(torch.float16)
masks, positions = random_tree(b.counts, b.contexts, 2)
path = torch.tensor([[0, 3, 7], [0, 1, 2]], dtype=torch.int32, device="cuda"), torch.tensor([3, 2], dtype=torch.int32, device="cuda")
frequencies = torch.rand(64, dtype=torch.float64, device="cuda")


def step(batch):
    q = ops.rotary_append(qkv, *batch.arrays, frequencies, False, 1.0, positions)
    out = ops.tree_attention(q, *batch.arrays, masks), ops.prompt_attention(q, *batch.arrays)
    ops.cache_accept(*batch.arrays, *path)
    return q, *out


torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step(b)
graph.replay()
want = step(other)
assert all(torch.equal(x, y) for x, y in zip(got, want))
for x, y in ((b.k_cache, other.k_cache), (b.v_cache, other.v_cache)):
    assert torch.equal(x.view(torch.int16), y.view(torch.int16))
print("replayed")
"""


def test_the_first_calls_of_a_process_can_be_captured(lib):
    run = subprocess.run([sys.executable, "-c", SCRIPT], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "PYTHONPATH": os.pathsep.join((ROOT, os.path.join(ROOT, "tests")))})
    assert run.returncode == 0 and "replayed" in run.stdout, run.stdout + run.stderr
