"""A process whose first call of the library is captured into a graph: the scratch pool is made during the capture."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thunderkittens-sm7x_b200")

CALLS = {
    "documents": """
q, k, v = (torch.randn(1, 4, 300, 64, device="cuda").half() for _ in range(3))
ids = torch.zeros(1, 300, dtype=torch.int32, device="cuda")
call = lambda: tk_b200.attention_masked(q, k, v, scale=0.1, doc_ids=ids)
""",
    "paged": """
cache = [torch.randint(0, 100, (400, 2, 32, 128), dtype=torch.uint8, device="cuda") for _ in range(2)]
scale = torch.full((400, 2), 2.0 ** -7, device="cuda")
q, table = torch.randn(2, 8, 128, device="cuda").half(), torch.arange(400, device="cuda").int().view(2, 200)
lens, starts = torch.tensor([6000, 5000], device="cuda").int(), torch.tensor([0, 1, 2], device="cuda").int()
call = lambda: tk_b200.attention_paged(q, *cache, scale, scale, table, lens, starts, scale=0.1)
""",
    "gemm_softmax": """
a, b = (torch.randn(512, 512, device="cuda").half() for _ in range(2))
call = lambda: tk_b200.gemm_rowsoftmax(a, b)[1]
""",
}


@pytest.mark.parametrize("name", CALLS)
def test_first_call_in_a_capture(name):
    code = f"""
import sys
sys.path.insert(0, {PKG!r})
import torch, tk_b200
{CALLS[name]}
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = call()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, call())
assert tk_b200.device_status() == 0
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
