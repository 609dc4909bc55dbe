"""The first call of a process, within the capture of a graph."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

SCRIPT = """
import sys, torch
sys.path.insert(0, {pkg!r})
import torch_npu as npu
g = torch.Generator(device="cuda").manual_seed(1)
k, v = (torch.randint(-127, 128, (9, 16, 2, 64), generator=g, device="cuda", dtype=torch.int8) for _ in range(2))
ks, vs = (torch.rand((9, 2, 16), generator=g, device="cuda") * 0.02 for _ in range(2))
q = torch.randn((2, 8, 64), generator=g, device="cuda", dtype=torch.bfloat16)
table = torch.randperm(8, generator=g, device="cuda").int().view(2, 4)
lens = torch.tensor([50, 64], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, lse = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
graph.replay()
want = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
torch.cuda.synchronize()
assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and bool(out.isfinite().all())
print("fine")
"""


def test_captured_first_call(dev):
    run = subprocess.run([sys.executable, "-c", SCRIPT.format(pkg=str(ROOT / "ascend-python_b200"))], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "fine" in run.stdout, run.stderr[-2000:]
