"""The first call of a process may be one that a graph captures: what the library sets up once does not end the capture, and
ids that are out of range are still reported when the graph runs."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

CHILD = """
import sys
sys.path[:0] = [{here!r}, {pkg!r}]
import torch
from ucmx import _native, ops
kind = {kind!r}
dev = "cuda:0"
g = torch.Generator().manual_seed(3)
k, v = (torch.randn((9, 16, 2, 64), generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
q = torch.randn((2, 8, 64), generator=g).to(torch.bfloat16).to(dev)
off, ids = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 3, 5], [4, 2, 8, 0, 1]))
cache = ops.QuantKvCache.alloc(9, 16, 2, 64, 4, dev) if kind != "bf16" else None
every = torch.arange(9, dtype=torch.int32, device=dev)
out = torch.zeros_like(q)
torch.cuda.synchronize()

def run():
    if kind == "bf16":
        return ops.block_attention(q, k, v, off, block_ids=ids, out=out)
    ops.quant_write_blocks(cache, k, v, every)
    return ops.quant_block_attention(q, cache, off, block_ids=ids, out=out)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    run()
graph.replay()
torch.cuda.synchronize()
assert _native.device_error() == 0
first = out.clone()
assert bool(first.abs().sum() > 0)
run()
torch.cuda.synchronize()
assert torch.equal(first, out)
ids[1] = 1000
graph.replay()
torch.cuda.synchronize()
assert _native.device_error() == 3
print("captured first: ok")
"""


@pytest.mark.parametrize("kind", ["bf16", "quant"])
def test_first_call_inside_a_capture(kind):
    code = CHILD.format(here=HERE, pkg=os.path.join(os.path.dirname(HERE), "unified-cache-management_b200"), kind=kind)
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "captured first: ok" in p.stdout, p.stdout + p.stderr
