"""A process whose first call of the library is captured into a graph: what outlives the graph is not part of it."""
import os
import subprocess
import sys

import pytest

import wgkv

pytestmark = pytest.mark.gpu

FIRST_CALL_CAPTURED = """
import sys
import torch
import wgkv

bits = sys.argv[1]
dev = "cuda"
lens = torch.full((1, 2), 20, dtype=torch.int32, device=dev)
table = torch.arange(4, dtype=torch.int32, device=dev).view(1, 2, 2)
q = torch.randn(1, 1, 4, 64, device=dev).bfloat16()
row = torch.randn(1, 2, 1, 64, device=dev).bfloat16()
far = torch.full((1, 2), 32, dtype=torch.int32, device=dev)  # behind the table's two pages
cache4 = torch.zeros(4, 16, 80, dtype=torch.uint8, device=dev)
k = torch.randn(4, 16, 64, device=dev).bfloat16()
step = ((lambda: wgkv.paged_decode_kv4(q, cache4, lens, table, 0.125)) if bits == "4" else
        (lambda: wgkv.paged_decode(q, k, k, lens, table, 0.125)))
junk = [torch.full((64,), 0x7f, dtype=torch.uint8, device=dev) for _ in range(100)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    junk_in_graph = torch.full((64,), 0x7f, dtype=torch.uint8, device=dev)
    del junk_in_graph  # memory that the graph's later allocations take
    out = step()
wgkv.check_errors()  # nothing has run yet
g.replay()
wgkv.check_errors()
assert torch.equal(out, step())
wgkv.kv4_append(row, row, cache4, far, table)  # dropped and flagged
g.replay()
try:
    wgkv.check_errors()
except AssertionError as e:
    assert "max_tokens_per_head" in str(e), e
else:
    raise SystemExit("the replay lost an error that was flagged before it")
wgkv.check_errors()
print("reported")
"""


@pytest.mark.parametrize("bits", ["4", "16"])
def test_errors_outlive_a_graph_whose_capture_was_the_first_call(bits):
    here = os.path.dirname(os.path.dirname(os.path.abspath(wgkv.__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED, bits], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": here})
    assert r.returncode == 0 and "reported" in r.stdout, r.stdout + r.stderr
