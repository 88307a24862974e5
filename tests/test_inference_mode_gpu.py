"""State that outlives a call, made inside torch.inference_mode() and used outside of it."""
import os
import subprocess
import sys

import pytest

import wgkv

pytestmark = pytest.mark.gpu

COMMON = """
import torch
import wgkv

dev = "cuda"
lens = torch.full((1, 2), 20, dtype=torch.int32, device=dev)
table = torch.arange(4, dtype=torch.int32, device=dev).view(1, 2, 2)
q = torch.randn(1, 1, 4, 64, device=dev).bfloat16()
row = torch.randn(1, 2, 1, 64, device=dev).bfloat16()
far = torch.full((1, 2), 32, dtype=torch.int32, device=dev)  # behind the table's two pages
cache4 = torch.zeros(4, 16, 80, dtype=torch.uint8, device=dev)
k = torch.randn(4, 16, 64, device=dev).bfloat16()
"""

ERRORS = COMMON + """
with torch.inference_mode():
    wgkv.kv4_append(row, row, cache4, far, table)
for _ in range(2):
    try:
        wgkv.check_errors()
    except AssertionError as e:
        assert _ == 0 and "max_tokens_per_head" in str(e), e
print("good")
"""


def run(script):
    here = os.path.dirname(os.path.dirname(os.path.abspath(wgkv.__file__)))
    r = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": here})
    assert r.returncode == 0 and "good" in r.stdout, r.stdout + r.stderr


def test_errors_of_calls_in_inference_mode_are_reported_and_reset():
    run(ERRORS)


SCRATCH = """
import torch
import wgkv

dev = "cuda"


def attend(batch, kv_heads, group, d):
    n = batch * kv_heads
    lens = torch.full((batch, kv_heads), 20, dtype=torch.int32, device=dev)
    table = torch.arange(2 * n, dtype=torch.int32, device=dev).view(batch, kv_heads, 2)
    q = torch.randn(batch, 1, kv_heads * group, d, device=dev).bfloat16()
    k = torch.randn(2 * n, 16, d, device=dev).bfloat16()
    return wgkv.paged_decode(q, k, k, lens, table, 0.125)


with torch.inference_mode():
    attend(1, 2, 8, 128)  # few counters, long partial results
attend(16, 8, 1, 64)      # more counters in the same scratch, which are set to zero first
wgkv.check_errors()
print("good")
"""


def test_scratch_made_in_inference_mode_serves_outside_of_it():
    run(SCRATCH)
