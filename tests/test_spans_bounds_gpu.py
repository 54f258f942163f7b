"""Attention over spans and eviction in the build that checks indices (GOPHERLLM_DEBUG_BOUNDS=1): a page number outside the cache is
recorded and never used."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = r'''
import sys
sys.path.insert(0, sys.argv[1])
import torch
from gopherllm_b200 import ops
assert ops.DEBUG_BOUNDS
ops.PREFIX_SPARED_BYTES = 0
dev = "cuda:0"
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
H, G, D, N = 4, 2, 64, 6

def seen(what):
    torch.cuda.synchronize()
    st = ops.bounds_status(clear=True)
    assert st and all(v[0] == "page number" and v[1] in (99, -3) and v[2] == N for v in st.values()), (what, st)

for dtype in (torch.bfloat16, torch.float32):
    k = torch.randn(N, G, 64, D, device=dev).to(dtype); v = torch.randn_like(k)
    for members in (2, 40):
        q = torch.randn(members, H * D, device=dev).to(dtype); out = torch.empty_like(q)
        plan = ops.prefix_plan([(list(range(members)), 128)], members, H, G, D, dtype, 10, dev)
        good = i32([[0, 1, 2 + b % 4] for b in range(members)])
        ops.attention_prefix(q, out, k, v, i32([130] * members), good, plan, H, G, D)
        torch.cuda.synchronize()
        assert ops.bounds_status() == {}, ops.bounds_status()
        for col, bad in ((1, 99), (2, -3)):
            t = good.clone(); t[:, col] = bad
            ops.attention_prefix(q, out, k, v, i32([130] * members), t, plan, H, G, D)
            seen(("prefix", dtype, members, col))
    w = torch.rand(N, G, 64, device=dev)
    for run in (1, 40):
        q = torch.randn(run, H * D, device=dev).to(dtype); out = torch.empty_like(q)
        # (runs: the attention kernels of prompts take page numbers as they are, so a bad one is given where only the weights go)
        if run == 1:
            ops.attention_weighed(q, out, k, v, w, i32([0]), i32([run]), i32([100]), i32([[3, 99, 0]]), H, G, D, run, 100 + run)
            seen(("weighed", dtype, run))
    for to in (None, i32([[4, 99]])):
        ops.cache_evict(k, v, w, i32([180]), i32([[0, 99, 2] if to is None else [0, 1, 2]]), 100, recent=10, to_pages=to)
        seen(("evict", dtype))
print("ok")
'''


def test_bad_pages_are_recorded_and_never_used():
    env = dict(os.environ, GOPHERLLM_DEBUG_BOUNDS="1")
    r = subprocess.run([sys.executable, "-c", SCRIPT, ROOT], env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout[-2000:] + r.stderr[-4000:]
