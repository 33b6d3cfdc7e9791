"""Waits for copies that run out in the attention of 8-bit caches and of drafted tokens: the rows are NaN, the status says so and the
device stays usable. GPT2Q_TEST_PAGED_STALL, read once by a process, makes every wait expect 16 bytes more than are copied, so each
runs out with no copy outstanding."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import torch
from smelt_b200.paged import PagedKV, STATUS_TIMEOUT

g = torch.Generator(device="cuda").manual_seed(1)
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")

def cache(kind, page, dim):
    shape = (240 // page, 2, page, dim)
    if kind == "i8":
        k = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g)
        s = torch.rand(shape[:3], device="cuda", generator=g) + 0.5
        return PagedKV(k, k, s, s)
    k = torch.empty(shape, dtype=getattr(torch, kind), device="cuda").normal_(generator=g)
    return PagedKV(k, k)

def check(out, lse, status, rows, stalls):
    nan = torch.isnan(out).flatten(1)
    assert torch.equal(nan.all(1), nan.any(1)) and torch.equal(nan.all(1), torch.isnan(lse).all(1))
    assert nan.all(1).tolist() == [stalls] * rows and int(status) == (STATUS_TIMEOUT if stalls else 0), (nan.all(1), int(status))

for io, kind, page, dim, stalls in (("bfloat16", "i8", 16, 64, True), ("float32", "i8", 5, 64, False)):
    kv = cache(kind, page, dim)
    q = torch.empty(2, 4, dim, dtype=getattr(torch, io), device="cuda").normal_(generator=g)
    table = torch.arange(240 // page, dtype=torch.int32, device="cuda")[None].repeat(2, 1)
    lse, status = torch.empty(2, 4, device="cuda"), i32([0])
    check(kv.attend(q, table, i32([240, 7]), lse=lse, status=status), lse, status, 2, stalls)
# drafted tokens: on tiles of 16-bit queries, many or few per row, and warp by warp
for io, kind, page, dim, nodes, stalls in (("bfloat16", "bfloat16", 16, 128, 40, True), ("float16", "float16", 8, 64, 100, True), ("bfloat16", "i8", 16, 128, 40, True),
                                           ("float16", "i8", 16, 64, 100, True), ("float32", "float16", 16, 64, 3, True), ("float32", "float16", 5, 64, 3, False)):
    kv = cache(kind, page, dim)
    q = torch.empty(nodes, 4, dim, dtype=getattr(torch, io), device="cuda").normal_(generator=g)
    table = torch.arange(240 // page, dtype=torch.int32, device="cuda")[None]
    lse, status = torch.empty(nodes, 4, device="cuda"), i32([0])
    check(kv.attend_tree(q, table, i32([100]), i32([0, nodes]), lse=lse, status=status), lse, status, nodes, stalls)
x = torch.ones(1000, device="cuda")
assert float((x + x).sum()) == 2000.0
print("done")
"""


def test_waits_that_run_out_are_reported():
    env = dict(os.environ, GPT2Q_TEST_PAGED_STALL="1", PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, env=env, capture_output=True, text=True, timeout=180)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stdout[-2000:] + r.stderr[-2000:]
