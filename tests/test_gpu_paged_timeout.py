"""A wait for copies that runs out in attention over paged caches: the warps give up as one, the rows are NaN, the status
says so, and the device stays usable. GPT2Q_TEST_PAGED_STALL, read once by a process, makes every wait expect 16 bytes more
than are copied, so each runs out after its bound (about a second) with no copy outstanding."""
import os
import subprocess
import sys

import pytest

from .helpers import TINY  # noqa: F401  (the model of the child)

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import numpy as np, torch
from smelt_b200.gpu import Gpu
from smelt_b200._ffi import Gpt2qError
from smelt_b200.paged import PagedKV, STATUS_TIMEOUT
from tests.helpers import TINY, make_pack

g = torch.Generator(device="cuda").manual_seed(1)
for io, cache in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)):
    for page, stalls in ((16, True), (5, False)):  # copied in boxes, and gathered key by key
        k = torch.empty(240 // page, 2, page, 64, dtype=cache, device="cuda").normal_(generator=g)
        q = torch.empty(3, 4, 64, dtype=io, device="cuda").normal_(generator=g)
        table = torch.arange(240 // page, dtype=torch.int32, device="cuda")[None].repeat(3, 1)
        lens = torch.tensor([240, 0, 7], dtype=torch.int32, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        lse = torch.empty(3, 4, device="cuda")
        out = PagedKV(k, k).attend(q, table, lens, status=status, lse=lse)
        nan = torch.isnan(out).flatten(1)
        assert torch.equal(nan.all(1), nan.any(1)) and torch.equal(nan.all(1), torch.isnan(lse).all(1))
        assert nan.all(1).tolist() == ([True, False, True] if stalls else [False] * 3), (page, nan.all(1))
        assert int(status) == (STATUS_TIMEOUT if stalls else 0)
        assert bool((out[1] == 0).all()) and bool(torch.isneginf(lse[1]).all())
with Gpu(make_pack(TINY, "auto")) as h:
    hd = TINY.n_embd // TINY.n_head
    for page, stalls in ((16, True), (5, False)):
        layers = [PagedKV(*(torch.zeros(40, TINY.n_head, page, hd, device="cuda") for _ in range(2))) for _ in range(TINY.n_layer)]
        table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
        try:
            h.decode_paged([3], [0], layers, table)
            assert not stalls
        except Gpt2qError as e:
            assert stalls and e.code == -5, e
    h.prefill([np.arange(5, dtype=np.uint32)])
print("done")
"""


def test_waits_that_run_out_are_reported():
    env = dict(os.environ, GPT2Q_TEST_PAGED_STALL="1", PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, env=env, capture_output=True, text=True, timeout=180)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stdout[-2000:] + r.stderr[-2000:]
