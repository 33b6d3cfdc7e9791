"""What a read of an 8-bit cache in 16 bits rounds: the product code * scale to fp32, then that to the type."""
import numpy as np
import pytest
import torch

from smelt_b200.paged import PagedKV

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


@pytest.mark.parametrize("to", [torch.float16, torch.bfloat16])
def test_a_product_whose_two_roundings_differ_from_one(to):
    rng = np.random.default_rng(1)
    n = 1 << 17
    scale = torch.from_numpy(rng.uniform(0.5, 1.0, n).astype(np.float32)).cuda().view(n // 16, 1, 16)
    code = torch.from_numpy(rng.integers(-127, 128, (n // 16, 1, 16, 64)).astype(np.int8)).cuda()
    kv = PagedKV(code, code.clone(), scale, scale.clone())
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    table = torch.arange(n // 16, dtype=torch.int32, device="cuda")[None]
    got, _ = kv.read(table, pos, seq=torch.zeros_like(pos), dtype=to)
    exact = (code.double() * scale.double()[..., None]).reshape(n, 1, 64)  # 32 bits: exact
    twice = exact.float().to(to)
    assert torch.equal(got, twice)
    # each rounding is off by half a step at the most
    err = (got.double() - exact).abs()
    assert bool((err <= exact.abs() * (torch.finfo(to).eps / 2 + 2.0 ** -24) * (1 + 2.0 ** -20)).all())
    if to == torch.float16:  # among eight million products some lie so near the middle of two numbers that the first rounding decides
        once = torch.from_numpy(exact.cpu().numpy().astype(np.float16))
        assert 0 < int((once != got.cpu()).sum()) < n
