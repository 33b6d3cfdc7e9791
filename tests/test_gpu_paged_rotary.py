"""Appends whose head or rotated dims are no multiples of 16 (element by element), or whose rotated part ends inside a head."""
import pytest

from .test_gpu_paged import _built, test_append_matches_definition as check  # noqa: F401

pytestmark = pytest.mark.gpu

CASES = [  # heads, kv heads, dim, rotated, page
    (4, 2, 80, 40, 16), (6, 2, 72, 24, 16), (4, 4, 72, 72, 7), (3, 3, 40, 8, 64), (2, 1, 256, 2, 16), (8, 8, 136, 72, 32),
    (4, 1, 128, 48, 16), (2, 2, 248, 240, 8),
]


@pytest.mark.parametrize("io,cache", [("bf16", "bf16"), ("f32", "f16"), ("f32", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,dim,rot,page", CASES)
@pytest.mark.parametrize("counts,start", [([1], 1000), ([70, 1, 33], 5)])
def test_partial_rotation(io, cache, interleaved, heads, kv, dim, rot, page, counts, start):
    check(io, cache, heads, kv, dim, rot, interleaved, page, "nhd", counts, start)
