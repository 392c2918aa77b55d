"""Attention cut into parts, each element within its own bound: one part lost, doubled or put on a wrong
maximum is seen in every kernel that makes parts and in every join."""
import pytest
import torch

from page_bounds import attention_bounds
from page_cases import D, Case
from test_gpu_pages import attend

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16

SHAPES = [
    # new tokens, cached before, n_kv, heads
    ([1], [9000], 1, 16),                           # a row each of 16 heads in many parts: joined by rows
    ([2, 1, 1], [6000, 20, 300], 2, 12),
    ([12], [7000], 1, 2),                           # tiles of 32 rows
    ([1 + i % 3 for i in range(40)], [(i * 397) % 3000 for i in range(40)], 2, 4),
    ([20], [9000], 1, 8),                           # large tiles in many parts: joined by dims
    ([20, 1], [5000, 900], 1, 8),
    ([40, 3], [3000, 100], 1, 8),                   # tiles of 256 bf16 rows
    ([300], [4000], 1, 2),                          # some tiles, equally many parts each
    ([190, 0, 70, 1, 120], [1500, 9, 100, 2500, 800], 2, 4),
    ([64 + i for i in range(66)], [(i * 53) % 900 for i in range(66)], 1, 2),  # more sequences than a wave plans
]


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,n_kv,heads", SHAPES)
def test_every_element_of_parts(gpu, new, ctx, n_kv, heads, rows, kv):
    case = Case(new, ctx, 64, n_kv, kv, seed=42)
    q = torch.randn(case.total, heads, D, generator=torch.Generator().manual_seed(13)).to(rows)
    want, tol = attention_bounds(case, q)
    off = (attend(case, q) - want).abs()
    worst = (off / tol).max()
    assert worst <= 1.0, f"{float(worst):.2f} of the bound, off by {float(off.max()):.2e}"
