"""Attention over V of large and small magnitudes: f32 sums of weights up to 2^8 each hold any length up to
2^88."""
import pytest
import torch

from page_cases import D, Case, attention_tolerance
from test_gpu_pages import attend

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,heads", [([1], [500], 2), ([6, 2], [3000, 40], 2), ([80, 3], [700, 30], 4), ([12], [7000], 16)])
@pytest.mark.parametrize("power", [85, -85])
def test_magnitudes_of_v(gpu, power, new, ctx, heads, rows, kv):
    """V times a power of two, scores that rise along the positions: the same result times that power"""
    case = Case(new, ctx, 32, 1, kv, seed=61, k_std=3.0)
    q = torch.randn(case.total, heads, D, generator=torch.Generator().manual_seed(15)).to(rows)
    want, worst, vmax = case.attention(q)
    assert vmax < 8  # below 2^88 after the scaling
    if kv == "fp8":
        e = case.host["ve"]
        case.host["ve"] = torch.where(e == 255, e, (e.int() + power).to(torch.uint8))
    else:
        case.host["v"] = (case.host["v"].double() * 2.0 ** power).bfloat16()
    got = attend(case, q) * 2.0 ** -power
    assert (got - want).abs().max() <= attention_tolerance(worst, vmax, rows)
