"""What V holds reaches every row that attends it: infinities and NaN in V alone (the scores are finite), in
whichever of a tile's rows."""
import math

import pytest
import torch

from page_cases import D, Case, attention_tolerance
from test_gpu_pages import attend

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("kv,bad", [("bf16", math.nan), ("bf16", math.inf), ("bf16", -math.inf), ("fp8", math.nan)])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,at", [(6, 40, 42), (12, 40, 41), (12, 900, 904), (100, 40, 50), (100, 40, 90),
                                        (100, 40, 139), (100, 1000, 1003), (130, 0, 0), (300, 0, 129)])
def test_not_finite_in_v_alone(gpu, new, ctx, at, rows, kv, bad):
    """one dim of V at position `at` of one KV head: that dim is not finite in every row that attends it, and
    everything else is what it was"""
    case = Case([new, 2], [ctx, 5], 16, 2, kv, seed=33)
    q = torch.randn(case.total, 4, D, generator=torch.Generator().manual_seed(11)).to(rows)
    want, worst, vmax = case.attention(q)
    page, off, dim = int(case.host["table"][0, at // 16]), at % 16, 77
    if kv == "fp8":
        case.host["v"].view(torch.uint8)[page, 1, off // 16, dim, off % 16] = 0x7F
    else:
        case.host["v"][page, 1, off // 16, dim, off % 16] = bad
    got = attend(case, q)
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[max(at - ctx, 0):new, 2:, dim] = True
    lost = hit & torch.isfinite(got)
    assert not lost.any(), f"finite in rows {sorted(set(lost.nonzero()[:, 0].tolist()))}"
    assert (got[~hit] - want[~hit]).abs().max() <= attention_tolerance(worst, vmax, rows)
