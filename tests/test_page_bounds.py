"""The bound of the attention tests sees a mistake of one part: planted in the 64-bit reference, without a
GPU."""
import pytest
import torch

from page_bounds import attention_bounds
from page_cases import D, Case

MISTAKES = {  # of 64 positions in the middle of the longest sequence
    "lost": lambda part: part * 0.0,
    "twice": lambda part: part * 2.0,
    "relative to another maximum": lambda part: part * 0.5,
}


@pytest.mark.parametrize("mistake", MISTAKES)
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new,ctx,n_kv,heads", [([1], [9000], 1, 16), ([20], [9000], 1, 4), ([190, 70], [1500, 100], 2, 4),
                                                ([300], [4000], 1, 1)])
def test_a_part_that_is_wrong_is_seen(new, ctx, n_kv, heads, rows, mistake):
    case = Case(new, ctx, 64, n_kv, "bf16", seed=41)
    q = torch.randn(case.total, heads, D, generator=torch.Generator().manual_seed(12)).to(rows)
    want, tol = attention_bounds(case, q)
    at = ctx[0] // 128 * 64

    def weigh(s, w):
        if s == 0:
            w = w.clone()
            w[:, at:at + 64] = MISTAKES[mistake](w[:, at:at + 64])
        return w

    got, _ = attention_bounds(case, q, weigh)
    bad = ((got - want).abs() > tol).any(-1).any(-1)  # rows
    assert bad[:new[0]].all() and not bad[new[0]:].any()
