"""Attention of sequences that are longer than their table: a position past the table has no page, so
it has no part in any row, whatever part of a step or block of positions the table ends in."""
import math

import pytest
import torch

from page_cases import D, Case, attention_tolerance
from test_gpu_pages import attend

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def over_the_table(case, q, lens):
    """f64 attention of q where sequence s is lens[s] long, and what the tolerance goes by"""
    out, worst, vmax = torch.zeros(q.shape, dtype=torch.float64), 0.0, 0.0
    group = q.shape[1] // case.n_kv
    for s, n in enumerate(case.new):
        a, have = case.starts[s], case.rows[s][0].shape[1]
        last = torch.arange(lens[s] - n, lens[s])
        hide = torch.arange(have)[None] > last[:, None]
        for h in range(q.shape[1]):
            k, v = (x[h // group] for x in case.rows[s])
            x = q[a:a + n, h].double()
            w = torch.softmax((x @ k.T / math.sqrt(D)).masked_fill(hide, -math.inf), -1)
            out[a:a + n, h] = torch.nan_to_num(w) @ v  # (a row without positions: zeros)
            worst = max(worst, float((x.abs() @ k.abs().T).max()) / math.sqrt(D))
            vmax = max(vmax, float(v.abs().max()))
    return out, worst, vmax


# page, pages of a table: capacities that end inside a step of 32 or of 64 positions, up to 256 (items that
# are never cut) and above
TABLES = [(16, 3), (16, 5), (32, 3), (16, 19), (32, 21)]


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("page,width", TABLES)
@pytest.mark.parametrize("new", [1, 5, 9, 40])
def test_length_past_the_table(gpu, new, page, width, rows, kv):
    """a few positions past it, so that only some rows are behind its end; more than a step; far past; the
    other sequence ends inside it. 2 q heads a KV head: tiles of 16, 32 and 128 or 256 rows"""
    cap = page * width
    case = Case([new, 3], [cap - new, 30], page, 2, kv, seed=31, lead=1, tail=1)
    assert case.host["table"].shape == (2, width)
    q = torch.randn(case.total, 4, D, generator=torch.Generator().manual_seed(9)).to(rows)
    for past in (0, 2, 12, 60, 200, (1 << 30) - cap, (1 << 31) - 1 - cap):
        lens = [cap + past, case.lens[1]]
        case.host["lens"] = torch.tensor(lens, dtype=torch.int32)
        want, worst, vmax = over_the_table(case, q, lens)
        got = attend(case, q)
        off = (got[1:-1] - want[1:-1]).abs().max()
        assert off <= attention_tolerance(worst, vmax, rows), f"{past} past the table: off by {off}"
        assert (got[0] == 7).all() and (got[-1] == 7).all()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_many_sequences_past_the_table(gpu, kv):
    """more sequences than one wave plans, each behind its table's end"""
    n, cap = 70, 48
    case = Case([1 + i % 3 for i in range(n)], [cap - 1 - i % 3 for i in range(n)], 16, 1, kv, seed=32)
    q = torch.randn(case.total, 2, D, generator=torch.Generator().manual_seed(10))
    lens = [cap + (i * 7) % 40 for i in range(n)]
    case.host["lens"] = torch.tensor(lens, dtype=torch.int32)
    want, worst, vmax = over_the_table(case, q, lens)
    assert (attend(case, q) - want).abs().max() <= attention_tolerance(worst, vmax, F32)
