"""Attention refuses an `out` that shares memory with q or the pages, and takes one that only lies between
their rows."""
import pytest
import torch

import qe
from page_cases import D, Case
from test_pages_refusals import ADDR, attend, c_pages

W = 4 * D * 4  # bytes of a row of 4 heads, f32
Q = ADDR + (1 << 22)
PAGES = 8 * 16 * 2 * D * 2  # bytes of k, and of v


def code(rows=4, q=Q, out=Q, qs=512, os=512, **pages):
    got = attend(c_pages(**{**dict(v=ADDR + (1 << 20)), **pages}), rows=rows, q=q, out=out, qs=qs, os=os)
    return got, qe.lib().qe_last_error()


@pytest.mark.parametrize("kw", [
    dict(), dict(rows=1), dict(out=Q + W), dict(out=Q + 3 * W + W - 16), dict(out=Q - W), dict(out=Q - 4 * W + 16),
    # rows apart: between q's rows, but too wide for the gap
    dict(qs=1020, os=1020, out=Q + W), dict(qs=1020, os=1020, out=Q - W), dict(qs=1024, os=1024, out=Q + W - 16),
    dict(qs=1024, os=1024, out=Q - 3 * 2 * W - W + 16),
    # rows differently far apart: they meet somewhere
    dict(qs=1024, os=1028, out=Q + W), dict(qs=2048, os=512, out=Q + W), dict(qs=512, os=2048, out=Q - 4 * W),
    dict(rows=1000, qs=1024, os=1536, out=Q + W),
    # the pages
    dict(q=Q, out=ADDR), dict(out=ADDR + PAGES - 16), dict(out=ADDR - 4 * W + 16), dict(out=ADDR + (1 << 20) + 16),
    dict(out=ADDR - 2 * W, qs=1024, os=4096), dict(out=ADDR - 65536, qs=512, os=65536 // 4),
    dict(out=ADDR + (1 << 21), kv_dtype=qe.QE_KV_FP8, k_exp=ADDR + (1 << 21) + W, v_exp=ADDR + (1 << 23)),
    dict(out=ADDR + (1 << 21), kv_dtype=qe.QE_KV_FP8, k_exp=ADDR + (1 << 23), v_exp=ADDR + (1 << 21) + 4 * W - 16),
    # offsets past 64 bits of bytes
    dict(rows=1 << 28, qs=(1 << 32) - 4, os=(1 << 32) - 4),
])
def test_out_over_what_is_read(kw):
    got, why = code(**kw)
    assert got == qe.QE_ERR_ARG and b"overlap" in why, kw


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
def test_out_between_the_rows_of_q(gpu, rows):
    """q and out as the two halves of each row of one buffer, either first, and right behind each other"""
    case = Case([5, 1, 20], [30, 100, 7], 16, 2, "bf16", seed=51)
    pages = case.pages()
    q = torch.randn(case.total, 4, D, generator=torch.Generator().manual_seed(14)).to(rows)
    work = torch.empty(qe.op_page_attention_work_bytes(4, 2, 20), dtype=torch.uint8, device="cuda")

    def run(qd, out):
        qd.copy_(q)
        qe.op_page_attention(pages, qd, out, work, 20)
        return out.cpu()

    want = run(torch.empty(case.total, 4, D, dtype=rows, device="cuda"), torch.empty(case.total, 4, D, dtype=rows, device="cuda"))
    both = torch.empty(case.total, 8, D, dtype=rows, device="cuda")
    assert torch.equal(run(both[:, :4], both[:, 4:]), want)
    assert torch.equal(run(both[:, 4:], both[:, :4]), want)
    both = torch.empty(2 * case.total, 4, D, dtype=rows, device="cuda")
    assert torch.equal(run(both[:case.total], both[case.total:]), want)
    with pytest.raises(qe.QeError, match="overlap"):
        qe.op_page_attention(pages, both[:case.total], both[1:case.total + 1], work, 20)
