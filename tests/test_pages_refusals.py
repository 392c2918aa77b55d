"""What the paged-cache and draft-check operators refuse, before anything reaches a device: runs
without a GPU."""
import ctypes

import pytest
import torch

import qe
from test_rust_binding import c_struct_fields, rust_struct_fields

ADDR = 1 << 20  # an aligned address that is never read


def c_pages(**kw):
    f = dict(k=ADDR, v=ADDR, k_exp=None, v_exp=None, table=ADDR, lens=ADDR, starts=ADDR, n_pages=8, page_size=16,
             n_kv_heads=2, n_seqs=2, table_stride=4, kv_dtype=qe.QE_KV_BF16)
    f.update(kw)
    return qe._CPages(*[f[n] for n, _ in qe._CPages._fields_])


BAD_PAGES = [
    (dict(k=None), qe.QE_ERR_ARG), (dict(v=None), qe.QE_ERR_ARG), (dict(table=None), qe.QE_ERR_ARG),
    (dict(lens=None), qe.QE_ERR_ARG), (dict(starts=None), qe.QE_ERR_ARG),
    (dict(kv_dtype=qe.QE_KV_FP8), qe.QE_ERR_ARG), (dict(kv_dtype=qe.QE_KV_F32), qe.QE_ERR_UNSUPPORTED),
    (dict(kv_dtype=9), qe.QE_ERR_UNSUPPORTED),
    (dict(page_size=0), qe.QE_ERR_ARG), (dict(page_size=8), qe.QE_ERR_ARG), (dict(page_size=48), qe.QE_ERR_ARG),
    (dict(page_size=1 << 17), qe.QE_ERR_ARG), (dict(n_pages=0), qe.QE_ERR_ARG), (dict(n_pages=1 << 31), qe.QE_ERR_ARG),
    (dict(n_kv_heads=0), qe.QE_ERR_ARG), (dict(n_kv_heads=1025), qe.QE_ERR_ARG), (dict(n_seqs=0), qe.QE_ERR_ARG),
    (dict(n_seqs=65537), qe.QE_ERR_ARG), (dict(table_stride=0), qe.QE_ERR_ARG),
    (dict(table_stride=1 << 27), qe.QE_ERR_ARG), (dict(k=ADDR + 8), qe.QE_ERR_ARG), (dict(v=ADDR + 2), qe.QE_ERR_ARG),
    (dict(table=ADDR + 1), qe.QE_ERR_ARG), (dict(lens=ADDR + 2), qe.QE_ERR_ARG),
    (dict(kv_dtype=qe.QE_KV_FP8, k_exp=ADDR, v_exp=ADDR + 3), qe.QE_ERR_ARG),
]


def calls(pages, rows=4, k=ADDR, v=ADDR, stride=256, dtype=qe.QE_KV_F32):
    L, p = qe.lib(), None if pages is None else ctypes.byref(pages)
    yield L.qe_op_page_append(p, k, v, rows, stride, dtype, None)
    yield L.qe_op_page_read(p, k, v, rows, stride, dtype, None)


def test_more_rows_than_a_launch_takes():
    assert list(calls(c_pages(n_kv_heads=1), rows=1 << 28, dtype=qe.QE_KV_BF16)) == [qe.QE_ERR_ARG] * 2
    assert list(calls(c_pages(n_kv_heads=1024), rows=(1 << 18) - 15, stride=1 << 17)) == [qe.QE_ERR_ARG] * 2


def attend(pages, rows=4, heads=4, q=ADDR, out=ADDR + 65536, qs=512, os=512, new=1, dtype=qe.QE_KV_F32, work=ADDR,
           size=None):
    L = qe.lib()
    size = L.qe_op_page_attention_work_bytes(heads, 2, new) if size is None else size
    return L.qe_op_page_attention(None if pages is None else ctypes.byref(pages), q, out, rows, heads, qs, os, new,
                                  dtype, work, size, None)


@pytest.mark.parametrize("kw,code", BAD_PAGES)
def test_pages_struct(kw, code):
    p = c_pages(**kw)
    assert list(calls(p)) == [code, code]
    assert attend(p) == code
    assert qe.lib().qe_last_error()


def test_rows_arguments():
    p = c_pages()
    for kw in (dict(k=None), dict(v=None), dict(k=ADDR + 4), dict(stride=255), dict(stride=258), dict(stride=1 << 33),
               dict(dtype=2), dict(dtype=-1), dict(rows=1 << 31), dict(dtype=qe.QE_KV_BF16, stride=260)):
        assert list(calls(p, **kw)) == [qe.QE_ERR_ARG] * 2, kw
    assert list(calls(None)) == [qe.QE_ERR_ARG] * 2
    assert list(calls(p, rows=0, k=None, v=None)) == [qe.QE_OK] * 2


def test_attention_arguments():
    p = c_pages()
    for kw in (dict(q=None), dict(out=None), dict(work=None), dict(heads=0), dict(heads=3), dict(heads=1 << 17),
               dict(q=ADDR + 8), dict(out=ADDR + 4), dict(work=ADDR + 8), dict(qs=511), dict(os=514), dict(qs=1 << 33),
               dict(dtype=2), dict(rows=1 << 31), dict(size=0)):
        assert attend(p, **kw) == qe.QE_ERR_ARG, kw
    assert attend(None) == qe.QE_ERR_ARG
    assert attend(p, rows=0, q=None, out=None, work=None) == qe.QE_OK
    L = qe.lib()
    assert L.qe_op_page_attention_work_bytes(3, 2, 1) == 0 and L.qe_op_page_attention_work_bytes(4, 0, 1) == 0
    assert L.qe_page_bytes(3, 16, 2, qe.QE_KV_BF16) == 3 * 16 * 2 * 128 * 2
    assert L.qe_page_bytes(3, 16, 2, qe.QE_KV_FP8) == 3 * 16 * 2 * 128 and L.qe_page_bytes(3, 16, 2, 0) == 0


def verify(logits=ADDR, rows=4, vocab=100, stride=100, starts=ADDR, seqs=1, drafts=ADDR, probs=None, pstride=0,
           accept=ADDR, sample=ADDR, tokens=ADDR, count=ADDR, work=ADDR, size=None):
    L = qe.lib()
    size = L.qe_op_verify_drafts_work_bytes(rows, seqs, vocab) if size is None else size
    return L.qe_op_verify_drafts(logits, rows, vocab, stride, starts, seqs, drafts, probs, pstride, accept, sample, None,
                                 tokens, count, None, work, size, None)


def test_verify_arguments():
    for kw in (dict(logits=None), dict(starts=None), dict(drafts=None), dict(accept=None), dict(sample=None),
               dict(tokens=None), dict(count=None), dict(work=None), dict(seqs=0), dict(seqs=65536), dict(vocab=0),
               dict(vocab=1 << 31, stride=1 << 31), dict(stride=99), dict(stride=1 << 33), dict(probs=ADDR, pstride=99),
               dict(rows=1 << 31, size=1 << 60), dict(size=0)):
        assert verify(**kw) == qe.QE_ERR_ARG, kw


def test_python_checks():
    """shapes, types and devices are refused in Python, before pointers are taken"""
    k = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)
    v = torch.zeros(4, 2, 1, 128, 16, dtype=torch.bfloat16)
    plan = (torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    e = torch.zeros(4, 2, 16, dtype=torch.uint8)
    f8 = (k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn))
    qe.Pages(k, v, *plan)
    qe.Pages(*f8, *plan, e, e)
    qe.Pages(f8[0].view(torch.uint8), f8[1].view(torch.uint8), *plan, e, e)
    bad = [(k.float(), v, *plan), (k, v[:, :, :, :, :8], *plan), (k, v.half(), *plan), (k[:, :, :, :64], v, *plan),
           (k[:, :, :12], v, *plan), (k.transpose(0, 1), v, *plan), (k, v, plan[0].long(), *plan[1:]),
           (k, v, plan[0][:1], *plan[1:]), (k, v, *plan[:2], plan[2][:2]), (k, v, *plan, e, e), (*f8, *plan),
           (*f8, *plan, e, e[:, :, :8]), (k, v, plan[0].T.contiguous().T, *plan[1:])]
    for args in bad:
        with pytest.raises(qe.QeError) as err:
            qe.Pages(*args)
        assert err.value.code == qe.QE_ERR_ARG
    with pytest.raises(qe.QeError) as err:
        qe.Pages.empty(4, 16, 2, *plan, kv_dtype=qe.QE_KV_F32)
    assert err.value.code == qe.QE_ERR_UNSUPPORTED
    p = qe.Pages(k, v, *plan)
    x = torch.zeros(5, 2, 128)
    w = torch.zeros(1 << 16, dtype=torch.uint8)
    for call in (lambda: qe.op_page_append(p, x, x), lambda: qe.op_page_read(p, x, x.double()),
                 lambda: qe.op_page_append(p, x[:, :1], x[:, :1]), lambda: qe.op_page_append(p, x.half(), x.half()),
                 lambda: qe.op_page_append(p, x.transpose(1, 2), x.transpose(1, 2)),
                 lambda: qe.op_page_attention(p, x, x, w), lambda: qe.op_page_attention(p, x, x[:4], w),
                 lambda: qe.op_page_attention(p, x.flatten(1), x.flatten(1), w),
                 lambda: qe.op_page_attention(p, x, x, w, -1)):
        with pytest.raises(qe.QeError) as err:
            call()
        assert err.value.code == qe.QE_ERR_ARG
    i, f = torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    good = dict(logits=torch.zeros(4, 10), starts=i[:2], drafts=i, accept=f, sample=f[:1], tokens=i, count=i[:1], work=w)
    for kw in ({}, dict(logits=f), dict(logits=torch.zeros(10, 4).T), dict(drafts=i.long()), dict(accept=f[:3]),
               dict(sample=f), dict(tokens=i[::2]), dict(count=i), dict(draft_probs=torch.zeros(4, 9)),
               dict(temperature=f), dict(logprobs=f.double()), dict(starts=i[:1])):
        with pytest.raises(qe.QeError) as err:
            qe.op_verify_drafts(**{**good, **kw})
        assert err.value.code == qe.QE_ERR_ARG, kw


def test_pages_struct_in_rust():
    fields = [n for n, _ in qe._CPages._fields_]
    assert c_struct_fields("qe_pages") == fields == rust_struct_fields("qe_pages")
