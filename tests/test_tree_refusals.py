"""What the draft-tree and eviction operators refuse, before anything reaches a device: runs without a
GPU."""
import ctypes

import pytest
import torch

import qe
from test_pages_refusals import ADDR, BAD_PAGES, c_pages

MB = 1 << 20


def tree(pages, parents=ADDR, rows=4, heads=4, q=ADDR + MB, out=ADDR + 2 * MB, qs=512, os=512, new=1, dtype=qe.QE_KV_F32,
         work=ADDR + 64 * MB, size=None):
    L = qe.lib()
    size = L.qe_op_page_attention_work_bytes(heads, 2, new) if size is None else size
    return L.qe_op_page_tree_attention(None if pages is None else ctypes.byref(pages), parents, q, out, rows, heads, qs, os,
                                       new, dtype, work, size, None)


def weigh(pages, rows=4, heads=4, q=ADDR + MB, qs=512, new=1, dtype=qe.QE_KV_F32, mass=ADDR + 2 * MB, stride=64,
          work=ADDR + 3 * MB, size=None):
    L = qe.lib()
    size = L.qe_op_page_weigh_work_bytes(rows, heads, 2, 2, 64, new) if size is None else size
    return L.qe_op_page_weigh(None if pages is None else ctypes.byref(pages), q, rows, heads, qs, new, dtype, mass, stride,
                              work, size, None)


def move(pages, src=ADDR + MB, heads=2, stride=8, count=ADDR + 2 * MB, first=None, mass=None, mstride=0):
    return qe.lib().qe_op_page_move(None if pages is None else ctypes.byref(pages), src, heads, stride, count, first, mass,
                                    mstride, None)


def keep(mass=ADDR, stride=100, lens=ADDR + MB, seqs=2, heads=2, keep=10, sinks=1, recent=2, kept=ADDR + 2 * MB, kstride=10,
         count=ADDR + 3 * MB):
    return qe.lib().qe_op_page_keep(mass, stride, lens, seqs, heads, keep, sinks, recent, kept, kstride, count, None)


def check(logits=ADDR, rows=4, vocab=100, stride=100, starts=ADDR + MB, seqs=1, parents=ADDR + 2 * MB, nodes=ADDR + 3 * MB,
          accept=ADDR + 4 * MB, sample=ADDR + 5 * MB, temperature=None, depth=0, tokens=ADDR + 6 * MB, path=ADDR + 7 * MB,
          count=ADDR + 8 * MB, logprobs=None, work=ADDR + 9 * MB, size=None):
    L = qe.lib()
    size = L.qe_op_verify_tree_work_bytes(rows, seqs, vocab) if size is None else size
    return L.qe_op_verify_tree(logits, rows, vocab, stride, starts, seqs, parents, nodes, accept, sample, temperature, depth,
                               tokens, path, count, logprobs, work, size, None)


@pytest.mark.parametrize("kw,code", BAD_PAGES)
def test_pages_struct(kw, code):
    p = c_pages(**kw)
    assert [tree(p), weigh(p, stride=1 << 20), move(p)] == [code] * 3
    assert qe.lib().qe_last_error()


def test_tree_arguments():
    p = c_pages()
    for kw in (dict(q=None), dict(out=None), dict(work=None), dict(parents=None), dict(parents=ADDR + 2), dict(heads=0),
               dict(heads=3), dict(heads=1 << 17), dict(q=ADDR + 8), dict(out=ADDR + 4), dict(work=ADDR + 8), dict(qs=511),
               dict(os=514), dict(qs=1 << 33), dict(dtype=2), dict(rows=1 << 31), dict(size=0), dict(new=65),
               dict(out=ADDR + MB), dict(out=ADDR + MB + 4096), dict(out=ADDR), dict(parents=ADDR + 2 * MB + 8188),
               dict(parents=ADDR + 64 * MB + 4), dict(work=ADDR - 16)):
        assert tree(p, **kw) == qe.QE_ERR_ARG, kw
    assert tree(None) == qe.QE_ERR_ARG
    assert tree(p, rows=0, q=None, out=None, work=None, parents=None) == qe.QE_OK


def test_weigh_arguments():
    p = c_pages()
    for kw in (dict(q=None), dict(mass=None), dict(work=None), dict(heads=0), dict(heads=3), dict(heads=1 << 17),
               dict(q=ADDR + 8), dict(mass=ADDR + 2), dict(work=ADDR + 8), dict(qs=511), dict(qs=514), dict(qs=1 << 33),
               dict(dtype=2), dict(rows=1 << 31), dict(size=0), dict(stride=63), dict(stride=1 << 31),
               dict(mass=ADDR), dict(mass=ADDR + MB + 8188), dict(mass=ADDR + MB - 1020), dict(work=ADDR + 2 * MB),
               dict(work=ADDR + 2 * MB + 1008)):
        assert weigh(p, **kw) == qe.QE_ERR_ARG, kw
    assert weigh(None) == qe.QE_ERR_ARG
    assert weigh(p, rows=0, q=None, mass=None, work=None) == qe.QE_OK
    L = qe.lib()
    assert L.qe_op_page_weigh_work_bytes(4, 3, 2, 1, 64, 1) == 0 and L.qe_op_page_weigh_work_bytes(4, 4, 0, 1, 64, 1) == 0


def test_move_arguments():
    p = c_pages()
    f8 = c_pages(kv_dtype=qe.QE_KV_FP8, k_exp=ADDR + 3 * MB, v_exp=ADDR + 4 * MB)
    for pages, kw in ((p, dict(src=None)), (p, dict(count=None)), (p, dict(heads=0)), (p, dict(heads=3)), (p, dict(stride=0)),
                      (p, dict(stride=1 << 31)), (p, dict(src=ADDR + MB + 1)), (p, dict(count=ADDR + 2)),
                      (p, dict(first=ADDR + MB + 2)), (p, dict(mass=ADDR + 5 * MB + 2, mstride=8)),
                      (p, dict(mass=ADDR + 5 * MB, mstride=0)), (p, dict(mass=ADDR + 5 * MB, mstride=1 << 31)),
                      (p, dict(src=ADDR + 8)), (p, dict(count=ADDR + 65536 - 4)), (p, dict(first=ADDR)),
                      (p, dict(mass=ADDR + MB, mstride=8)), (p, dict(mass=ADDR, mstride=8)),
                      (f8, dict(src=ADDR + 3 * MB)), (f8, dict(mass=ADDR + 4 * MB, mstride=8)),
                      (c_pages(n_kv_heads=1024, n_seqs=512), dict(heads=1))):
        assert move(pages, **kw) == qe.QE_ERR_ARG, kw
    assert move(None) == qe.QE_ERR_ARG


def test_keep_arguments():
    for kw in (dict(mass=None), dict(lens=None), dict(kept=None), dict(count=None), dict(seqs=0), dict(seqs=65537),
               dict(heads=0), dict(heads=1025), dict(seqs=1 << 12, heads=1 << 10), dict(stride=0), dict(stride=1 << 31),
               dict(kstride=1 << 31), dict(keep=0), dict(keep=11), dict(sinks=11), dict(sinks=5, recent=6), dict(recent=1 << 63),
               dict(mass=ADDR + 2), dict(lens=ADDR + MB + 1), dict(kept=ADDR + 2 * MB + 3), dict(count=ADDR + 3 * MB + 1),
               dict(kept=ADDR + 1596), dict(kept=ADDR + MB), dict(count=ADDR), dict(count=ADDR + MB + 4),
               dict(count=ADDR + 2 * MB + 156)):
        assert keep(**kw) == qe.QE_ERR_ARG, kw


def test_check_arguments():
    for kw in (dict(logits=None), dict(starts=None), dict(parents=None), dict(nodes=None), dict(accept=None), dict(sample=None),
               dict(tokens=None), dict(path=None), dict(count=None), dict(work=None), dict(seqs=0), dict(seqs=65536),
               dict(vocab=0), dict(vocab=1 << 31, stride=1 << 31), dict(stride=99), dict(stride=1 << 33),
               dict(rows=1 << 31, size=1 << 60), dict(size=0), dict(work=ADDR + 9 * MB + 8), dict(parents=ADDR + 2),
               dict(path=ADDR + 7 * MB + 2), dict(logprobs=ADDR + 3), dict(temperature=ADDR + 1),
               dict(tokens=ADDR), dict(path=ADDR + 6 * MB), dict(logprobs=ADDR + 4 * MB), dict(work=ADDR + 2 * MB),
               dict(count=ADDR + 9 * MB + 8), dict(tokens=ADDR + 5 * MB), dict(logprobs=ADDR + 6 * MB + 12)):
        assert check(**kw) == qe.QE_ERR_ARG, kw


def test_python_checks():
    """shapes, types and devices are refused in Python, before pointers are taken"""
    k = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)
    v = torch.zeros(4, 2, 1, 128, 16, dtype=torch.bfloat16)
    p = qe.Pages(k, v, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    x, w = torch.zeros(5, 4, 128), torch.zeros(1 << 16, dtype=torch.uint8)
    i, f, m = torch.zeros(5, dtype=torch.int32), torch.zeros(5), torch.zeros(2, 2, 48)
    two, kept = i[:2], torch.zeros(2, 2, 9, dtype=torch.int32)
    calls = [lambda: qe.op_page_tree_attention(p, i, x, x, w), lambda: qe.op_page_tree_attention(p, i[:4], x, x, w),
             lambda: qe.op_page_tree_attention(p, i.long(), x, x, w), lambda: qe.op_page_tree_attention(p, i, x, x[:4], w),
             lambda: qe.op_page_tree_attention(p, i, x.half(), x.half(), w),
             lambda: qe.op_page_tree_attention(p, i, x, x, w, -1),
             lambda: qe.op_page_weigh(p, x, m, w), lambda: qe.op_page_weigh(p, x, m.double(), w),
             lambda: qe.op_page_weigh(p, x, m[:1], w), lambda: qe.op_page_weigh(p, x, m[0], w),
             lambda: qe.op_page_weigh(p, x, m.transpose(0, 1), w, -2), lambda: qe.op_page_weigh(p, x.half(), m, w),
             lambda: qe.op_page_weigh(p, x, m[:, :, ::2], w),
             lambda: qe.op_page_keep(m, two, kept, two, 4), lambda: qe.op_page_keep(m, i, kept, two, 4),
             lambda: qe.op_page_keep(m, two, kept.long(), two, 4), lambda: qe.op_page_keep(m, two, kept[0], two, 4),
             lambda: qe.op_page_keep(m, two, kept, two.long(), 4), lambda: qe.op_page_keep(m.half(), two, kept, two, 4),
             lambda: qe.op_page_keep(m, two, kept, two, 4, -1),
             lambda: qe.op_page_move(p, kept, two), lambda: qe.op_page_move(p, kept[:, :1], two),
             lambda: qe.op_page_move(p, kept[0, 0], two), lambda: qe.op_page_move(p, kept.long(), two),
             lambda: qe.op_page_move(p, kept, i), lambda: qe.op_page_move(p, kept, two, first=i),
             lambda: qe.op_page_move(p, kept, two, mass=f), lambda: qe.op_page_move(p, kept[:, 0], two)]
    for n, call in enumerate(calls):
        with pytest.raises(qe.QeError) as err:
            call()
        assert err.value.code == qe.QE_ERR_ARG, n
    good = dict(logits=torch.zeros(5, 10), starts=i[:2], parents=i, nodes=i, accept=f, sample=f[:1], tokens=i,
                path=torch.zeros(1, 64, dtype=torch.int32), count=i[:1], work=w)
    for kw in ({}, dict(logits=f), dict(logits=torch.zeros(10, 5).T), dict(nodes=i.long()), dict(accept=f[:3]),
               dict(sample=f), dict(tokens=i[::2]), dict(count=i), dict(parents=f), dict(path=i), dict(max_depth=-1),
               dict(temperature=f), dict(logprobs=f.double()), dict(starts=i[:1])):
        with pytest.raises(qe.QeError) as err:
            qe.op_verify_tree(**{**good, **kw})
        assert err.value.code == qe.QE_ERR_ARG, kw


def test_nodes_of_a_tree():
    """the count of nodes of a tree in the header and here"""
    text = open(qe.os.path.join(qe.os.path.dirname(qe._HERE), "include", "qe.h")).read()
    assert f"#define QE_TREE_NODES {qe.QE_TREE_NODES}\n" in text
