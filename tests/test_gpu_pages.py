"""Paged K/V cache on the GPU: rows into pages and back, and the attention over them, against plain
64-bit references."""
import math

import pytest
import torch

import qe
from page_cases import D, Case, attention_tolerance, pow2_rows

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def spaced(rows, heads, dtype, gap, fill=7.0):
    """rows [rows, heads, 128] whose rows lie heads * 128 + gap elements apart, and what they lie in"""
    base = torch.full((rows + 1, heads * D + gap), fill, dtype=dtype, device="cuda")
    return base[:rows, :heads * D].unflatten(1, (heads, D)), base


def attend(case, q, max_new=None, gap=0, stream=None):
    """out of op_page_attention as f64 on the host; rows of no sequence hold 7"""
    heads = q.shape[1]
    pages = case.pages()
    qd, _ = spaced(q.shape[0], heads, q.dtype, gap)
    qd.copy_(q)
    out, _ = spaced(q.shape[0], heads, q.dtype, 2 * gap)
    out.fill_(7.0)
    most = max(case.new) if max_new is None else max_new
    work = torch.empty(qe.op_page_attention_work_bytes(heads, case.n_kv, most), dtype=torch.uint8, device="cuda")
    work.fill_(0xFF)
    qe.op_page_attention(pages, qd, out, work, most, stream)
    torch.cuda.synchronize()
    return out.cpu().double()


def check_attention(case, heads, rows, max_new=None, gap=0, q_std=1.0, seed=3):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(case.total, heads, D, generator=g) * q_std).to(rows)
    want, worst, vmax = case.attention(q)
    got = attend(case, q, max_new, gap)
    mine = torch.zeros(case.total, dtype=torch.bool)
    mine[case.starts[0]:case.starts[-1]] = True
    assert torch.isfinite(got).all()
    assert (got[~mine] == 7.0).all(), "rows of no sequence were written"
    off = (got[mine] - want[mine]).abs().max() if mine.any() else 0.0
    assert off <= attention_tolerance(worst, vmax, rows), f"off by {off}"


# ---- rows into pages and back ----

APPEND = [
    # new tokens, cached before, page, n_kv
    ([1], [0], 16, 1),
    ([1, 1, 1], [15, 16, 300], 16, 8),
    ([5, 0, 33, 1], [14, 7, 0, 63], 64, 2),
    ([130, 16, 17], [3, 0, 31], 32, 3),
    ([300], [129], 256, 2),
]


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,page,n_kv", APPEND)
def test_append_and_read(gpu, new, ctx, page, n_kv, kv, rows):
    case = Case(new, ctx, page, n_kv, kv, seed=1, lead=2, tail=3)
    pages = case.pages()
    g = torch.Generator().manual_seed(2)
    x = {n: (torch.randn(case.total, n_kv, D, generator=g) * 3).to(rows) for n in "kv"}
    dev = {}
    for n in "kv":
        dev[n], _ = spaced(case.total, n_kv, rows, 24)
        dev[n].copy_(x[n])
    qe.op_page_append(pages, dev["k"], dev["v"])
    # the pages as they should be: the case's, with the new rows in their places
    want = {n: None if t is None else t.clone() for n, t in case.host.items()}
    bits = torch.uint8 if kv == "fp8" else torch.int16
    back = {n: torch.full((case.total, n_kv, D), 7.0, dtype=torch.float64) for n in "kv"}
    for s, n_new in enumerate(new):
        for i in range(n_new):
            t, pos = case.starts[s] + i, ctx[s] + i
            at, off = int(want["table"][s, pos // page]), pos % page
            for n in "kv":
                if kv == "fp8":
                    y, e = pow2_rows(x[n][t].double())
                    want[n + "e"][at, :, off] = e
                    back[n][t] = y * torch.exp2(e.double() - 127)[..., None]
                    y = y.to(torch.float8_e4m3fn)
                else:
                    y = x[n][t].bfloat16()
                    back[n][t] = y.double()
                if n == "k":
                    want["k"].view(bits)[at, :, off] = y.view(bits)
                else:
                    want["v"].view(bits)[at, :, off // 16, :, off % 16] = y.view(bits)
    for n in ("k", "v", "ke", "ve"):
        if want[n] is not None:
            a, b = case.dev[n].cpu(), want[n]
            if n in "kv":
                a, b = a.view(bits), b.view(bits)
            assert torch.equal(a, b), n
    out = {n: spaced(case.total, n_kv, rows, 8)[0] for n in "kv"}
    qe.op_page_read(pages, out["k"], out["v"])
    for n in "kv":
        assert torch.equal(out[n].cpu(), back[n].to(rows)), n


def test_append_special_values(gpu):
    """rows of zeros, of subnormals, with infinities and NaN, at the edge of the scale's steps and of
    f32's range, and ties between two e4m3 values"""
    g = torch.Generator().manual_seed(4)
    rows = []
    rows.append(torch.zeros(D))
    rows.append(torch.randn(D, generator=g) * 1e-42)
    rows.append(torch.cat([torch.tensor([math.inf, -math.inf, math.nan]), torch.randn(D - 3, generator=g)]))
    rows.append(torch.full((D,), math.inf))
    for top in (448.0, 448.0001, 447.99, 1.75, 1.7500001, 3.4e38, 2.0 ** -120, 2.0 ** -126):
        rows.append(torch.cat([torch.tensor([top, -top]), torch.randn(D - 2, generator=g) * top * 0.1]))
    ties = torch.arange(D).float() * 0.0 + 1.0625  # halfway between 1.0 and 1.125
    ties[1::2] = 1.1875                            # halfway between 1.125 and 1.25
    ties[0] = 448.0
    rows.append(ties)
    small = torch.full((D,), 2.0 ** -10)  # half of the smallest e4m3 step: to zero; 1.5 of it: up to even
    small[0], small[1] = 448.0, 3 * 2.0 ** -10
    rows.append(small)
    x = torch.stack(rows)[:, None].contiguous()
    case = Case([len(rows)], [0], 16, 1, "fp8", seed=1)
    pages = case.pages()
    xd = x.cuda()
    qe.op_page_append(pages, xd, -xd)
    for n, sign in (("k", 1), ("v", -1)):
        y, e = pow2_rows(x.double() * sign)
        got_e = case.dev[n + "e"].cpu()
        for i in range(len(rows)):
            at, off = int(case.host["table"][0, i // 16]), i % 16
            assert int(got_e[at, 0, off]) == int(e[i, 0]), (n, i)
            raw = case.dev[n].view(torch.uint8).cpu().view(torch.float8_e4m3fn)
            z = raw[at, 0, off] if n == "k" else raw.view(torch.uint8)[at, 0, off // 16, :, off % 16].contiguous().view(
                torch.float8_e4m3fn)
            z = z.double()
            assert torch.equal(torch.isnan(z), torch.isnan(y[i, 0])), (n, i)
            assert torch.equal(torch.nan_to_num(z), torch.nan_to_num(y[i, 0])), (n, i)
    case = Case([3], [0], 16, 1, "bf16", seed=1)
    pages = case.pages()
    x = torch.randn(3, 1, D, generator=g)
    x[0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.39e38])
    xd, out = x.cuda(), [torch.empty(3, 1, D, device="cuda") for _ in "kv"]
    qe.op_page_append(pages, xd, xd)
    qe.op_page_read(pages, *out)
    for o in out:
        torch.testing.assert_close(o.cpu(), x.bfloat16().float(), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("entry", [-1, 1 << 30, -(1 << 31)])
def test_pages_that_are_not_there(gpu, entry):
    """append writes nothing there, read gives zeros, attention leaves the positions out; a sequence
    with no page at all gives zeros; lengths past the table and negative positions are the same"""
    new, ctx = [20, 5, 3], [30, 0, 40]
    holes = [(0, 1, entry), (0, 3, entry), (1, 0, entry)]
    case = Case(new, ctx, 16, 2, "fp8", seed=5, holes=holes)
    for rows in (F32, BF16):
        check_attention(case, 4, rows)
    pages = case.pages()
    x = torch.randn(case.total, 2, D, device="cuda")
    before = {n: case.dev[n].view(torch.uint8).clone() for n in ("k", "v", "ke", "ve")}
    qe.op_page_append(pages, x, x)
    named = set(int(p) for p in case.host["table"].flatten() if 0 <= p < case.n_pages)
    for n, t in before.items():
        for at in range(case.n_pages):
            if at not in named:
                assert torch.equal(case.dev[n].view(torch.uint8)[at], t[at]), (n, at)
    k, v = torch.full_like(x, 9.0), torch.full_like(x, 9.0)
    qe.op_page_read(pages, k, v)
    for s, n_new in enumerate(new):
        for i in range(n_new):
            t = case.starts[s] + i
            there = bool(case.seen[s][ctx[s] + i])
            assert bool((k[t] == 0).all()) != there and bool((v[t] == 0).all()) != there


def test_a_plan_that_does_not_fit(gpu):
    """a length past the table: the positions behind it have no page; a length below the number of new
    rows: rows before position 0 attend nothing"""
    case = Case([4, 6], [12, 10], 16, 1, "bf16", seed=6)
    q = torch.randn(case.total, 2, D)
    case.host["lens"] = torch.tensor([1 << 30, 3], dtype=torch.int32)
    got = attend(case, q)
    k, v = (x[0] for x in case.rows[0])
    assert case.lens[0] == 16
    table = case.host["table"]
    if table.shape[1] == 1:
        for t in range(4):
            w = torch.softmax(q[t].double() @ k.T / math.sqrt(D), -1) @ v
            assert (got[t] - w).abs().max() < 1e-4
    assert (got[4:7] == 0).all()
    k, v = (x[0] for x in case.rows[1])
    for i in range(3):
        w = torch.softmax(q[7 + i].double() @ k[:i + 1].T / math.sqrt(D), -1) @ v[:i + 1]
        assert (got[7 + i] - w).abs().max() < 1e-4
    x = torch.randn(case.total, 1, D, device="cuda")
    pages = case.pages()
    k, v = torch.full_like(x, 9.0), torch.full_like(x, 9.0)
    qe.op_page_append(pages, x, x)
    qe.op_page_read(pages, k, v)
    assert (k[:7] == 0).all() and (v[:7] == 0).all()
    assert torch.equal(k[7:], x[7:].bfloat16().float())


# ---- attention ----

SHAPES = [
    # new tokens, cached before, page, n_kv, heads
    ([1], [0], 16, 8, 16),
    ([1], [196], 64, 8, 16),
    ([1, 1, 1, 1, 1], [0, 15, 16, 63, 700], 16, 2, 8),
    ([5, 5], [60, 123], 32, 2, 4),
    ([3, 0, 7, 1], [125, 20, 0, 64], 16, 1, 3),
    ([8, 2], [500, 90], 128, 1, 16),
    ([17], [47], 16, 2, 2),
    ([70, 1, 33], [10, 300, 0], 32, 2, 4),
    ([129, 64], [0, 191], 64, 1, 2),
    ([200, 1, 1], [77, 130, 5], 256, 1, 5),
    ([31], [1000], 16, 2, 8),
]


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,page,n_kv,heads", SHAPES)
def test_attention(gpu, new, ctx, page, n_kv, heads, kv, rows):
    check_attention(Case(new, ctx, page, n_kv, kv, seed=11, lead=1, tail=2, spare=1), heads, rows, gap=16)


@pytest.mark.parametrize("max_new", [0, 1, 9, 400])
@pytest.mark.parametrize("rows", [F32, BF16])
def test_attention_any_max_new(gpu, max_new, rows):
    """max_new only chooses how the work is cut up"""
    check_attention(Case([150, 1, 4], [20, 200, 61], 16, 2, "fp8", seed=12), 4, rows, max_new=max_new)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_attention_long(gpu, kv):
    """a long axis: many runs that are joined, and sequences of one and a few tokens beside it"""
    check_attention(Case([1, 1, 2], [9000, 3, 4100], 64, 1, kv, seed=13), 2, F32)


@pytest.mark.parametrize("rows", [F32, BF16])
def test_attention_peaked_scores(gpu, rows):
    """scores of some hundred: weights of 1 and of nothing, maxima that rise along the positions"""
    check_attention(Case([40, 1], [90, 260], 16, 1, "bf16", seed=14, k_std=6.0), 2, rows, q_std=6.0)


@pytest.mark.parametrize("n_seqs", [300])
def test_attention_many_sequences(gpu, n_seqs):
    new = [(i * 7) % 3 for i in range(n_seqs)]
    ctx = [(i * 37) % 90 for i in range(n_seqs)]
    check_attention(Case(new, ctx, 16, 1, "bf16", seed=15), 2, F32)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,heads", [(6, 2), (100, 2)])
def test_values_that_are_masked(gpu, bad, rows, new, heads):
    """NaN and infinities in K and V of a later token reach only the rows that attend it"""
    case = Case([new], [40], 16, 1, "bf16", seed=16)
    at = 40 + new // 2
    for n in "kv":
        page, off = int(case.host["table"][0, at // 16]), at % 16
        if n == "k":
            case.host["k"][page, 0, off, 5] = bad
        else:
            case.host["v"][page, 0, off // 16, 9, off % 16] = bad
    q = torch.randn(new, heads, D, generator=torch.Generator().manual_seed(7)).to(rows)
    want, worst, vmax = case.attention(q)
    got = attend(case, q)
    tol = attention_tolerance(worst, vmax, rows)
    assert (got[:new // 2] - want[:new // 2]).abs().max() <= tol
    assert not torch.isfinite(got[new // 2:]).all()


def test_query_that_is_not_finite(gpu):
    """a NaN in one row's query stays in that row and head"""
    case = Case([9, 40], [50, 3], 16, 1, "bf16", seed=17)
    q = torch.randn(case.total, 4, D, generator=torch.Generator().manual_seed(8))
    want, worst, vmax = case.attention(q)
    bad = q.clone()
    bad[4, 2, 7] = math.nan
    bad[30, 1, 0] = math.nan
    got = attend(case, bad)
    hit = torch.zeros(case.total, 4, dtype=torch.bool)
    hit[4, 2] = hit[30, 1] = True
    assert torch.isnan(got[hit]).all()
    assert (got[~hit] - want[~hit]).abs().max() <= attention_tolerance(worst, vmax, F32)


@pytest.mark.parametrize("new", [[1, 1, 1], [90, 3, 50]])
def test_same_result_every_time(gpu, new):
    """the cut of the work is fixed by the plan: bit-identical results"""
    case = Case(new, [700, 30, 300], 32, 2, "fp8", seed=18)
    q = torch.randn(case.total, 8, D)
    a = attend(case, q)
    for _ in range(3):
        assert torch.equal(attend(case, q), a)


def test_pages_past_32_bits(gpu):
    """pages whose bytes lie beyond 4 GiB: offsets are 64 bits wide"""
    n_kv, page = 8, 256
    n_pages = (5 << 30) // (n_kv * page * D * 2)
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([600], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 600], dtype=torch.int32, device="cuda")
    pages = qe.Pages.empty(n_pages, page, n_kv, table, lens, starts)
    k, v = (torch.randn(600, n_kv, D, device="cuda").bfloat16() for _ in "kv")
    qe.op_page_append(pages, k, v)
    out = [torch.empty_like(k) for _ in "kv"]
    qe.op_page_read(pages, *out)
    assert torch.equal(out[0], k) and torch.equal(out[1], v)
    q = torch.randn(600, n_kv, D, device="cuda")
    o = torch.empty_like(q)
    work = torch.empty(qe.op_page_attention_work_bytes(n_kv, n_kv, 600), dtype=torch.uint8, device="cuda")
    qe.op_page_attention(pages, q, o, work, 600)
    w = torch.softmax(q[599, 3].double() @ k[:, 3].double().T / math.sqrt(D), -1) @ v[:, 3].double()
    assert (o[599, 3].double() - w).abs().max() < 1e-4


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("n_seqs,most,longest", [(65, 1, 2000), (65, 3, 5000), (64, 2, 300), (1500, 2, 40), (70, 100, 30)])
def test_attention_of_batches(gpu, n_seqs, most, longest, rows, kv):
    """batches on both sides of what a wave plans alone, with sequences that have no new token; items dealt
    out whole and, where one sequence is much longer than the rest, cut"""
    new = [i % (most + 1) for i in range(n_seqs)]
    ctx = [(i * 37) % 40 for i in range(n_seqs)]
    ctx[n_seqs // 2] = longest
    new[n_seqs // 2] = most
    check_attention(Case(new, ctx, 32, 1, kv, seed=19, lead=3, tail=20), 2, rows, gap=8)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_append_to_many_sequences(gpu, kv):
    """more sequences than the search keeps on chip"""
    n_seqs = 1500
    case = Case([i % 3 for i in range(n_seqs)], [(i * 11) % 30 for i in range(n_seqs)], 16, 1, kv, seed=20, lead=1, tail=9)
    pages = case.pages()
    x = torch.randn(case.total, 1, D, generator=torch.Generator().manual_seed(4))
    k, v = (torch.full_like(x, 9.0).cuda() for _ in "kv")
    qe.op_page_append(pages, x.cuda(), -x.cuda())
    qe.op_page_read(pages, k, v)
    if kv == "fp8":
        y, e = pow2_rows(x.double())
        y = (y * torch.exp2(e.double() - 127)[..., None]).float()
    else:
        y = x.bfloat16().float()
    mine = slice(case.starts[0], case.starts[-1])
    assert torch.equal(k.cpu()[mine], y[mine]) and torch.equal(v.cpu()[mine], -y[mine])
    for t in (k, v):
        assert (t[:case.starts[0]] == 9).all() and (t[case.starts[-1]:] == 9).all()


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,heads", [(6, 2), (100, 2)])
def test_e4m3_values_that_are_masked(gpu, rows, new, heads):
    """NaN in e4m3 pages at a later token reaches only the rows that attend it"""
    case = Case([new], [40], 16, 1, "fp8", seed=16)
    at = 40 + new // 2
    page, off = int(case.host["table"][0, at // 16]), at % 16
    q = torch.randn(new, heads, D, generator=torch.Generator().manual_seed(7)).to(rows)
    want, worst, vmax = case.attention(q)
    case.host["k"].view(torch.uint8)[page, 0, off, 5] = 0x7F
    case.host["v"].view(torch.uint8)[page, 0, off // 16, 9, off % 16] = 0xFF
    got = attend(case, q)
    assert (got[:new // 2] - want[:new // 2]).abs().max() <= attention_tolerance(worst, vmax, rows)
    assert torch.isnan(got[new // 2:]).any(-1).all()


def test_calls_on_two_streams(gpu):
    """two plans on two streams at once, each with work of its own, as eager calls and as graphs"""
    cases = [Case([1, 3, 2], [900, 40, 333], 16, 2, "bf16", seed=23), Case([150, 20], [60, 700], 32, 2, "fp8", seed=24)]
    qs = [torch.randn(c.total, 4, D, generator=torch.Generator().manual_seed(5)) for c in cases]
    alone = [attend(c, q) for c, q in zip(cases, qs)]
    pages, qd = [c.pages() for c in cases], [q.cuda() for q in qs]
    outs = [torch.empty_like(q) for q in qd]
    works = [torch.empty(qe.op_page_attention_work_bytes(4, 2, max(c.new)), dtype=torch.uint8, device="cuda") for c in cases]
    streams, graphs = [torch.cuda.Stream() for _ in cases], []
    torch.cuda.synchronize()

    def call(i):
        qe.op_page_attention(pages[i], qd[i], outs[i], works[i], max(cases[i].new))

    def same():
        torch.cuda.synchronize()
        for o, a in zip(outs, alone):
            assert torch.equal(o.cpu().double(), a)
            o.zero_()
        torch.cuda.synchronize()

    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                call(i)
    same()
    for i, st in enumerate(streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=st):
            call(i)
    torch.cuda.synchronize()
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
        same()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx", [([1 + i % 3 for i in range(40)], [(i * 397) % 3000 for i in range(40)]),
                                     ([1, 0, 4, 1], [12000, 50, 700, 5000]),
                                     ([190, 0, 70, 1, 120], [1500, 9, 100, 2500, 800])])
def test_attention_of_ragged_batches(gpu, new, ctx, rows, kv):
    """few sequences of very different lengths: parts of one size that end with their item"""
    check_attention(Case(new, ctx, 64, 2, kv, seed=25, lead=2, tail=5), 4, rows, gap=8)


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,n_kv,heads", [([1], [9000], 1, 16), ([12], [7000], 1, 2), ([2, 1, 1], [6000, 20, 300], 2, 12),
                                                ([20, 1], [5000, 900], 1, 8), ([20], [9000], 1, 16), ([40, 3], [3000, 100], 1, 8)])
def test_attention_of_many_parts(gpu, new, ctx, n_kv, heads, rows):
    """a long axis and many q heads of a KV head: parts that the workgroups join together"""
    check_attention(Case(new, ctx, 64, n_kv, "bf16", seed=26, lead=1), heads, rows)
