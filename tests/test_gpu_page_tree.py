"""Attention of trees of drafted tokens over the paged cache, against plain 64-bit references."""
import math

import pytest
import torch

import qe
from page_cases import D, Case, attention_tolerance
from test_gpu_pages import BF16, F32, spaced
from tree_cases import family, packed, random_tree, tree_attention

pytestmark = pytest.mark.gpu


def attend(case, parents, q, max_new=None, gap=0):
    """out of op_page_tree_attention as f64 on the host; rows of no sequence hold 7"""
    heads = q.shape[1]
    pages = case.pages()
    qd, _ = spaced(q.shape[0], heads, q.dtype, gap)
    qd.copy_(q)
    out, _ = spaced(q.shape[0], heads, q.dtype, 2 * gap)
    out.fill_(7.0)
    most = min(64, max(case.new)) if max_new is None else max_new
    work = torch.empty(qe.op_page_attention_work_bytes(heads, case.n_kv, most), dtype=torch.uint8, device="cuda")
    work.fill_(0xFF)
    qe.op_page_tree_attention(pages, parents.cuda(), qd, out, work, most)
    torch.cuda.synchronize()
    return out.cpu().double()


def check(case, trees, heads, rows, max_new=None, gap=0, q_std=1.0, seed=3):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(case.total, heads, D, generator=g) * q_std).to(rows)
    want, worst, vmax = tree_attention(case, trees, q)
    got = attend(case, packed(case, trees), q, max_new, gap)
    mine = torch.zeros(case.total, dtype=torch.bool)
    mine[case.starts[0]:case.starts[-1]] = True
    assert torch.isfinite(got).all()
    assert (got[~mine] == 7.0).all(), "rows of no sequence were written"
    off = (got[mine] - want[mine]).abs().max() if mine.any() else 0.0
    assert off <= attention_tolerance(worst, vmax, rows), f"off by {off}"


SHAPES = [
    # nodes, cached before, page, n_kv, heads
    ([1], [0], 16, 8, 16),
    ([13], [184], 64, 8, 16),
    ([1, 5, 1, 9, 2], [0, 15, 16, 63, 700], 16, 2, 8),
    ([16, 3], [60, 123], 32, 2, 2),
    ([3, 0, 7, 1], [125, 20, 0, 64], 16, 1, 3),
    ([33, 2], [500, 90], 128, 1, 16),
    ([17], [47], 16, 2, 2),
    ([64, 1, 33], [10, 300, 0], 32, 2, 4),
    ([64, 50], [0, 191], 64, 1, 2),
    ([61, 1, 1], [77, 130, 5], 256, 1, 5),
    ([31], [1000], 16, 2, 8),
    ([64, 64], [1200, 31], 64, 1, 8),
]


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,page,n_kv,heads", SHAPES)
def test_trees(gpu, new, ctx, page, n_kv, heads, kv, rows):
    case = Case(new, ctx, page, n_kv, kv, seed=61, lead=1, tail=2, spare=1)
    check(case, [random_tree(n, 100 + i) for i, n in enumerate(new)], heads, rows, gap=16)


@pytest.mark.parametrize("max_new", [0, 1, 9, 64])
@pytest.mark.parametrize("rows", [F32, BF16])
def test_any_max_new(gpu, max_new, rows):
    """max_new only chooses how the work is cut up"""
    new = [60, 1, 4]
    check(Case(new, [20, 200, 61], 16, 2, "fp8", seed=62), [random_tree(n, n) for n in new], 4, rows, max_new=max_new)


KINDS = {
    "chain": lambda n: [i - 1 for i in range(n)],
    "star": lambda n: [-1] + [0] * (n - 1),
    "forest": lambda n: random_tree(n, 5, roots=n // 3 + 1),
    "alone": lambda n: [-1] * n,
    "two chains": lambda n: [i - 2 if i > 1 else i - 1 for i in range(n)],
    "no parents by other values": lambda n: [(-7, i, n + 3, 1 << 30, -(1 << 31), 0 if i else -1)[i % 6] for i in range(n)],
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kv,rows,heads", [("bf16", F32, 2), ("fp8", BF16, 4), ("bf16", BF16, 16), ("fp8", F32, 8)])
def test_kinds_of_trees(gpu, kind, kv, rows, heads):
    new = [64, 20, 7]
    check(Case(new, [100, 0, 333], 16, 2, kv, seed=63), [KINDS[kind](n) for n in new], heads, rows)


@pytest.mark.parametrize("rows", [F32, BF16])
def test_a_chain_is_causal(gpu, rows):
    """chains give what op_page_attention gives, within both's error"""
    case = Case([30, 5], [200, 900], 32, 2, "bf16", seed=64)
    q = torch.randn(case.total, 4, D, generator=torch.Generator().manual_seed(3)).to(rows)
    want, worst, vmax = case.attention(q)
    got = attend(case, packed(case, [KINDS["chain"](n) for n in case.new]), q)
    assert (got - want).abs().max() <= attention_tolerance(worst, vmax, rows)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,n_kv,heads", [([1, 9, 2], [9000, 3, 4100], 1, 2), ([12], [7000], 1, 2), ([64, 3], [6000, 100], 1, 8),
                                                ([20], [9000], 1, 16)])
def test_long(gpu, new, ctx, n_kv, heads, rows, kv):
    """a long axis: many parts that are joined"""
    check(Case(new, ctx, 64, n_kv, kv, seed=65, lead=1), [random_tree(n, n) for n in new], heads, rows)


@pytest.mark.parametrize("rows", [F32, BF16])
def test_peaked_scores(gpu, rows):
    """scores of some hundred: weights of 1 and of nothing"""
    new = [40, 6]
    check(Case(new, [90, 260], 16, 1, "bf16", seed=66, k_std=6.0), [random_tree(n, n) for n in new], 2, rows, q_std=6.0)


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("n_seqs,most", [(70, 3), (300, 2), (66, 64)])
def test_many_sequences(gpu, n_seqs, most, rows):
    new = [(i * 7) % (most + 1) for i in range(n_seqs)]
    ctx = [(i * 37) % 90 for i in range(n_seqs)]
    ctx[n_seqs // 2] = 900
    check(Case(new, ctx, 16, 1, "bf16", seed=67), [random_tree(n, i) for i, n in enumerate(new)], 2, rows)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("n,heads", [(9, 2), (64, 2), (60, 8)])
def test_values_of_other_branches(gpu, bad, rows, n, heads, kv):
    """NaN and infinities in K and V of a node reach that node and those below it, and no other"""
    case = Case([n], [40], 16, 1, kv, seed=68)
    tree = random_tree(n, 11)
    q = torch.randn(n, heads, D, generator=torch.Generator().manual_seed(7)).to(rows)
    want, worst, vmax = tree_attention(case, [tree], q)
    node = n // 3
    page, off = int(case.host["table"][0, (40 + node) // 16]), (40 + node) % 16
    k, v = case.host["k"], case.host["v"]
    if kv == "fp8":
        k.view(torch.uint8)[page, 0, off, 5] = 0x7F
        v.view(torch.uint8)[page, 0, off // 16, 9, off % 16] = 0xFF
    else:
        k[page, 0, off, 5] = bad
        v[page, 0, off // 16, 9, off % 16] = bad
    got = attend(case, packed(case, [tree]), q)
    hit = torch.tensor([node in family(tree, i) for i in range(n)])
    assert hit.any() and not hit.all()
    assert (got[~hit] - want[~hit]).abs().max() <= attention_tolerance(worst, vmax, rows)
    if math.isnan(bad) or kv == "fp8":  # (an infinite score may be -inf, which weighs nothing)
        assert not torch.isfinite(got[hit]).all(-1).any()


def test_only_v_is_not_finite(gpu):
    """infinity in V alone: in the dim it is in, of the rows that attend it"""
    for n, heads, rows in ((9, 2, F32), (64, 2, F32), (64, 4, BF16), (20, 1, BF16)):
        case = Case([n], [70], 16, 1, "bf16", seed=69)
        tree = random_tree(n, 12)
        q = torch.randn(n, heads, D, generator=torch.Generator().manual_seed(7)).to(rows)
        want, worst, vmax = tree_attention(case, [tree], q)
        hit = torch.zeros(n, heads, D, dtype=torch.bool)
        for node, d in ((2, 9), (n - 3, 100), (n // 2, 64)):
            at = 70 + node
            case.host["v"][int(case.host["table"][0, at // 16]), 0, at % 16 // 16, d, at % 16] = math.inf
            for i in range(n):
                if node in family(tree, i):
                    hit[i, :, d] = True
        got = attend(case, packed(case, [tree]), q)
        assert (got[hit] == math.inf).all()
        assert (got[~hit] - want[~hit]).abs().max() <= attention_tolerance(worst, vmax, rows)


@pytest.mark.parametrize("entry", [-1, 1 << 30, -(1 << 31)])
def test_pages_that_are_not_there(gpu, entry):
    """in the context and among the nodes; a sequence with no page at all gives zeros"""
    new, ctx = [20, 5, 60], [30, 0, 40]
    case = Case(new, ctx, 16, 2, "fp8", seed=70, holes=[(0, 1, entry), (0, 2, entry), (1, 0, entry), (2, 4, entry)])
    for rows in (F32, BF16):
        check(case, [random_tree(n, n) for n in new], 4, rows)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("n,heads", [(8, 2), (15, 4), (50, 4)])
def test_a_plan_that_does_not_fit(gpu, n, heads, rows, kv):
    """nodes past the table, lengths far past it, and lengths below the number of nodes"""
    case = Case([n, 5], [80 - n, 30], 16, 2, kv, seed=71, lead=1, tail=1)
    trees = [random_tree(n, 3), random_tree(5, 4)]
    q = torch.randn(case.total, heads, D, generator=torch.Generator().manual_seed(9)).to(rows)
    for lens in ([80, 35], [83, 35], [80 + n, 3], [140, 0], [1 << 30, 5], [(1 << 31) - 1, -4], [n - 2, 35], [-(1 << 31), 1]):
        case.host["lens"] = torch.tensor(lens, dtype=torch.int32)
        want, worst, vmax = tree_attention(case, trees, q, lens)
        got = attend(case, packed(case, trees), q)
        assert (got[1:-1] - want[1:-1]).abs().max() <= attention_tolerance(worst, vmax, rows), lens
        assert (got[0] == 7).all() and (got[-1] == 7).all()


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("max_new", [0, 5, 64])
def test_more_nodes_than_a_tree_has(gpu, max_new, rows):
    """rows behind a sequence's first 64 are zeros, whatever they hang on"""
    new = [100, 3]
    case = Case(new, [50, 20], 16, 1, "bf16", seed=72)
    check(case, [random_tree(n, n) for n in new], 2, rows, max_new=max_new)


@pytest.mark.parametrize("new", [[1, 1, 1], [64, 3, 50], [12, 16, 9]])
def test_same_result_every_time(gpu, new):
    case = Case(new, [700, 30, 300], 32, 2, "fp8", seed=73)
    q = torch.randn(case.total, 8, D)
    parents = packed(case, [random_tree(n, n) for n in new])
    a = attend(case, parents, q)
    for _ in range(3):
        assert torch.equal(attend(case, parents, q), a)


def test_calls_on_two_streams(gpu):
    """two plans on two streams at once, each with work of its own, as eager calls and as graphs"""
    cases = [Case([1, 13, 2], [900, 40, 333], 16, 2, "bf16", seed=74), Case([64, 20], [60, 700], 32, 2, "fp8", seed=75)]
    qs = [torch.randn(c.total, 4, D, generator=torch.Generator().manual_seed(5)) for c in cases]
    parents = [packed(c, [random_tree(n, n) for n in c.new]) for c in cases]
    alone = [attend(c, p, q) for c, p, q in zip(cases, parents, qs)]
    pages, qd, pd = [c.pages() for c in cases], [q.cuda() for q in qs], [p.cuda() for p in parents]
    outs = [torch.empty_like(q) for q in qd]
    works = [torch.empty(qe.op_page_attention_work_bytes(4, 2, max(c.new)), dtype=torch.uint8, device="cuda") for c in cases]
    streams, graphs = [torch.cuda.Stream() for _ in cases], []
    torch.cuda.synchronize()

    def call(i):
        qe.op_page_tree_attention(pages[i], pd[i], qd[i], outs[i], works[i], max(cases[i].new))

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
@pytest.mark.parametrize("new,ctx,n_kv,heads", [([20], [1500], 1, 2), ([11], [3000], 1, 3), ([13], [9000], 1, 4), ([64], [5000], 1, 1),
                                                ([21, 3, 17], [7000, 40, 2500], 1, 3), ([17, 32], [2600, 4000], 2, 4),
                                                ([33, 1], [16000, 16000], 1, 1)])
def test_half_filled_tiles_over_a_long_axis(gpu, new, ctx, n_kv, heads, kv):
    """33 to 64 f32 rows a KV head, whose items are cut into 17 to 32, 33 to 64 and more parts"""
    check(Case(new, ctx, 64, n_kv, kv, seed=76, lead=1, tail=1), [random_tree(n, n) for n in new], heads, F32, gap=16)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_half_filled_tiles_of_many_sequences(gpu, kv):
    """33 to 64 f32 rows a KV head of more sequences than a wave has lanes, one of them long, and rows behind the 64th node"""
    new = [(i * 7) % 31 for i in range(70)]
    ctx = [(i * 37) % 200 for i in range(70)]
    new[33], ctx[33], new[50] = 30, 6000, 70
    check(Case(new, ctx, 32, 1, kv, seed=77), [random_tree(n, i) for i, n in enumerate(new)], 2, F32, max_new=30)
