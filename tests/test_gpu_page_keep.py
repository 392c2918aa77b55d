"""Weights added up per position, the choice of what to keep, and the move of kept rows, against plain
references."""
import math

import numpy as np
import pytest
import torch

import qe
from page_cases import D, Case
from test_gpu_pages import BF16, F32, spaced

pytestmark = pytest.mark.gpu

KEYS = ("k", "v", "ke", "ve")


# ---- weigh ----

def weights(case, q, lens=None):
    """what is added to mass [n_seqs, n_kv, positions] in f64, and the largest sum of |q k| / sqrt(128)"""
    positions = case.host["table"].shape[1] * case.page
    out, worst = torch.zeros(len(case.new), case.n_kv, positions, dtype=torch.float64), 0.0
    group = q.shape[1] // case.n_kv
    for s, n in enumerate(case.new):
        have = case.lens[s]
        last = torch.arange(n) + (have if lens is None else lens[s]) - n
        hide = (torch.arange(have)[None] > last[:, None]) | ~case.seen[s][None]
        for h in range(q.shape[1]) if n else ():
            k = case.rows[s][0][h // group]
            x = q[case.starts[s]:case.starts[s] + n, h].double()
            w = torch.softmax((x @ k.T / math.sqrt(D)).masked_fill(hide, -math.inf), -1)
            out[s, h // group, :have] += torch.nan_to_num(w, nan=0.0).sum(0)
            worst = max(worst, float((x.abs() @ k.abs().T).max()) / math.sqrt(D))
    return out, worst


def tolerance(added, before, worst, rows):
    """Of an entry. A score is a sum of 128 products in f32, off by at most 64 x 2^-24 of the sum of
    magnitudes (`worst`); with the exponential's rounding and its argument's a weight by (64 + 4) x 2^-24 of
    it, numerator and denominator. The denominator adds up at most 2^10 values one after another (2^-14),
    the entry `rows` weights and what was there (each sum half a step: 2^-24). bf16 rows are exact."""
    return added * (2 * (64 + 4) * 2.0 ** -24 * worst + 2.0 ** -13 + (rows + 8) * 2.0 ** -24) + 2.0 ** -23 * before + 1e-30


def weigh(case, q, before, max_new=None, gap=0, stream=None):
    pages = case.pages()
    qd, _ = spaced(q.shape[0], q.shape[1], q.dtype, gap)
    qd.copy_(q)
    mass = before.cuda()
    most = max(case.new) if max_new is None else max_new
    positions = case.host["table"].shape[1] * case.page
    size = qe.op_page_weigh_work_bytes(q.shape[0], q.shape[1], case.n_kv, len(case.new), positions, most)
    work = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    qe.op_page_weigh(pages, qd, mass, work, most, stream)
    torch.cuda.synchronize()
    return mass.cpu()


def check_weigh(case, heads, rows, max_new=None, gap=0, spare=0, q_std=1.0, lens=None):
    g = torch.Generator().manual_seed(4)
    q = (torch.randn(case.total, heads, D, generator=g) * q_std).to(rows)
    added, worst = weights(case, q, lens)
    added = torch.nn.functional.pad(added, (0, spare))
    before = torch.rand(added.shape, generator=g)
    got = weigh(case, q, before, max_new, gap).double()
    tol = tolerance(added, before.double() + added, worst, max(case.new) * heads // case.n_kv)
    off = (got - before.double() - added).abs() - tol
    assert (off <= 0).all(), f"off by {float(off.max())} over the tolerance"
    none = added == 0
    assert torch.equal(got[none], before.double()[none]), "an entry that nothing is added to was changed"


WEIGH = [
    # new tokens, cached before, page, n_kv, heads
    ([1], [0], 16, 8, 16),
    ([1], [196], 64, 8, 16),
    ([1, 1, 1, 1, 1], [0, 15, 16, 63, 700], 16, 2, 8),
    ([5, 5], [60, 123], 32, 2, 4),
    ([3, 0, 7, 1], [125, 20, 0, 64], 16, 1, 3),
    ([8, 2], [500, 90], 128, 1, 16),
    ([32], [900], 64, 2, 4),
    ([70, 1, 33], [10, 300, 0], 32, 2, 4),
    ([129, 64], [0, 191], 64, 1, 2),
    ([200, 1, 1], [77, 130, 5], 256, 1, 5),
    ([1, 2], [5000, 30], 64, 1, 16),
]


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,page,n_kv,heads", WEIGH)
def test_weigh(gpu, new, ctx, page, n_kv, heads, kv, rows):
    check_weigh(Case(new, ctx, page, n_kv, kv, seed=81, lead=1, tail=2, spare=1), heads, rows, gap=16, spare=5)


@pytest.mark.parametrize("max_new", [0, 1, 9, 400])
@pytest.mark.parametrize("rows", [F32, BF16])
def test_weigh_any_max_new(gpu, max_new, rows):
    check_weigh(Case([150, 1, 4], [20, 200, 61], 16, 2, "fp8", seed=82), 4, rows, max_new=max_new)


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,heads", [([1, 3], [20000, 4], 2), ([40], [9000], 4), ([300], [3500], 2)])
def test_weigh_long(gpu, new, ctx, heads, rows):
    check_weigh(Case(new, ctx, 64, 1, "bf16", seed=83), heads, rows)


@pytest.mark.parametrize("rows", [F32, BF16])
def test_weigh_peaked_scores(gpu, rows):
    check_weigh(Case([40, 1], [90, 260], 16, 1, "bf16", seed=84, k_std=6.0), 2, rows, q_std=6.0)


@pytest.mark.parametrize("n_seqs,most", [(70, 1), (300, 2), (66, 20)])
def test_weigh_many_sequences(gpu, n_seqs, most):
    new = [(i * 7) % (most + 1) for i in range(n_seqs)]
    check_weigh(Case(new, [(i * 37) % 90 for i in range(n_seqs)], 16, 1, "bf16", seed=85), 2, F32)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new,ctx,page,heads", [([100, 31], [156, 0], 16, 2), ([100, 31], [157, 0], 16, 2), ([200, 3], [56, 250], 64, 4),
                                                ([17, 64], [238, 5], 256, 1), ([256], [0], 32, 6)])
def test_weigh_a_block_of_positions(gpu, new, ctx, page, heads, rows, kv):
    """tables that hold just what one workgroup has, and a little more"""
    check_weigh(Case(new, ctx, page, 1, kv, seed=94, lead=2, tail=1), heads, rows, gap=8)


@pytest.mark.parametrize("entry", [-1, 1 << 30, -(1 << 31)])
@pytest.mark.parametrize("new", [[20, 5, 3], [1, 1, 1], [100, 5, 80]])
def test_weigh_pages_that_are_not_there(gpu, entry, new):
    """such positions get nothing, and rows that attend nothing give nothing"""
    holes = [(0, 1, entry), (1, 0, entry), (2, 2, entry)]
    for rows in (F32, BF16):
        check_weigh(Case(new, [30, 0, 40], 16, 2, "fp8", seed=86, holes=holes), 4, rows)


@pytest.mark.parametrize("n", [1, 6, 50])
def test_weigh_a_plan_that_does_not_fit(gpu, n):
    """lengths past the table and below the number of new rows"""
    case = Case([n, 5], [80 - n, 30], 16, 2, "bf16", seed=87, lead=1, tail=1)
    for lens in ([80, 35], [83, 35], [80 + n, 3], [140, 0], [1 << 30, 5], [(1 << 31) - 1, -4], [-(1 << 31), 1]):
        case.host["lens"] = torch.tensor(lens, dtype=torch.int32)
        check_weigh(case, 4, F32, lens=lens)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n,heads", [(6, 2), (100, 2)])
def test_weigh_values_that_are_masked(gpu, bad, n, heads):
    """NaN and infinities in K of a later token: the rows before it weigh as ever, and nothing is written
    behind the last row's position"""
    case = Case([n], [40], 16, 1, "bf16", seed=88)
    at = 40 + n - 1
    q = torch.randn(n, heads, D, generator=torch.Generator().manual_seed(7))
    page, off = int(case.host["table"][0, at // 16]), at % 16
    case.host["k"][page, 0, off, 5] = bad
    case.host["lens"][0] -= 1  # every row one position earlier: none attends it
    added, worst = weights(case, q, [int(case.host["lens"][0])])
    added[..., at:] = 0
    got = weigh(case, q, torch.zeros(added.shape)).double()
    assert ((got - added).abs() <= tolerance(added, added, worst, n * heads)).all()


def test_weigh_query_that_is_not_finite(gpu):
    """a NaN in one row's query spoils the entries that this row attends, in its KV head"""
    for n, ctx, row in (([9, 40], [50, 3], 30), ([1, 1], [50, 70], 1), ([100, 30], [5, 80], 110)):
        case = Case(n, ctx, 16, 2, "bf16", seed=89)
        q = torch.randn(case.total, 4, D, generator=torch.Generator().manual_seed(8))
        added, worst = weights(case, q)
        q[row, 1, 0] = math.nan
        got = weigh(case, q, torch.zeros(added.shape)).double()
        s = 1 if row >= n[0] else 0
        end = ctx[s] + (row - case.starts[s]) + 1
        assert torch.isnan(got[s, 0, :end]).all()
        got[s, 0, :end] = added[s, 0, :end]
        assert ((got - added).abs() <= tolerance(added, added, worst, max(n) * 2)).all()


def test_weigh_same_result_every_time(gpu):
    for new in ([1, 1, 1], [90, 3, 50]):
        case = Case(new, [700, 30, 300], 32, 2, "fp8", seed=90)
        q = torch.randn(case.total, 8, D)
        zero = torch.zeros(3, 2, case.host["table"].shape[1] * 32)
        a = weigh(case, q, zero)
        for _ in range(3):
            assert torch.equal(weigh(case, q, zero), a)


# ---- keep ----

def kept_of(mass, lens, keep, sinks, recent):
    """kept [n_seqs, n_kv, keep] and count by sorting"""
    n_seqs, n_kv, stride = mass.shape
    kept, count = np.full((n_seqs, n_kv, keep), -1), np.zeros(n_seqs, np.int64)
    for s in range(n_seqs):
        ln = min(max(int(lens[s]), 0), stride)
        n = count[s] = min(ln, keep)
        a = min(sinks, n)
        b = min(recent, n - a)
        for h in range(n_kv):
            row = mass[s, h].astype(np.float64)
            row = np.where(np.isnan(row), -np.inf, row)
            nan = np.isnan(mass[s, h])
            mid = np.arange(a, ln - b)
            mid = mid[np.lexsort((mid, -row[mid], nan[mid]))][:n - a - b]
            kept[s, h, :n] = np.concatenate([np.arange(a), np.sort(mid), np.arange(ln - b, ln)])
    return kept, count


def check_keep(mass, lens, keep, sinks=0, recent=0, wide=0):
    n_seqs, n_kv, _ = mass.shape
    kept = torch.full((n_seqs, n_kv, keep + wide), 77, dtype=torch.int32, device="cuda")
    count = torch.full((n_seqs,), 77, dtype=torch.int32, device="cuda")
    qe.op_page_keep(torch.from_numpy(mass).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), kept, count,
                    keep, sinks=sinks, recent=recent)
    want = kept_of(mass, lens, keep, sinks, recent)
    np.testing.assert_array_equal(count.cpu().numpy(), want[1])
    np.testing.assert_array_equal(kept[..., :keep].cpu().numpy(), want[0])
    assert (kept[..., keep:] == 77).all()


@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (7, 4, 3), (64, 4, 16), (500, 0, 100), (1000, 4, 0), (1500, 1500, 0),
                                               (1024, 0, 1024), (3000, 4, 128)])
@pytest.mark.parametrize("values", ["spread", "ties", "equal"])
def test_keep(gpu, keep, sinks, recent, values):
    rng = np.random.default_rng([keep, sinks])
    lens = [2500, 0, 1, 7, 1024, 1025, 1023, 2047, 64, -5, 2499]
    mass = np.exp(rng.standard_normal((len(lens), 3, 2500)) * 2).astype(np.float32)
    if values == "ties":
        mass = np.round(mass * 4) / 4
    elif values == "equal":
        mass[:] = 0.25
    check_keep(mass.astype(np.float32), lens, keep, sinks, recent, wide=3)


@pytest.mark.parametrize("n,keep", [(70000, 5000), (33333, 33000), (200001, 1024), (131072, 1)])
def test_keep_long(gpu, n, keep):
    rng = np.random.default_rng(n)
    mass = np.exp(rng.standard_normal((2, 2, n)) * 2).astype(np.float32)
    mass[0] = np.round(mass[0] * 8) / 8
    check_keep(mass, [n, n - 77], keep, min(4, keep - 1), keep // 8)


def test_keep_special_values(gpu):
    """NaN below everything, infinities, signs and zeros, subnormals; lengths past the row"""
    rng = np.random.default_rng(3)
    pool = np.array([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0, -1.0, 1e-45, -1e-45, 3.4e38, -3.4e38, 1e-38], np.float32)
    mass = rng.choice(pool, (4, 2, 700)).astype(np.float32)
    for keep in (1, 50, 200, 400, 600, 699, 700, 900):
        check_keep(mass, [700, 650, 1 << 30, (1 << 31) - 1], keep, 0, min(keep, 3))


# ---- move ----

def move_host(case, src, count, first, mass):
    """the case's pages and mass after the move, row by row on the host"""
    got = {n: None if t is None else t.clone() for n, t in case.host.items()}
    mass = None if mass is None else mass.clone()
    n_kv, page = case.n_kv, case.page
    table = case.host["table"]
    bits = torch.uint8 if case.kv == "fp8" else torch.int16

    def slot(s, pos):
        if pos < 0 or pos >= table.shape[1] * page:
            return None
        at = int(table[s, pos // page])
        return (at, pos % page) if 0 <= at < case.n_pages else None

    for s in range(len(case.new)):
        base = 0 if first is None else int(first[s])
        n = min(max(int(count[s]), 0), src.shape[-1])
        for h in range(n_kv):
            row = src[s] if src.dim() == 2 else src[s, h]
            for i in range(n):
                a, b = slot(s, base + int(row[i])), slot(s, base + i)
                if int(row[i]) < 0:
                    continue
                if a and b:
                    got["k"].view(bits)[b[0], h, b[1]] = case.host["k"].view(bits)[a[0], h, a[1]]
                    got["v"].view(bits)[b[0], h, b[1] // 16, :, b[1] % 16] = case.host["v"].view(bits)[a[0], h, a[1] // 16, :, a[1] % 16]
                    for e in ("ke", "ve"):
                        if got[e] is not None:
                            got[e][b[0], h, b[1]] = case.host[e][a[0], h, a[1]]
            if mass is not None:
                old = mass[s, h].clone()
                width = mass.shape[2]
                mass[s, h, max(base + n, 0):max(0, min(int(case.host["lens"][s]), width))] = 0.0
                for i in range(n):
                    x, y = base + int(row[i]), base + i
                    if int(row[i]) >= 0 and 0 <= x < width and 0 <= y < width:
                        mass[s, h, y] = old[x]
                    elif 0 <= y < width:
                        mass[s, h, y] = old[y]
    return got, mass


def check_move(case, src, count, first=None, mass=None):
    want, want_mass = move_host(case, src, count, first, mass)
    pages = case.pages()
    md = None if mass is None else mass.cuda()
    ints = lambda x: torch.as_tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    qe.op_page_move(pages, src.int().cuda(), ints(count), first=None if first is None else ints(first), mass=md)
    bits = torch.uint8 if case.kv == "fp8" else torch.int16
    for n in KEYS:
        if want[n] is not None:
            a, b = case.dev[n].cpu(), want[n]
            if n in "kv":
                a, b = a.view(bits), b.view(bits)
            assert torch.equal(a, b), n
    if mass is not None:
        assert torch.equal(md.cpu(), want_mass)


def chosen(g, heads, n, of):
    """[heads, n] ascending positions of `of`"""
    return torch.stack([torch.randperm(of, generator=g)[:n].sort()[0] for _ in range(heads)])


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("lens,page,n_kv,share", [([40], 16, 1, 0.5), ([700, 33, 5], 16, 2, 0.3), ([1000, 999], 64, 3, 0.9),
                                                  ([513, 1, 300], 256, 2, 0.1), ([1500], 32, 2, 0.6)])
def test_move_what_is_kept(gpu, lens, page, n_kv, share, kv):
    g = torch.Generator().manual_seed(5)
    case = Case([0] * len(lens), lens, page, n_kv, kv, seed=91, spare=1)
    count = [max(1, int(ln * share)) for ln in lens]
    src = torch.full((len(lens), n_kv, max(count) + 3), -1)
    for s, n in enumerate(count):
        src[s, :, :n] = chosen(g, n_kv, n, lens[s])
    mass = torch.rand(len(lens), n_kv, case.host["table"].shape[1] * page, generator=g)
    check_move(case, src, count, mass=mass)
    check_move(case, src, count)
    check_move(case, src[:, 0].contiguous(), count, mass=mass)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page", [16, 64])
def test_move_paths(gpu, page, kv):
    """accepted nodes put one after another behind lengths of every alignment"""
    g = torch.Generator().manual_seed(6)
    ctx = list(range(0, 70, 3))
    new = [1 + i % 64 for i in range(0, 23 * 5, 5)][:len(ctx)]
    ctx = ctx[:len(new)]
    case = Case(new, ctx, page, 2, kv, seed=92)
    src, count = torch.full((len(new), 64), -1), []
    for s, n in enumerate(new):
        m = int(torch.randint(0, n + 1, (1,), generator=g))
        src[s, :m] = chosen(g, 1, m, n)[0]
        count.append(m)
    mass = torch.rand(len(new), 2, case.host["table"].shape[1] * page, generator=g)
    check_move(case, src, count, ctx)
    check_move(case, src, count, ctx, mass)


def test_move_at_the_edges(gpu):
    """counts of nothing, below 0 and above what there is; all rows where they are; pages that are not
    there, positions past the table and before the start"""
    holes = [(0, 2, -1), (1, 1, 1 << 30), (2, 0, -5)]
    case = Case([0] * 4, [100, 60, 40, 90], 16, 2, "fp8", seed=93, holes=holes)
    g = torch.Generator().manual_seed(7)
    src = torch.stack([chosen(g, 2, 30, ln) for ln in (100, 60, 40, 112)])
    mass = torch.rand(4, 2, 112, generator=g)
    for count in ([30, 30, 30, 30], [0, -3, 1, 1 << 30], [5, 30, 17, 16]):
        check_move(case, src, count, mass=mass)
        check_move(case, src, count, [0, 20, -7, 60], mass)
    same = torch.arange(30).expand(4, 2, 30).contiguous()
    check_move(case, same, [30, 20, 10, 0], mass=mass)
    case.host["lens"] = torch.tensor([1 << 30, -5, 0, 112], dtype=torch.int32)
    check_move(case, src, [30, 2, 3, 4], mass=mass)
    check_move(case, src, [30, 2, 3, 4], mass=mass[..., :50].contiguous())


def test_move_past_32_bits(gpu):
    """pages whose bytes lie beyond 4 GiB"""
    n_kv, page = 8, 256
    n_pages = (5 << 30) // (n_kv * page * D * 2)
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([600], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 600], dtype=torch.int32, device="cuda")
    pages = qe.Pages.empty(n_pages, page, n_kv, table, lens, starts)
    k, v = (torch.randn(600, n_kv, D, device="cuda").bfloat16() for _ in "kv")
    qe.op_page_append(pages, k, v)
    at = torch.randperm(600, generator=torch.Generator().manual_seed(1))[:300].sort()[0]
    qe.op_page_move(pages, at[None].int().cuda(), torch.tensor([300], dtype=torch.int32, device="cuda"))
    out = [torch.empty_like(k) for _ in "kv"]
    qe.op_page_read(pages, *out)
    assert torch.equal(out[0][:300], k[at.cuda()]) and torch.equal(out[1][:300], v[at.cuda()])
    assert torch.equal(out[0][300:], k[300:]) and torch.equal(out[1][300:], v[300:])


def widened(src, wide):
    """src with -1 behind each row, up to `wide` of them"""
    return torch.nn.functional.pad(src, (0, wide - src.shape[-1]), value=-1)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page", [16, 64])
def test_move_paths_of_wide_rows(gpu, page, kv):
    """what test_move_paths moves, of a src that has room for more"""
    g = torch.Generator().manual_seed(16)
    new = [1 + i % 64 for i in range(0, 23 * 5, 5)]
    ctx = list(range(0, 3 * len(new), 3))
    case = Case(new, ctx, page, 2, kv, seed=95)
    src, count = torch.full((len(new), 90), -1), []
    for s, n in enumerate(new):
        m = int(torch.randint(0, n + 1, (1,), generator=g))
        src[s, :m] = chosen(g, 1, m, n)[0]
        count.append(m)
    mass = torch.rand(len(new), 2, case.host["table"].shape[1] * page, generator=g)
    check_move(case, src, count, ctx)
    check_move(case, src, count, ctx, mass)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page,share", [(16, 0.4), (64, 0.95), (256, 0.7)])
def test_move_of_many_rows_from_any_start(gpu, page, share, kv):
    """counts of 65 to some 600 behind a first of every alignment to the runs of 16, and before the start"""
    g = torch.Generator().manual_seed(17)
    first = [*range(16), 64 + 9, -1, -16, -21, -100]
    lens = [200 + 29 * (i * 7 % len(first)) for i in range(len(first))]
    case = Case([0] * len(first), lens, page, 1, kv, seed=96, spare=1)
    count = [max(65, int((ln - f) * share)) for ln, f in zip(lens, first)]
    src = torch.stack([widened(chosen(g, 1, n, ln - f), max(count) + 1) for n, ln, f in zip(count, lens, first)])
    mass = torch.rand(len(first), 1, case.host["table"].shape[1] * page, generator=g)
    check_move(case, src, count, first)
    check_move(case, src, count, first, mass)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_move_of_many_rows_at_the_edges(gpu, kv):
    """pages that are not there as source and destination, positions past the table and past mass, counts of
    nothing, below 0 and above what src holds; all rows where they are"""
    holes = [(0, 2, -1), (0, 9, 1 << 30), (1, 1, -(1 << 31)), (1, 2, -1), (2, 0, -5), (3, 5, -1)]
    case = Case([0] * 4, [300, 260, 140, 290], 16, 2, kv, seed=97, holes=holes)
    g = torch.Generator().manual_seed(18)
    src = torch.stack([widened(chosen(g, 2, n, ln), 150) for n, ln in ((150, 300), (150, 260), (120, 140), (150, 390))])
    mass = torch.rand(4, 2, case.host["table"].shape[1] * 16, generator=g)
    for count in ([150, 149, 120, 150], [0, -3, 1, 1 << 30], [-(1 << 31), 70, 65, 16]):
        check_move(case, src, count, mass=mass)
        check_move(case, src, count, [0, 20, -7, 60], mass)
        check_move(case, src, count, [290, 1 << 30, -(1 << 31), (1 << 31) - 1], mass)
    same = torch.arange(100).expand(4, 2, 100).contiguous()
    check_move(case, same, [100, 70, 10, 0], mass=mass)
    case.host["lens"] = torch.tensor([1 << 30, -5, 0, 304], dtype=torch.int32)
    check_move(case, src, [130, 2, 3, 80], mass=mass)
    check_move(case, src, [130, 66, 70, 80], mass=mass[..., :90].contiguous())


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("first", [0, 5])
def test_move_of_thousands_of_rows(gpu, first, kv):
    """counts around 2048 rows, of which the kernel finds the places at a time, and of more than twice that"""
    g = torch.Generator().manual_seed(19)
    count, lens = [2047, 2048, 2049, 4999, 2043], [2100, 4100, 2070, 5600, 3000]
    case = Case([0] * 5, lens, 64, 1, kv, seed=98)
    src = torch.stack([widened(chosen(g, 1, n, ln - first), 5000) for n, ln in zip(count, lens)])
    mass = torch.rand(5, 1, case.host["table"].shape[1] * 64, generator=g)
    check_move(case, src, count, [first] * 5, mass)


def test_move_by_one(gpu):
    """a cache at its bound that drops one position of each head: all rows behind it move by one"""
    case = Case([0] * 2, [600, 577], 64, 2, "fp8", seed=99)
    src = torch.stack([torch.stack([torch.cat([torch.arange(d), torch.arange(d + 1, 600)]) for d in drop])
                       for drop in ((0, 300), (17, 575))])
    mass = torch.rand(2, 2, case.host["table"].shape[1] * 64, generator=torch.Generator().manual_seed(20))
    check_move(case, src, [599, 576], mass=mass)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("new,ctx,heads,max_new", [([1, 1], [700, 90], 4, 1), ([8, 3], [300, 20], 2, 8), ([70, 9], [500, 100], 2, 70),
                                                   ([90, 40], [20, 0], 1, 90), ([30], [200], 2, 3)])
def test_weigh_the_last_bits_of_f32_rows(gpu, new, ctx, heads, max_new, kv):
    """scores that only the lowest 8 bits of q decide: q has whole numbers from 2^23 on, in pairs that differ by at most
    60, and each position's K takes the difference of one pair. Few rows, many, one block of positions, and more rows than
    max_new says."""
    case = Case(new, ctx, 16, 1, kv, seed=100)
    g = torch.Generator().manual_seed(21)
    for s, ln in enumerate(case.lens):
        for j in range(ln):
            row = torch.zeros(D)
            i, sign = int(torch.randint(0, 64, (1,), generator=g)), 1 - 2 * (j % 2)
            row[2 * i], row[2 * i + 1] = sign, -sign
            page, off = int(case.host["table"][s, j // 16]), j % 16
            case.host["k"][page, 0, off] = row.to(case.host["k"].dtype)
            if kv == "fp8":
                case.host["ke"][page, 0, off] = 127
            case.rows[s][0][0, j] = row.double()
    q = (2 ** 23 + 256 * torch.randint(0, 2 ** 14, (case.total, heads, 64, 1), generator=g)
         + torch.randint(0, 61, (case.total, heads, 64, 2), generator=g)).flatten(2).float()
    added, _ = weights(case, q)
    got = weigh(case, q, torch.zeros(added.shape), max_new).double()
    # Sums of whole numbers below 2^24 are exact. The exponent's argument is at most 60 log2(e) / sqrt(128) = 7.7, a
    # difference 15.4, each rounded, and c too: 2^-19, in numerator and denominator; the exponential 2^-23; at most 2^10
    # values are summed one after another for a row (2^-14) and the rows' weights for an entry (2^-16)
    assert ((got - added).abs() <= added * (2.0 ** -17 + 2.0 ** -13)).all()
