"""The draft-tree and eviction operators together, as a serving loop calls them, eagerly and as captured
graphs that are replayed on plans that change in place."""
import math

import pytest
import torch

import qe
from page_cases import D, Case, attention_tolerance
from test_gpu_page_keep import kept_of, tolerance, weights
from tree_cases import packed, random_tree

pytestmark = pytest.mark.gpu


class Trees:
    """a pass of serving with a tree of 13 nodes for each of three sequences: append, attention, logits, check,
    move; `ctx` is on the device and grows by what was accepted"""

    def __init__(self, kv, rows):
        self.heads, self.n_kv, self.n, self.seqs, self.vocab = 4, 2, 13, 3, 3000
        t = self.n * self.seqs
        self.case = Case([self.n] * self.seqs, [60, 20, 90], 16, self.n_kv, kv, seed=101, spare=5)
        used = set(self.case.host["table"].flatten().tolist())
        self.case.n_pages += 20  # room for the steps
        for m, x in self.case.host.items():
            if m in ("k", "v", "ke", "ve") and x is not None:
                self.case.host[m] = torch.cat([x, x[:1].expand(20, *x.shape[1:])]).contiguous()
        free = [i for i in range(self.case.n_pages) if i not in used]
        for s in range(self.seqs):
            for i in range(self.case.host["table"].shape[1]):
                if self.case.host["table"][s, i] < 0 and free:
                    self.case.host["table"][s, i] = free.pop()
        self.pages = self.case.pages()
        self.g = torch.Generator().manual_seed(102)
        self.parents = packed(self.case, [random_tree(self.n, s, width=4) for s in range(self.seqs)]).cuda()
        new = dict(device="cuda")
        self.k, self.v = (torch.empty(t, self.n_kv, D, dtype=rows, **new) for _ in "kv")
        self.q, self.out = (torch.empty(t, self.heads, D, dtype=rows, **new) for _ in "qo")
        self.w = (torch.randn(self.heads * D, self.vocab, generator=self.g) * 0.4).cuda()
        self.logits = torch.empty(t, self.vocab, **new)
        self.nodes = torch.empty(t, dtype=torch.int32, **new)
        self.accept, self.sample = torch.empty(t, **new), torch.empty(self.seqs, **new)
        self.tokens, self.count = torch.empty(t, dtype=torch.int32, **new), torch.empty(self.seqs, dtype=torch.int32, **new)
        self.path = torch.empty(self.seqs, qe.QE_TREE_NODES, dtype=torch.int32, **new)
        self.lps = torch.empty(t, **new)
        self.ctx = torch.tensor([60, 20, 90], dtype=torch.int32, **new)
        self.work = [torch.empty(b, dtype=torch.uint8, **new) for b in (
            qe.op_page_attention_work_bytes(self.heads, self.n_kv, self.n),
            qe.op_verify_tree_work_bytes(t, self.seqs, self.vocab))]

    def fill(self):
        for x in (self.k, self.v, self.q):
            x.copy_(torch.randn(x.shape, generator=self.g))
        self.nodes.copy_(torch.randint(0, self.vocab, self.nodes.shape, generator=self.g))
        self.accept.copy_(torch.rand(self.accept.shape, generator=self.g) * 2e-4)
        self.sample.copy_(torch.rand(self.sample.shape, generator=self.g))

    def step(self):
        torch.add(self.ctx, self.n, out=self.case.dev["lens"])
        qe.op_page_append(self.pages, self.k, self.v)
        qe.op_page_tree_attention(self.pages, self.parents, self.q, self.out, self.work[0], self.n)
        torch.mm(self.out.float().flatten(1), self.w, out=self.logits)
        qe.op_verify_tree(self.logits, self.case.dev["starts"], self.parents, self.nodes, self.accept, self.sample,
                          self.tokens, self.path, self.count, self.work[1], logprobs=self.lps, max_depth=6)
        qe.op_page_move(self.pages, self.path, self.count, first=self.ctx)
        self.ctx.add_(self.count)

    def state(self):
        torch.cuda.synchronize()
        d = self.case.dev
        return [x.clone() for x in (self.out, self.tokens, self.path, self.count, self.lps, self.ctx, d["k"].view(torch.uint8),
                                    d["v"].view(torch.uint8)) + ((d["ke"], d["ve"]) if d["ke"] is not None else ())]


@pytest.mark.parametrize("kv,rows", [("fp8", torch.float32), ("bf16", torch.bfloat16)])
def test_a_pass_with_trees_as_a_graph(gpu, kv, rows):
    """replays equal eager passes from the same state, with eager work between them"""
    a, b = Trees(kv, rows), Trees(kv, rows)
    side = torch.cuda.Stream()
    for x in (a, b):
        x.fill()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a.step()
    torch.cuda.synchronize()
    deeper = 0
    for i in range(4):
        for x in (a, b):
            x.fill()
        graph.replay()
        b.step()
        for x, y in zip(a.state(), b.state()):
            assert torch.equal(x, y), i
        deeper += int((a.count > 1).sum())
        torch.randn(1000, device="cuda").sum()
    assert deeper > 0


@pytest.mark.parametrize("kv", ["fp8", "bf16"])
def test_what_a_tree_leaves_is_a_chain(gpu, kv):
    """after the move, causal attention of the accepted nodes' queries over the cache gives what the tree gave them"""
    x = Trees(kv, torch.float32)
    for _ in range(3):
        x.fill()
        ctx = x.ctx.clone()
        x.step()
        count, path = x.count.tolist(), x.path.cpu()
        rows = [s * x.n + int(path[s, i]) for s in range(x.seqs) for i in range(count[s])]
        starts = [0]
        for c in count:
            starts.append(starts[-1] + c)
        q = x.q[rows].contiguous()
        out = torch.empty_like(q)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        d = x.case.dev
        pages = qe.Pages(d["k"], d["v"], d["table"], x.ctx, ints(starts), d["ke"], d["ve"])
        work = torch.empty(qe.op_page_attention_work_bytes(x.heads, x.n_kv, x.n), dtype=torch.uint8, device="cuda")
        qe.op_page_attention(pages, q, out, work, x.n)
        assert torch.equal(x.ctx, ctx + x.count)
        # both are within the tolerance of the same sums; |q k| of a row of 128 at most 128 x 5 x 5 / sqrt(128)
        tol = 2 * attention_tolerance(128 * 25 / math.sqrt(D), 5.0, torch.float32)
        assert (out - x.out[rows]).abs().max() <= tol


@pytest.mark.parametrize("kv", ["fp8", "bf16"])
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
def test_a_cache_of_bounded_size(gpu, kv, rows):
    """weigh, keep, move: mass is the weights' sum, what is kept follows from it, and attention over what was
    moved is attention over the kept positions; then a decode step goes on from there"""
    heads, n_kv, keep, sinks, recent = 4, 2, 150, 4, 30
    case = Case([20, 1, 33], [300, 90, 500], 16, n_kv, kv, seed=103, spare=1)
    pages = case.pages()
    q = torch.randn(case.total, heads, D, generator=torch.Generator().manual_seed(9)).to(rows)
    positions = case.host["table"].shape[1] * 16
    mass = torch.zeros(3, n_kv, positions, device="cuda")
    work = torch.empty(qe.op_page_weigh_work_bytes(case.total, heads, n_kv, 3, positions, 33), dtype=torch.uint8, device="cuda")
    qe.op_page_weigh(pages, q.cuda(), mass, work, 33)
    added, worst = weights(case, q)
    assert ((mass.cpu().double() - added).abs() <= tolerance(added, added, worst, 66)).all()
    # every row's weights add up to 1
    total = mass.sum(-1).cpu()
    for s, n in enumerate(case.new):
        assert (total[s] - n * heads // n_kv).abs().max() <= n * heads // n_kv * 2.0 ** -12
    kept = torch.empty(3, n_kv, keep, dtype=torch.int32, device="cuda")
    count = torch.empty(3, dtype=torch.int32, device="cuda")
    qe.op_page_keep(mass, case.dev["lens"], kept, count, keep, sinks=sinks, recent=recent)
    want, n = kept_of(mass.cpu().numpy(), case.lens, keep, sinks, recent)
    assert (kept.cpu().numpy() == want).all() and (count.cpu().numpy() == n).all()
    before = mass.clone()
    qe.op_page_move(pages, kept, count, mass=mass)
    for s in range(3):
        for h in range(n_kv):
            at = torch.from_numpy(want[s, h, :n[s]]).cuda()
            assert torch.equal(mass[s, h, :n[s]], before[s, h, at]) and (mass[s, h, n[s]:] == 0).all()
    # one more token a sequence
    g = torch.Generator().manual_seed(10)
    k, v, q = (torch.randn(3, m, D, generator=g).to(rows) for m in (n_kv, n_kv, heads))
    lens = count + 1
    plan = qe.Pages(case.dev["k"], case.dev["v"], case.dev["table"], lens, torch.arange(4, dtype=torch.int32, device="cuda"),
                    case.dev["ke"], case.dev["ve"])
    qe.op_page_append(plan, k.cuda(), v.cuda())
    stored = [torch.empty(3, n_kv, D, dtype=rows, device="cuda") for _ in "kv"]
    qe.op_page_read(plan, *stored)
    stored = [x.cpu().double() for x in stored]
    out = torch.empty(3, heads, D, dtype=rows, device="cuda")
    work = torch.empty(qe.op_page_attention_work_bytes(heads, n_kv, 1), dtype=torch.uint8, device="cuda")
    qe.op_page_attention(plan, q.cuda(), out, work, 1)
    for s in range(3):
        for h in range(heads):
            at = torch.from_numpy(want[s, h // 2, :n[s]])
            ks, vs = (torch.cat([case.rows[s][i][h // 2][at], stored[i][s, h // 2][None]]) for i in range(2))
            x = q[s, h].double()
            p = torch.softmax(ks @ x / math.sqrt(D), 0) @ vs
            tol = attention_tolerance(float((ks.abs() @ x.abs()).max()) / math.sqrt(D), float(vs.abs().max()), rows)
            assert (out[s, h].cpu().double() - p).abs().max() <= tol


def test_a_bounded_cache_as_a_graph(gpu):
    """a decode step that weighs, keeps and moves every time, captured and replayed: equal to eager steps"""
    heads, n_kv, keep = 8, 2, 100

    def make():
        case = Case([1, 1], [100, 80], 16, n_kv, "bf16", seed=104, spare=2)
        pages = case.pages()
        case.dev["table"].copy_(torch.arange(2 * case.host["table"].shape[1], dtype=torch.int32).view(2, -1) % case.n_pages)
        positions = case.host["table"].shape[1] * 16
        d = dict(case=case, pages=pages, mass=torch.zeros(2, n_kv, positions, device="cuda"),
                 k=torch.empty(2, n_kv, D, device="cuda"), v=torch.empty(2, n_kv, D, device="cuda"),
                 q=torch.empty(2, heads, D, device="cuda"), out=torch.empty(2, heads, D, device="cuda"),
                 kept=torch.empty(2, n_kv, keep, dtype=torch.int32, device="cuda"),
                 count=torch.tensor([100, 80], dtype=torch.int32, device="cuda"), g=torch.Generator().manual_seed(11),
                 w1=torch.empty(qe.op_page_attention_work_bytes(heads, n_kv, 1), dtype=torch.uint8, device="cuda"),
                 w2=torch.empty(qe.op_page_weigh_work_bytes(2, heads, n_kv, 2, positions, 1), dtype=torch.uint8, device="cuda"))
        return d

    def fill(d):
        for n in "kvq":
            d[n].copy_(torch.randn(d[n].shape, generator=d["g"]))

    def step(d):
        lens = d["case"].dev["lens"]
        torch.add(d["count"], 1, out=lens)
        qe.op_page_append(d["pages"], d["k"], d["v"])
        qe.op_page_attention(d["pages"], d["q"], d["out"], d["w1"], 1)
        qe.op_page_weigh(d["pages"], d["q"], d["mass"], d["w2"], 1)
        qe.op_page_keep(d["mass"], lens, d["kept"], d["count"], keep, sinks=2, recent=10)
        qe.op_page_move(d["pages"], d["kept"], d["count"], mass=d["mass"])

    # (pages of the two sequences must not be shared)
    a, b = make(), make()
    assert len(set(a["case"].dev["table"].flatten().tolist())) >= 2 * -(-(keep + 1) // 16)
    for d in (a, b):
        table = torch.stack([torch.arange(7), torch.arange(7, 14)]).int()
        assert a["case"].n_pages >= 14 and d["case"].dev["table"].shape[1] >= 7
        d["case"].dev["table"].fill_(-1)
        d["case"].dev["table"][:, :7] = table.cuda()
        d["case"].dev["k"].copy_(torch.randn(d["case"].dev["k"].shape, generator=torch.Generator().manual_seed(1)))
        d["case"].dev["v"].copy_(torch.randn(d["case"].dev["v"].shape, generator=torch.Generator().manual_seed(2)))
    side = torch.cuda.Stream()
    for d in (a, b):
        fill(d)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a)
    step(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(a)
    torch.cuda.synchronize()
    for i in range(5):
        for d in (a, b):
            fill(d)
        graph.replay()
        step(b)
        torch.cuda.synchronize()
        for n in ("out", "mass", "kept", "count"):
            assert torch.isfinite(a[n].float()).all() and torch.equal(a[n], b[n]), (i, n)
        for n in "kv":
            assert torch.equal(a["case"].dev[n].view(torch.int16), b["case"].dev[n].view(torch.int16)), (i, n)
        torch.randn(1000, device="cuda").sum()
    assert a["count"].tolist() == [100, 86]


def test_two_loops_on_two_streams(gpu):
    """two serving loops with trees on two streams at once, as graphs, each with work of its own: equal to each alone"""
    kinds = [("fp8", torch.float32), ("bf16", torch.bfloat16)]
    alone, both = [Trees(*k) for k in kinds], [Trees(*k) for k in kinds]
    streams, graphs = [torch.cuda.Stream() for _ in kinds], []
    for x in alone + both:
        x.fill()
    torch.cuda.synchronize()
    for x, st in zip(both, streams):
        with torch.cuda.stream(st):
            x.step()
    for x in alone:
        x.step()
    torch.cuda.synchronize()
    for x, st in zip(both, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=st):
            x.step()
    torch.cuda.synchronize()
    for i in range(4):
        for x in alone + both:
            x.fill()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for x, y in zip(alone, both):
            x.step()
            for a, b in zip(x.state(), y.state()):
                assert torch.equal(a, b), i


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 70]])
def test_weights_of_two_plans_on_two_streams(gpu, new):
    cases = [Case(new, [700, 30, 300], 32, 2, kv, seed=105 + i) for i, kv in enumerate(("fp8", "bf16"))]
    q = torch.randn(sum(new), 8, D, generator=torch.Generator().manual_seed(3)).cuda()
    pages = [c.pages() for c in cases]
    positions = [c.host["table"].shape[1] * 32 for c in cases]
    size = [qe.op_page_weigh_work_bytes(sum(new), 8, 2, 3, p, max(new)) for p in positions]
    work = [torch.empty(s, dtype=torch.uint8, device="cuda") for s in size]
    mass = [torch.zeros(3, 2, p, device="cuda") for p in positions]
    alone = [torch.zeros_like(m) for m in mass]
    for i in range(2):
        for _ in range(6):
            qe.op_page_weigh(pages[i], q, alone[i], work[i], max(new))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(6):
        for i, st in enumerate(streams):
            qe.op_page_weigh(pages[i], q, mass[i], work[i], max(new), stream=st)
    torch.cuda.synchronize()
    for a, b in zip(alone, mass):
        assert torch.equal(a, b)
