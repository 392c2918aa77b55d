"""qe_op_verify_drafts against the rule in numpy's 64 bits, and the whole pass of speculative serving
(append, attention, check) as one captured graph."""
import math

import numpy as np
import pytest
import torch

import qe
from page_cases import D, Case

pytestmark = pytest.mark.gpu

NONE = 0xFFFFFFFF


def target(x, temp):
    """log p of one row of logits, by the documented rules"""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    lp = np.full(x.shape, -np.inf)
    if not temp > 0 or top == -np.inf:
        lp[int(x.argmax()) if top > -np.inf else 0] = 0.0
        return lp
    if top == np.inf:
        lp[x == np.inf] = -np.log((x == np.inf).sum())
        return lp
    with np.errstate(invalid="ignore"):
        z = np.where(x == -np.inf, -np.inf, (x - top) / np.float64(np.float32(temp)))
    return z - np.log(np.exp(z).sum())


def reference(logits, starts, drafts, probs, accept, sample, temps):
    rows, vocab = logits.shape
    tokens, count, lps = np.full(rows, 77, np.int64), np.zeros(len(starts) - 1, np.int64), np.full(rows, 5.0)
    drawn = {}  # row: (weights, aim, log p)
    for s in range(len(starts) - 1):
        for r in range(starts[s], starts[s + 1]):
            tokens[r], lps[r] = NONE, 0.0
        for r in range(starts[s], starts[s + 1]):
            lp = target(logits[r], temps[s])
            p, d, last = np.exp(lp), int(drafts[r]), r == starts[s + 1] - 1
            q = np.zeros(vocab)
            if not last:
                if probs is not None:
                    q = np.where(probs[r] > 0, probs[r].astype(np.float64), 0.0)
                elif d < vocab:
                    q[d] = 1.0
                if d < vocab and np.float64(accept[r]) * q[d] < p[d]:
                    tokens[r], lps[r] = d, lp[d]
                    continue
            w = np.maximum(p - q, 0.0)
            if not w.sum() > 0:
                w = p
            c = np.cumsum(w)
            hit = np.nonzero((c > np.float64(sample[s]) * c[-1]) & (w > 0))[0]
            tok = int(hit[0]) if len(hit) else int(np.nonzero(w > 0)[0][-1])
            tokens[r], lps[r], count[s] = tok, lp[tok], r - starts[s] + 1
            drawn[r] = w, np.float64(sample[s]) * c[-1], lp
            break
    return tokens, count, lps, drawn


def settle(got, want, lps, drawn):
    """A running sum of n weights in 64 bits is off by at most n 2^-53 of the whole sum, whatever the
    order. Where the aim lies that near to a token's border (numbers such as 0.5 among equal weights do)
    the token on its other side is as right: then `want` takes it."""
    for r in np.nonzero(got != want)[0]:
        if r in drawn:
            w, aim, lp = drawn[r]
            tok = got[r]
            if tok < len(w) and w[tok] > 0:
                c, slack = np.cumsum(w), 2 * len(w) * 2.0 ** -53 * w.sum()
                if c[tok] - w[tok] - slack <= aim <= c[tok] + slack:
                    want[r], lps[r] = tok, lp[tok]


def check(logits, starts, drafts, probs, accept, sample, temps=None, gap=0):
    rows, vocab = logits.shape
    n = len(starts) - 1
    want = reference(logits, starts, drafts, probs, accept, sample, np.ones(n) if temps is None else temps)

    def spaced(x):
        base = torch.full((rows, vocab + gap), math.inf, device="cuda")
        base[:, :vocab] = torch.from_numpy(x)
        return base[:, :vocab]

    def dev(x, dtype):
        return torch.from_numpy(np.asarray(x).astype(dtype)).cuda()

    tokens = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    count = torch.full((n,), 77, dtype=torch.int32, device="cuda")
    lps = torch.full((rows,), 5.0, device="cuda")
    work = torch.empty(qe.op_verify_drafts_work_bytes(rows, n, vocab), dtype=torch.uint8, device="cuda")
    work.fill_(0xFF)
    qe.op_verify_drafts(spaced(logits), dev(starts, np.int32), dev(np.asarray(drafts, np.uint32).view(np.int32), np.int32),
                        dev(accept, np.float32), dev(sample, np.float32), tokens, count, work,
                        draft_probs=None if probs is None else spaced(probs),
                        temperature=None if temps is None else dev(temps, np.float32), logprobs=lps)
    got = tokens.cpu().numpy().view(np.uint32).astype(np.int64)
    settle(got, want[0], want[2], want[3])
    np.testing.assert_array_equal(got, want[0])
    np.testing.assert_array_equal(count.cpu().numpy(), want[1])
    # log p in 64 bits, rounded once to f32: half a step, plus 64-bit noise
    np.testing.assert_allclose(lps.cpu().numpy().astype(np.float64), want[2], rtol=2.0 ** -23, atol=1e-12)


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4097, 33001, 151936])
@pytest.mark.parametrize("dense", [False, True])
def test_against_the_rule(gpu, vocab, dense):
    rng = np.random.default_rng([vocab, dense])
    rows_of = [1, 5, 0, 2, 9, 1, 3, 8, 4]
    starts = [2]
    for k in rows_of:
        starts.append(starts[-1] + k)
    rows = starts[-1] + 1
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    probs = softmax(x + rng.standard_normal(x.shape) * 0.5) if dense else None
    near = x if probs is None else np.log(np.maximum(probs, 1e-30))
    drafts = np.argmax(near + rng.gumbel(size=x.shape) * (1.0 if dense else 0.1), -1).astype(np.uint32)
    temps = np.array([1.0, 0.7, 1.0, 0.0, 1.5, 0.3, 1.0, 0.9, 1.0], np.float32)
    check(x, starts, drafts, probs, rng.random(rows, np.float32), rng.random(len(rows_of), np.float32), temps, gap=5)


@pytest.mark.parametrize("dense", [False, True])
def test_rows_at_the_edges(gpu, dense):
    """NaN, infinities, nothing above -inf, ties, drafts out of range or impossible, p = q, numbers 0 and
    just below 1, temperatures that are not above 0, tiny and infinite"""
    vocab = 3001
    rng = np.random.default_rng(8)
    base = rng.standard_normal(vocab).astype(np.float32)
    kinds = []
    r = base.copy(); r[::3] = np.nan; kinds.append(r)
    kinds.append(np.full(vocab, -np.inf, np.float32))
    kinds.append(np.full(vocab, np.nan, np.float32))
    r = base.copy(); r[[7, 2900]] = np.inf; kinds.append(r)
    r = np.full(vocab, -np.inf, np.float32); r[2999] = -3.0; kinds.append(r)
    kinds.append(np.zeros(vocab, np.float32))
    r = base.copy(); r[[5, 1800]] = 40.0; kinds.append(r)
    r = base.copy(); r[11] = 200.0; kinds.append(r)  # p is 1 there and nothing elsewhere
    kinds.append((base * 1e30).astype(np.float32))
    u_last = np.nextafter(np.float32(1), np.float32(0))
    logits, starts, drafts, accept, sample, temps, probs = [], [0], [], [], [], [], []
    for k in kinds:
        for d in (0, 11, 2999, vocab, NONE):
            for u, v in ((0.0, 0.0), (0.5, u_last), (u_last, 0.5)):
                for t in (1.0, 0.0, -1.0, np.nan, np.inf, 1e-38):
                    logits += [k, base]
                    q = np.zeros(vocab, np.float32)
                    q[min(d, vocab - 1)] = 1.0
                    if d == 11:  # the draft model is the target
                        q = np.exp(target(k, t)).astype(np.float32)
                    if d == 2999:
                        q = np.where(base > 0, base, np.nan).astype(np.float32)
                    probs += [q, q]
                    drafts += [d, d]
                    accept += [u, u]
                    sample.append(v)
                    temps.append(t)
                    starts.append(len(logits))
    check(np.stack(logits), starts, np.array(drafts, np.uint32), np.stack(probs) if dense else None,
          np.array(accept, np.float32), np.array(sample, np.float32), np.array(temps, np.float32))


@pytest.mark.parametrize("dense", [False, True])
def test_what_is_emitted_follows_the_target(gpu, dense):
    """the first token of 60,000 two-row sequences has the target's distribution whatever the draft's"""
    n, vocab = 60000, 11
    rng = np.random.default_rng(12)
    x = np.tile((rng.standard_normal(vocab) * 1.2).astype(np.float32), (2 * n, 1))
    q = softmax((rng.standard_normal(vocab) * 1.2).astype(np.float32)[None])[0]
    d = rng.choice(vocab, size=2 * n, p=q.astype(np.float64) / q.astype(np.float64).sum()) if dense else np.full(2 * n, 4)
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a).astype(t)).cuda()  # noqa: E731
    tokens = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
    count = torch.zeros(n, dtype=torch.int32, device="cuda")
    work = torch.empty(qe.op_verify_drafts_work_bytes(2 * n, n, vocab), dtype=torch.uint8, device="cuda")
    qe.op_verify_drafts(dev(x, np.float32), dev(np.arange(n + 1) * 2, np.int32), dev(d, np.int32),
                        dev(rng.random(2 * n, np.float32), np.float32), dev(rng.random(n, np.float32), np.float32),
                        tokens, count, work, draft_probs=dev(np.tile(q, (2 * n, 1)), np.float32) if dense else None)
    first = tokens.cpu().numpy()[::2]
    p = np.exp(target(x[0], 1.0))
    share = np.bincount(first, minlength=vocab) / n
    # 5 standard deviations of a share of n draws
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-9).all(), (share, p)


@pytest.mark.parametrize("dense", [False, True])
def test_long_runs_of_drafts(gpu, dense):
    """sequences of more drafts than are looked at together, that stop at the border, behind it and not at all"""
    rng = np.random.default_rng([5, dense])
    rows_of, wrong = [150, 64, 65, 129, 200], [140, 63, 64, 999, 64]
    starts = np.concatenate([[0], np.cumsum(rows_of)])
    x = (rng.standard_normal((starts[-1], 40)) * 4).astype(np.float32)
    drafts = x.argmax(-1).astype(np.uint32)
    for s, w in enumerate(wrong):
        if w < rows_of[s]:
            drafts[starts[s] + w] = x[starts[s] + w].argmin()
    probs = np.zeros_like(x) if dense else None
    if dense:
        probs[np.arange(len(x)), drafts] = 1.0
    check(x, starts, drafts, probs, np.full(len(x), 0.5, np.float32), rng.random(5, np.float32), np.zeros(5, np.float32))


def test_more_rows_than_a_grid_is_wide(gpu):
    """70,002 rows: greedy, two a sequence"""
    rng = np.random.default_rng(6)
    n, vocab = 35001, 7
    x = rng.standard_normal((2 * n, vocab)).astype(np.float32)
    best = x.argmax(-1)
    drafts = rng.integers(0, vocab, 2 * n)
    yes = drafts[::2] == best[::2]
    dev = lambda a, t: torch.from_numpy(a.astype(t)).cuda()  # noqa: E731
    tokens = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
    count = torch.zeros(n, dtype=torch.int32, device="cuda")
    work = torch.empty(qe.op_verify_drafts_work_bytes(2 * n, n, vocab), dtype=torch.uint8, device="cuda")
    qe.op_verify_drafts(dev(x, np.float32), dev(np.arange(n + 1) * 2, np.int32), dev(drafts, np.int32),
                        dev(np.full(2 * n, 0.5), np.float32), dev(np.full(n, 0.5), np.float32), tokens, count, work,
                        temperature=torch.zeros(n, device="cuda"))
    got = tokens.cpu().numpy()
    np.testing.assert_array_equal(count.cpu().numpy(), 1 + yes)
    np.testing.assert_array_equal(got[::2], best[::2])
    np.testing.assert_array_equal(got[1::2], np.where(yes, best[1::2], -1))


@pytest.mark.parametrize("kv,rows", [("fp8", torch.float32), ("bf16", torch.bfloat16)])
def test_a_pass_of_speculative_serving_as_a_graph(gpu, kv, rows):
    """append, attention, projection to logits and the check of the drafts, captured once on a stream of
    its own and replayed on plans that change in place, with eager work between the replays: every
    replay equals the same calls made eagerly"""
    heads, n_kv, page, vocab, seqs, k = 4, 2, 16, 5000, 3, 3
    n = seqs * (k + 1)
    case = Case([k + 1] * seqs, [60, 20, 90], page, n_kv, kv, seed=21, spare=2)
    used = set(case.host["table"].flatten().tolist())
    free = [i for i in range(case.n_pages) if i not in used]
    for s in range(seqs):  # room for the steps: pages of their own behind the sequences' last
        for i in range(case.host["table"].shape[1]):
            if case.host["table"][s, i] < 0 and free:
                case.host["table"][s, i] = free.pop()
    pages = case.pages()
    g = torch.Generator().manual_seed(22)
    new = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = {m: torch.empty(n, n_kv, D, dtype=rows, device="cuda") for m in "kv"}
    q, out = (torch.empty(n, heads, D, dtype=rows, device="cuda") for _ in range(2))
    w = (new(heads * D, vocab) * 0.3).cuda()
    logits = torch.empty(n, vocab, device="cuda")
    drafts = torch.empty(n, dtype=torch.int32, device="cuda")
    accept, sample = torch.empty(n, device="cuda"), torch.empty(seqs, device="cuda")
    tokens, count = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(seqs, dtype=torch.int32, device="cuda")
    lps = torch.empty(n, device="cuda")
    work = [torch.empty(b, dtype=torch.uint8, device="cuda") for b in (
        qe.op_page_attention_work_bytes(heads, n_kv, k + 1), qe.op_verify_drafts_work_bytes(n, seqs, vocab))]

    def fill():
        for t in (x["k"], x["v"], q):
            t.copy_(new(*t.shape))
        drafts.copy_(torch.randint(0, vocab, (n,), generator=g))
        accept.copy_(torch.rand(n, generator=g) * 1e-3)
        sample.copy_(torch.rand(seqs, generator=g))

    def step():
        qe.op_page_append(pages, x["k"], x["v"])
        qe.op_page_attention(pages, q, out, work[0], k + 1)
        torch.mm(out.float().flatten(1), w, out=logits)
        qe.op_verify_drafts(logits, case.dev["starts"], drafts, accept, sample, tokens, count, work[1], logprobs=lps)

    def state():
        torch.cuda.synchronize()
        return [t.clone() for t in (out, tokens, count, lps, case.dev["k"].view(torch.uint8), case.dev["v"].view(torch.uint8))]

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(5):
        fill()
        case.dev["lens"].add_(torch.tensor([1, 3, 0], dtype=torch.int32, device="cuda"))
        if i == 3:  # a sequence that has ended
            case.dev["starts"].copy_(torch.tensor([0, 4, 4, 8], dtype=torch.int32))
        keep = [case.dev[m].clone() for m in ("k", "v")]
        graph.replay()
        got = state()
        for m, t in zip(("k", "v"), keep):
            case.dev[m].view(torch.uint8).copy_(t.view(torch.uint8))
        for t in (out, tokens, count, lps):
            t.fill_(0) if i < 3 else None  # from then on the last rows belong to no sequence
        step()
        want = state()
        for a, b in zip(got, want):
            ok = a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a
            assert torch.equal(ok, b), i
        torch.randn(1000, device="cuda").sum()
