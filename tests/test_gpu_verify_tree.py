"""qe_op_verify_tree against the rule in numpy's 64 bits."""
import math

import numpy as np
import pytest
import torch

import qe
from test_gpu_verify_drafts import NONE, settle, target
from tree_cases import random_tree

pytestmark = pytest.mark.gpu


def reference(logits, starts, parents, nodes, accept, sample, temps, max_depth=0):
    rows, vocab = logits.shape
    n = len(starts) - 1
    tokens, lps = np.full(rows, 77, np.int64), np.full(rows, 5.0)
    path, count, drawn = np.full((n, 64), -1, np.int64), np.zeros(n, np.int64), {}
    for s in range(n):
        a, b = starts[s], starts[s + 1]
        if b <= a:
            continue
        tokens[a:b], lps[a:b] = NONE, 0.0
        at, way = a, [0]
        while True:
            lp = target(logits[a + way[-1]], temps[s])
            p = np.exp(lp)
            q, left, taken = p.copy(), 1.0, None
            for c in range(way[-1] + 1, min(b - a, 64)):
                if parents[a + c] != way[-1] or (max_depth and len(way) > max_depth):
                    continue
                d = int(nodes[a + c])
                mine = q[d] if d < vocab else 0.0
                if np.float64(accept[a + c]) * left < mine:
                    taken = c
                    break
                left -= mine
                if d < vocab:
                    q[d] = 0.0
            if taken is None:
                break
            tokens[at], lps[at] = nodes[a + taken], lp[nodes[a + taken]]
            way.append(taken)
            at += 1
        if not q.sum() > 0:
            q = p
        c = np.cumsum(q)
        hit = np.nonzero((c > np.float64(sample[s]) * c[-1]) & (q > 0))[0]
        tok = int(hit[0]) if len(hit) else int(np.nonzero(q > 0)[0][-1])
        tokens[at], lps[at], count[s] = tok, lp[tok], len(way)
        path[s, :len(way)] = way
        drawn[at] = q, np.float64(sample[s]) * c[-1], lp
    return tokens, path, count, lps, drawn


def call(logits, starts, parents, nodes, accept, sample, temps, max_depth=0, gap=0):
    rows, vocab = logits.shape
    n = len(starts) - 1
    base = torch.full((rows, vocab + gap), math.inf, device="cuda")
    base[:, :vocab] = torch.from_numpy(logits)
    dev = lambda x, t: torch.from_numpy(np.ascontiguousarray(x).astype(t)).cuda()  # noqa: E731
    tokens, count = (torch.full((m,), 77, dtype=torch.int32, device="cuda") for m in (rows, n))
    path, lps = torch.full((n, 64), 77, dtype=torch.int32, device="cuda"), torch.full((rows,), 5.0, device="cuda")
    work = torch.empty(qe.op_verify_tree_work_bytes(rows, n, vocab), dtype=torch.uint8, device="cuda")
    work.fill_(0xFF)
    qe.op_verify_tree(base[:, :vocab], dev(starts, np.int32), dev(parents, np.int32),
                      dev(np.asarray(nodes, np.uint32).view(np.int32), np.int32), dev(accept, np.float32),
                      dev(sample, np.float32), tokens, path, count, work,
                      temperature=None if temps is None else dev(temps, np.float32), logprobs=lps, max_depth=max_depth)
    return (tokens.cpu().numpy().view(np.uint32).astype(np.int64), path.cpu().numpy(), count.cpu().numpy(),
            lps.cpu().numpy().astype(np.float64))


def check(logits, starts, parents, nodes, accept, sample, temps=None, max_depth=0, gap=0):
    n = len(starts) - 1
    tokens, path, count, lps, drawn = reference(logits, starts, parents, nodes, accept, sample,
                                                np.ones(n) if temps is None else temps, max_depth)
    got = call(logits, starts, parents, nodes, accept, sample, temps, max_depth, gap)
    np.testing.assert_array_equal(got[1], path)
    np.testing.assert_array_equal(got[2], count)
    settle(got[0], tokens, lps, drawn)
    np.testing.assert_array_equal(got[0], tokens)
    # log p in 64 bits, rounded once to f32: half a step, plus 64-bit noise
    np.testing.assert_allclose(got[3], lps, rtol=2.0 ** -23, atol=1e-12)
    return count


def likely(rng, logits, starts, parents, share=0.85):
    """nodes' tokens: a parent's likeliest in the order of its children, some at random"""
    rows, vocab = logits.shape
    nodes = rng.integers(0, vocab, rows).astype(np.uint32)
    for a, b in zip(starts[:-1], starts[1:]):
        seen = {}
        for i in range(a, b):
            p = parents[i]
            if 0 <= p < i - a:
                rank = seen[p] = seen.get(p, -1) + 1
                if rng.random() < share:
                    nodes[i] = np.argsort(-logits[a + p])[min(rank, vocab - 1)]
    return nodes


@pytest.mark.parametrize("max_depth", [0, 2, 63])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4097, 33001, 151936])
def test_against_the_rule(gpu, vocab, max_depth):
    rng = np.random.default_rng([vocab, 3])
    sizes = [1, 13, 0, 2, 64, 1, 3, 30, 5]
    starts = np.concatenate([[2], 2 + np.cumsum(sizes)])
    rows = starts[-1] + 1
    parents = np.full(rows, -1)
    for s, m in enumerate(sizes):
        parents[starts[s]:starts[s] + m] = random_tree(m, s)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    temps = np.array([1.0, 0.7, 1.0, 0.0, 1.5, 0.3, 1.0, 0.9, 1.0], np.float32)
    check(x, starts, parents, likely(rng, x, starts, parents), rng.random(rows, np.float32), rng.random(len(sizes), np.float32),
          temps, max_depth, gap=5)


def test_rows_at_the_edges(gpu):
    """NaN, infinities, nothing above -inf, ties, tokens out of range or impossible, the same token twice,
    numbers 0 and just below 1, temperatures that are not above 0, tiny and infinite"""
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
    logits, starts, parents, nodes, accept, sample, temps = [], [0], [], [], [], [], []
    for k in kinds:
        for family in ((0, 5, 11), (11, 11, 2999), (2999, vocab, NONE), (7, 2900, 7), (5, 1800, 0)):
            for u, v in ((0.0, 0.0), (0.5, u_last), (u_last, 0.5)):
                for t in (1.0, 0.0, -1.0, np.nan, np.inf, 1e-38):
                    logits += [k, base, k, base]
                    parents += [-1, 0, 0, 0]
                    nodes += [0, *family]
                    accept += [u] * 4
                    sample.append(v)
                    temps.append(t)
                    starts.append(len(logits))
    check(np.stack(logits), np.array(starts), np.array(parents), np.array(nodes, np.uint32), np.array(accept, np.float32),
          np.array(sample, np.float32), np.array(temps, np.float32))


def test_what_is_emitted_follows_the_target(gpu):
    """the first token of 60,000 trees has the target's distribution, whatever the children, and the second
    that of the row it follows"""
    n, vocab = 60000, 11
    rng = np.random.default_rng(12)
    x = (rng.standard_normal((4, vocab)) * 1.2).astype(np.float32)
    # root, three children (tokens 4, 9, 4 again), the last two rows below the first child
    parents, nodes = [-1, 0, 0, 0, 1, 1], [0, 4, 9, 4, 2, 7]
    rows = np.stack([x[0], x[1], x[2], x[2], x[3], x[3]])
    got = call(np.tile(rows, (n, 1)), np.arange(n + 1) * 6, np.tile(parents, n), np.tile(nodes, n),
               rng.random(6 * n, np.float32), rng.random(n, np.float32), None)
    tokens = got[0].reshape(n, 6)
    for seen, row in ((tokens[:, 0], x[0]), (tokens[got[1][:, 1] == 1, 1], x[1])):
        p = np.exp(target(row, 1.0))
        share = np.bincount(seen, minlength=vocab) / len(seen)
        # 5 standard deviations of a share of that many draws
        assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / len(seen)) + 1e-9).all(), (share, p)


@pytest.mark.parametrize("depth", [0, 1, 40, 63])
def test_long_paths(gpu, depth):
    """greedy chains and combs of 64 nodes that are accepted to the end, or to max_depth; rows behind the
    first 64 are never reached"""
    rng = np.random.default_rng(5)
    sizes = [64, 64, 80, 63]
    starts = np.concatenate([[0], np.cumsum(sizes)])
    parents = np.concatenate([np.arange(-1, 63), [i - 2 if i > 1 else i - 1 for i in range(64)], np.arange(-1, 79),
                              np.arange(-1, 62)])
    x = (rng.standard_normal((starts[-1], 40)) * 4).astype(np.float32)
    nodes = np.zeros(starts[-1], np.uint32)
    for s in range(4):
        for i in range(1, sizes[s]):
            nodes[starts[s] + i] = x[starts[s] + parents[starts[s] + i]].argmax()
    count = check(x, starts, parents, nodes, np.full(len(x), 0.5, np.float32), rng.random(4, np.float32),
                  np.zeros(4, np.float32), depth)
    np.testing.assert_array_equal(count, np.minimum([64, 33, 64, 63], depth + 1 if depth else 99))


def test_trees_that_are_not(gpu):
    """parents that are no earlier node: such nodes are never reached; a second root is not either"""
    rng = np.random.default_rng(6)
    parents = np.array([5, 0, 2, 3, 4, 99, -1, 6, 1, 1 << 30, 0, 0])
    x = (rng.standard_normal((24, 50)) * 2).astype(np.float32)
    starts = np.array([0, 12, 24])
    both = np.concatenate([parents, parents])
    for u in (0.0, 0.3, 0.9):
        nodes = np.array([x[max(0, min(int(p), 11)) + 12 * (i // 12)].argmax() for i, p in enumerate(both)], np.uint32)
        check(x, starts, both, nodes, np.full(24, u, np.float32), np.array([0.2, 0.8], np.float32))


def test_many_trees(gpu):
    """more rows than a grid is wide, and more sequences than there are CUs"""
    rng = np.random.default_rng(7)
    n, vocab = 22000, 7
    x = rng.standard_normal((3 * n, vocab)).astype(np.float32)
    parents = np.tile([-1, 0, 0], n)
    nodes = rng.integers(0, vocab, 3 * n).astype(np.uint32)
    got = call(x, np.arange(n + 1) * 3, parents, nodes, np.full(3 * n, 0.5), np.full(n, 0.5), np.zeros(n))
    best = x.argmax(-1)
    one, two = nodes[1::3] == best[::3], nodes[2::3] == best[::3]
    np.testing.assert_array_equal(got[2], 1 + (one | two))
    np.testing.assert_array_equal(got[1][:, 1], np.where(one, 1, np.where(two, 2, -1)))
    np.testing.assert_array_equal(got[0][::3], best[::3])
    np.testing.assert_array_equal(got[0][1::3], np.where(one, best[1::3], np.where(two, best[2::3], NONE)))


@pytest.mark.parametrize("max_depth,n", [(1, 8), (3, 12), (7, 18)])
def test_large_trees_level_by_level(gpu, max_depth, n):
    """so many rows that the check goes from level to level instead of summing all of them; trees that end at
    every depth, single roots, no rows, more rows than a tree has, greedy ones, rows that are not finite"""
    rng = np.random.default_rng([n, 5])
    vocab = 70001
    sizes = [64, 1, 0, 80, 64, 2] + [64] * (n - 6)
    starts = np.concatenate([[1], 1 + np.cumsum(sizes)])
    rows = starts[-1] + 2
    parents = np.full(rows, -1)
    for s, m in enumerate(sizes):
        parents[starts[s]:starts[s] + m] = random_tree(m, s, width=4)
    x = rng.standard_normal((rows, vocab), dtype=np.float32) * 2
    nodes = rng.integers(0, vocab, rows).astype(np.uint32)
    for a, b in zip(starts[:-1], starts[1:]):
        seen = {}
        for i in range(a, b):
            p = parents[i]
            if 0 <= p < i - a:
                rank = seen[p] = seen.get(p, -1) + 1
                if rank < 3 and rng.random() < 0.9:
                    x[a + p, nodes[i]] = 14.0 - rank
    x[starts[0], 5::7] = np.nan
    x[starts[4], 100:200] = np.inf
    nodes[starts[4] + 1] = 150
    temps = np.array([(0.7, 1.0, 0.0, 1.3, 0.9)[i % 5] for i in range(n)], np.float32)
    count = check(x, starts, parents, nodes, rng.random(rows, np.float32), rng.random(n, np.float32), temps, max_depth)
    assert count.max() > 1


@pytest.mark.parametrize("vocab", [262144, 262145, 400003, 1 << 20])
def test_large_vocabularies(gpu, vocab):
    """more chunks than a wave holds in registers, up to the largest"""
    rng = np.random.default_rng([vocab, 9])
    starts, parents = np.array([0, 5, 9]), np.array([-1, 0, 0, 1, 1, -1, 0, 1, 2])
    x = rng.standard_normal((9, vocab), dtype=np.float32)
    nodes = rng.integers(0, vocab, 9).astype(np.uint32)
    nodes[[1, 6]] = [vocab - 1, vocab // 2]
    x[0, vocab - 1] = x[5, vocab // 2] = 16.0
    for depth in (0, 1):
        check(x, starts, parents, nodes, np.full(9, 0.2, np.float32), np.array([0.3, 0.999], np.float32),
              np.array([1.0, 0.8], np.float32), depth)


def few_tokens(n, vocab, at, values):
    """rows [n, vocab] that are -inf but for the tokens `at` (each row's own, or the same for all), with `values`"""
    x = np.full((n, vocab), -np.inf, np.float32)
    x[np.arange(n)[:, None], np.broadcast_to(at, values.shape)] = values
    return x


# trees: few, whose rows are all summed first; many, which go level by level
@pytest.mark.parametrize("n", [200, 700])
@pytest.mark.parametrize("children", [(3, 900), (900, 3, 2047), (5, 4, 3, 2, 1)])
def test_chunks_of_which_all_is_refused(gpu, n, children):
    """logits masked to a few tokens (a row of 2048 that holds only refused children has nothing left, whatever
    its sums leave by rounding): the draw is one of the others, from the first number on"""
    rng = np.random.default_rng([n, len(children)])
    vocab, m = 6000, len(children)
    others = (2500, 5999)
    x = few_tokens(n, vocab, np.array(children + others), (rng.standard_normal((n, m + 2)) * 1.5).astype(np.float32))
    logits = np.repeat(x, 1 + m, 0)
    starts = np.arange(n + 1) * (1 + m)
    u_last = np.nextafter(np.float32(1), np.float32(0))
    for v in (0.0, 1e-30, 0.5, u_last):
        args = (logits, starts, np.tile([-1] + [0] * m, n), np.tile([0, *children], n), np.full(len(logits), u_last, np.float32),
                np.full(n, v, np.float32))
        count = check(*args, max_depth=1)
        assert (count == 1).all()
        if v in (0.0, u_last):
            np.testing.assert_array_equal(call(*args, None, 1)[0][::1 + m], others[0] if v == 0.0 else others[1])


@pytest.mark.parametrize("n", [200, 900])
def test_little_is_left_of_a_chunk(gpu, n):
    """two refused children that are all but 1e-14 of a chunk: what is left of it is drawn by its own sum, which the
    difference from the chunk's would give to a few percent"""
    rng = np.random.default_rng([n, 4])
    vocab = 5000
    # (each refused child leaves about 1e-7 of what there was, which a number just below 1 refuses)
    values = np.stack([np.zeros(n), np.full(n, -16.0), np.full(n, -32.0), np.full(n, -32.0)], 1) + rng.random((n, 4)) * 0.2
    values[:, 3] += rng.standard_normal(n)
    values = values.astype(np.float32)
    logits = np.repeat(few_tokens(n, vocab, np.array([70, 1500, 1999, 2048]), values), 3, 0)
    w = np.exp(values[:, 2:].astype(np.float64) - values[:, 3:])
    border = w[:, 0] / w.sum(1)
    u_last = np.nextafter(np.float32(1), np.float32(0))
    for side, token in ((1 - 2.0 ** -12, 1999), (1 + 2.0 ** -12, 2048)):
        args = (logits, np.arange(n + 1) * 3, np.tile([-1, 0, 0], n), np.tile([0, 70, 1500], n), np.full(3 * n, u_last, np.float32),
                (border * side).astype(np.float32))
        np.testing.assert_array_equal(call(*args, None, 1)[0][::3], token)
        check(*args, max_depth=1)


@pytest.mark.parametrize("n,vocab", [(1500, 5000), (560, 20001)])
def test_many_trees_level_by_level(gpu, n, vocab):
    """so many trees that a wave has a chunk of the level's row: trees of 1 to 5 nodes, none, and rows without weight"""
    rng = np.random.default_rng([n, 6])
    sizes = rng.integers(0, 6, n)
    starts = np.concatenate([[0], np.cumsum(sizes)])
    rows = int(starts[-1])
    parents = np.concatenate([np.asarray(random_tree(int(m), s, width=3), np.int64) for s, m in enumerate(sizes)])
    x = rng.standard_normal((rows, vocab), dtype=np.float32)
    nodes = rng.integers(0, vocab, rows).astype(np.uint32)
    for a, b in zip(starts[:-1], starts[1:]):
        for i in range(a + 1, b):
            x[a + parents[i], nodes[i]] = 10.0
    x[rng.integers(0, rows, 20)] = -np.inf
    x[rng.integers(0, rows, 20), ::3] = np.nan
    temps = np.array([(0.7, 1.0, 0.0, 1.3)[i % 4] for i in range(n)], np.float32)
    count = check(x, starts, parents, nodes, rng.random(rows, np.float32), rng.random(n, np.float32), temps, 2)
    assert set(count) == {0, 1, 2, 3}


@pytest.mark.parametrize("n", [4, 40])
@pytest.mark.parametrize("vocab", [262145, 1 << 20])
def test_few_tokens_of_a_large_vocabulary(gpu, vocab, n):
    """logits masked to a few tokens, some in one chunk with refused children only; trees whose rows are summed first (4 of
    the smaller vocabulary), and level by level, with four waves and with one for a chunk"""
    rng = np.random.default_rng([vocab, n])
    at = np.array([5, 2047, 4096, 4097, 130000, 131071, 200000, vocab - 2, vocab - 1])
    x = few_tokens(n, vocab, at, (rng.standard_normal((n, len(at))) * 1.5).astype(np.float32))
    children = np.stack([rng.permutation(at)[:4] for _ in range(n)])
    children[0], children[1], children[2] = at[:4], at[[0, 1, 7, 8]], at[2:6]
    logits = np.repeat(x, 5, 0)
    u_last = np.nextafter(np.float32(1), np.float32(0))
    nodes = np.concatenate([np.zeros((n, 1), np.int64), children], 1).ravel()
    for v in (0.0, 0.4, u_last):
        count = check(logits, np.arange(n + 1) * 5, np.tile([-1, 0, 0, 0, 0], n), nodes, np.full(5 * n, u_last, np.float32),
                      np.full(n, v, np.float32), max_depth=1)
        assert (count == 1).all()
