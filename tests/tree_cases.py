"""Random trees of drafts and the 64-bit attention of their nodes over a Case's pages."""
import math
import random

import torch

from page_cases import D


def random_tree(n, seed, width=6, roots=1):
    """parents of n nodes: -1 for the first `roots`, else one of the `width` nodes before"""
    rng = random.Random(seed)
    return [-1 if i < roots else rng.randrange(max(0, i - width), i) for i in range(n)]


def family(parents, i):
    """node i and its ancestors; a parent that is not an earlier node is none"""
    got = [i]
    while 0 <= parents[got[-1]] < got[-1]:
        got.append(parents[got[-1]])
    return got


def packed(case, trees, fill=-1):
    """the trees' parents in the case's packed rows"""
    p = torch.full((case.total,), fill, dtype=torch.int32)
    for s, tree in enumerate(trees):
        p[case.starts[s]:case.starts[s] + len(tree)] = torch.tensor(tree, dtype=torch.int32)
    return p


def tree_attention(case, trees, q, lens=None):
    """f64 attention of q [rows, heads, 128] (rows of no sequence: NaN), and the largest sum of |q k| /
    sqrt(128) and |v| that enter it. lens: lengths in place of the case's (positions past the case's rows
    are not there)."""
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    group, worst, vmax = q.shape[1] // case.n_kv, 0.0, 0.0
    for s, n in enumerate(case.new):
        if n == 0:
            continue
        a, have = case.starts[s], case.lens[s]
        first = (case.lens[s] if lens is None else lens[s]) - n
        seen = torch.zeros(n, have, dtype=torch.bool)
        for i in range(min(n, 64)):
            if first + i < 0:
                continue
            seen[i, :max(first, 0)] = True
            for j in family(trees[s], i):
                if 0 <= first + j < have:
                    seen[i, first + j] = True
        seen &= case.seen[s][None]
        for h in range(q.shape[1]):
            k, v = (x[h // group] for x in case.rows[s])
            x = q[a:a + n, h].double()
            w = (x @ k.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
            w = torch.nan_to_num(torch.softmax(w, -1), nan=0.0)  # (a row that attends nothing: zeros)
            out[a:a + n, h] = w @ v
            worst = max(worst, float((x.abs() @ k.abs().T).max()) / math.sqrt(D))
            vmax = max(vmax, float(v.abs().max()))
    return out, worst, vmax
