"""The measured work of the draft-tree and eviction operators over the paged K/V cache.

One pass of speculative serving with trees of drafts is: append the nodes' K/V, attend with each node
seeing the cached positions and its ancestors, check the tree against the target's probabilities, and
move the accepted path's rows to where the next tokens continue. A cache of bounded size adds up the
attention weight each position gets, picks the positions to keep and moves them to the front. Kinds
(a case's "kind"):
  tree       attention of the nodes of a tree per sequence (op_page_tree_attention)
  check      trees of drafts against softmax(logits / T), from given random numbers (op_verify_tree)
  move       kept rows of K, V and mass to the front, in place (op_page_move)
  weigh      the softmax weight that each position gets from new tokens, added up (op_page_weigh)
  keep       the positions to keep by that weight (op_page_keep)

Pages: k [n_pages][n_kv][page_size][128] and v [n_pages][n_kv][page_size / 16][128][16] (16
positions transposed). e4m3 pages have one exponent byte e per (position, KV head) row in
[n_pages][n_kv][page_size], and the row's values are the stored ones times 2^(e - 127). The plan:
table [n_seqs][pages of a sequence], lens (each sequence's length, the new tokens included), starts
(its rows in the packed rows: starts[s] .. starts[s + 1]).
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

D = 128
NODES = 64      # nodes of a tree at most
VOCAB = 151936  # of the Qwen3-0.6B architecture the engine serves


def listed():
    return [
        # one chat a little past a 130-token prompt, a small tree: latency
        dict(name="tree_1x13", kind="tree", n_seqs=1, new=13, ctx=184, heads=16, n_kv=8, page=64, kv="bf16", rows="f32"),
        # a batch of chats, ragged lengths and trees
        dict(name="tree_16x26", kind="tree", n_seqs=16, new=26, ctx=2048, heads=16, n_kv=8, page=16, kv="fp8", rows="f32"),
        # large trees over long chats
        dict(name="tree_32x61", kind="tree", n_seqs=32, new=61, ctx=8192, heads=32, n_kv=8, page=64, kv="bf16", rows="bf16"),
        # one chat's tree against the target
        dict(name="check_1x13", kind="check", n_seqs=1, new=13, vocab=VOCAB),
        # a batch with large trees
        dict(name="check_24x48", kind="check", n_seqs=24, new=48, vocab=VOCAB),
        # the accepted paths of a batch of trees
        dict(name="move_paths_48", kind="move", n_seqs=48, new=30, ctx=1024, keep=0, n_kv=8, page=64, kv="fp8"),
        # long chats cut down to what each KV head keeps
        dict(name="move_evicted", kind="move", n_seqs=6, new=0, ctx=8192, keep=2048, n_kv=8, page=64, kv="bf16"),
        # one decode step of a batch of chats
        dict(name="weigh_decode_40", kind="weigh", n_seqs=40, new=1, ctx=4096, heads=32, n_kv=8, page=64, kv="fp8", rows="bf16"),
        # the last 32 tokens of long prompts look back over them
        dict(name="weigh_window", kind="weigh", n_seqs=4, new=32, ctx=16000, heads=16, n_kv=8, page=64, kv="bf16", rows="bf16"),
        # prompt chunks, every token counted
        dict(name="weigh_chunks", kind="weigh", n_seqs=3, new=1024, ctx=4096, heads=16, n_kv=8, page=32, kv="bf16", rows="f32"),
        # one chat that has reached its bound
        dict(name="keep_1", kind="keep", n_seqs=1, ctx=4500, n_kv=8, keep=1024, sinks=4, recent=128),
        # long prompts after prefill
        dict(name="keep_32", kind="keep", n_seqs=32, ctx=32000, n_kv=8, keep=4096, sinks=4, recent=512),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "check", "move", "weigh", "weigh", "keep"])
    kv, rows = rng.choice(["bf16", "fp8"]), rng.choice(["f32", "bf16"])
    page = rng.choice([16, 32, 64, 128, 256])
    shape = rng.randrange(1 << 20)
    heads, n_kv = rng.choice([(16, 8), (16, 8), (32, 8), (8, 8), (64, 8), (24, 8), (12, 2), (16, 1)])
    if kind == "tree":
        new = _log_int(rng, 1, NODES)
        ctx = rng.choice([0, _log_int(rng, 16, 16000), _log_int(rng, 16, 16000)])
        # at most about half of the largest listed case's work
        cost, kept = new * (ctx + new) * heads, (ctx + new) * n_kv
        n_seqs = _log_int(rng, 1, max(1, min(48, int(2.5e8 // cost), 1_000_000 // kept)))
        return dict(kind=kind, n_seqs=n_seqs, new=new, ctx=ctx, heads=heads, n_kv=n_kv, page=page, kv=kv, rows=rows,
                    shape=shape)
    if kind == "check":
        new, vocab = _log_int(rng, 1, NODES), rng.choice([VOCAB, _log_int(rng, 1000, 200_000)])
        return dict(kind=kind, n_seqs=_log_int(rng, 1, max(1, min(48, 1000 * VOCAB // (new * vocab)))), new=new,
                    vocab=vocab, shape=shape)
    if kind == "move":
        if rng.random() < 0.4:
            return dict(kind=kind, n_seqs=_log_int(rng, 1, 64), new=_log_int(rng, 1, NODES), ctx=_log_int(rng, 1, 3000),
                        keep=0, n_kv=n_kv, page=page, kv=kv, shape=shape)
        ctx = _log_int(rng, 64, 20000)
        return dict(kind=kind, n_seqs=_log_int(rng, 1, max(1, min(32, 400_000 // (ctx * n_kv)))), new=0, ctx=ctx,
                    keep=max(1, int(ctx * rng.uniform(0.1, 0.8))), n_kv=n_kv, page=page, kv=kv, shape=shape)
    if kind == "weigh":
        new = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 65, 1024)])
        ctx = rng.choice([0, _log_int(rng, 16, 16000), _log_int(rng, 16, 16000)])
        cost, kept = new * (ctx + new) * heads, (ctx + new) * n_kv
        n_seqs = _log_int(rng, 1, max(1, min(48, int(1.5e8 // cost), 600_000 // kept)))
        return dict(kind=kind, n_seqs=n_seqs, new=new, ctx=ctx, heads=heads, n_kv=n_kv, page=page, kv=kv, rows=rows,
                    shape=shape)
    ctx = _log_int(rng, 32, 60000)
    keep = max(1, int(ctx * rng.uniform(0.05, 1.1)))
    sinks = min(keep, rng.choice([0, 1, 4]))
    return dict(kind=kind, n_seqs=_log_int(rng, 1, max(1, min(64, 4_000_000 // (ctx * n_kv)))), ctx=ctx, n_kv=n_kv,
                keep=keep, sinks=sinks, recent=rng.choice([0, min(keep - sinks, keep // 4)]), shape=shape)


def _lengths(case):
    """(new rows, length with them) of each sequence: the first has the most of both, the others are
    ragged."""
    rng = random.Random(case.get("shape", 1) * 7919 + 5)
    new = case.get("new", 0)
    got = [(new, case["ctx"] + new)]
    for _ in range(case["n_seqs"] - 1):
        n = rng.randint(max(1, new // 2), new) if new else 0
        got.append((n, rng.randint(case["ctx"] // 4, case["ctx"]) + n))
    return got


def _trees(case):
    """parents of each sequence's nodes: -1 for the root, else an earlier node, most often a recent one
    (some six levels)."""
    rng = random.Random(case.get("shape", 1) * 7919 + 6)
    counts = [case["new"]] + [rng.randint(max(1, case["new"] // 2), case["new"]) for _ in range(case["n_seqs"] - 1)]
    if case["kind"] != "check":
        counts = [n for n, _ in _lengths(case)]
    trees = []
    for n in counts:
        parents, depth = [-1], [0]
        for i in range(1, n):
            p = rng.randrange(max(0, i - 9), i)
            while depth[p] >= 7:
                p = parents[p]
            parents.append(p)
            depth.append(depth[p] + 1)
        trees.append((parents, depth))
    return trees


def _paths(case):
    """an accepted path of each tree: the root, then children"""
    rng = random.Random(case.get("shape", 1) * 7919 + 8)
    got = []
    for parents, _ in _trees(case):
        path = [0]
        while rng.random() < 0.75:
            children = [i for i, p in enumerate(parents) if p == path[-1]]
            if not children:
                break
            path.append(rng.choice(children))
        got.append(path)
    return got


def _kept_counts(case):
    return [min(case["keep"], ln) for _, ln in _lengths(case)]


def work(case):
    kind = case["kind"]
    if kind == "check":
        # the logits of the root and of the accepted nodes, two more for each tree
        rows = sum(min(1 + max(d), 3) for _, d in _trees(case))
        return {"bytes": 4.0 * rows * case["vocab"], "flops": 4.0 * rows * case["vocab"]}
    if kind == "keep":
        values = case["n_kv"] * sum(ln for _, ln in _lengths(case))
        return {"bytes": 4.0 * (values + case["n_kv"] * sum(_kept_counts(case))), "flops": 1.0 * values}
    el = 2 if case["kv"] == "bf16" else 1
    row = case["n_kv"] * (D * el + (1 if el == 1 else 0))  # K, or V, of one position
    if kind == "move":
        if case["new"]:
            moved = [sum(i != p for i, p in enumerate(path)) for path in _paths(case)]
            return {"bytes": 4.0 * row * max(1, sum(moved)), "flops": 0.0}
        rows = sum(_kept_counts(case))
        return {"bytes": float(rows * (4 * row + 12 * case["n_kv"])), "flops": 0.0}
    lengths, io = _lengths(case), (4 if case["rows"] == "f32" else 2)
    t, positions = sum(n for n, _ in lengths), sum(ln for _, ln in lengths)
    if kind == "tree":
        pairs = sum(n * (ln - n) + sum(d + 1 for d in tree[1]) for (n, ln), tree in zip(lengths, _trees(case)))
        return {"bytes": float(2 * positions * row + 2 * t * case["heads"] * D * io),
                "flops": 4.0 * D * case["heads"] * pairs}
    pairs = sum(n * (2 * ln - n + 1) // 2 for n, ln in lengths)
    return {"bytes": float(positions * (row + 8 * case["n_kv"]) + t * case["heads"] * D * io),
            "flops": 2.0 * D * case["heads"] * pairs}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + 29) % (1 << 62))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pow2(e):
    """2^e for whole e in -126 .. 127, exactly"""
    return ((e.int() + 127) << 23).view(torch.float32)


def _raw(x):
    """pages as whole numbers of their width, which indexing takes for every type"""
    return x.view(torch.uint8 if x.element_size() == 1 else torch.int16)


def _quantise(x):
    """e4m3 values and exponent bytes of rows x [..., 128] (f32): the smallest power of two that
    brings a row's largest magnitude to at most 448."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(m == 0, torch.zeros_like(e), e).clamp(-126, 126)
    return (x * _pow2(-e.unsqueeze(-1))).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _filled_pages(case, g, n_pages):
    """Pages as a serving program finds them: every slot holds the rows of some token. K has a few
    channels that are larger than the others, as keys have."""
    shape = (n_pages, case["n_kv"], case["page"], D)
    gain = 0.6 + 0.5 * torch.rand(D, device="cuda", generator=g)
    gain[::19] *= 3.0
    k = torch.randn(shape, device="cuda", generator=g).mul_(gain)
    v = torch.randn(shape, device="cuda", generator=g)
    if case["kv"] == "fp8":
        (k, ke), (v, ve) = _quantise(k), _quantise(v)
    else:
        k, v, ke, ve = k.bfloat16(), v.bfloat16(), None, None
    v = _raw(v).unflatten(2, (-1, 16)).transpose(3, 4).contiguous()
    return dict(k=k, v=v.view(k.dtype), ke=ke, ve=ve)


def _packed(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


def _mass(case, g, positions):
    """accumulated attention weight: most of it on few positions, equal values among them"""
    x = torch.randn(case["n_seqs"], case["n_kv"], positions, device="cuda", generator=g).mul_(1.5).exp_()
    x = x.mul_(64).round_().div_(64)
    live = torch.arange(positions, device="cuda") < _ints([ln for _, ln in _lengths(case)])[:, None, None]
    return x.mul_(live)


def _prepare_pages(case, seed):
    g, kind = _generator(seed), case["kind"]
    lengths, ps = _lengths(case), case["page"]
    need = [-(-ln // ps) for _, ln in lengths]
    n_pages = sum(need) + 3
    s = dict(kind=kind, page=ps, n_kv=case["n_kv"], n_pages=n_pages, new=case["new"], **_filled_pages(case, g, n_pages))
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    at, rows = 0, []
    for n in need:
        rows.append(torch.nn.functional.pad(order[at:at + n], (0, max(need) - n)))
        at += n
    s["table"] = torch.stack(rows).contiguous()
    s["lens"] = _ints([ln for _, ln in lengths])
    starts = _packed([n for n, _ in lengths])
    s["starts"], t, positions = _ints(starts), starts[-1], max(need) * ps
    if kind in ("tree", "weigh"):
        dt = torch.float32 if case["rows"] == "f32" else torch.bfloat16
        s["q"] = torch.randn(t, case["heads"], D, device="cuda", generator=g).mul_(1.4).to(dt)
    if kind == "tree":
        trees = _trees(case)
        s["parents"] = _ints([p for parents, _ in trees for p in parents])
        s["out"] = torch.empty_like(s["q"])
    if kind == "weigh":
        s["mass"] = torch.rand(case["n_seqs"], case["n_kv"], positions, device="cuda", generator=g)
        s["mass"].mul_(torch.arange(positions, device="cuda") < (s["lens"] - (s["starts"][1:] - s["starts"][:-1]))[:, None, None])
    if kind == "move":
        s["mass"] = None
        if case["new"]:  # the accepted paths, from where the trees' rows begin
            paths = _paths(case)
            s["src"] = _ints([p + [-1] * (NODES - len(p)) for p in paths])
            s["count"] = _ints([len(p) for p in paths])
            s["first"] = _ints([ln - n for n, ln in lengths])
        else:  # what each KV head keeps of the whole sequence: the largest of some weights
            counts = _kept_counts(case)
            s["mass"] = _mass(case, g, positions)
            w = torch.rand(case["n_seqs"], case["n_kv"], positions, device="cuda", generator=g)
            w.masked_fill_(torch.arange(positions, device="cuda") >= s["lens"][:, None, None], -1.0)
            w = w.argsort(-1, descending=True)
            rows = []
            for i, n in enumerate(counts):
                rows.append(torch.nn.functional.pad(w[i, :, :n].sort(-1)[0], (0, case["keep"] - n), value=-1))
            s["src"], s["count"], s["first"] = torch.stack(rows).int().contiguous(), _ints(counts), None
    if own:
        qe = importlib.import_module("mac-gpu-compiler_amd.qe")
        s["qe"] = qe
        s["pages"] = qe.Pages(s["k"], s["v"], s["table"], s["lens"], s["starts"], s["ke"], s["ve"])
        size = 0
        if kind == "tree":
            size = qe.op_page_attention_work_bytes(case["heads"], case["n_kv"], case["new"])
        elif kind == "weigh":
            size = qe.op_page_weigh_work_bytes(t, case["heads"], case["n_kv"], case["n_seqs"], positions, case["new"])
        s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return s


def _prepare_check(case, seed):
    g, vocab, n = _generator(seed), case["vocab"], case["n_seqs"]
    trees = _trees(case)
    starts = _packed([len(p) for p, _ in trees])
    t = starts[-1]
    # logits: a spread body, a few likely tokens, and a part of the vocabulary that may not be emitted
    x = torch.randn(t, vocab, device="cuda", generator=g).mul_(1.7)
    top = torch.randint(0, vocab, (t, 12), device="cuda", generator=g)
    x.scatter_add_(1, top, 6.0 + 6.0 * torch.rand(t, 12, device="cuda", generator=g))
    x[:, -max(1, vocab // 500):] = -math.inf
    # a node's children are the likely tokens of its row in order, now and then another one
    row, rank = [], []
    for a, (parents, _) in zip(starts, trees):
        seen = {}
        for p in parents:
            row.append(a + max(p, 0))
            rank.append(min(seen.get(p, 0), 7))
            seen[p] = seen.get(p, 0) + 1
    likely = x.topk(8, -1)[1][_ints(row).long(), _ints(rank).long()]
    other = torch.randint(0, vocab, (t,), device="cuda", generator=g)
    s = dict(kind="check", logits=x, starts=_ints(starts), parents=_ints([p for tree, _ in trees for p in tree]),
             new=case["new"], depth=max(max(d) for _, d in trees))
    s["nodes"] = torch.where(torch.rand(t, device="cuda", generator=g) < 0.85, likely, other).to(torch.int32)
    s["temperature"] = torch.tensor([(0.7, 1.0, 0.0, 1.3, 0.9)[i % 5] for i in range(n)], device="cuda")
    s["accept"] = torch.rand(t, device="cuda", generator=g)
    s["sample"] = torch.rand(n, device="cuda", generator=g)
    s["tokens"] = torch.empty(t, dtype=torch.int32, device="cuda")
    s["path"] = torch.empty(n, NODES, dtype=torch.int32, device="cuda")
    s["count"] = torch.empty(n, dtype=torch.int32, device="cuda")
    s["logprobs"] = torch.empty(t, device="cuda")
    if own:
        qe = importlib.import_module("mac-gpu-compiler_amd.qe")
        s["qe"] = qe
        s["work"] = torch.empty(qe.op_verify_tree_work_bytes(t, n, vocab), dtype=torch.uint8, device="cuda")
    return s


def _prepare_keep(case, seed):
    g = _generator(seed)
    lens = [ln for _, ln in _lengths(case)]
    s = dict(kind="keep", keep=case["keep"], sinks=case["sinks"], recent=case["recent"], lens=_ints(lens))
    s["mass"] = _mass(case, g, max(lens))
    s["kept"] = torch.empty(case["n_seqs"], case["n_kv"], case["keep"], dtype=torch.int32, device="cuda")
    s["count"] = torch.empty(case["n_seqs"], dtype=torch.int32, device="cuda")
    if own:
        s["qe"] = importlib.import_module("mac-gpu-compiler_amd.qe")
    return s


def prepare(case, seed):
    return {"check": _prepare_check, "keep": _prepare_keep}.get(case["kind"], _prepare_pages)(case, seed)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _positions(s, name):
    """K (or V) of every position of the table's rows in f32: [seq][n_kv][position][128]"""
    x = _raw(s[name])[s["table"].long()].view(s[name].dtype).float()
    if name == "v":
        x = x.transpose(4, 5).flatten(3, 4)
    if s["ke"] is not None:
        x = x.mul_(_pow2(s[name + "e"][s["table"].long()].int().unsqueeze(-1) - 127))
    return x.transpose(1, 2).flatten(2, 3)


def _scores(s, hidden):
    """softmax weights [seq][n_kv][group][new][position] of the new tokens, with 0 where a (seq, new,
    position) is hidden; the rows of a sequence that has fewer than `new` come out as those of others"""
    starts = s["starts"].long()
    n_seqs, n_kv, new, (t, heads, _) = starts.shape[0] - 1, s["n_kv"], s["new"], s["q"].shape
    k = _positions(s, "k")
    i = torch.arange(new, device="cuda")
    q = s["q"].float()[(starts[:-1, None] + i).clamp(max=t - 1)]
    group = heads // n_kv
    q = q.unflatten(2, (n_kv, group)).permute(0, 2, 3, 1, 4).reshape(n_seqs, n_kv, group * new, D)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).div_(math.sqrt(D))
    x = x.unflatten(2, (group, new)).masked_fill_(hidden[:, None, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    return x.div_(x.sum(-1, keepdim=True))


def _family(s):
    """[seq][new][new]: whether the second node is the first or one of its ancestors"""
    starts, new = s["starts"].long(), s["new"]
    i = torch.arange(new, device="cuda")
    real = i < (starts[1:] - starts[:-1])[:, None]
    p = s["parents"].long()[(starts[:-1, None] + i).clamp(max=s["parents"].shape[0] - 1)].masked_fill(~real, -1)
    a = (p[:, :, None] == i) | (i[:, None] == i)
    for _ in range(6):
        a = torch.matmul(a.float(), a.float()) > 0
    return a


def _tree(s):
    starts, lens, new = s["starts"].long(), s["lens"].long(), s["new"]
    t, heads, _ = s["q"].shape
    n_seqs, first = starts.shape[0] - 1, lens - (starts[1:] - starts[:-1])
    at = torch.arange(s["table"].shape[1] * s["page"], device="cuda") - first[:, None]  # [seq][position], of the nodes
    family = _family(s).gather(2, at.clamp(0, new - 1)[:, None].expand(-1, new, -1))
    hidden = (at[:, None] >= 0) & ((at[:, None] >= new) | ~family)
    x = _scores(s, hidden)
    o = torch.matmul(x.flatten(2, 3), _positions(s, "v")).unflatten(2, x.shape[2:4])
    o = o.permute(0, 3, 1, 2, 4).reshape(n_seqs, new, heads, D)
    row = torch.arange(t, device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    return o[seq, row - starts[seq]].to(s["q"].dtype)


def _weigh(s):
    starts, lens, new = s["starts"].long(), s["lens"].long(), s["new"]
    count = starts[1:] - starts[:-1]
    i = torch.arange(new, device="cuda")
    last = (lens - count)[:, None] + i
    hidden = torch.arange(s["mass"].shape[2], device="cuda") > last[:, :, None]
    x = _scores(s, hidden)
    x = x.mul_((i < count[:, None])[:, None, None, :, None])
    s["mass"].add_(x.sum((2, 3)))
    return s["mass"]


def _check(s):
    starts, new = s["starts"].long(), s["new"]
    n, (t, vocab) = starts.shape[0] - 1, s["logits"].shape
    i, seq = torch.arange(new, device="cuda"), torch.arange(n, device="cuda")
    rows = (starts[:-1, None] + i).clamp(max=t - 1)  # [seq][node]
    real = i < (starts[1:] - starts[:-1])[:, None]
    parents, nodes, accept = (s[k][rows] for k in ("parents", "nodes", "accept"))
    nodes = nodes.long()
    twin = (nodes[:, :, None] == nodes[:, None, :]) & (i[None, :] < i[:, None])  # an earlier node of the same token
    temp = s["temperature"].double()[:, None]
    greedy = temp == 0
    cur, going = torch.zeros(n, dtype=torch.long, device="cuda"), torch.ones(n, dtype=torch.bool, device="cuda")
    tokens, logp = torch.full((t + 1,), -1, device="cuda"), torch.zeros(t + 1, dtype=torch.float64, device="cuda")
    path = torch.full((n, NODES), -1, device="cuda")
    path[:, 0] = 0
    count = torch.ones(n, dtype=torch.long, device="cuda")
    for level in range(s["depth"] + 1):
        x = s["logits"][rows[seq, cur]].double()
        best = x.argmax(-1, keepdim=True)
        x = x.sub_(x.amax(-1, keepdim=True)).div_(temp.masked_fill(greedy, 1.0))
        x = x.masked_fill_(greedy, -math.inf).scatter_(1, best, 0.0)
        w = x.exp()
        total = w.sum(-1, keepdim=True)
        p = w.div_(total)
        child = (parents == cur[:, None]) & real & (level < s["depth"])
        mine = p.gather(1, nodes) * (child & ~(twin & child[:, None, :]).any(-1))
        left = 1.0 - (mine.cumsum(-1) - mine)
        taken = child & (accept.double() * left < mine)
        some, next_ = taken.any(-1), taken.int().argmax(-1)
        tried = torch.zeros(n, vocab + 1, device="cuda", dtype=torch.bool)
        tried.scatter_(1, torch.where(child, nodes, vocab), True)
        rest = p.masked_fill(tried[:, :vocab], 0.0)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
        cum = rest.cumsum(-1)
        end = vocab - 1 - (rest > 0).flip(-1).to(torch.int8).argmax(-1)
        token = torch.minimum((cum <= s["sample"].double()[:, None] * rest.sum(-1, keepdim=True)).sum(-1), end)
        token = torch.where(some, nodes[seq, next_], token)
        at = torch.where(going, starts[:-1] + level, t)
        tokens[at] = token
        logp[at] = (x.gather(1, token[:, None]) - total.log())[:, 0]
        going = going & some
        cur = torch.where(going, next_, cur)
        if level < NODES - 1:
            path[:, level + 1] = torch.where(going, next_, -1)
        count += going
    return {"tokens": tokens[:t].int(), "path": path.int(), "count": count.int(), "logprobs": logp[:t].float()}


def _move(s):
    count, src = s["count"].long(), s["src"].long()
    if src.dim() == 2:
        src = src[:, None].expand(-1, s["n_kv"], -1)
    base = torch.zeros_like(count) if s["first"] is None else s["first"].long()
    n_seqs, n_kv, most = src.shape
    i = torch.arange(most, device="cuda")
    live = (i < count[:, None])[:, None].expand(-1, n_kv, -1)
    seq, head, at = torch.nonzero(live, as_tuple=True)
    a, b = base[seq] + src[seq, head, at], base[seq] + at
    ps, table = s["page"], s["table"].long()
    pa, pb = table[seq, a // ps], table[seq, b // ps]
    a_off, b_off = a % ps, b % ps
    k, v = _raw(s["k"]), _raw(s["v"])
    k[pb, head, b_off] = k[pa, head, a_off]
    v[pb, head, b_off // 16, :, b_off % 16] = v[pa, head, a_off // 16, :, a_off % 16]
    for e in ("ke", "ve"):
        if s[e] is not None:
            s[e][pb, head, b_off] = s[e][pa, head, a_off]
    if s["mass"] is not None:
        m = s["mass"][seq, head, a]
        j = torch.arange(s["mass"].shape[2], device="cuda")
        s["mass"].masked_fill_(((j >= (base + count)[:, None]) & (j < s["lens"][:, None]))[:, None], 0.0)
        s["mass"][seq, head, b] = m
    return {n: s[n] for n in ("k", "v", "ke", "ve", "mass")}


def _keep(s):
    mass, lens, keep = s["mass"], s["lens"].long(), s["keep"]
    positions = mass.shape[2]
    j, count = torch.arange(positions, device="cuda"), lens.clamp(max=keep)
    always = (j < s["sinks"]) | (j >= (lens - s["recent"])[:, None])
    x = mass.masked_fill(always[:, None], math.inf).masked_fill((j >= lens[:, None])[:, None], -math.inf)
    order = x.sort(dim=-1, descending=True, stable=True)[1][..., :keep]
    order = torch.nn.functional.pad(order, (0, keep - order.shape[2]), value=positions)
    i = torch.arange(keep, device="cuda")
    order = order.masked_fill((i >= count[:, None])[:, None], positions).sort(-1)[0]
    s["kept"].copy_(order.masked_fill(order == positions, -1))
    s["count"].copy_(count)
    return {"kept": s["kept"], "count": s["count"]}


def run(s):
    kind = s["kind"]
    if not own:
        return {"tree": _tree, "check": _check, "move": _move, "weigh": _weigh, "keep": _keep}[kind](s)
    qe = s["qe"]
    if kind == "tree":
        qe.op_page_tree_attention(s["pages"], s["parents"], s["q"], s["out"], s["work"], s["new"])
        return s["out"]
    if kind == "check":
        qe.op_verify_tree(s["logits"], s["starts"], s["parents"], s["nodes"], s["accept"], s["sample"], s["tokens"],
                          s["path"], s["count"], s["work"], temperature=s["temperature"], logprobs=s["logprobs"],
                          max_depth=s["depth"])
        return {n: s[n] for n in ("tokens", "path", "count", "logprobs")}
    if kind == "move":
        qe.op_page_move(s["pages"], s["src"], s["count"], first=s["first"], mass=s["mass"])
        return {n: s[n] for n in ("k", "v", "ke", "ve", "mass")}
    if kind == "weigh":
        qe.op_page_weigh(s["pages"], s["q"], s["mass"], s["work"], s["new"])
        return s["mass"]
    qe.op_page_keep(s["mass"], s["lens"], s["kept"], s["count"], s["keep"], sinks=s["sinks"], recent=s["recent"])
    return {"kept": s["kept"], "count": s["count"]}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, a sequence at a time
# ---------------------------------------------------------------------------------------------
def _rows64(s, name, i, ln):
    """K or V rows [n_kv][position][128] of sequence i in 64 bits"""
    pos = torch.arange(ln, device="cuda")
    page, off = s["table"][i].long()[pos // s["page"]], pos % s["page"]
    x = _raw(s[name])
    x = x[page, :, off] if name == "k" else x[page, :, off // 16, :, off % 16]
    x = x.view(s[name].dtype).double()
    if s["ke"] is not None:
        x = x * torch.exp2(s[name + "e"][page, :, off].double() - 127)[..., None]
    return x.transpose(0, 1).contiguous()


def _exact_attention(s, trees):
    tree = trees is not None
    got = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda") if tree else s["mass"].double()
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    group = s["q"].shape[1] // s["n_kv"]
    for i, ln in enumerate(lens):
        a, n = starts[i], starts[i + 1] - starts[i]
        seen = torch.zeros(n, ln, dtype=torch.bool)
        for t in range(n):
            seen[t, :ln - n if tree else ln - n + t + 1] = True
            node = t
            while tree and node >= 0:
                seen[t, ln - n + node] = True
                node = trees[i][0][node]
        hidden = ~seen.cuda()
        k = _rows64(s, "k", i, ln)
        v = _rows64(s, "v", i, ln) if tree else None
        for h in range(s["q"].shape[1]):
            x = s["q"][a:a + n, h].double() @ k[h // group].T.contiguous() / math.sqrt(D)
            x = torch.softmax(x.masked_fill_(hidden, -math.inf), -1)
            if tree:
                got[a:a + n, h] = x @ v[h // group]
            else:
                got[i, h // group, :ln] += x.sum(0)
    return got


def _exact_check(s):
    starts = s["starts"].tolist()
    n, t = len(starts) - 1, s["logits"].shape[0]
    parents, nodes, accept = s["parents"].tolist(), s["nodes"].tolist(), s["accept"].tolist()
    tokens, logps, counts, paths = [-1] * t, [0.0] * t, [0] * n, []
    for i in range(n):
        a, b, temp = starts[i], starts[i + 1], float(s["temperature"][i])
        path, at = [0], a
        while True:
            x = s["logits"][a + path[-1]].double()
            if temp == 0:
                logp = torch.full_like(x, -math.inf)
                logp[int(x.argmax())] = 0.0
            else:
                logp = torch.log_softmax(x / temp, -1)
            p = logp.exp()
            left, picked, q = 1.0, None, p.clone()
            for c in range(a, b):
                if parents[c] != path[-1]:
                    continue
                mine = float(q[nodes[c]])
                if accept[c] * left < mine:
                    picked = c
                    break
                left -= mine
                q[nodes[c]] = 0.0
            if picked is None:
                break
            tokens[at], logps[at] = nodes[picked], float(logp[nodes[picked]])
            path.append(picked - a)
            at += 1
        if float(q.sum()) <= 0:
            q = p
        cum = torch.cumsum(q, -1)
        hit = torch.nonzero((cum > float(s["sample"][i]) * float(cum[-1])) & (q > 0))
        tok = int(hit[0]) if len(hit) else int(torch.nonzero(q > 0)[-1])
        tokens[at], logps[at], counts[i] = tok, float(logp[tok]), len(path)
        paths.append(path + [-1] * (NODES - len(path)))
    return {"tokens": _ints(tokens), "path": _ints(paths), "count": _ints(counts),
            "logprobs": torch.tensor(logps, dtype=torch.float64, device="cuda")}


def _exact_move(s):
    """slot after slot, as whole rows"""
    lens, counts = s["lens"].tolist(), s["count"].tolist()
    got = {n: None if s[n] is None else s[n].clone() for n in ("k", "v", "ke", "ve", "mass")}
    for i, ln in enumerate(lens):
        base = 0 if s["first"] is None else int(s["first"][i])
        for h in range(s["n_kv"]):
            src = s["src"][i] if s["src"].dim() == 2 else s["src"][i, h]
            a = base + src[:counts[i]].long()
            b = base + torch.arange(counts[i], device="cuda")
            (pa, oa), (pb, ob) = ((s["table"][i].long()[x // s["page"]], x % s["page"]) for x in (a, b))
            _raw(got["k"])[pb, h, ob] = _raw(s["k"])[pa, h, oa]
            _raw(got["v"])[pb, h, ob // 16, :, ob % 16] = _raw(s["v"])[pa, h, oa // 16, :, oa % 16]
            for e in ("ke", "ve"):
                if s[e] is not None:
                    got[e][pb, h, ob] = s[e][pa, h, oa]
            if s["mass"] is not None:
                got["mass"][i, h, base + counts[i]:ln] = 0.0
                got["mass"][i, h, b] = s["mass"][i, h, a]
    return {n: x.double() if n in ("k", "v", "mass") and x is not None else x for n, x in got.items()}


def _exact_keep(s):
    kept, counts = [], []
    for i, ln in enumerate(s["lens"].tolist()):
        n = min(ln, s["keep"])
        counts.append(n)
        sinks = min(s["sinks"], n)
        recent = min(s["recent"], n - sinks)
        for row in s["mass"][i].cpu().numpy().astype(np.float64):
            middle = np.arange(sinks, ln - recent)
            middle = middle[np.lexsort((middle, -row[middle]))][:n - sinks - recent]
            got = np.full(s["keep"], -1, dtype=np.int32)
            got[:n] = np.concatenate([np.arange(sinks), np.sort(middle), np.arange(ln - recent, ln)])
            kept.append(got)
    return {"kept": torch.from_numpy(np.stack(kept)).cuda().view(s["kept"].shape), "count": _ints(counts)}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "keep":
        return _exact_keep(s)
    if kind == "check":
        return _exact_check(s)
    if kind == "move":
        return _exact_move(s)
    return _exact_attention(s, _trees(case) if kind == "tree" else None)
