"""Inputs and 64-bit references of the paged-cache operators' tests (qe.Pages, include/qe.h)."""
import math

import torch

import qe

D = 128


def pow2_rows(x):
    """(e4m3 values as f64, exponent byte) of rows x [..., 128] f64, by the definition: the smallest
    power of two for which the largest finite magnitude is at most 448 of it, nearest value with ties
    to even, NaN for what is not finite."""
    fine = torch.isfinite(x)
    big = torch.where(fine, x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.zeros_like(big)
    for i, a in enumerate(big.flatten().tolist()):
        n = 0
        if a > 0:
            m, p = math.frexp(a)  # a = m 2^p, 0.5 <= m < 1; 448 = 0.875 * 2^9
            n = max(p - 9 if m <= 0.875 else p - 8, -126)
        e.view(-1)[i] = n
    y = torch.where(fine, x, torch.zeros_like(x)) / torch.exp2(e)[..., None]
    step = torch.exp2((torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))) - 3).clamp(min=-9))
    y = torch.round(y / step) * step
    return torch.where(fine, y, torch.full_like(y, math.nan)), (e + 127).to(torch.uint8)


class Case:
    """Pages of random rows with garbage (NaN) wherever no position of the plan lies, a random page
    order, and the logical rows k, v [seq][n_kv, length, 128] (f64, as stored)."""

    def __init__(self, new, ctx, page=16, n_kv=2, kv="bf16", seed=0, holes=(), lead=0, tail=0, spare=0, k_std=1.0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.ctx, self.page, self.n_kv, self.kv = list(new), list(ctx), page, n_kv, kv
        n = len(self.new)
        lens = [a + b for a, b in zip(self.new, self.ctx)]
        width = max(1, max(-(-ln // page) for ln in lens)) + spare
        self.n_pages = sum(-(-ln // page) for ln in lens) + 2
        order = torch.randperm(self.n_pages, generator=g).tolist()
        table = torch.full((n, width), -1, dtype=torch.int32)
        raw = torch.float8_e4m3fn if kv == "fp8" else torch.bfloat16
        k = torch.full((self.n_pages, n_kv, page, D), math.nan).to(raw)
        v = torch.full((self.n_pages, n_kv, page // 16, D, 16), math.nan).to(raw)
        ke = torch.full((self.n_pages, n_kv, page), 255, dtype=torch.uint8) if kv == "fp8" else None
        ve = None if ke is None else ke.clone()
        bits = torch.uint8 if kv == "fp8" else torch.int16
        self.rows = []
        for s, ln in enumerate(lens):
            pair = []
            for name, std in (("k", k_std), ("v", 1.0)):
                x = torch.randn(ln, n_kv, D, generator=g) * std
                if kv == "fp8":
                    y, e = pow2_rows(x.double())
                    pair.append((y.to(torch.float8_e4m3fn), e, y * torch.exp2(e.double() - 127)[..., None]))
                else:
                    y = x.bfloat16()
                    pair.append((y, None, y.double()))
            for i in range(-(-ln // page)):
                table[s, i] = order.pop()
                at, m = int(table[s, i]), min(page, ln - i * page)
                off = torch.arange(m)
                part = slice(i * page, i * page + m)
                k.view(bits)[at, :, :m] = pair[0][0][part].view(bits).transpose(0, 1)
                v.view(bits)[at, :, off // 16, :, off % 16] = pair[1][0][part].view(bits)
                if ke is not None:
                    ke[at, :, :m] = pair[0][1][part].T
                    ve[at, :, :m] = pair[1][1][part].T
            self.rows.append([p[2].transpose(0, 1) for p in pair])
        self.seen = [torch.ones(ln, dtype=torch.bool) for ln in lens]
        for s, i, entry in holes:  # page i of sequence s is not there
            table[s, i] = entry
            self.seen[s][i * page:(i + 1) * page] = False
        starts = [lead]
        for m in self.new:
            starts.append(starts[-1] + m)
        self.lens, self.starts, self.total = lens, starts, starts[-1] + tail
        self.host = dict(k=k, v=v, ke=ke, ve=ve, table=table, lens=torch.tensor(lens, dtype=torch.int32),
                         starts=torch.tensor(starts, dtype=torch.int32))

    def pages(self):
        self.dev = {n: None if t is None else t.cuda() for n, t in self.host.items()}
        d = self.dev
        return qe.Pages(d["k"], d["v"], d["table"], d["lens"], d["starts"], d["ke"], d["ve"])

    def attention(self, q):
        """f64 attention of q [rows, heads, 128] (rows of no sequence: NaN), and the largest sum of
        |q k| / sqrt(128) and |v| that enter it, which its rounding errors go by."""
        out = torch.full(q.shape, math.nan, dtype=torch.float64)
        group, worst, vmax = q.shape[1] // self.n_kv, 0.0, 0.0
        for s, n in enumerate(self.new):
            a, ln = self.starts[s], self.lens[s]
            if n == 0:
                continue
            pos = torch.arange(ln - n, ln)
            hide = (torch.arange(ln)[None] > pos[:, None]) | ~self.seen[s][None]
            for h in range(q.shape[1]):
                k, v = (x[h // group] for x in self.rows[s])
                x = q[a:a + n, h].double()
                w = (x @ k.T / math.sqrt(D)).masked_fill(hide, -math.inf)
                m = w.amax(-1, keepdim=True)
                w = torch.exp(w - torch.where(m == -math.inf, torch.zeros_like(m), m))
                w = w.masked_fill(hide, 0.0)
                den = w.sum(-1, keepdim=True)
                out[a:a + n, h] = torch.where(den > 0, w @ v / den.clamp(min=1e-300), torch.zeros(()).double())
                worst = max(worst, float((x.abs() @ k.abs().T).max()) / math.sqrt(D))
                vmax = max(vmax, float(v.abs().max()))
        return out, worst, vmax


def attention_tolerance(worst, vmax, rows):
    """Largest error of an output element. A score is a sum of 128 products in f32 in some order, off
    by at most 64 x 2^-24 of the sum of magnitudes (`worst`); with it a weight is off relatively by
    that much, by the exponential's rounding and its argument's (2^-24 of |score| <= worst, twice
    over), and numerator and denominator both: twice the sum, plus 2^-20 for the sums over positions.
    bf16 rows: the weights rounded to bf16 (2^-8) and the output (2^-8)."""
    tol = vmax * (2 * (64 + 4) * 2.0 ** -24 * worst + 2.0 ** -20)
    return tol + (vmax * 2 * 2.0 ** -8 if rows == torch.bfloat16 else 0.0)
