"""64-bit attention over a Case's pages with a bound for each output element, tight enough to see one lost
part of a long axis."""
import math

import torch

from page_cases import D


def attention_bounds(case, q, weigh=None):
    """f64 attention of q [rows, heads, 128], and how far each element of the result may be off. weigh(s, w)
    may change the weights [new, positions] of a sequence: a planted mistake.

    With p the weights over their sum, each element is sum p v. Let A = sum p |v| and B = sqrt(sum (p v)^2).
    - A score is off by at most 64 x 2^-24 of the row's largest sum of |q k| / sqrt(128); with the
      exponential and its argument's rounding a weight by (64 + 4) x 2^-24 of it, numerator and denominator:
      twice that, times A.
    - A sum in f32 takes at most 1024 additions one after another (32 blocks of 16 weights a lane, and the
      parts), so it is off by at most 2^10 x 2^-24 of the sum of magnitudes; again both: 2^-13 A.
    - bf16 rows: every weight of the numerator is rounded by at most 2^-8 of itself, up or down at random:
      the sum of such errors passes 8 x 2^-8 B with a chance of 2 exp(-32) an element (Hoeffding). The
      density of weights changes over a rounding step by a share of 2^-7 at most, so that the mean error is
      below 2^-14. The output: 2^-8 of it."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // case.n_kv
    for s, n in enumerate(case.new):
        if n == 0:
            continue
        a, ln = case.starts[s], case.lens[s]
        hide = (torch.arange(ln)[None] > torch.arange(ln - n, ln)[:, None]) | ~case.seen[s][None]
        for h in range(q.shape[1]):
            k, v = (x[h // group] for x in case.rows[s])
            x = q[a:a + n, h].double()
            w = (x @ k.T / math.sqrt(D)).masked_fill(hide, -math.inf)
            w = torch.exp(w - w.amax(-1, keepdim=True)).masked_fill(hide, 0.0)  # (every row has positions)
            if weigh:
                w = weigh(s, w)
            p = w / w.sum(-1, keepdim=True)
            o, mean = p @ v, p @ v.abs()
            worst = (x.abs() @ k.abs().T).masked_fill(hide, 0.0).amax(-1, keepdim=True) / math.sqrt(D)
            e = mean * (2 * (64 + 4) * 2.0 ** -24 * worst + 2.0 ** -13)
            if q.dtype == torch.bfloat16:
                e = e + 8 * 2.0 ** -8 * torch.sqrt((p * p) @ (v * v)) + 2.0 ** -14 * mean + 2.0 ** -8 * o.abs()
            out[a:a + n, h], tol[a:a + n, h] = o, e
    return out, tol
