"""Tree attention, accumulated weights and eviction in 64 bits, request by
request and in the order of the formulas (TEST INFRASTRUCTURE ONLY).

For a request with ``p`` cached tokens and ``n`` drafts at positions p .. p+n-1,
draft i sees position k if k < p, or k = p + j with bit j of its mask set.
``bounds`` gives, beside the values, what rounding may move them by:

* a logit is a sum of 576 exact products accumulated in fp32 in an order that
  is not known: off by at most 576 * 2^-23 of the sum of their magnitudes
  (2^-23, not 2^-24, for accumulators that truncate), times scale * log2(e);
* the base-2 lse moves by at most the largest of its logits' errors, plus the
  exponential's and the sum's (2^-18 is far above both) and one rounding;
* a weight moves relatively by ln 2 times its logit's and the lse's error;
* P is rounded to bf16 before the second product, half a step, 2^-8 of each
  weight at most, and divided by the rounded weights' sum: that moves the
  output by at most 2^-8 of sum w |c| and 2^-8 of itself; its own rounding by
  2^-8 of itself once more.
"""

from __future__ import annotations

import math

import torch

PAGE = 64
LOG2E = 1.4426950408889634


def slots(block_row: torch.Tensor, n: int) -> torch.Tensor:
    pos = torch.arange(n)
    return block_row.long()[pos // PAGE] * PAGE + pos % PAGE


def sees(mask_row, p: int, n: int) -> torch.Tensor:
    bits = [(int(mask_row[j // 64]) >> (j % 64)) & 1 if j // 64 < len(mask_row) else 0 for j in range(n)]
    return torch.cat([torch.ones(p, dtype=torch.bool), torch.tensor(bits, dtype=torch.bool)])


def _request(q_nope, q_pe, ckv, kpe, prefix, table, cu, mask, scale, b):
    lo, hi, p = int(cu[b]), int(cu[b + 1]), int(prefix[b])
    n = hi - lo
    s = slots(table[b], p + n)
    c = ckv.reshape(-1, 512)[s].double()
    k = torch.cat([c, kpe.reshape(-1, 64)[s].double()], 1)
    q = torch.cat([q_nope[lo:hi], q_pe[lo:hi]], 2).double()
    see = torch.stack([sees(mask[i].tolist(), p, n) for i in range(lo, hi)]) if n else torch.zeros(0, p, dtype=torch.bool)
    see = see[:, None, :].expand(n, q.shape[1], p + n)
    x = torch.einsum("ihd,kd->ihk", q, k) * (scale * LOG2E)
    x = torch.where(see, x, -math.inf)
    off = torch.einsum("ihd,kd->ihk", q.abs(), k.abs()) * (576 * 2.0 ** -23 * scale * LOG2E)
    off = torch.where(see, off, 0.0)
    return lo, hi, c, x, off


def tree_reference(q_nope, q_pe, ckv, kpe, prefix, table, cu, mask, scale):
    """(output, lse, output bound, lse bound), float64; rows of no request are NaN."""
    T, H = q_nope.shape[:2]
    out = torch.full((T, H, 512), math.nan, dtype=torch.float64)
    lse = torch.full((T, H), math.nan, dtype=torch.float64)
    out_off, lse_off = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(len(prefix)):
        lo, hi, c, x, off = _request(q_nope, q_pe, ckv, kpe, prefix, table, cu, mask, scale, b)
        if hi <= lo:
            continue
        # For masked rows.  Of a visible one a finite logit leaves nothing infinite; with a logit of
        # -inf its infinities count as nothing here, which the operator does not define.
        c = torch.where(torch.isfinite(c), c, 0.0)
        top = x.amax(-1, keepdim=True) if x.shape[-1] else torch.full((*x.shape[:2], 1), -math.inf)
        top = torch.where(top == -math.inf, 0.0, top)
        e = torch.exp2(x - top)
        total = e.sum(-1, keepdim=True)
        w = e / torch.where(total == 0, 1.0, total)
        out[lo:hi] = w @ c
        lse[lo:hi] = torch.where(total == 0, -math.inf, top + total.log2()).squeeze(-1)
        worst = off.amax(-1)
        seen = torch.where(torch.isfinite(lse[lo:hi]), lse[lo:hi].abs(), 0.0)
        lse_off[lo:hi] = worst + 2.0 ** -18 + seen * 2.0 ** -23
        spread = w @ c.abs()
        out_off[lo:hi] = spread * (2.0 ** -8 + 2 * math.log(2) * worst + 2.0 ** -17)[..., None] + out[lo:hi].abs() * 2.0 ** -7
    return out, lse, out_off, lse_off


def weights_reference(q_nope, q_pe, ckv, kpe, prefix, table, cu, mask, scale, lse, acc):
    """(accumulators, bound), float64, from the lse that the call is given."""
    new, off_all = acc.double().clone(), torch.zeros(acc.shape, dtype=torch.float64)
    for b in range(len(prefix)):
        lo, hi, _, x, off = _request(q_nope, q_pe, ckv, kpe, prefix, table, cu, mask, scale, b)
        if hi <= lo:
            continue
        given = lse[lo:hi].double()[..., None]
        w = torch.where(given == -math.inf, 0.0, torch.exp2(x - torch.where(given == -math.inf, 0.0, given)))
        n = x.shape[-1]
        rows = w.shape[0] * w.shape[1]
        # the exponent's argument is rounded once more; sums of `rows` terms in fp32
        rel = math.log(2) * (off + (x.abs().nan_to_num(posinf=0.0) + given.abs().nan_to_num(posinf=0.0)) * 2.0 ** -23) + 2.0 ** -21
        new[b, :n] += w.sum((0, 1))
        off_all[b, :n] = (w * (rel + rows * 2.0 ** -24)).sum((0, 1)) + new[b, :n].abs() * 2.0 ** -23
    return new, off_all


def evict_reference(acc, seq_lens, budget, sink, recent):
    """Kept positions per request, ascending (lists)."""
    kept = []
    for b, n in enumerate(seq_lens.tolist()):
        if n <= budget:
            kept.append(list(range(n)))
            continue
        row = acc[b].tolist()
        key = [(0, 0.0) if v != v else (1, -v) for v in row[:n]]  # NaN first, then larger first
        middle = sorted(range(sink, n - recent), key=lambda i: (key[i], i))
        kept.append(sorted([*range(sink), *middle[:budget - sink - recent], *range(n - recent, n)]))
    return kept
