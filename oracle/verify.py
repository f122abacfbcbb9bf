"""Verification of drafted tokens by its definition, request by request (TEST
INFRASTRUCTURE ONLY): the target's distribution p after a row, and after each
rejection what is left of it as a distribution of its own, in exact fractions
where asked (small vocabularies) and in 64 bits otherwise."""

from __future__ import annotations

from fractions import Fraction

import torch


def verify_reference(target, draft, tokens, parents, cu, accept_u, sample_u, width, exact=False):
    """(paths, accepted, next tokens) as lists."""
    num = (lambda x: Fraction(float(x))) if exact else float  # noqa: E731
    paths, accepted, following = [], [], []
    for b in range(len(cu) - 1):
        lo, n = int(cu[b]), int(cu[b + 1] - cu[b])
        path, node = [], 0
        if n == 0:
            paths.append([-1] * width)
            accepted.append(0)
            following.append(-1)
            continue
        p = [num(x) for x in target[lo]]
        for j in range(1, n):
            if int(parents[lo + j]) != node or len(path) == width:
                continue
            x = int(tokens[lo + j])
            q = [num(v) for v in draft[lo + node]] if draft is not None else None
            if num(accept_u[lo + j]) * (q[x] if q is not None else 1) < p[x]:
                path.append(j)
                node = j
                p = [num(v) for v in target[lo + node]]
                continue
            # p is a distribution here: its sum is 1 by assumption, or by the division
            left = [max(v - w, 0) for v, w in zip(p, q)] if q is not None else [0 if i == x else v for i, v in enumerate(p)]
            whole = sum(left) if q is not None else 1 - p[x]
            gone = sum(left) == 0
            p = [v / whole for v in left] if not gone else [0 * v for v in left]
        if sum(p) == 0:
            p = [num(v) for v in target[lo + node]]
        mark, run, token = num(sample_u[b]) * sum(p), 0, -1
        for v, w in enumerate(p):
            run += w
            if run > mark:
                token = v
                break
        paths.append(path + [-1] * (width - len(path)))
        accepted.append(len(path))
        following.append(token)
    return paths, accepted, following


def random_case(batch, most, vocab, branch, certain, seed, dyadic=False):
    """(target, draft or None, tokens, parents, cu, accept_u, sample_u) on the CPU: trees of up to `most` rows, drafts near the
    target.  `dyadic`: probabilities that are multiples of 2^-8, with many zeros and ties."""
    g = torch.Generator().manual_seed(seed)
    counts = [int(torch.randint(1, most + 1, (1,), generator=g)) for _ in range(batch)]
    if batch > 2:
        counts[1] = 0
    total = sum(counts)

    def rows(x):
        if not dyadic:
            return torch.softmax(x, 1)
        parts = torch.multinomial(torch.softmax(x, 1), 256, replacement=True, generator=g)
        return torch.zeros(total, vocab).scatter_add_(1, parts, torch.full(parts.shape, 2.0 ** -8))

    x = torch.randn(total, vocab, generator=g) * 2
    target, draft = rows(x), rows(x + 0.5 * torch.randn(total, vocab, generator=g))
    parents, tokens = [], []
    cu = torch.tensor([0, *counts]).cumsum(0)
    for b, n in enumerate(counts):
        kids = [0] * n
        for j in range(n):
            free = [i for i in range(j) if kids[i] < branch]
            par = -1 if j == 0 else free[int(torch.randint(len(free), (1,), generator=g))]
            parents.append(par)
            at = draft[cu[b] + max(par, 0)]
            tokens.append(int(at.argsort(descending=True)[kids[par] % vocab]) if certain and par >= 0
                          else int(torch.multinomial(at, 1, generator=g)))
            if par >= 0:
                kids[par] += 1
    u, s = torch.rand(total, generator=g), torch.rand(batch, generator=g)
    if dyadic:
        u, s = (u * 64).floor() / 64, (s * 64).floor() / 64
    return target, None if certain else draft, torch.tensor(tokens), torch.tensor(parents), cu, u, s
