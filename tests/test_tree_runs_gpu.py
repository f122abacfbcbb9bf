"""GPU parity of tree attention and accumulated weights where one CTA walks a
long run of one request's tiles, where many requests make the join take each
of its forms, and where a row sees nothing for whole tiles.  The batches draw
their pages from a small pool, so that the oracle stays quick."""

import math

import pytest
import torch

from dsa_b200 import tree
from oracle import tree as otree
from test_tree_gpu import SCALE, Case, run, weigh

pytestmark = pytest.mark.gpu

LEAD = 3  # units that a group counts beside its tiles (attention)


class Pooled(Case):
    """Page k of every request is one of `variants` pages that all requests'
    page k are drawn from."""

    def __init__(self, prefixes, drafts, heads, seed, device, variants=3, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        normal = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
        need = [(p + n + 63) // 64 for p, n in zip(prefixes, drafts)]
        width, T, words = max(need), sum(drafts), (max(drafts) + 63) // 64
        self.variants = variants
        self.ckv, self.kpe = normal(width * variants, 64, 512), normal(width * variants, 64, 64)
        self.table = torch.arange(width, dtype=torch.int32) * variants + torch.randint(
            0, variants, (len(need), width), generator=g, dtype=torch.int32)
        self.table[torch.arange(width) >= torch.tensor(need)[:, None]] = -1
        rows = []
        for n in drafts:
            parents = [int(torch.randint(-1, j, (1,), generator=g)) if j and j % 3 == 0 else j - 1 for j in range(n)]
            rows += [r + [0] * (words - len(r)) for r in (tree.masks_from_parents(parents) if n else [])]
        self.q_nope = (normal(T, heads, 512).float() * scale).to(torch.bfloat16)
        self.q_pe = normal(T, heads, 64)
        self.prefix = torch.tensor(prefixes, dtype=torch.int32)
        self.cu = torch.tensor([0, *drafts]).cumsum(0).int()
        self.mask = torch.tensor(rows, dtype=torch.int64).reshape(T, words)
        self.device, self.T, self.H, self.B = device, T, heads, len(prefixes)
        self.drafts = drafts

    def pieces(self, lead):
        """Per CTA the tiles of each request that its slice has (of one group,
        for the attention): {(cta, request, group): tiles}."""
        sms = torch.cuda.get_device_properties(self.device).multi_processor_count
        tiles = [(p + n + 63) // 64 if n else 0 for p, n in zip(self.prefix.tolist(), self.drafts)]
        groups = [(n * self.H + 63) // 64 for n in self.drafts]
        total = sum(g * (t + lead) for g, t in zip(groups, tiles) if t)
        start = [total // sms * c + total % sms * c // sms for c in range(sms + 1)]
        at, out = 0, {}
        for b, (t, g) in enumerate(zip(tiles, groups)):
            if not t:
                continue
            for c in range(sms):
                if start[c + 1] <= at or start[c] >= at + g * (t + lead):
                    continue
                if lead:
                    for k in range(g):
                        lo = max(start[c], at + k * (t + lead) + lead)
                        hi = min(start[c + 1], at + (k + 1) * (t + lead))
                        if hi > lo:
                            out[c, b, k] = hi - lo
                else:  # a tile belongs to the slice that its first unit falls into
                    lo, hi = max(0, -(-(start[c] - at) // g)), min(t, -(-(start[c + 1] - at) // g))
                    if hi > lo:
                        out[c, b, 0] = hi - lo
            at += g * (t + lead)
        return out

    def check_rms(self, out):
        """Two roundings to bf16 by half a step (2^-8) at most, of the weights and
        of the output, neither correlated with the values: over a request the
        error's rms stays below sqrt(2) 2^-8 of the output's."""
        want = self.reference()[0]
        for b in range(self.B):
            lo, hi = int(self.cu[b]), int(self.cu[b + 1])
            if hi > lo:
                err = (out[lo:hi].cpu().double() - want[lo:hi]).square().mean().sqrt()
                assert err <= math.sqrt(2) * 2.0 ** -8 * want[lo:hi].square().mean().sqrt(), (b, float(err))


def lengths(n, lo, hi, seed):
    return torch.randint(lo, hi + 1, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("profile", ["rising", "falling", "steps"])
@pytest.mark.parametrize("drafts", [3, 5])  # one group of rows, two
def test_rescaling_within_long_runs(cuda_device, profile, drafts):
    """Logits whose level moves along the context by more than the rescaling
    threshold (8), up in some rows and down in others, within one CTA's run."""
    c = Pooled(lengths(160, 600, 1500, 1), [drafts] * 160, 16, 2, cuda_device, scale=0.05)
    longest = max(c.pieces(LEAD).values())
    assert longest >= 8, longest
    pages = c.ckv.shape[0] // c.variants
    pos = torch.arange(pages * 64)
    g = torch.Generator().manual_seed(3)
    level = {"rising": pos / 1500 * 6 - 3, "falling": 3 - pos / 1500 * 6,
             "steps": (torch.rand(pages, generator=g) * 6 - 3).repeat_interleave(64)}[profile]
    # scale * 64 * log2(e) = 6.7 a unit: 40 over a context
    at = level.reshape(pages, 1, 64, 1).expand(pages, c.variants, 64, 64)
    c.kpe = (at + 0.02 * torch.randn(at.shape, generator=g)).reshape(-1, 64, 64).to(torch.bfloat16)
    c.q_pe[:] = torch.tensor([1.0, 0.5, -1.0, 0.25])[torch.arange(16) % 4][:, None]
    out, lse = run(c)
    c.check(out, lse)
    c.check_rms(out)


def test_rows_that_see_nothing_for_whole_tiles(cuda_device):
    """No prefix, drafts over three pages: most rows see nothing in the first
    tile, some only their last, some nothing at all."""
    c = Pooled([0] * 120, [150] * 120, 1, 4, cuda_device)
    c.mask.zero_()
    for b in range(120):
        for j in range(150):
            row = c.mask[150 * b + j]
            kind = (b + j) % 5
            if kind == 0:
                continue                                                # nothing
            seen = [j] if kind == 1 else ([149] if kind == 2 else ([70 + j % 20, j] if kind == 3 else [j // 2, 149]))
            for k in seen:
                row[k // 64] |= (1 << (k % 64)) if k % 64 < 63 else -(1 << 63)
    assert max(c.pieces(LEAD).values()) == 3  # whole groups
    out, lse = run(c)
    c.check(out, lse)
    assert torch.isinf(lse.cpu()).sum() == 120 * 30
    lse, acc, new = weigh(c, lse=lse)
    want, off = otree.weights_reference(c.q_nope, c.q_pe, c.ckv, c.kpe, c.prefix, c.table, c.cu, c.mask, SCALE,
                                        lse.cpu(), acc.cpu())
    assert ((new.cpu().double() - want).abs() <= off).all()


@pytest.mark.parametrize("drafts,most", [(1, 16), (8, 8), (9, 8)])  # one group of rows, two, three; tiles a run
def test_weights_over_many_runs_of_tiles(cuda_device, drafts, most):
    n = 150 if drafts == 1 else 100
    c = Pooled(lengths(n, 1100, 2500, 5), [drafts] * n, 16, 6, cuda_device)
    pieces = list(c.pieces(0).values())
    assert max(pieces) > most and any(p > most and p % most for p in pieces), pieces
    lse, acc, out = weigh(c)
    want, off = otree.weights_reference(c.q_nope, c.q_pe, c.ckv, c.kpe, c.prefix, c.table, c.cu, c.mask, SCALE,
                                        lse.cpu(), acc.cpu())
    assert ((out.cpu().double() - want).abs() <= off).all()
    twice = acc.clone()
    weigh(c, acc=twice, lse=lse, out=twice)
    assert torch.equal(twice, out)


@pytest.mark.parametrize("requests,drafts,heads,bound", [
    (3, 2, 16, 10),        # a row a block, 512 threads
    (9, 2, 16, 32),        # a row a block
    (15, 2, 16, 32),
    (25, 4, 16, 96),       # two rows
    (50, 4, 16, 296),      # four
    (60, 5, 24, 296),      # drafts split between groups
    (100, 4, 16, 296),
    (300, 4, 16, None),    # by record
])
def test_every_form_of_the_join(cuda_device, requests, drafts, heads, bound):
    """One request is much longer than the others, so that its groups have many
    records; some requests begin or end within a slice."""
    prefixes = lengths(requests - 1, 1, 300, 7)
    prefixes.insert(requests // 3, 40_000 if requests > 100 else 20_000)
    c = Pooled(prefixes, [drafts] * requests, heads, 8, cuda_device, variants=1 if requests > 100 else 2)
    groups = requests * drafts * heads // 64 + requests
    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    tiers = [10, 32, 96, 2 * sms]
    assert next((t for t in tiers if groups <= t), None) == (2 * sms if bound == 296 else bound)
    records = [k for k in c.pieces(LEAD) if k[1] == requests // 3 and k[2] == 0]
    assert len(records) > 8, len(records)
    out, lse = run(c)
    c.check(out, lse)
    c.check_rms(out)
    again = run(c)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    # The long request alone: other slices, the same sums up to their roundings.
    b = requests // 3
    lo, hi = int(c.cu[b]), int(c.cu[b + 1])
    alone = Pooled.__new__(Pooled)
    alone.__dict__.update(c.__dict__, q_nope=c.q_nope[lo:hi], q_pe=c.q_pe[lo:hi], prefix=c.prefix[b:b + 1], B=1, T=hi - lo,
                          table=c.table[b:b + 1], cu=c.cu[b:b + 2] - lo, mask=c.mask[lo:hi], drafts=[drafts])
    o, l = run(alone)
    bound_o, bound_l = c.reference()[2:]
    assert ((o - out[lo:hi]).cpu().double().abs() <= 2 * bound_o[lo:hi]).all()
    assert ((l - lse[lo:hi]).cpu().double().abs() <= 2 * bound_l[lo:hi]).all()
    apart = (o.double() - out[lo:hi].double()).square().mean().sqrt()
    assert apart <= 2 * math.sqrt(2) * 2.0 ** -8 * out[lo:hi].double().square().mean().sqrt()


@pytest.mark.parametrize("prefixes,drafts,heads", [
    ([1000, 77, 0], [300, 129, 65], 16),   # five words of mask, chains with branches
    ([30], [1000], 3),                      # 16 words, drafts over 16 pages
    ([5000], [512], 16),                    # a prompt's chunk
])
def test_more_than_64_drafts(cuda_device, prefixes, drafts, heads):
    c = Pooled(prefixes, drafts, heads, 9, cuda_device)
    if len(prefixes) == 1 and heads == 16:  # causal
        c.mask = torch.tensor(tree.masks_from_parents(list(range(-1, drafts[0] - 1))))
    out, lse = run(c)
    c.check(out, lse)
    c.check_rms(out)
    lse, acc, new = weigh(c, lse=lse)
    want, off = otree.weights_reference(c.q_nope, c.q_pe, c.ckv, c.kpe, c.prefix, c.table, c.cu, c.mask, SCALE,
                                        lse.cpu(), acc.cpu())
    assert ((new.cpu().double() - want).abs() <= off).all()


def test_logits_of_the_weights_are_not_shrunk(cuda_device):
    """The tensor core truncates its accumulator at each step of 16 products, by
    half a unit in the last place on average, at most 2^-24 of the partial sum.
    Partial sums grow towards the logit in proportion to their steps, so that
    three sums of 12 steps shrink it by at most 6.5 * 2^-24 = 3.9e-7 of itself
    (one of 36 steps: at most 1.1e-6, 4.7e-7 as measured)."""
    n = 40_000
    c = Pooled([n], [1], 1, 10, cuda_device, variants=1)
    acc = torch.zeros(1, c.table.shape[1] * 64, device=cuda_device)
    out = weigh(c, acc=acc, lse=torch.zeros(1, 1, device=cuda_device))[2][0, :n].cpu().double()
    k = torch.cat([c.ckv, c.kpe], -1)[c.table[0].long()].reshape(-1, 576)[:n].double()
    x = k @ torch.cat([c.q_nope, c.q_pe], -1).reshape(576).double() * (SCALE * otree.LOG2E)
    shrunk = -((out.log2() - x) * x).sum() / x.square().sum()  # the error's part along x
    assert abs(float(shrunk)) <= 6.5 * 2.0 ** -24, float(shrunk)
