"""GPU parity of tree attention (dsa_b200.tree.run) and of the accumulated
attention weights (dsa_b200.evict.accumulate) with the 64-bit oracle, whose
error bounds are the tolerances, at the sizes and masks where they can go
wrong."""

import math

import pytest
import torch

from dsa_b200 import DsaError, evict, tree
from oracle import tree as otree

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(192.0)


class Case:
    """Seeded inputs on the CPU (`host`) and the device; drafts form a random tree."""

    def __init__(self, prefixes, drafts, heads, seed=0, device="cuda", extra_pages=2, words=None, scale=1.0, tail=0):
        g = torch.Generator().manual_seed(seed)
        normal = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
        B, T = len(prefixes), sum(drafts)
        need = [(p + n + 63) // 64 for p, n in zip(prefixes, drafts)]
        width = max(1, max(need))
        pool = sum(need) + extra_pages
        perm = torch.randperm(pool, generator=g)
        table = torch.full((B, width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = perm[at:at + n].int()
            at += n
        words = words or max(1, (max(drafts) + 63) // 64)
        rows = []
        for n in drafts:
            parents = [int(torch.randint(-1, j, (1,), generator=g)) if j and j % 3 == 0 else j - 1 for j in range(n)]
            rows += [r + [0] * (words - len(r)) for r in (tree.masks_from_parents(parents) if n else [])]
        total = T + tail
        rows += [[-1] * words] * tail
        self.q_nope = (normal(total, heads, 512).float() * scale).to(torch.bfloat16)
        self.q_pe = normal(total, heads, 64)
        self.ckv, self.kpe = normal(pool, 64, 512), normal(pool, 64, 64)
        self.prefix = torch.tensor(prefixes, dtype=torch.int32)
        self.table = table
        self.cu = torch.tensor([0, *drafts]).cumsum(0).int()
        self.mask = torch.tensor(rows, dtype=torch.int64).reshape(total, words)
        self.device, self.T, self.H, self.B = device, total, heads, B

    def args(self):
        return [t.to(self.device) for t in (self.q_nope, self.q_pe, self.ckv, self.kpe, self.prefix, self.table, self.cu,
                                            self.mask)]

    def outs(self):
        return (torch.full((self.T, self.H, 512), 7.0, dtype=torch.bfloat16, device=self.device),
                torch.full((self.T, self.H), 7.0, device=self.device))

    def reference(self):
        return otree.tree_reference(self.q_nope, self.q_pe, self.ckv, self.kpe, self.prefix, self.table, self.cu,
                                    self.mask, SCALE)

    def check(self, out, lse):
        ro, rl, bo, bl = self.reference()
        mine = ~torch.isnan(rl)
        out, lse = out.cpu().double(), lse.cpu().double()
        assert torch.equal(lse[mine] == -math.inf, rl[mine] == -math.inf)
        fin = mine & (rl != -math.inf)
        assert ((lse - rl).abs() <= bl)[fin].all(), float((lse - rl).abs()[fin].max())
        bad = ((out - ro).abs() > bo)[mine]
        assert not bad.any(), (int(bad.sum()), float((out - ro).abs()[mine].max()))
        assert (out[~mine] == 7).all() and (lse[~mine] == 7).all()


def run(c, args=None):
    out, lse = c.outs()
    tree.run(*(args or c.args()), SCALE, out, lse)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("prefixes,drafts,heads", [
    ([0], [1], 16),                        # the draft alone
    ([1], [1], 1),                         # one head
    ([63], [1], 16), ([64], [1], 16), ([65], [2], 16),   # the page's border
    ([300], [4], 16),                      # one full group
    ([300], [5], 16),                      # a partial second group
    ([100, 5, 700], [3, 0, 4], 16),        # a request without drafts
    ([130], [7], 5),                       # rows that split a draft's heads between groups
    ([70, 200], [2, 1], 128),              # all heads
    ([190], [70], 3),                      # two mask words, drafts across pages
    ([10, 2000, 900, 64, 0], [1, 2, 9, 3, 6], 8),
    ([9000], [9], 16),                     # several groups over several slices
    ([20000], [1], 16),                    # one group over all slices
])
def test_matches_the_oracle(cuda_device, prefixes, drafts, heads):
    c = Case(prefixes, drafts, heads, seed=len(prefixes) + sum(prefixes), device=cuda_device)
    c.check(*run(c))


def test_many_requests(cuda_device):
    g = torch.Generator().manual_seed(3)
    prefixes = torch.randint(0, 200, (401,), generator=g).tolist()
    drafts = torch.randint(0, 6, (401,), generator=g).tolist()
    c = Case(prefixes, drafts, 4, seed=5, device=cuda_device)
    c.check(*run(c))


def test_rows_that_see_nothing(cuda_device):
    c = Case([0, 40], [6, 3], 16, seed=9, device=cuda_device)
    c.mask[1] = 0       # nothing at all: output 0, lse -inf
    c.mask[2, 0] = 1    # the first draft only, not itself
    c.mask[7] = 0       # the prefix only
    out, lse = run(c)
    c.check(out, lse)
    assert (lse[1] == -math.inf).all() and (out[1] == 0).all()


def test_masked_places_may_hold_anything(cuda_device):
    c = Case([70, 0], [9, 5], 16, seed=11, device=cuda_device)
    c.mask[:, 0] &= ~0b100  # nobody sees the third draft of either request
    for b, p in ((0, 70), (1, 0)):
        s = int(otree.slots(c.table[b], p + 3)[-1])
        c.ckv.view(-1, 512)[s, ::3] = math.nan
        c.ckv.view(-1, 512)[s, 1::3] = math.inf
        c.kpe.view(-1, 64)[s] = -math.inf
    used = torch.zeros(c.ckv.shape[0] * 64, dtype=torch.bool)
    for b, n in ((0, 79), (1, 5)):
        used[otree.slots(c.table[b], n)] = True
    c.ckv.view(-1, 512)[~used] = math.nan   # behind the last token, and pages of nobody
    c.kpe.view(-1, 64)[~used] = math.inf
    out, lse = run(c)
    assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()
    # A masked row gives nothing to any logit it is not in: the oracle masks it too.
    c.ckv, c.kpe = c.ckv.nan_to_num(0, 0, 0), c.kpe.nan_to_num(0, 0, 0)
    c.check(out, lse)


def test_a_draft_that_only_some_rows_see_is_nan_to_those_alone(cuda_device):
    c = Case([100], [4], 16, seed=12, device=cuda_device)
    c.mask[:, 0] = torch.tensor([1, 3, 5, 9])  # all follow draft 0; drafts 1, 2, 3 see themselves
    s = int(otree.slots(c.table[0], 102)[-1])  # draft 1
    c.ckv.view(-1, 512)[s, 5] = math.nan
    out, lse = run(c)
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    for i in (0, 2, 3):
        assert torch.isfinite(out[i].float()).all() and torch.isfinite(lse[i]).all()


def test_rising_logits_move_the_maximum(cuda_device):
    """Logits that grow along the context by far more than the rescaling
    threshold, so that O is rescaled again and again."""
    c = Case([1500], [3], 16, seed=13, device=cuda_device, scale=0.05)
    s = otree.slots(c.table[0], 1500)
    ramp = torch.linspace(-3, 3, 1500)[:, None]
    c.q_pe[:] = 1.0
    c.kpe.view(-1, 64)[s] = (ramp * torch.ones(1, 64)).to(torch.bfloat16)
    c.check(*run(c))
    c.kpe.view(-1, 64)[s] = (-ramp * torch.ones(1, 64)).to(torch.bfloat16)
    c.check(*run(c))


def test_strided_caches_and_wide_tables(cuda_device):
    c = Case([200, 77], [3, 5], 16, seed=14, device=cuda_device)
    args = c.args()
    both = torch.full((c.ckv.shape[0], 67, 584), math.nan, dtype=torch.bfloat16, device=cuda_device)
    both[:, :64, :512], both[:, :64, 512:576] = args[2], args[3]
    args[2], args[3] = both[:, :64, :512], both[:, :64, 512:576]
    wide = torch.full((c.B, 40), -1, dtype=torch.int64, device=cuda_device)
    wide[:, :c.table.shape[1]] = args[5]
    args[5], args[6] = wide, args[6].long()
    qs = torch.empty(c.T, 2 * c.H, 512, dtype=torch.bfloat16, device=cuda_device)[:, ::2]
    qs.copy_(args[0])
    args[0] = qs
    c.check(*run(c, args))


def test_rows_behind_the_last_request_are_left(cuda_device):
    c = Case([64, 3], [2, 2], 16, seed=15, device=cuda_device, tail=3)
    out, lse = run(c)
    assert (out[4:] == 7).all() and (lse[4:] == 7).all()
    c.check(out, lse)


def test_pages_outside_the_pool_are_masked_and_reported(cuda_device):
    c = Case([200], [2], 16, seed=16, device=cuda_device)
    args = c.args()
    args[5][0, 1] = c.ckv.shape[0] + 5
    out, lse = c.outs()
    with pytest.raises(DsaError, match="page pool"):
        tree.run(*args, SCALE, out, lse)
    assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()
    assert tree.device_status(cuda_device) == 0


@pytest.mark.parametrize("prefix,cu", [([-3], [0, 2]), ([100000], [0, 2]), ([10], [0, 3]), ([10], [2, 0]), ([10], [-1, 2])])
def test_lengths_that_do_not_fit_are_reported(cuda_device, prefix, cu):
    c = Case([10], [2], 16, seed=17, device=cuda_device)
    args = c.args()
    args[4] = torch.tensor(prefix, dtype=torch.int32, device=cuda_device)
    args[6] = torch.tensor(cu, dtype=torch.int32, device=cuda_device)
    out, lse = c.outs()
    with pytest.raises(DsaError, match="seq_len"):
        tree.run(*args, SCALE, out, lse)
    c.check(*run(c))  # the workspace is as good as before


def test_graphs_streams_and_repeats_give_the_same_bits(cuda_device):
    c = Case([3000, 500, 0], [9, 2, 3], 16, seed=18, device=cuda_device)
    args = c.args()
    out, lse = run(c, args)
    for _ in range(3):
        o2, l2 = run(c, args)
        assert torch.equal(out, o2) and torch.equal(lse, l2)
    side = torch.cuda.Stream(cuda_device)
    o3, l3 = c.outs()
    with torch.cuda.stream(side):
        tree.run(*args, SCALE, o3, l3)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        o4, l4 = c.outs()
        with torch.cuda.graph(graph, stream=side):
            tree.run(*args, SCALE, o4, l4)
    assert torch.equal(out, o3) and torch.equal(lse, l3)
    args[4][0] = 10  # the lengths of the replay are the device's
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    c.prefix[0] = 10
    c.check(o4, l4)


def weigh(c, args=None, acc=None, lse=None, out=None):
    args = args or c.args()
    if lse is None:
        lse = run(c, args)[1]
    if acc is None:
        acc = torch.rand(c.B, args[5].shape[1] * 64, generator=torch.Generator().manual_seed(1)).to(c.device)
    if out is None:
        out = torch.full_like(acc, 7.0)
    evict.accumulate(*args, SCALE, lse, acc, out)
    torch.cuda.synchronize()
    return lse, acc, out


@pytest.mark.parametrize("prefixes,drafts,heads", [
    ([0], [1], 16), ([63], [1], 16), ([64], [1], 1), ([300], [5], 16), ([100, 5, 700], [3, 0, 4], 16),
    ([130], [7], 5), ([190], [70], 3), ([70, 200], [2, 1], 128), ([9000], [9], 16), ([20000], [1], 16),
    ([10, 2000, 900, 64, 0], [1, 2, 9, 3, 6], 8),
])
def test_weights_match_the_oracle(cuda_device, prefixes, drafts, heads):
    c = Case(prefixes, drafts, heads, seed=len(prefixes) + sum(prefixes), device=cuda_device)
    lse, acc, out = weigh(c)
    want, off = otree.weights_reference(c.q_nope, c.q_pe, c.ckv, c.kpe, c.prefix, c.table, c.cu, c.mask, SCALE,
                                        lse.cpu(), acc.cpu())
    err = (out.cpu().double() - want).abs()
    assert (err <= off).all(), (float(err.max()), float(off.max()))
    # every row's weights sum to one, up to the errors of its weights
    given = (out - acc).cpu().double().sum(1)
    rows = torch.tensor([n * heads for n in drafts], dtype=torch.float64)
    assert ((given - rows).abs() <= off.sum(1) + acc.cpu().double().sum(1) * 2.0 ** -23 + rows * 2.0 ** -10).all()


def test_weights_in_place_repeat_and_skip_what_saw_nothing(cuda_device):
    c = Case([0, 2500], [3, 9], 16, seed=21, device=cuda_device)
    c.mask[1] = 0
    args = c.args()
    used = torch.zeros(c.ckv.shape[0] * 64, dtype=torch.bool)
    used[otree.slots(c.table[0], 3)] = True
    used[otree.slots(c.table[1], 2509)] = True
    args[2].view(-1, 512)[~used.to(cuda_device)] = math.nan
    lse, acc, out = weigh(c, args)
    assert torch.isfinite(out).all()
    twice = acc.clone()
    weigh(c, args, acc=twice, lse=lse, out=twice)
    assert torch.equal(twice, out)
    again = weigh(c, args, acc=acc, lse=lse)[2]
    assert torch.equal(again, out)
    strided = torch.full((c.B, acc.shape[1] + 5), 3.0, device=cuda_device)
    view = strided[:, :acc.shape[1]]
    weigh(c, args, acc=acc, lse=lse, out=view)
    assert torch.equal(view, out) and (strided[:, acc.shape[1]:] == 3).all()


def test_inputs_in_other_layouts_give_the_same_bits(cuda_device):
    c = Case([70, 900], [5, 3], 16, seed=31, device=cuda_device)
    args = c.args()
    out, lse = run(c, args)
    _, acc, weights = weigh(c, args, lse=lse)
    apart = lambda t: torch.stack((t, t), -1)[..., 0]  # noqa: E731  every second element
    assert not any(apart(args[i]).is_contiguous() for i in (0, 1, 4, 7))
    other = [apart(args[0]), apart(args[1]), args[2], args[3], apart(args[4]), apart(args[5].long()),
             apart(args[6].long()), apart(args[7])]
    o, l = run(c, other)
    assert torch.equal(o, out) and torch.equal(l, lse)
    assert torch.equal(weigh(c, other, acc=acc, lse=apart(lse))[2], weights)


def test_a_page_that_a_request_has_twice_and_another_shares(cuda_device):
    c = Case([200, 130], [3, 2], 16, seed=32, device=cuda_device)
    c.table[0, 1] = c.table[0, 0]
    c.table[1, 0] = c.table[0, 2]
    c.check(*run(c))
    lse, acc, out = weigh(c)
    want, off = otree.weights_reference(c.q_nope, c.q_pe, c.ckv, c.kpe, c.prefix, c.table, c.cu, c.mask, SCALE,
                                        lse.cpu(), acc.cpu())
    assert ((out.cpu().double() - want).abs() <= off).all()


def test_no_drafts_at_all(cuda_device):
    c = Case([5, 70], [1, 1], 16, seed=22, device=cuda_device)
    args = c.args()
    acc = torch.rand(2, args[5].shape[1] * 64, device=cuda_device)
    out = torch.zeros_like(acc)
    args[6].zero_()
    o, l = c.outs()
    tree.run(*args, SCALE, o, l)
    evict.accumulate(*args, SCALE, l, acc, out)
    assert (o == 7).all() and (l == 7).all() and torch.equal(out, acc)
    args[0], args[1], args[7] = args[0][:0], args[1][:0], args[7][:0]
    out.zero_()
    tree.run(*args, SCALE, o[:0], l[:0])
    evict.accumulate(*args, SCALE, l[:0], acc, out)
    assert torch.equal(out, acc)


def test_pages_behind_four_gigabytes(cuda_device):
    """Page offsets that pass 32 bits, in a pool of 70000 pages (4.6 GB of ckv)."""
    c = Case([300, 90], [4, 2], 16, seed=23, device=cuda_device)
    args = c.args()
    need = [int((t >= 0).sum()) for t in c.table]
    ckv = torch.zeros(70000, 64, 512, dtype=torch.bfloat16, device=cuda_device)
    kpe = torch.zeros(70000, 64, 64, dtype=torch.bfloat16, device=cuda_device)
    far = torch.full_like(args[5], -1)
    at = 69999
    for b, n in enumerate(need):
        for k in range(n):
            far[b, k] = at
            ckv[at], kpe[at] = args[2][args[5][b, k]], args[3][args[5][b, k]]
            at -= 700
    near = run(c, args)
    args[2], args[3], args[5] = ckv, kpe, far
    out, lse = run(c, args)
    c.check(out, lse)
    assert torch.equal(out, near[0]) and torch.equal(lse, near[1])
    acc = torch.rand(2, far.shape[1] * 64, device=cuda_device)
    got = weigh(c, args, acc=acc, lse=lse)[2]
    assert torch.equal(got, weigh(c, c.args(), acc=acc, lse=lse)[2])


def test_two_streams_and_two_graphs_at_once(cuda_device):
    cases = [Case([4000, 900, 2500], [9, 2, 5], 16, seed=24, device=cuda_device),
             Case([700, 6000], [20, 3], 8, seed=25, device=cuda_device)]
    args = [c.args() for c in cases]
    want = [run(c, a) for c, a in zip(cases, args)]
    accs = [weigh(c, a, lse=w[1]) for c, a, w in zip(cases, args, want)]
    streams = [torch.cuda.Stream(cuda_device) for _ in cases]
    outs = [c.outs() for c in cases]
    news = [torch.zeros_like(a[1]) for a in accs]
    graphs = []
    for c, a, o, w, n, s in zip(cases, args, outs, accs, news, streams):
        s.wait_stream(torch.cuda.current_stream(cuda_device))
        with torch.cuda.stream(s):
            tree.run(*a, SCALE, *o)
            evict.accumulate(*a, SCALE, o[1], w[1], n)
            s.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=s):
                tree.run(*a, SCALE, *o)
                evict.accumulate(*a, SCALE, o[1], w[1], n)
    for together in (False, True):
        for t in [*outs[0], *outs[1], *news]:
            t.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for c, a, o, w, n, s, g in zip(cases, args, outs, accs, news, streams, graphs):
                with torch.cuda.stream(s):
                    if together:
                        g.replay()
                    else:
                        tree.run(*a, SCALE, *o)
                        evict.accumulate(*a, SCALE, o[1], w[1], n)
        torch.cuda.synchronize()
        for o, w, n, a in zip(outs, want, news, accs):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1]) and torch.equal(n, a[2])


def test_other_requests_non_finite_queries_do_not_leak(cuda_device):
    """A group's columns behind its rows hold the next request's queries."""
    c = Case([500, 300], [1, 2], 16, seed=26, device=cuda_device)
    args = c.args()
    good = run(c, args)
    args[0] = args[0].clone()
    args[0][1:] = math.nan
    out, lse = run(c, args)
    assert torch.equal(out[0], good[0][0]) and torch.equal(lse[0], good[1][0])
    assert torch.isnan(out[1:]).all() and torch.isnan(lse[1:]).all()
    acc = torch.zeros(2, args[5].shape[1] * 64, device=cuda_device)
    got = weigh(c, args, acc=acc, lse=lse)[2]
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1, :300]).all() and (got[1, 302:] == 0).all()


def test_refusals(cuda_device):
    c = Case([100, 20], [3, 2], 16, seed=27, device=cuda_device)
    q, pe, ckv, kpe, prefix, table, cu, mask = c.args()
    out, lse = c.outs()
    good = dict(q_nope=q, q_pe=pe, ckv_cache=ckv, kpe_cache=kpe, prefix_lens=prefix, block_table=table, cu_drafts=cu,
                tree_mask=mask, sm_scale=SCALE)
    tree.run(**good, output=out, lse=lse)
    acc = torch.zeros(2, table.shape[1] * 64, device=cuda_device)
    evict.accumulate(**good, lse=lse, acc=acc, out=acc)
    wrong = [dict(q_nope=q.float()), dict(q_nope=q[:, :, :511]), dict(q_nope=q.cpu()), dict(q_pe=pe[1:]), dict(q_pe=pe.half()),
             dict(q_nope=q.repeat(1, 9, 1), q_pe=pe.repeat(1, 9, 1)), dict(ckv_cache=ckv.flatten(0, 1)), dict(ckv_cache=ckv[1:]),
             dict(kpe_cache=kpe[:, :, :32]), dict(prefix_lens=prefix.long()), dict(prefix_lens=prefix[:1]),
             dict(block_table=table.float()), dict(block_table=table[0]), dict(block_table=table[:1]), dict(cu_drafts=cu[:-1]),
             dict(cu_drafts=cu.float()), dict(tree_mask=mask.int()), dict(tree_mask=mask[:, 0]), dict(tree_mask=mask[1:]),
             dict(tree_mask=mask[:, :0]), dict(block_table=table.cpu())]
    for change in wrong:
        with pytest.raises(ValueError):
            tree.run(**{**good, **change}, output=out, lse=lse)
        with pytest.raises(ValueError):
            evict.accumulate(**{**good, **change}, lse=lse, acc=acc, out=acc)
    for o, l in ((out.float(), lse), (out[1:], lse), (out.transpose(0, 1), lse), (out, lse.double()), (out, lse[:, :8]),
                 (out.cpu(), lse), (out, lse.t().contiguous().t())):
        with pytest.raises(ValueError):
            tree.run(**good, output=o, lse=l)
    for l, a, o in ((lse.double(), acc, acc), (lse[1:], acc, acc), (lse, acc.double(), acc), (lse, acc[:, :-1], acc),
                    (lse, acc, acc[:1]), (lse, acc.t().contiguous().t(), acc), (lse, acc, acc.cpu()),
                    (lse, acc[:1].expand(2, -1), acc)):
        with pytest.raises(ValueError):
            evict.accumulate(**good, lse=l, acc=a, out=o)


def test_weights_of_accepted_drafts_alone(cuda_device):
    """Rejected rows get an lse of -inf; the accepted ones need not be the first."""
    c = Case([130, 61, 2000], [4, 9, 6], 16, seed=41, device=cuda_device)
    for b, parents in enumerate(([-1, 0, 0, 0], [-1, -1, 0, 1, 2, 2, 4, 3, 6], [-1, 0, 0, 1, 1, 3])):
        c.mask[int(c.cu[b]):int(c.cu[b + 1])] = torch.tensor(tree.masks_from_parents(parents))
    accepted = torch.zeros(19, dtype=torch.bool)
    accepted[[0, 3, 4 + 0, 4 + 2, 4 + 4, 4 + 6, 4 + 8]] = True  # {0, 3}, {0, 2, 4, 6, 8} and none
    args = c.args()
    lse = run(c, args)[1].masked_fill(~accepted.to(cuda_device)[:, None], -math.inf)
    acc = torch.zeros(3, args[5].shape[1] * 64, device=cuda_device)
    out = weigh(c, args, acc=acc, lse=lse)[2].cpu()
    want, off = otree.weights_reference(c.q_nope, c.q_pe, c.ckv, c.kpe, c.prefix, c.table, c.cu, c.mask, SCALE,
                                        lse.cpu(), acc.cpu())
    assert ((out.double() - want).abs() <= off).all()
    # An accepted row's weights sum to 2^(its lse - the given one); the test's own sum is in 64 bits.
    lse_off = (torch.exp2(c.reference()[3]) - 1)[accepted].sum()
    assert ((out.double().sum(1) - torch.tensor([2 * 16.0, 5 * 16.0, 0.0])).abs() <= off.sum(1) + lse_off).all()
    assert (out[0, 133] > 0) and (out[0, 131:133] == 0).all() and (out[2] == 0).all()


def test_two_threads_on_one_stream(cuda_device, monkeypatch):
    """A call is two launches that share the stream's records: another thread's
    must not come between them."""
    import threading

    monkeypatch.setattr(tree, "_CHECK", False)
    cases = [Case([4000, 900, 2500], [9, 2, 5], 16, seed=42, device=cuda_device),
             Case([700, 6000, 64], [20, 3, 1], 8, seed=43, device=cuda_device)]
    args = [c.args() for c in cases]
    want = [run(c, a) for c, a in zip(cases, args)]
    outs = [[c.outs() for _ in range(150)] for c in cases]
    torch.cuda.synchronize()
    start, errors = threading.Barrier(2), []

    def calls(a, mine):
        try:
            start.wait()
            for o in mine:
                tree.run(*a, SCALE, *o)
        except Exception as e:  # noqa: BLE001  raised below, in the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=calls, args=x) for x in zip(args, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert tree.device_status(cuda_device) == 0
    for w, mine in zip(want, outs):
        for o in mine:
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


def test_back_to_back_and_concurrent_calls_without_waits(cuda_device, monkeypatch):
    """Eager calls that nothing waits between: attention, weights and eviction
    overlap the next launch on their stream, and those of another stream."""
    monkeypatch.setattr(tree, "_CHECK", False)
    cases = [Case([4000, 900, 2500], [9, 2, 5], 16, seed=44, device=cuda_device),
             Case([700, 6000], [20, 3], 8, seed=45, device=cuda_device)]
    args = [c.args() for c in cases]
    state = []
    for c, a in zip(cases, args):
        out, lse = run(c, a)
        _, acc, new = weigh(c, a, lse=lse)
        B, budget = c.B, 256
        caches = [torch.cat([t, torch.zeros(B * 4, *t.shape[1:], dtype=t.dtype, device=t.device)]) for t in a[2:4]]
        fresh = (a[2].shape[0] + torch.arange(B * 4, device=cuda_device)).int().reshape(B, 4)
        lens = (a[4] + a[6][1:] - a[6][:-1]).int()
        keep, kept = (torch.empty(B, budget, dtype=torch.int32, device=cuda_device),
                      torch.empty(B, dtype=torch.int32, device=cuda_device))
        new2 = torch.empty(B, 256, device=cuda_device)

        def step(a=a, c=c, caches=caches, out=out, lse=lse, acc=acc, new=new, lens=lens, fresh=fresh, keep=keep, kept=kept,
                 new2=new2):
            rows = (*a[:2], *caches, *a[4:], SCALE)
            tree.run(*rows, out, lse)
            evict.accumulate(*rows, lse, acc, new)
            evict.run(new, lens, a[5], fresh, *caches, None, 3, 20, keep, kept, new2)

        step()
        torch.cuda.synchronize()
        mine = [out, lse, new, keep, kept, new2, *caches]
        state.append((step, mine, [t.clone() for t in mine]))
        kept_ = otree.evict_reference(new.cpu(), lens.cpu(), budget, 3, 20)
        assert all(keep[b, :len(k)].tolist() == k for b, k in enumerate(kept_))
    streams = [torch.cuda.Stream(cuda_device) for _ in cases]
    for s, (step, _, _) in zip(streams, state):
        s.wait_stream(torch.cuda.current_stream(cuda_device))
        with torch.cuda.stream(s):
            step()  # the stream's workspaces exist
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (_, mine, _) in zip(streams, state):
            for t in mine[:6]:
                t.zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for s, (step, _, _) in zip(streams, state):
                with torch.cuda.stream(s):
                    step()
        torch.cuda.synchronize()
        for _, mine, want in state:
            assert all(torch.equal(x, y) for x, y in zip(mine, want))
    assert tree.device_status(cuda_device) == 0 and evict.device_status(cuda_device) == 0


def test_rows_before_the_first_request_are_left(cuda_device):
    c = Case([130, 0, 20], [5, 3, 2], 16, seed=46, device=cuda_device, tail=4)
    for name in ("q_nope", "q_pe", "mask"):  # the four rows of no request go first
        setattr(c, name, getattr(c, name).roll(4, 0))
    c.cu = c.cu + 4
    out, lse = run(c)
    c.check(out, lse)  # the first rows too: NaN in the reference, left as they were
    assert (out[:4] == 7).all() and (lse[:4] == 7).all()
    lse, acc, new = weigh(c, lse=lse)
    want, off = otree.weights_reference(c.q_nope, c.q_pe, c.ckv, c.kpe, c.prefix, c.table, c.cu, c.mask, SCALE,
                                        lse.cpu(), acc.cpu())
    assert ((new.cpu().double() - want).abs() <= off).all()


def test_output_over_the_queries(cuda_device):
    """A group's rows are written after its queries were read, by the CTA that
    read them or by the join, so the output may take the queries' place."""
    c = Case([3000, 500, 0, 64], [9, 2, 3, 30], 16, seed=47, device=cuda_device)
    args = c.args()
    out, lse = run(c, args)
    for _ in range(5):
        q = args[0].clone()
        tree.run(q, *args[1:], SCALE, q, lse)
        assert torch.equal(q, out)


def test_outputs_over_inputs_are_refused(cuda_device):
    c = Case([100, 20], [3, 2], 16, seed=48, device=cuda_device)
    args = c.args()
    out, lse = c.outs()
    tree.run(*args, SCALE, out, lse)
    acc = torch.zeros(2, args[5].shape[1] * 64, device=cuda_device)
    shifted = torch.empty(6, 16, 512, dtype=torch.bfloat16, device=cuda_device)
    shifted[:5] = args[0]
    for q, o, l in ((shifted[:5], shifted[1:], lse), (args[0], args[2].view(-1)[:out.numel()].view(out.shape), lse),
                    (args[0], out, out.view(torch.float32).view(-1)[:80].view(5, 16)),
                    (args[0], out, args[0].view(torch.float32).view(-1)[:80].view(5, 16))):
        with pytest.raises(ValueError, match="share memory"):
            tree.run(q, *args[1:], SCALE, o, l)
    big = torch.zeros(2 * acc.numel(), device=cuda_device)
    for l, o in ((big[:80].view(5, 16), big[64:64 + acc.numel()].view(acc.shape)),
                 (lse, args[3].view(torch.float32).view(-1)[:acc.numel()].view(acc.shape))):
        with pytest.raises(ValueError, match="share"):
            evict.accumulate(*args, SCALE, l, acc, o)
