"""GPU tests of eviction (dsa_b200.evict.run): the kept positions and every
moved byte equal the oracle's, and the decode loop that uses it with the tree
attention, the accumulated weights, the indexer and the sparse attention."""

import math

import pytest
import torch

from dsa_b200 import DsaError, attention, cache, evict, indexer, tree, workloads
from oracle import attention as oatt
from oracle import compare
from oracle import indexer as oix
from oracle import tree as otree

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, seq, budget, device, seed=0, pool=None, width=None, new_width=None, shared=False):
        g = torch.Generator().manual_seed(seed)
        need = [(n + 63) // 64 for n in seq]
        fresh = [(min(n, budget) + 63) // 64 for n in seq]
        width = width or max(1, max(need))
        new_width = new_width or (budget + 63) // 64
        old = 40 if shared else sum(need)
        pool = old + sum(fresh) + 2
        perm = torch.randperm(pool, generator=g)
        self.table = torch.full((len(seq), width), -1, dtype=torch.int32)
        self.new_table = torch.full((len(seq), new_width), -1, dtype=torch.int32)
        at, to = 0, old
        for b in range(len(seq)):
            self.table[b, :need[b]] = perm[torch.randint(0, old, (need[b],), generator=g) if shared
                                           else slice(at, at + need[b])].int()
            self.new_table[b, :fresh[b]] = perm[to:to + fresh[b]].int()
            at, to = at + need[b], to + fresh[b]
        self.acc = torch.randn(len(seq), width * 64, generator=g).mul(2).exp()
        self.seq = torch.tensor(seq, dtype=torch.int32)
        self.ckv = torch.randint(-32768, 32768, (pool, 64, 512), generator=g, dtype=torch.int16).view(torch.bfloat16)
        self.kpe = torch.randint(-32768, 32768, (pool, 64, 64), generator=g, dtype=torch.int16).view(torch.bfloat16)
        self.index = torch.randint(0, 256, (pool, 64, 1, 132), generator=g, dtype=torch.uint8)
        self.budget, self.device = budget, device

    def run(self, sink, recent, index=True, acc=None, new_acc=None):
        d = self.device
        got = {"ckv": self.ckv.to(d), "kpe": self.kpe.to(d), "index": self.index.to(d),
               "keep": torch.full((len(self.seq), self.budget), 7, dtype=torch.int32, device=d),
               "seq": torch.full((len(self.seq),), 7, dtype=torch.int32, device=d),
               "acc": torch.full((len(self.seq), self.new_table.shape[1] * 64), 7.0, device=d) if new_acc is None else new_acc}
        evict.run(self.acc.to(d) if acc is None else acc, self.seq.to(d), self.table.to(d), self.new_table.to(d), got["ckv"],
                  got["kpe"], got["index"] if index else None, sink, recent, got["keep"], got["seq"], got["acc"])
        torch.cuda.synchronize()
        return {k: v.cpu() for k, v in got.items()}

    def check(self, got, sink, recent, index=True):
        kept = otree.evict_reference(self.acc, self.seq, self.budget, sink, recent)
        ckv, kpe = self.ckv.view(torch.int16).reshape(-1, 512).clone(), self.kpe.view(torch.int16).reshape(-1, 64).clone()
        pages = self.index.reshape(-1, 64 * 132).clone()
        for b, pos in enumerate(kept):
            n, pos = len(pos), torch.tensor(pos, dtype=torch.long)
            assert got["seq"][b] == n
            assert torch.equal(got["keep"][b, :n].long(), pos) and (got["keep"][b, n:] == -1).all()
            want = torch.zeros(got["acc"].shape[1])
            want[:n] = self.acc[b, pos]
            assert torch.equal(got["acc"][b].view(torch.int32), want.view(torch.int32))
            src = self.table[b].long()[pos // 64] * 64 + pos % 64
            dst = otree.slots(self.new_table[b], n)
            ckv[dst], kpe[dst] = ckv[src], kpe[src]
            if index:
                keys, scales = pages[:, :8192].unflatten(1, (64, 128)), pages[:, 8192:].unflatten(1, (64, 4))
                keys[dst // 64, dst % 64] = keys[src // 64, src % 64]
                scales[dst // 64, dst % 64] = scales[src // 64, src % 64]
        assert torch.equal(got["ckv"].view(torch.int16).reshape(-1, 512), ckv)
        assert torch.equal(got["kpe"].view(torch.int16).reshape(-1, 64), kpe)
        assert torch.equal(got["index"].reshape(-1, 64 * 132), pages)


@pytest.mark.parametrize("seq,budget,sink,recent", [
    ([1], 1, 0, 0), ([2], 1, 0, 0), ([2], 1, 1, 0), ([2], 1, 0, 1),
    ([0, 5, 100], 64, 4, 8),                 # all within the budget
    ([64, 65, 66, 0], 64, 4, 8),             # at the budget's border
    ([500], 100, 0, 0), ([500], 100, 40, 60),  # no token between is kept
    ([500], 100, 100, 0), ([5001], 1024, 4, 64),
    ([3000, 64, 1999, 20000, 1], 515, 5, 77),  # odd sizes, four tokens a warp
    ([9000] * 40, 63, 1, 2),                 # more requests: smaller clusters
    ([700] * 400, 130, 3, 11),
])
def test_matches_the_oracle(cuda_device, seq, budget, sink, recent):
    c = Case(seq, budget, cuda_device, seed=sum(seq) % 1000)
    c.check(c.run(sink, recent), sink, recent)


def test_equal_weights_keep_the_earlier(cuda_device):
    c = Case([4000, 9000, 300], 200, cuda_device, seed=1)
    c.acc[:] = 0.25
    c.acc[1, 100:8000:7] = 0.0
    c.acc[2] = (torch.arange(c.acc.shape[1]) % 3).float()
    c.check(c.run(3, 50), 3, 50)


def test_signed_zeros_infinities_subnormals_and_nan(cuda_device):
    c = Case([2000, 2000, 2000, 2000], 300, cuda_device, seed=2)
    c.acc[0, ::5] = math.nan                  # more NaN than the budget
    c.acc[1, ::50] = math.nan
    c.acc[1, 1::40] = math.inf
    c.acc[1, 2::3] = -math.inf
    c.acc[2] = 0.0
    c.acc[2, ::2] = -0.0                      # equal to 0
    c.acc[3] = torch.arange(c.acc.shape[1]).flip(0).int().view(torch.float32)  # subnormal
    c.check(c.run(2, 9), 2, 9)


def test_neighbouring_floats_are_told_apart(cuda_device):
    """Keys that differ in their last ten bits only: all three radix passes."""
    c = Case([30000], 1000, cuda_device, seed=3)
    bits = torch.randint(0, 3000, (1, c.acc.shape[1]), generator=torch.Generator().manual_seed(4), dtype=torch.int32)
    c.acc = (bits + 0x3F800000).view(torch.float32)
    c.check(c.run(0, 0), 0, 0)
    c.acc = -c.acc
    c.check(c.run(0, 0), 0, 0)


def test_contexts_longer_than_the_cluster_can_hold(cuda_device):
    c = Case([450_000, 300_000], 2000, cuda_device, seed=5, shared=True)  # 16 CTAs a request: it fits
    c.check(c.run(10, 500), 10, 500)
    c = Case([450_000, *[70] * 78, 300_000], 2000, cuda_device, seed=5, shared=True)  # 2 CTAs: it does not
    c.check(c.run(10, 500), 10, 500)


def test_wide_tables_strided_weights_and_no_index_cache(cuda_device):
    c = Case([900, 20], 300, cuda_device, seed=6, width=33, new_width=9)
    got = c.run(4, 4, index=False)
    c.check(got, 4, 4, index=False)
    wide = torch.full((2, c.acc.shape[1] + 3), math.inf, device=cuda_device)
    wide[:, :-3] = c.acc.to(cuda_device)
    target = torch.full((2, 9 * 64 + 1), 5.0, device=cuda_device)
    got = c.run(4, 4, acc=wide[:, :-3], new_acc=target[:, :-1])
    c.check(got, 4, 4)
    assert (target[:, -1] == 5).all()


def test_tables_and_lengths_in_other_layouts(cuda_device):
    c = Case([900, 70, 300], 256, cuda_device, seed=41)
    apart = lambda t: torch.stack((t, t), -1)[..., 0]  # noqa: E731  every second element
    c.seq, c.table, c.new_table = apart(c.seq), apart(c.table.long()), apart(c.new_table.long())
    c.check(c.run(4, 16), 4, 16)


def test_strided_caches(cuda_device):
    c = Case([900, 400], 300, cuda_device, seed=7)
    both = torch.zeros(c.ckv.shape[0], 64, 576, dtype=torch.bfloat16)
    both[:, :, :512], both[:, :, 512:] = c.ckv, c.kpe
    both = both.to(cuda_device)
    keep = torch.empty(2, 300, dtype=torch.int32, device=cuda_device)
    seq = torch.empty(2, dtype=torch.int32, device=cuda_device)
    acc = torch.empty(2, c.new_table.shape[1] * 64, device=cuda_device)
    evict.run(c.acc.to(cuda_device), c.seq.to(cuda_device), c.table.to(cuda_device).long(),
              c.new_table.to(cuda_device), both[:, :, :512], both[:, :, 512:], None, 4, 4, keep, seq, acc)
    got = {"ckv": both[:, :, :512].cpu().contiguous(), "kpe": both[:, :, 512:].cpu().contiguous(), "index": c.index,
           "keep": keep.cpu(), "seq": seq.cpu(), "acc": acc.cpu()}
    c.check(got, 4, 4, index=False)


def test_bad_lengths_and_pages_are_reported(cuda_device):
    c = Case([900, 400], 300, cuda_device, seed=8)
    c.seq[0] = 100_000
    with pytest.raises(DsaError, match="seq_len"):
        c.run(0, 0)
    c.seq[0] = -5
    with pytest.raises(DsaError, match="seq_len"):
        c.run(0, 0)
    c = Case([900, 400], 300, cuda_device, seed=8)
    c.table[0, 2] = c.ckv.shape[0]
    with pytest.raises(DsaError, match="page"):
        c.run(0, 0)
    c = Case([900, 400], 300, cuda_device, seed=8)
    c.new_table[1, 2] = -1
    with pytest.raises(DsaError, match="page"):
        c.run(0, 0)
    assert evict.device_status(cuda_device) == 0


def test_new_pages_that_are_in_use_are_refused(cuda_device):
    c = Case([900, 400], 300, cuda_device, seed=9)
    c.new_table[0, 1] = c.table[1, 3]
    with pytest.raises(ValueError, match="still in use"):
        c.run(0, 0)
    c = Case([900, 400], 300, cuda_device, seed=9)
    c.new_table[0, 1] = c.new_table[1, 0]
    with pytest.raises(ValueError, match="twice"):
        c.run(0, 0)


def test_refusals(cuda_device):
    c = Case([900, 400], 300, cuda_device, seed=10)
    d = cuda_device
    good = dict(acc=c.acc.to(d), seq_lens=c.seq.to(d), block_table=c.table.to(d), new_block_table=c.new_table.to(d),
                ckv_cache=c.ckv.to(d), kpe_cache=c.kpe.to(d), k_index_cache_fp8=c.index.to(d), num_sink=1, num_recent=1,
                keep=torch.empty(2, 300, dtype=torch.int32, device=d), new_seq_lens=torch.empty(2, dtype=torch.int32, device=d),
                new_acc=torch.empty(2, 320, device=d))
    evict.run(**good)
    for change in (dict(num_sink=-1), dict(num_sink=200, num_recent=101), dict(keep=good["keep"][:, :0]),
                   dict(keep=torch.empty(2, 321, dtype=torch.int32, device=d)), dict(keep=good["keep"].long()),
                   dict(acc=good["acc"][:, 1:]), dict(acc=good["acc"].double()), dict(new_acc=good["new_acc"][:, :-1]),
                   dict(new_acc=good["acc"][:, :320], acc=good["acc"]), dict(new_acc=good["acc"][:, 64:384]), dict(seq_lens=good["seq_lens"].long()),
                   dict(new_seq_lens=good["new_seq_lens"][:1]), dict(block_table=good["block_table"].float()),
                   dict(kpe_cache=good["kpe_cache"][1:]), dict(ckv_cache=good["ckv_cache"].half()),
                   dict(k_index_cache_fp8=good["k_index_cache_fp8"][1:]), dict(acc=good["acc"].cpu()),
                   dict(new_block_table=good["new_block_table"][:1])):
        with pytest.raises(ValueError):
            evict.run(**{**good, **change})


def test_graph_and_side_stream(cuda_device):
    c = Case([900, 5000], 300, cuda_device, seed=11)
    d = cuda_device
    ckv, kpe, index = c.ckv.to(d), c.kpe.to(d), c.index.to(d)
    ins = [c.acc.to(d), c.seq.to(d), c.table.to(d), c.new_table.to(d)]
    keep = torch.empty(2, 300, dtype=torch.int32, device=d)
    seq, acc = torch.empty(2, dtype=torch.int32, device=d), torch.empty(2, 320, device=d)
    side = torch.cuda.Stream(d)
    side.wait_stream(torch.cuda.current_stream(d))
    with torch.cuda.stream(side):
        evict.run(*ins, ckv, kpe, index, 4, 10, keep, seq, acc)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            evict.run(*ins, ckv, kpe, index, 4, 10, keep, seq, acc)
    c.acc = c.acc.flip(1).contiguous()
    c.seq[0] = 250
    ins[0].copy_(c.acc)
    ins[1].copy_(c.seq)
    for t, host in ((ckv, c.ckv), (kpe, c.kpe), (index, c.index)):
        t.copy_(host)
    graph.replay()
    torch.cuda.synchronize()
    c.check({"ckv": ckv.cpu(), "kpe": kpe.cpu(), "index": index.cpu(), "keep": keep.cpu(), "seq": seq.cpu(),
             "acc": acc.cpu()}, 4, 10)


def test_a_decode_loop_with_eviction(cuda_device):
    """Keys are written, drafts verified, their weights accumulated, the caches
    brought down to the budget; then drafts, indexer and sparse attention run on
    the new pages and give what they give on the kept tokens alone."""
    d, lens, drafts, budget, scale = cuda_device, [5000, 2600, 700], [4, 3, 2], 2400, 1 / math.sqrt(192)
    g = torch.Generator().manual_seed(12)
    dec = workloads.make_decode_inputs([n + 64 for n in lens], seed=12, device=d,
                                       pool_pages=sum((n + 127) // 64 for n in lens) + 3 * 40)
    ix = dec.indexer
    prefix = torch.tensor(lens, dtype=torch.int32, device=d)
    cu = torch.tensor([0, *drafts], device=d).cumsum(0).int()
    mask = torch.tensor([r for n in drafts for r in tree.masks_from_parents(list(range(-1, n - 1)))], device=d)
    T = sum(drafts)
    qn, qp = (torch.randn(T, 16, w, generator=g).to(torch.bfloat16).to(d) for w in (512, 64))
    bt = ix.block_table
    new_slots = torch.cat([bt[b].long()[(torch.arange(n, device=d) + lens[b]) // 64] * 64
                           + (torch.arange(n, device=d) + lens[b]) % 64 for b, n in enumerate(drafts)])
    cache.write_index_k(torch.randn(T, 128, generator=g).to(torch.bfloat16).to(d), new_slots, ix.k_index_cache_fp8)

    acc = torch.zeros(3, bt.shape[1] * 64, device=d)
    out, lse = torch.empty(T, 16, 512, dtype=torch.bfloat16, device=d), torch.empty(T, 16, device=d)
    step = (qn, qp, dec.ckv_cache, dec.kpe_cache, prefix, bt, cu, mask, scale)
    tree.run(*step, out, lse)
    evict.accumulate(*step, lse, acc, acc)
    total = acc.sum(1).cpu()
    assert torch.allclose(total, torch.tensor(drafts) * 16.0, rtol=1e-3)

    seq = prefix + torch.tensor(drafts, dtype=torch.int32, device=d)
    used = {int(x) for b, n in enumerate(seq.tolist()) for x in bt[b, :(n + 63) // 64]}
    free = torch.tensor([x for x in range(dec.ckv_cache.shape[0]) if x not in used], dtype=torch.int32)
    wide = (budget + 63) // 64 + 1  # room for the next drafts
    new_bt = free[:3 * wide].reshape(3, wide).to(d)
    keep = torch.empty(3, budget, dtype=torch.int32, device=d)
    new_seq, new_acc = torch.empty_like(seq), torch.empty(3, wide * 64, device=d)
    evict.run(acc, seq, bt, new_bt, dec.ckv_cache, dec.kpe_cache, ix.k_index_cache_fp8, 4, 64, keep, new_seq, new_acc)
    kept = otree.evict_reference(acc.cpu(), seq.cpu(), budget, 4, 64)
    assert new_seq.tolist() == [len(k) for k in kept]
    for b, k in enumerate(kept):
        assert keep[b, :len(k)].tolist() == k

    # The next drafts on the new pages, against a cache that holds the kept tokens alone.
    qn2, qp2 = (torch.randn(T, 16, w, generator=g).to(torch.bfloat16).to(d) for w in (512, 64))
    plain_ckv, plain_kpe = torch.zeros(3 * wide, 64, 512, dtype=torch.bfloat16), torch.zeros(3 * wide, 64, 64, dtype=torch.bfloat16)
    plain_bt = torch.arange(3 * wide, dtype=torch.int32).reshape(3, wide)
    for b, k in enumerate(kept):
        src = bt[b].cpu().long()[torch.tensor(k) // 64] * 64 + torch.tensor(k) % 64
        dst = otree.slots(plain_bt[b], len(k))
        plain_ckv.view(-1, 512)[dst] = dec.ckv_cache.cpu().reshape(-1, 512)[src]
        plain_kpe.view(-1, 64)[dst] = dec.kpe_cache.cpu().reshape(-1, 64)[src]
        drafts_at = torch.arange(drafts[b]) + len(k)
        for cache_, rows, table in ((plain_ckv, 512, plain_bt), (plain_kpe, 64, plain_bt)):
            fresh = torch.randn(drafts[b], rows, generator=torch.Generator().manual_seed(b)).to(torch.bfloat16)
            cache_.view(-1, rows)[table[b].long()[drafts_at // 64] * 64 + drafts_at % 64] = fresh
            mine = dec.ckv_cache if rows == 512 else dec.kpe_cache
            mine.view(-1, rows)[(new_bt[b].cpu().long()[drafts_at // 64] * 64 + drafts_at % 64).to(d)] = fresh.to(d)
    o2, l2 = torch.empty_like(out), torch.empty_like(lse)
    tree.run(qn2, qp2, dec.ckv_cache, dec.kpe_cache, new_seq, new_bt, cu, mask, scale, o2, l2)
    o3, l3 = torch.empty_like(out), torch.empty_like(lse)
    tree.run(qn2, qp2, plain_ckv.to(d), plain_kpe.to(d), new_seq, plain_bt.to(d), cu, mask, scale, o3, l3)
    assert torch.equal(o2, o3) and torch.equal(l2, l3)

    topk = torch.full((3, 2048), 7, dtype=torch.int32, device=d)
    indexer.run(ix.q_index_fp8, ix.k_index_cache_fp8, ix.weights, new_seq, new_bt, topk)
    ref, scores = oix.indexer_reference(ix.q_index_fp8.cpu(), ix.k_index_cache_fp8.cpu(), ix.weights.cpu(), new_seq.cpu(),
                                        new_bt.cpu())
    ku = ix.k_index_cache_fp8.cpu().view(torch.uint8).reshape(-1)
    bounds = [oix.score_error_bound(ix.q_index_fp8[b].cpu(), ku, ix.weights[b].cpu(), int(new_seq[b]), new_bt[b].cpu().long())
              for b in range(3)]
    rep = compare.compare_topk(topk.cpu(), ref, scores, bounds, new_seq.cpu(), new_bt.cpu(), ix.num_pages)
    assert rep.ok, rep.problems[:5]
    so, sl = torch.empty(3, 16, 512, dtype=torch.bfloat16, device=d), torch.empty(3, 16, device=d)
    attention.run(dec.q_nope, dec.q_pe, dec.ckv_cache, dec.kpe_cache, topk, scale, so, sl)
    ro, rl = oatt.attention_reference(dec.q_nope, dec.q_pe, dec.ckv_cache, dec.kpe_cache, topk, scale)
    assert compare.harness_close(so.cpu(), ro, 1e-2, 1e-2).ok and compare.harness_close(sl.cpu(), rl, 1e-3, 1e-3).ok


def test_pages_behind_four_gigabytes(cuda_device):
    c = Case([900, 400], 300, cuda_device, seed=13)
    ckv = torch.zeros(70000, 64, 512, dtype=torch.bfloat16, device=cuda_device)
    kpe = torch.zeros(70000, 64, 64, dtype=torch.bfloat16, device=cuda_device)
    index = torch.zeros(70000, 64, 1, 132, dtype=torch.uint8, device=cuda_device)
    pages = c.ckv.shape[0]
    to = 69999 - 500 * torch.arange(pages)
    ckv[to.to(cuda_device)], kpe[to.to(cuda_device)] = c.ckv.to(cuda_device), c.kpe.to(cuda_device)
    index[to.to(cuda_device)] = c.index.to(cuda_device)
    far = lambda t: torch.where(t >= 0, to[t.clamp(min=0).long()], -1).to(cuda_device)  # noqa: E731
    keep = torch.empty(2, 300, dtype=torch.int32, device=cuda_device)
    seq, acc = torch.empty(2, dtype=torch.int32, device=cuda_device), torch.empty(2, 320, device=cuda_device)
    evict.run(c.acc.to(cuda_device), c.seq.to(cuda_device), far(c.table), far(c.new_table), ckv, kpe, index, 4, 4, keep, seq, acc)
    back = to.to(cuda_device)
    c.check({"ckv": ckv[back].cpu(), "kpe": kpe[back].cpu(), "index": index[back].cpu(), "keep": keep.cpu(),
             "seq": seq.cpu(), "acc": acc.cpu()}, 4, 4)


def test_a_whole_step_in_one_graph(cuda_device):
    """Attention, accumulation and eviction captured together and replayed for new lengths."""
    d, scale = cuda_device, 1 / math.sqrt(192)
    g = torch.Generator().manual_seed(14)
    dec = workloads.make_decode_inputs([3000, 1200], seed=14, device=d, pool_pages=120)
    used = {int(x) for x in dec.indexer.block_table.flatten() if x >= 0}
    free = torch.tensor([x for x in range(120) if x not in used][:20], dtype=torch.int32)
    new_bt = free.reshape(2, 10).to(d)
    cu = torch.tensor([0, 2, 5], dtype=torch.int32, device=d)
    mask = torch.tensor(tree.masks_from_parents([-1, 0]) + tree.masks_from_parents([-1, 0, 0]), device=d)
    qn, qp = (torch.randn(5, 16, w, generator=g).to(torch.bfloat16).to(d) for w in (512, 64))
    prefix = torch.tensor([2900, 1100], dtype=torch.int32, device=d)
    seq = torch.empty_like(prefix)
    bt = dec.indexer.block_table
    acc, new_acc = torch.zeros(2, bt.shape[1] * 64, device=d), torch.zeros(2, 640, device=d)
    out, lse = torch.zeros(5, 16, 512, dtype=torch.bfloat16, device=d), torch.zeros(5, 16, device=d)
    keep, new_seq = torch.zeros(2, 600, dtype=torch.int32, device=d), torch.zeros_like(seq)

    def step():
        rows = (qn, qp, dec.ckv_cache, dec.kpe_cache, prefix, bt, cu, mask, scale)
        tree.run(*rows, out, lse)
        evict.accumulate(*rows, lse, acc, acc)
        torch.add(prefix, cu[1:] - cu[:-1], out=seq)
        evict.run(acc, seq, bt, new_bt, dec.ckv_cache, dec.kpe_cache, dec.indexer.k_index_cache_fp8, 4, 32, keep, new_seq, new_acc)

    side = torch.cuda.Stream(d)
    side.wait_stream(torch.cuda.current_stream(d))
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    for lengths in ([2900, 1100], [700, 400]):
        prefix.copy_(torch.tensor(lengths, dtype=torch.int32))
        acc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        a, got = acc.cpu(), (keep.cpu(), new_seq.cpu(), new_acc.cpu())
        kept = otree.evict_reference(a, seq.cpu(), 600, 4, 32)
        for b, k in enumerate(kept):
            assert int(got[1][b]) == len(k) and got[0][b, :len(k)].tolist() == k
            assert torch.equal(got[2][b, :len(k)], a[b, k])
        assert torch.allclose(a.sum(1), torch.tensor([32.0, 48.0]), rtol=1e-3)


def test_lengths_in_place(cuda_device):
    """new_seq_lens may be seq_lens: eager, and captured and replayed until
    every request is within the budget."""
    d = cuda_device
    for seq, budget in (([5001, 70, 30000, 1999, 0], 515), ([9000] * 40, 63), ([650, 700] * 200, 130)):
        c = Case(seq, budget, d, seed=51)
        rest = dict(acc=c.acc.to(d), block_table=c.table.to(d), new_block_table=c.new_table.to(d), num_sink=3, num_recent=11)
        for _ in range(5):
            caches = dict(ckv_cache=c.ckv.to(d), kpe_cache=c.kpe.to(d), k_index_cache_fp8=c.index.to(d))
            lens = c.seq.to(d)
            keep = torch.full((len(seq), budget), 7, dtype=torch.int32, device=d)
            acc = torch.full((len(seq), c.new_table.shape[1] * 64), 7.0, device=d)
            evict.run(**rest, **caches, seq_lens=lens, keep=keep, new_seq_lens=lens, new_acc=acc)
            torch.cuda.synchronize()
            c.check({"ckv": caches["ckv_cache"].cpu(), "kpe": caches["kpe_cache"].cpu(),
                     "index": caches["k_index_cache_fp8"].cpu(), "keep": keep.cpu(), "seq": lens.cpu(), "acc": acc.cpu()}, 3, 11)
    lens.copy_(c.seq)
    side = torch.cuda.Stream(d)
    side.wait_stream(torch.cuda.current_stream(d))
    with torch.cuda.stream(side):
        evict.run(**rest, **caches, seq_lens=lens, keep=keep, new_seq_lens=lens, new_acc=acc)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            evict.run(**rest, **caches, seq_lens=lens, keep=keep, new_seq_lens=lens, new_acc=acc)
    for grown in (1, 40, 500):  # as a decode loop lengthens them
        lens.add_(grown)
        lens.clamp_(max=c.table.shape[1] * 64)
        want = lens.cpu()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(lens.cpu(), want.clamp(max=budget))
        kept = otree.evict_reference(c.acc, want, budget, 3, 11)
        for b, k in enumerate(kept):
            assert keep[b, :len(k)].tolist() == k


def test_outputs_over_inputs_are_refused(cuda_device):
    d = cuda_device
    c = Case([900, 400], 300, d, seed=52)
    lens = torch.tensor([900, 400, 0], dtype=torch.int32, device=d)
    table = c.table.to(d)
    good = dict(acc=c.acc.to(d), seq_lens=lens[:2], block_table=table, new_block_table=c.new_table.to(d), ckv_cache=c.ckv.to(d),
                kpe_cache=c.kpe.to(d), k_index_cache_fp8=c.index.to(d), num_sink=1, num_recent=1,
                keep=torch.empty(2, 300, dtype=torch.int32, device=d), new_seq_lens=torch.empty(2, dtype=torch.int32, device=d),
                new_acc=torch.empty(2, 320, device=d))
    evict.run(**good)
    for change in (dict(new_seq_lens=lens[1:]), dict(new_seq_lens=table.view(-1)[:2]), dict(new_seq_lens=good["keep"].view(-1)[3:5]),
                   dict(keep=good["acc"].view(torch.int32).view(-1)[:600].view(2, 300)),
                   dict(keep=good["new_acc"].view(torch.int32).view(-1)[:600].view(2, 300))):
        with pytest.raises(ValueError, match="share memory"):
            evict.run(**{**good, **change})


def test_dense_and_sparse_agree_up_to_the_selection_size(cuda_device):
    """Where a draft sees at most 2048 tokens the indexer selects them all, and
    tree attention is the sparse attention's function."""
    d = cuda_device
    lens = [2048, 1500, 63, 1]
    dec = workloads.make_decode_inputs(lens, seed=53, device=d)
    ix = dec.indexer
    topk = torch.full((4, 2048), 7, dtype=torch.int32, device=d)
    indexer.run(ix.q_index_fp8, ix.k_index_cache_fp8, ix.weights, ix.seq_lens, ix.block_table, topk)
    so, sl = torch.empty(4, 16, 512, dtype=torch.bfloat16, device=d), torch.empty(4, 16, device=d)
    attention.run(dec.q_nope, dec.q_pe, dec.ckv_cache, dec.kpe_cache, topk, dec.sm_scale, so, sl)
    o, l = torch.empty_like(so), torch.empty_like(sl)
    rows = (dec.q_nope, dec.q_pe, dec.ckv_cache, dec.kpe_cache, torch.tensor(lens, dtype=torch.int32, device=d) - 1,
            ix.block_table, torch.arange(5, dtype=torch.int32, device=d), torch.ones(4, 1, dtype=torch.int64, device=d))
    tree.run(*rows, dec.sm_scale, o, l)
    host = [t.cpu() for t in rows]
    ro, rl, bo, bl = otree.tree_reference(*host, dec.sm_scale)
    assert ((o.cpu().double() - ro).abs() <= bo).all() and ((l.cpu().double() - rl).abs() <= bl).all()
    # The sparse attention's own tolerance (its harness's) on the same values.
    assert compare.harness_close(so.cpu(), ro.float(), 1e-2, 1e-2).ok and compare.harness_close(sl.cpu(), rl.float(), 1e-3, 1e-3).ok


def test_scalars_of_other_types(cuda_device):
    """A scale and counts that are numpy's or tensors, as the sparse attention takes them."""
    import numpy as np
    d = cuda_device
    dec = workloads.make_decode_inputs([900, 400], seed=54, device=d, pool_pages=64)
    bt = dec.indexer.block_table
    rows = (dec.q_nope, dec.q_pe, dec.ckv_cache, dec.kpe_cache, torch.tensor([899, 399], dtype=torch.int32, device=d), bt,
            torch.arange(3, dtype=torch.int32, device=d), torch.ones(2, 1, dtype=torch.int64, device=d))
    want = None
    for scale in (0.0625, np.float32(0.0625), np.float64(0.0625), torch.tensor(0.0625), torch.tensor([0.0625], device=d)):
        out, lse = torch.zeros(2, 16, 512, dtype=torch.bfloat16, device=d), torch.zeros(2, 16, device=d)
        acc = torch.zeros(2, bt.shape[1] * 64, device=d)
        tree.run(*rows, scale, out, lse)
        evict.accumulate(*rows, scale, lse, acc, acc)
        want = want or (out, lse, acc)
        assert all(torch.equal(a, b) for a, b in zip(want, (out, lse, acc)))
    c = Case([900, 400], 300, d, seed=55)
    c.check(c.run(np.int64(4), torch.tensor(16)), 4, 16)
    with pytest.raises(TypeError):
        c.run(4.0, 16)
