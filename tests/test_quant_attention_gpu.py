"""GPU parity of attention over the 8-bit latent cache (dsa_b200.quant.attend,
attend_sparse) with the 64-bit oracle, whose error bounds are the tolerances, at
the sizes and masks where it can go wrong."""

import math

import pytest
import torch

from dsa_b200 import DsaError, quant, tree
from oracle import quant as oq

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(192.0)


def cache_of(pages, seed, spread=0.3):
    """Latents as a norm leaves them, scales that differ from token to token."""
    g = torch.Generator().manual_seed(seed)
    cache = torch.zeros(pages, quant.PAGE_BYTES, dtype=torch.uint8)
    codes, kpe, scales = oq.pieces(cache)
    codes[:] = (torch.randn(codes.shape, generator=g) * 140).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    kpe[:] = torch.randn(kpe.shape, generator=g).bfloat16()
    scales[:] = torch.exp(torch.randn(scales.shape, generator=g) * spread) / 140
    return cache


def break_tokens(cache, slots):
    """NaN codes, infinite position parts and scales at these slots."""
    codes, kpe, scales = oq.pieces(cache)
    p, t = slots // 64, slots % 64
    codes[p, t] = 0x7F
    codes[p, t, ::2] = 0xFF
    kpe[p, t] = math.inf
    scales[p, t] = math.nan
    scales[p[::2], t[::2]] = math.inf
    scales[p[::3], t[::3]] = 0


@pytest.fixture(params=[0, 520], autouse=True, ids=["narrow", "wide"])
def _table_width(request, monkeypatch):
    """Every test with tables as wide as the lengths, where small calls run as clusters, and far wider, where all run as slices."""
    monkeypatch.setattr(Dense, "width", request.param)


class Dense:
    width = 0

    def __init__(self, lens, rows, heads, seed=0, spread=0.3, extra=2, tail=0, q_scale=1.0, hidden="broken"):
        g = torch.Generator().manual_seed(seed)
        need = [max(1, (n + 63) // 64) for n in lens]
        pool, width = sum(need) + extra, max(max(need) + 1, self.width)
        perm = torch.randperm(pool, generator=g)
        self.table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n].int()
            at += n
        self.cache = cache_of(pool, seed + 1, spread)
        behind = [self.table[b, n // 64] * 64 + torch.arange(n % 64, 64) for b, n in enumerate(lens) if n % 64]
        if hidden == "broken" and behind:
            break_tokens(self.cache, torch.cat(behind).long())
        total = (len(lens) if rows is None else sum(rows)) + tail
        self.q_nope = (torch.randn(total, heads, 512, generator=g) * q_scale).bfloat16()
        self.q_pe = torch.randn(total, heads, 64, generator=g).bfloat16()
        self.seq = torch.tensor(lens, dtype=torch.int32)
        self.cu = None if rows is None else torch.tensor([0, *rows]).cumsum(0).int()
        self.shape = (total, heads)

    def args(self, device="cuda"):
        return [None if t is None else t.to(device) for t in (self.q_nope, self.q_pe, self.cache, self.seq, self.table, self.cu)]

    def outs(self, device="cuda"):
        return torch.full((*self.shape, 512), 7.0, dtype=torch.bfloat16, device=device), torch.full(self.shape, 7.0, device=device)

    def reference(self, scale=SCALE):
        return oq.attend_reference(self.q_nope, self.q_pe, self.cache, self.seq, self.table, self.cu, scale)

    def check(self, out, lse, scale=SCALE):
        compare(out, lse, *self.reference(scale))


def compare(out, lse, ro, rl, bo, bl):
    out, lse = out.cpu().double(), lse.cpu().double()
    mine = ~torch.isnan(rl)
    assert torch.equal(lse[mine] == -math.inf, rl[mine] == -math.inf)
    fin = mine & (rl != -math.inf)
    assert ((lse - rl).abs() <= bl)[fin].all(), float((lse - rl).abs()[fin].max())
    bad = ~((out - ro).abs() <= bo)[mine]
    assert not bad.any(), (int(bad.sum()), float((out - ro).abs()[mine].max()))
    assert (out[~mine] == 7).all() and (lse[~mine] == 7).all()


def run(c, scale=SCALE):
    out, lse = c.outs()
    quant.attend(*c.args(), scale, out, lse)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("lens,rows,heads", [
    ([1], None, 16), ([1], None, 1), ([63], None, 16), ([64], None, 16), ([65], None, 16), ([127], None, 16), ([128], None, 16),
    ([129], None, 16), ([1000], None, 16), ([3000], None, 16), ([0, 5, 0, 700, 0], None, 16), ([513, 64, 1, 300], None, 8),
    ([400, 900], None, 3), ([257, 130], None, 24), ([640, 100], None, 32), ([300], None, 33), ([1100, 90], None, 128),
    ([100], [1], 16), ([100, 200], [2, 0], 16), ([700, 130, 64], [3, 1, 5], 16), ([260, 129], [4, 9], 8), ([50], [50], 16),
    ([200, 190, 1, 0], [65, 40, 1, 0], 5), ([128, 256], [2, 2], 128), ([383, 2], [7, 2], 17), ([3], [5], 16), ([0, 40], [2, 3], 16),
    ([20000], None, 16), ([20000], [3], 16),
])
def test_dense(cuda_device, lens, rows, heads):
    c = Dense(lens, rows, heads, seed=len(lens) + heads)
    c.check(*run(c))


@pytest.mark.parametrize("requests", [15, 16, 33, 34, 74, 75, 148, 149])
def test_clusters_of_all_sizes(cuda_device, requests):
    """Numbers of groups at which the clusters become smaller, and end; contexts of no token to nine tiles."""
    g = torch.Generator().manual_seed(requests)
    lens = torch.randint(0, 1100 if requests < 20 else 500, (requests,), generator=g).tolist()
    c = Dense([0, *lens[1:]], None, 16, seed=requests)
    c.check(*run(c))


@pytest.mark.parametrize("rows", [None, 1])
def test_many_short_requests(cuda_device, rows):
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 200, (700,), generator=g).tolist()
    c = Dense(lens, rows if rows is None else [i % 3 for i in range(700)], 16, seed=5)
    c.check(*run(c))


@pytest.mark.parametrize("heads", [16, 64])
def test_long_runs_of_one_request_beside_others(cuda_device, heads):
    """Slices of many tiles, segments that end inside them, records of many slices."""
    c = Dense([40000, 130, 1, 9000], [1, 2, 1, 3], heads, seed=7)
    c.check(*run(c))


@pytest.mark.parametrize("spread", [0.0, 3.0])
@pytest.mark.parametrize("q_scale", [1e-30, 0.0, 6.0])
def test_scales_and_queries_of_all_sizes(cuda_device, spread, q_scale):
    """Scales spread over e^10 and more, peaked and flat weights, queries of zeros."""
    c = Dense([2000, 300], [1, 2], 16, seed=9, spread=spread, q_scale=q_scale)
    c.check(*run(c))


def test_maximum_grows_along_the_context(cuda_device):
    """Logits that rise from tile to tile, scales that grow and shrink by powers of two, rows of zeros with any scale."""
    c = Dense([4000], None, 16, seed=11, q_scale=2.0)
    _, kpe, scales = oq.pieces(c.cache)
    codes, _, _ = oq.pieces(c.cache)
    for t in range(4000):
        p, i = int(c.table[0, t // 64]), t % 64
        scales[p, i] *= 2.0 ** ((t // 300) % 14 - 7)
        if t % 97 == 0:
            codes[p, i] = 0
            scales[p, i] = [0.0, 1.0, 2.0 ** -120][t % 3]
        kpe[p, i] = (kpe[p, i].float() + 0.002 * t * torch.sign(c.q_pe[0, t % 16].float())).bfloat16()
    c.check(*run(c))


def test_one_heavy_token_beside_many_light_ones(cuda_device):
    """A first token with a weight 2^19 times the others', which hold a good part of it together: they still count."""
    n = 30000
    c = Dense([n], None, 16, seed=13, q_scale=0.02)
    codes, kpe, scales = oq.pieces(c.cache)
    kpe[:] = 0
    kpe[int(c.table[0, 0]), 0] = torch.sign(c.q_pe[0, 0].float()).bfloat16() * 2.0
    c.q_pe[:] = c.q_pe[:, :1]
    scale = 19 / oq.LOG2E / float((c.q_pe[0, 0].float().abs() * 2).sum())
    c.check(*run(c, scale), scale)


def test_rows_of_a_chain_are_those_of_single_tokens(cuda_device):
    c = Dense([900, 333], [4, 3], 16, seed=15)
    out, lse = run(c)
    single = Dense([900, 333], [4, 3], 16, seed=15)
    single.seq = torch.tensor([897, 898, 899, 900, 331, 332, 333], dtype=torch.int32)
    single.table = c.table[[0, 0, 0, 0, 1, 1, 1]]
    single.cu = None
    o2, l2 = run(single)
    assert torch.allclose(lse, l2, atol=1e-4, rtol=0) and torch.allclose(out.float(), o2.float(), atol=2e-2, rtol=2e-2)


def test_short_contexts_agree_with_bf16(cuda_device):
    """The same function as tree attention over the cache read back."""
    c = Dense([500, 64, 1], None, 16, seed=17, hidden="")
    out, lse = run(c)
    pool = c.cache.shape[0]
    ckv = torch.zeros(pool, 64, 512, dtype=torch.bfloat16, device="cuda")
    kpe = torch.zeros(pool, 64, 64, dtype=torch.bfloat16, device="cuda")
    everything = torch.arange(pool, dtype=torch.int32, device="cuda")[None]
    quant.read(c.cache.cuda(), everything, torch.zeros(1, dtype=torch.int32, device="cuda"),
               torch.tensor([0, 64 * pool], dtype=torch.int32, device="cuda"), ckv.view(-1, 512), kpe.view(-1, 64))
    o2, l2 = c.outs()
    tree.run(c.q_nope.cuda(), c.q_pe.cuda(), ckv, kpe, c.seq.cuda() - 1, c.table.cuda(), torch.arange(4, device="cuda"),
             torch.ones(3, 1, dtype=torch.int64, device="cuda"), SCALE, o2, l2)
    assert torch.allclose(lse, l2, atol=3e-2, rtol=0) and torch.allclose(out.float(), o2.float(), atol=3e-2, rtol=3e-2)


def test_nan_where_it_is_seen(cuda_device):
    """A visible broken token makes the rows that see it NaN, the others not."""
    c = Dense([300, 300], [3, 1], 16, seed=19)
    broken = c.table[0, 298 // 64] * 64 + 298 % 64  # seen by the first request's last two rows
    codes, _, _ = oq.pieces(c.cache)
    codes[int(broken) // 64, int(broken) % 64, 5] = 0x7F
    out, lse = run(c)
    assert torch.isnan(out[1:3]).all() and torch.isnan(lse[1:3]).all()
    ro, rl, bo, bl = c.reference()
    keep = torch.tensor([0, 3])
    compare(out[keep.cuda()], lse[keep.cuda()], ro[keep], rl[keep], bo[keep], bl[keep])
    c = Dense([300], None, 16, seed=20)
    c.q_nope[0, 3, 7] = math.nan
    c.q_nope[0, 4, 8] = math.inf
    out, lse = run(c)
    assert torch.isnan(out[0, 3:5]).all() and not torch.isnan(out[0, :3]).any() and not torch.isnan(out[0, 5:]).any()


def test_rows_outside_are_left(cuda_device):
    c = Dense([300, 90], [2, 1], 16, seed=21, tail=3)
    c.check(*run(c))


def test_reports_and_masks_what_does_not_fit(cuda_device):
    c = Dense([300, 90], None, 16, seed=23)
    c.table[0, 2] = 1 << 20
    out, lse = c.outs()
    with pytest.raises(DsaError, match="pool"):
        quant.attend(*c.args(), SCALE, out, lse)
    see = torch.ones(300, dtype=torch.bool)
    see[128:192] = False
    pos = torch.arange(300)
    slot = c.table[0].long().clamp(max=c.cache.shape[0] - 1)[pos // 64] * 64 + pos % 64
    ro, rl, bo, bl = oq._softmax(c.q_nope[0], c.q_pe[0], *oq.rows(c.cache, slot), oq.scales_of(c.cache, slot), see, SCALE)
    compare(out[0].cpu(), lse[0].cpu(), ro, rl, bo, bl)
    c = Dense([300, 90], None, 16, seed=24)
    c.seq[1] = 10 ** 6
    with pytest.raises(DsaError, match="seq_len"):
        quant.attend(*c.args(), SCALE, *c.outs())
    c = Dense([300, 90], [2, 1], 16, seed=25)
    c.cu = torch.tensor([0, 3, 2], dtype=torch.int32)
    out, lse = c.outs()
    with pytest.raises(DsaError, match="seq_len"):
        quant.attend(*c.args(), SCALE, out, lse)


def test_output_in_place_of_queries(cuda_device):
    c = Dense([3000, 64, 700], [2, 1, 3], 16, seed=27)
    out, lse = run(c)
    args = c.args()
    l2 = torch.zeros_like(lse)
    quant.attend(*args, SCALE, args[0], l2)
    assert torch.equal(args[0], out) and torch.equal(l2, lse)


def sparse_case(T, heads, topk, pages, seed, holes=0.0, empty=()):
    g = torch.Generator().manual_seed(seed)
    picked = torch.randint(0, pages * 64, (T, topk), generator=g).int()
    picked[torch.rand(T, topk, generator=g) < holes] = -1
    for i in empty:
        picked[i] = -1
    cache = cache_of(pages, seed)
    unused = torch.ones(pages * 64, dtype=torch.bool)
    unused[picked[picked >= 0].long()] = False
    if unused.any():
        break_tokens(cache, torch.nonzero(unused)[:, 0])
    return (torch.randn(T, heads, 512, generator=g).bfloat16(), torch.randn(T, heads, 64, generator=g).bfloat16(), cache, picked)


@pytest.mark.parametrize("T,heads,topk,pages,holes,empty", [
    (1, 16, 2048, 40, 0.0, ()), (3, 16, 2048, 70, 0.3, (1,)), (2, 16, 1, 1, 0.0, ()), (2, 16, 127, 3, 0.1, ()), (2, 16, 128, 3, 0.0, ()),
    (4, 1, 129, 9, 0.5, (0, 3)), (5, 33, 300, 20, 0.2, ()), (2, 128, 2048, 50, 0.9, ()), (160, 16, 2048, 500, 0.1, (7, 150)),
    (700, 8, 64, 30, 0.95, ()), (1, 16, 65536, 900, 0.0, ()),
    # rows of more than 16 heads that make many tiles
    (75, 17, 1111, 60, 0.1, (0, 40)), (40, 33, 2048, 300, 0.0, ()), (20, 128, 1025, 90, 0.7, (19,)), (161, 128, 64, 30, 0.2, ()),
    (2, 24, 65536, 900, 0.1, ()),
])
def test_sparse(cuda_device, T, heads, topk, pages, holes, empty):
    case = sparse_case(T, heads, topk, pages, T + topk, holes, empty)
    out, lse = torch.full((T, heads, 512), 7.0).bfloat16().cuda(), torch.full((T, heads), 7.0).cuda()
    quant.attend_sparse(*[t.cuda() for t in case], SCALE, out, lse)
    compare(out, lse, *oq.sparse_reference(*case, SCALE))


@pytest.mark.parametrize("T,heads,topk,empty", [(1, 16, 1, ()), (3, 16, 300, (1,)), (14, 20, 129, (0, 13)), (30, 128, 256, ())])
def test_sparse_with_empty_room(cuda_device, T, heads, topk, empty):
    """Selections of few slots in rows of many give what rows without the room give, but for the order of their sums."""
    case = sparse_case(T, heads, topk, 20, T + topk, 0.2, empty)
    for room in (0, 4200):
        wide = (*case[:3], torch.cat([case[3], torch.full((T, room), -1, dtype=torch.int32)], 1))
        out, lse = torch.full((T, heads, 512), 7.0).bfloat16().cuda(), torch.full((T, heads), 7.0).cuda()
        quant.attend_sparse(*[t.cuda() for t in wide], SCALE, out, lse)
        compare(out, lse, *oq.sparse_reference(*case, SCALE))


def test_sparse_reports_bad_indices(cuda_device):
    case = list(sparse_case(2, 16, 256, 4, 3))
    want = [t.clone() for t in case]
    want[3][1, 77] = want[3][1, 200] = -1
    case[3][1, 77], case[3][1, 200] = 256, -5
    out, lse = torch.zeros(2, 16, 512).bfloat16().cuda(), torch.zeros(2, 16).cuda()
    with pytest.raises(DsaError, match="index"):
        quant.attend_sparse(*[t.cuda() for t in case], SCALE, out, lse)
    compare(out, lse, *oq.sparse_reference(*want, SCALE))


def test_all_tokens_selected_is_dense(cuda_device):
    c = Dense([700], None, 16, seed=29)
    out, lse = run(c)
    pos = torch.arange(700)
    picked = (c.table[0].long()[pos // 64] * 64 + pos % 64).int()[torch.randperm(700)][None]
    o2, l2 = c.outs()
    quant.attend_sparse(c.q_nope.cuda(), c.q_pe.cuda(), c.cache.cuda(), picked.cuda(), SCALE, o2, l2)
    c.check(o2, l2)
    assert torch.allclose(lse, l2, atol=1e-4, rtol=0)


def test_refusals(cuda_device):
    c = Dense([300, 90], [2, 1], 16, seed=31)
    good = [*c.args(), SCALE, *c.outs()]
    quant.attend(*good)
    for k, bad in ((0, good[0].float()), (0, good[0][:, :, :500]), (1, good[1][:2]), (2, good[2][:, 1:]), (2, good[2].cpu()), (3, good[3][:1]),
                   (3, good[3].float()), (4, good[4][0]), (5, good[5][:2]), (5, None), (7, good[7].float()), (7, good[7][:2]),
                   (8, good[8].double()), (0, good[0].repeat(1, 9, 1)), (8, good[8].T)):
        args = list(good)
        args[k] = bad
        with pytest.raises(ValueError, match="dsa_quant.attend"):
            quant.attend(*args)
    with pytest.raises(ValueError, match="share memory"):
        quant.attend(*good[:7], good[2].flatten()[:3 * 16 * 1024].view(torch.bfloat16).reshape(3, 16, 512), good[8])
    case = [t.cuda() for t in sparse_case(2, 16, 256, 4, 3)]
    outs = torch.zeros(2, 16, 512).bfloat16().cuda(), torch.zeros(2, 16).cuda()
    for k, bad in ((3, case[3][:1]), (3, case[3].float()), (3, case[3].cpu()), (2, case[2][:, :9])):
        args = list(case)
        args[k] = bad
        with pytest.raises(ValueError, match="dsa_quant.attend_sparse"):
            quant.attend_sparse(*args, SCALE, *outs)


def test_strided_queries_and_other_index_types(cuda_device):
    c = Dense([300, 1000], [2, 1], 16, seed=33)
    out, lse = run(c)
    wide = torch.zeros(3, 16, 600, dtype=torch.bfloat16, device="cuda")
    wide[:, :, 3:515], wide[:, :, 515:579] = c.q_nope.cuda(), c.q_pe.cuda()
    o2, l2 = c.outs()
    args = c.args()
    quant.attend(wide[:, :, 3:515], wide[:, :, 515:579], args[2].view(-1, 64, 644), args[3].long(),
                 torch.cat([args[4], args[4]], 1)[:, :args[4].shape[1]], args[5].long(), torch.tensor(SCALE), o2, l2)
    assert torch.equal(out, o2) and torch.allclose(lse, l2, atol=1e-6, rtol=0)


def test_streams_graphs_and_repetition(cuda_device):
    """Calls on two streams at once, a captured and replayed one with new lengths, all bit for bit what a single call gives."""
    a, b = Dense([3000, 64, 700], [2, 1, 3], 16, seed=35), Dense([9000], None, 64, seed=36)
    want = [run(c) for c in (a, b)]
    args, outs = [c.args() for c in (a, b)], [c.outs() for c in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, x, o in zip(streams, args, outs):
            with torch.cuda.stream(s):
                quant.attend(*x, SCALE, *o)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(streams[0]), torch.cuda.graph(graph, stream=streams[0]):
        quant.attend(*args[0], SCALE, *outs[0])
    for lens in ([3000, 64, 700], [1500, 3, 699], [2, 1, 4]):
        a.seq = torch.tensor(lens, dtype=torch.int32)
        args[0][3].copy_(a.seq)
        a2 = Dense([3000, 64, 700], [2, 1, 3], 16, seed=35, hidden="")
        a2.seq = a.seq
        args[0][2].copy_(a2.cache)
        graph.replay()
        torch.cuda.synchronize()
        a2.check(*outs[0])
