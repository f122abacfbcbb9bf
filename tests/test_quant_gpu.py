"""GPU parity of the 8-bit latent cache (dsa_b200.quant.write, read) with the
64-bit oracle: codes exactly, the rest within the roundings that the formulas
take."""

import math

import pytest
import torch

from dsa_b200 import DsaError, quant
from oracle import quant as oq
from test_quant import angles, kv_rows

pytestmark = pytest.mark.gpu

# fp32: a sum of 512 squares (each step 2^-24, twice: the product's and the sum's), the mean, root, quotient and two products
SCALE_RTOL = (512 + 8) * 2.0 ** -24


def written(device, n, pages, seed, norm=True, rope=True, interleaved=False, strided=False, slots=None):
    g = torch.Generator().manual_seed(seed + 50)
    kv = kv_rows(n, seed)
    w = (1 + 0.3 * torch.randn(512, generator=g)).bfloat16() if norm else None
    table = angles(300, seed) if rope else None
    pos = torch.randint(0, 300, (n,), generator=g) if rope else None
    if slots is None:
        slots = torch.randperm(pages * 64, generator=g)[:n]
        slots[::7] = -1
    cache = torch.full((pages, quant.PAGE_BYTES), 0x5A, dtype=torch.uint8, device=device)
    on = kv.to(device)
    if strided:
        wide = torch.zeros(n, 1536 + 576, dtype=torch.bfloat16, device=device)
        wide[:, 1528:2104] = on
        on = wide[:, 1528:2104]
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    args = (on, slots.to(device), cache, to(w), 1e-6, to(pos), to(table), interleaved)
    return args, oq.write_rows(kv, w, 1e-6, pos, table, interleaved), slots


def check(cache, want, slots, least=0.0):
    code, scale, e = want
    cache = cache.cpu()
    codes, kpe, scales = oq.pieces(cache)
    real = slots >= 0
    p, t = slots[real] // 64, slots[real] % 64
    assert torch.equal(codes[p, t], code[real])
    assert ((scales[p, t].double() - scale[real]).abs() <= SCALE_RTOL * scale[real]).all()
    # A product and an FMA in fp32, 2^-24 of |b sin| and of the result, |b| at most sqrt 2 of the row's largest rotated
    # value (a rotation keeps a pair's length); then half a step of bf16.
    off = (kpe[p, t].double() - e[real]).abs()
    assert (off <= 2.0 ** -8 * e[real].abs() + 2.0 ** -22 * e[real].abs().amax(1, keepdim=True) + least).all()
    untouched = torch.ones(codes.shape[:2], dtype=torch.bool)
    untouched[p, t] = False
    assert (codes[untouched] == 0x5A).all() and (kpe.view(torch.uint8)[untouched] == 0x5A).all()
    assert (scales.view(torch.uint8).reshape(*scales.shape, 4)[untouched] == 0x5A).all()


@pytest.mark.parametrize("n,pages", [(1, 1), (3, 2), (33, 1), (64, 5), (1001, 17), (5003, 80)])
@pytest.mark.parametrize("norm,rope,interleaved,strided", [(True, True, False, True), (True, True, True, False),
                                                           (False, False, False, False), (False, True, True, True),
                                                           (True, False, False, True)])
def test_write(cuda_device, n, pages, norm, rope, interleaved, strided):
    args, want, slots = written(cuda_device, n, pages, n + pages, norm, rope, interleaved, strided)
    quant.write(*args)
    check(args[2], want, slots)


def test_write_ties_zeros_and_what_is_not_finite(cuda_device):
    """Quotients that are borders of e4m3 exactly, rows of zeros, tiny rows, infinities and NaN."""
    kv = torch.zeros(8, 576)
    # 448 t / M with M = 448 * 2^k: t itself; 17, 19, ... are halfway between codes from 16 to 32
    kv[0, :32], kv[0, 100] = torch.arange(1, 64, 2).float(), 448.0
    kv[1, :512], kv[1, 1] = torch.arange(512).float() * 2.0 ** -10, 448 * 2.0 ** -6
    kv[3, 5], kv[4, 6], kv[5, 7] = math.inf, -math.inf, math.nan
    kv[6, :512] = 2.0 ** -125  # the scale would be below 2^-126
    kv[7, :512], kv[7, 3] = 1.5e38, -3e38
    kv = kv.bfloat16()
    cache = torch.zeros(1, quant.PAGE_BYTES, dtype=torch.uint8, device=cuda_device)
    quant.write(kv.to(cuda_device), torch.arange(8, device=cuda_device), cache)
    codes, _, scales = oq.pieces(cache.cpu())
    want, scale, _ = oq.write_rows(kv)
    assert torch.equal(codes[0, :8], want)
    assert ((scales[0, :8].double() - scale).abs() <= 2.0 ** -23 * scale).all()


@pytest.mark.parametrize("norm", [False, True])
def test_write_keeps_the_sign_of_zeros(cuda_device, norm):
    kv = kv_rows(40, 3)
    kv[:, ::3], kv[:, 1::5] = -0.0, 0.0
    w = torch.randn(512, generator=torch.Generator().manual_seed(4)).bfloat16() if norm else None
    cache = torch.zeros(1, quant.PAGE_BYTES, dtype=torch.uint8, device=cuda_device)
    quant.write(kv.to(cuda_device), torch.arange(40, device=cuda_device), cache, None if w is None else w.to(cuda_device))
    assert torch.equal(oq.pieces(cache.cpu())[0][0, :40], oq.write_rows(kv, w)[0])
@pytest.mark.parametrize("eps", [1e-6, 0.0, 1e-30, 1e30])
@pytest.mark.parametrize("spread", [0.0, 6.0])
def test_write_of_rows_of_all_sizes_with_a_norm(cuda_device, eps, spread):
    """Latents and weights whose squares and products leave fp32's range on either side, where the scale is an ordinary number;
    rows whose scale is beyond it."""
    g = torch.Generator().manual_seed(int(spread) + 1)
    sizes = [2.0 ** e for e in (-132, -126, -110, -75, -63, -50, -20, 0, 20, 40, 59, 60, 63, 64, 80, 100, 120, 124)]
    kv = torch.randn(len(sizes) + 5, 576, generator=g) * torch.exp(spread * torch.randn(len(sizes) + 5, 576, generator=g).clamp(-3, 3) / 3)
    kv[:len(sizes)] *= torch.tensor(sizes)[:, None]
    kv = kv.clamp(-3e38, 3e38)
    kv[len(sizes)] = 0
    kv[len(sizes) + 1, :512] = 0
    kv[len(sizes) + 1, 7] = 3e38  # one value alone
    kv[len(sizes) + 2, :512] = 1e-38
    kv[len(sizes) + 3, 9], kv[len(sizes) + 4, 9] = math.inf, math.nan
    kv = kv.bfloat16()
    for size in (1.0, 1e-36, 1e-20, 1e20, 1e36):
        w = ((1 + 0.3 * torch.randn(512, generator=g)) * size).bfloat16()
        cache = torch.zeros(1, quant.PAGE_BYTES, dtype=torch.uint8, device=cuda_device)
        quant.write(kv.to(cuda_device), torch.arange(len(kv), device=cuda_device), cache, w.to(cuda_device), eps)
        codes, _, scales = oq.pieces(cache.cpu())
        want, scale, _ = oq.write_rows(kv, w, float(torch.tensor(eps, dtype=torch.float32)))
        n = len(kv)
        # where the scale is within its own error of the border, either is right
        border = ((scale / 2.0 ** -126 - 1).abs() < 2 * SCALE_RTOL) & (codes[0, :n] == 0).all(1)
        assert torch.equal(codes[0, :n][~border], want[~border])
        assert ((scales[0, :n].double() - scale).abs() <= SCALE_RTOL * scale)[~border].all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_write_of_rows_out_of_range_among_others(cuda_device, interleaved):
    """Many rows a warp, some of them beyond fp32's squares or below its products, zeros, padding, slots and positions outside."""
    args, _, slots = written(cuda_device, 20001, 320, 11, True, True, interleaved, True)
    kv, pos = args[0].cpu(), args[5].cpu()
    kv[::97] *= 1e25
    kv[5::101] *= 1e-37
    kv[7::89, :512] = 0
    pos[11::1000], slots[13::1000] = 300, 320 * 64
    args[0].copy_(kv)
    args[5].copy_(pos)
    args[1].copy_(slots)
    with pytest.raises(DsaError, match="outside"):
        quant.write(*args)
    kept = torch.where((pos < 300) & (slots < 320 * 64), slots, -1)
    want = oq.write_rows(kv, args[3].cpu(), float(torch.tensor(1e-6)), pos.clamp(max=299), args[6].cpu(), interleaved)
    # The position parts of the smallest rows are subnormal numbers of bf16: steps of 2^-133, whatever the value; and fp32's of 2^-149.
    check(args[2], want, kept, 2.0 ** -134 + 2.0 ** -148)


def test_write_reports_what_does_not_fit(cuda_device):
    args, want, slots = written(cuda_device, 20, 2, 3)
    for k, bad in ((1, 128), (5, -1), (5, 300)):
        changed = [a.clone() if torch.is_tensor(a) else a for a in args]
        changed[k][4] = bad
        kept = slots.clone()
        kept[4] = -1
        with pytest.raises(DsaError, match="outside"):
            quant.write(*changed)
        check(changed[2], want, kept)


def test_write_refuses(cuda_device):
    args, _, _ = written(cuda_device, 20, 2, 3)
    for k, bad in ((0, args[0].float()), (0, args[0][:, :575]), (0, args[0].T), (1, args[1][:5]), (1, args[1].float()),
                   (2, args[2][:, :100]), (2, args[2].float()), (3, args[3].float()), (3, args[3][:500]), (5, None), (6, None),
                   (6, args[6].double()), (6, args[6][:, :32]), (1, args[1].cpu()), (6, args[6].cpu())):
        changed = list(args)
        changed[k] = bad
        with pytest.raises(ValueError, match="dsa_quant.write"):
            quant.write(*changed)
    inside = args[2].flatten()[:20 * 1152].view(torch.bfloat16).reshape(20, 576)
    with pytest.raises(ValueError, match="share memory"):
        quant.write(inside, *args[1:])


def test_write_in_a_graph_and_on_another_stream(cuda_device):
    args, want, slots = written(cuda_device, 300, 6, 9, True, True, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        quant.write(*args)
    torch.cuda.synchronize()
    check(args[2], want, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        quant.write(*args)
    args[2].fill_(0x5A)
    graph.replay()
    torch.cuda.synchronize()
    check(args[2], want, slots)


def filled(device, pages, seed):
    """A cache of random rows, some NaN among them."""
    g = torch.Generator().manual_seed(seed)
    cache = torch.zeros(pages, quant.PAGE_BYTES, dtype=torch.uint8)
    codes, kpe, scales = oq.pieces(cache)
    codes[:] = torch.randint(0, 256, codes.shape, generator=g).to(torch.uint8)
    kpe[:] = torch.randn(kpe.shape, generator=g).bfloat16()
    scales[:] = torch.exp(torch.randn(scales.shape, generator=g) - 4)
    return cache


@pytest.mark.parametrize("lens,starts", [([1], [0]), ([5], [63]), ([0, 130, 0, 0, 7, 64], [0, 17, 5, 0, 127, 64]), ([1000, 1, 333], [0, 500, 64]),
                                         ([2] * 70, list(range(70))), ([0] * 40 + [9] + [0] * 40, [3] * 81)])
@pytest.mark.parametrize("together", [False, True])
def test_read(cuda_device, lens, starts, together):
    g = torch.Generator().manual_seed(len(lens))
    need = [max(1, (s + n + 63) // 64) for s, n in zip(starts, lens)]
    pool, width = sum(need) + 2, max(need)
    perm, table, at = torch.randperm(pool, generator=g), torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n].int()
        at += n
    cache = filled(cuda_device, pool, 4)
    front, total = 2, sum(lens) + 5  # rows before the first and behind the last request
    cu = torch.tensor([front] + [front + sum(lens[:i + 1]) for i in range(len(lens))])
    if together:
        both = torch.full((total, 584), 7.0, dtype=torch.bfloat16, device=cuda_device)
        ckv, kpe = both[:, :512], both[:, 512:576]
    else:
        ckv = torch.full((total, 512), 7.0, dtype=torch.bfloat16, device=cuda_device)
        kpe = torch.full((total, 64), 7.0, dtype=torch.bfloat16, device=cuda_device)
    on = [t.to(cuda_device) for t in (cache, table, torch.tensor(starts), cu)]
    quant.read(*on, ckv, kpe)
    if total > 7:
        slot = torch.cat([table[b].long()[(s + torch.arange(n)) // 64] * 64 + (s + torch.arange(n)) % 64
                          for b, (s, n) in enumerate(zip(starts, lens)) if n])
        c, e = oq.rows(cache, slot)
        got = ckv.cpu()[front:-3].double()
        assert torch.equal(torch.isnan(got), torch.isnan(c))
        c, got = c.nan_to_num(), got.nan_to_num()
        assert ((got - c).abs() <= (2.0 ** -8 + 2.0 ** -23) * c.abs()).all()  # fp32, then half a step of bf16
        assert torch.equal(kpe.cpu()[front:-3].double(), e)
    for t in (ckv, kpe):
        assert (t[:front] == 7).all() and (t[-3:] == 7).all()
    if together:
        assert (both[:, 576:] == 7).all()


def test_read_reports_what_does_not_exist(cuda_device):
    cache = filled(cuda_device, 3, 5).to(cuda_device)
    table = torch.tensor([[0, 3], [-1, 2]], device=cuda_device)
    ckv, kpe = (torch.full((8, n), 7.0, dtype=torch.bfloat16, device=cuda_device) for n in (512, 64))
    starts, cu = torch.tensor([62, 126], device=cuda_device), torch.tensor([0, 4, 8], device=cuda_device)
    with pytest.raises(DsaError, match="pool"):
        quant.read(cache, table, starts, cu, ckv, kpe)
    assert (ckv[2:4] == 0).all() and (kpe[2:4] == 0).all() and (ckv[6:] == 0).all()  # page 3; behind the table
    assert (kpe[:2] != 0).any() and (kpe[4:6] != 0).any()
    with pytest.raises(DsaError, match="seq_len"):
        quant.read(cache, torch.tensor([[0, 1], [1, 2]], device=cuda_device), torch.tensor([-1, 0], device=cuda_device), cu, ckv, kpe)


def test_read_refuses(cuda_device):
    cache = filled(cuda_device, 3, 5).to(cuda_device)
    ckv, kpe = (torch.zeros(8, n, dtype=torch.bfloat16, device=cuda_device) for n in (512, 64))
    args = [cache, torch.tensor([[0, 1]], device=cuda_device), torch.tensor([0], device=cuda_device),
            torch.tensor([0, 8], device=cuda_device), ckv, kpe]
    quant.read(*args)
    for k, bad in ((0, cache[:, :-4]), (1, args[1][0]), (1, args[1].float()), (2, args[3]), (3, args[2]), (4, ckv.float()), (4, ckv[:, :500]),
                   (5, kpe[:7]), (5, kpe.cpu()), (4, ckv.T), (2, args[2].float())):
        changed = list(args)
        changed[k] = bad
        with pytest.raises(ValueError, match="dsa_quant.read"):
            quant.read(*changed)
    inside = cache.flatten()[:8 * 1024].view(torch.bfloat16).reshape(8, 512)
    with pytest.raises(ValueError, match="share memory"):
        quant.read(*args[:4], inside, kpe)


def test_written_rows_come_back(cuda_device):
    """write, then read: half a step of the codes and of bf16 away from the normalised rows."""
    n = 500
    kv = kv_rows(n, 8, spread=2)
    w = (1 + 0.2 * torch.randn(512, generator=torch.Generator().manual_seed(1))).bfloat16()
    table = torch.randperm(9, generator=torch.Generator().manual_seed(2))[None].int()
    slots = table[0].long()[torch.arange(n) // 64] * 64 + torch.arange(n) % 64
    cache = torch.zeros(9, quant.PAGE_BYTES, dtype=torch.uint8, device=cuda_device)
    quant.write(kv.to(cuda_device), slots.to(cuda_device), cache, w.to(cuda_device))
    out = torch.zeros(n, 576, dtype=torch.bfloat16, device=cuda_device)
    quant.read(cache, table.to(cuda_device), torch.tensor([0], device=cuda_device), torch.tensor([0, n], device=cuda_device),
               out[:, :512], out[:, 512:])
    c = kv[:, :512].double()
    y = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-6) * w.double()
    top = y.abs().amax(1, keepdim=True)
    off = (out[:, :512].cpu().double() - y).abs()
    # code: half a step, 2^-4 of the value or 2^-10 of the scale; then bf16's, and the scale's own error
    assert (off <= (2.0 ** -4 + 2.0 ** -8 * 1.07 + SCALE_RTOL) * y.abs() + 2.0 ** -10 * top / 448).all()
    assert torch.equal(out[:, 512:].cpu(), kv[:, 512:])
