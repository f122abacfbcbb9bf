"""How exactly the attention over the 8-bit latent cache takes its weights: in four
8-bit parts, which outputs in bf16 hide unless tokens cancel."""

import math

import pytest
import torch

from dsa_b200 import quant
from oracle import quant as oq

SCALE = 1.0 / math.sqrt(192.0)
N = 256
# Each part is half a step off what the one before leaves, which may pass a power of two by an eighth with the weight's lower bits:
# the four leave 2^-14 of a weight.  The lower half's rounding is 2^-18, the product's and the exponential's 2^-22 and less.
WEIGHT = 2.0 ** -14 + 2.0 ** -17


def in_parts(w, without=None):
    """float64 sums of a weight's parts (`without` one of them), as the kernel takes them."""
    bits = lambda x, t: x.half().view(torch.int16).to(torch.int32) if t is torch.float16 else x.view(torch.int32)  # noqa: E731
    e5m2 = lambda x: ((bits(x, torch.float16) + 0x80) & ~0xFF).to(torch.int16).view(torch.float16).float()  # noqa: E731
    half = lambda x: x.half().float()  # noqa: E731
    upper = (bits(w, torch.float32) & ~0x1FFF).view(torch.float32)
    h, low = half(upper), half(w - upper)
    parts = [e5m2(h)]
    parts.append(e5m2(h - parts[0]))
    rest = half(half(h - parts[0] - parts[1] + low) * 128)
    parts.append(e5m2(rest))
    parts.append(e5m2(rest - parts[2]))
    units = [1.0, 1.0, 1 / 128, 1 / 128]
    return sum(p.double() * u for k, (p, u) in enumerate(zip(parts, units)) if k != without)


def test_four_parts_hold_a_weight():
    """2^-14 of a weight or half a step of the last part, 2^-24; the lower half's rounding, 2^-18 of the weight, or 2^-25 as the
    upper half's."""
    w = torch.exp2(torch.rand(1 << 20, generator=torch.Generator().manual_seed(0)) * 44 - 29)
    off = (in_parts(w) - w.double()).abs()
    assert (off <= (w * 2.0 ** -14).clamp(min=2.0 ** -24) + 2.0 ** -18 * w + 2.0 ** -24).all()


def pairs(logits, seed=0):
    """A cache of 128 pairs of tokens with opposite codes in four dims of their own and scales that differ by up to 2^-10: what
    is left of a pair in the output shows its weights' errors a thousand times as large.  (cache, scales, base-2 logits)"""
    g = torch.Generator().manual_seed(seed)
    cache = torch.zeros(N // 64, quant.PAGE_BYTES, dtype=torch.uint8)
    codes, kpe, scales = oq.pieces(cache)
    at = torch.arange(N)
    for j in range(4):
        codes[at // 64, at % 64, 4 * (at // 2) + j] = torch.where(at % 2 == 0, 0x7E, 0xFE).to(torch.uint8)  # 448, -448
    s = torch.exp(torch.rand(N // 2, generator=g) * 2 - 1)
    both = torch.stack([s, s * (1 - 2.0 ** -10 * torch.rand(N // 2, generator=g))], 1).flatten()
    scales[:] = both.view(N // 64, 64)
    x = -torch.randint(0, 60 if logits else 1, (N // 2,), generator=g).repeat_interleave(2).bfloat16()
    kpe[:, :, 0] = x.view(N // 64, 64)
    return cache, both, x.double() * SCALE * oq.LOG2E


def wanted(scales, x, others=()):
    """(outputs, bounds) [512] of any row with these logits, and with `others` that have no part in the outputs."""
    lse = torch.logsumexp(torch.cat([x, *others]) / oq.LOG2E, 0) * oq.LOG2E
    w = torch.exp2(x - lse) * scales.double() * 448
    out = (w[0::2] - w[1::2]).repeat_interleave(4)
    return out, WEIGHT * (w[0::2] + w[1::2]).repeat_interleave(4) + (2.0 ** -8 + 2.0 ** -16) * out.abs()


@pytest.mark.parametrize("logits", [False, True])
def test_the_bound_shows_each_part(logits):
    """(The first part is the same for both tokens of a pair; without it every output of ordinary rows is wrong.)"""
    _, scales, x = pairs(logits)
    out, bound = wanted(scales, x)
    w = torch.exp2(x - x.max()).float() * scales * 32 / scales.max()
    lse = torch.logsumexp(x / oq.LOG2E, 0) * oq.LOG2E
    unit = 448 * float(scales.max()) / 32 * 2.0 ** float(x.max() - lse)
    for without in (None, 1, 2, 3):
        got = in_parts(w, without) * unit
        fine = ((got[0::2] - got[1::2]).repeat_interleave(4) - out).abs() <= bound
        assert fine.all() if without is None else (~fine).float().mean() > 0.05


@pytest.mark.gpu
@pytest.mark.parametrize("logits", [False, True])
@pytest.mark.parametrize("rows,heads,pages", [(1, 16, 4), (1, 16, 900), (1, 128, 4), (2, 128, 900), (3, 24, 900)])
def test_pairs_that_cancel(cuda_device, logits, rows, heads, pages):
    """Dense, as clusters (tables as wide as the context) and slices, groups of 16 rows and of 32."""
    cache, scales, x = pairs(logits)
    table = torch.zeros(1, pages, dtype=torch.int32)
    table[0, :4] = torch.arange(4)
    q_pe = torch.zeros(rows, heads, 64, dtype=torch.bfloat16)
    q_pe[:, :, 0] = 1
    on = [t.to(cuda_device) for t in (torch.zeros(rows, heads, 512, dtype=torch.bfloat16), q_pe, cache)]
    out, lse = torch.zeros(rows, heads, 512, dtype=torch.bfloat16, device=cuda_device), torch.zeros(rows, heads, device=cuda_device)
    quant.attend(*on, torch.tensor([N], device=cuda_device), table.to(cuda_device),
                 torch.tensor([0, rows], device=cuda_device), SCALE, out, lse)
    want, bound = wanted(scales, x)
    assert ((out[-1].cpu().double() - want).abs() <= bound).all()  # the last row sees all pairs whole


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads", [(1, 16), (200, 16), (100, 128)])
def test_selected_pairs_that_cancel(cuda_device, rows, heads):
    cache, scales, x = pairs(True)
    picked = torch.stack([torch.randperm(N, generator=torch.Generator().manual_seed(i)) for i in range(rows)])
    q_pe = torch.zeros(rows, heads, 64, dtype=torch.bfloat16)
    q_pe[:, :, 0] = 1
    out, lse = torch.zeros(rows, heads, 512, dtype=torch.bfloat16, device=cuda_device), torch.zeros(rows, heads, device=cuda_device)
    quant.attend_sparse(torch.zeros(rows, heads, 512, dtype=torch.bfloat16, device=cuda_device), q_pe.to(cuda_device),
                        cache.to(cuda_device), picked.to(cuda_device), SCALE, out, lse)
    want, bound = wanted(scales, x)
    assert ((out.cpu().double() - want).abs() <= bound).all()


KINDS = {  # (their scale, factor of the pairs' scales, their base-2 logit, their codes)
    "heavy": (2.0 ** 24, 1.0, -100.0, "random"), "heavier": (2.0 ** 45, 1.0, -140.0, "random"),
    "zeros": (1.0, 2.0 ** -24, 0.0, "zeros"), "light": (2.0 ** -100, 1.0, 0.0, "random"),
}


def among_others(kind, first, seed=3):
    """The pairs behind or before a tile of tokens that have next to no part in the outputs: scales far above the pairs' and no
    weight, rows of zeros with the scale that they are written with, scales far below."""
    scale, by, logit, what = KINDS[kind]
    cache, scales, x = pairs(True)
    more = torch.zeros(2, quant.PAGE_BYTES, dtype=torch.uint8)
    codes, kpe, s = oq.pieces(more)
    if what == "random":
        g = torch.Generator().manual_seed(seed)
        codes[:] = (torch.randn(codes.shape, generator=g) * 140).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    s[:] = scale
    kpe[:, :, 0] = round(logit / (SCALE * oq.LOG2E))
    oq.pieces(cache)[2].mul_(by)
    other = kpe[:, :, 0].double().flatten() * SCALE * oq.LOG2E
    out, bound = wanted(scales * by, x, (other,))
    # what the others do add
    lse = torch.logsumexp(torch.cat([x, other]) / oq.LOG2E, 0) * oq.LOG2E
    bound = bound + scale * 448 * 2.0 ** float(other.max() - lse) * 128 * (what == "random")
    cache = torch.cat([cache, more])
    return cache, torch.tensor([4, 5, 0, 1, 2, 3] if first else [0, 1, 2, 3, 4, 5], dtype=torch.int32)[None], out, bound


def unit_queries(rows, heads, device):
    q_pe = torch.zeros(rows, heads, 64, dtype=torch.bfloat16, device=device)
    q_pe[:, :, 0] = 1
    return (torch.zeros(rows, heads, 512, dtype=torch.bfloat16, device=device), q_pe,
            torch.zeros(rows, heads, 512, dtype=torch.bfloat16, device=device), torch.zeros(rows, heads, device=device))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("heads,pages", [(16, 6), (16, 900), (24, 900), (128, 6)])
def test_tokens_that_do_not_count_take_nothing(cuda_device, kind, first, heads, pages):
    cache, table, want, bound = among_others(kind, first)
    q_nope, q_pe, out, lse = unit_queries(1, heads, cuda_device)
    wide = torch.zeros(1, pages, dtype=torch.int32)
    wide[:, :6] = table
    quant.attend(q_nope, q_pe, cache.to(cuda_device), torch.tensor([N + 128], device=cuda_device), wide.to(cuda_device), None, SCALE,
                 out, lse)
    assert ((out[0].cpu().double() - want).abs() <= bound).all()
    picked = (table[0].long()[:, None] * 64 + torch.arange(64)).flatten()[None].repeat(1 if heads == 16 else 100, 1)
    q_nope, q_pe, out, lse = unit_queries(len(picked), heads, cuda_device)
    quant.attend_sparse(q_nope, q_pe, cache.to(cuda_device), picked.to(cuda_device), SCALE, out, lse)
    assert ((out.cpu().double() - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [5, 900])
def test_later_drafts_take_nothing(cuda_device, pages):
    """Drafts of large scales that a chain's first row does not see."""
    cache, scales, x = pairs(True)
    more = torch.zeros(1, quant.PAGE_BYTES, dtype=torch.uint8)
    codes, _, s = oq.pieces(more)
    codes[:], s[:] = 0x7E, 2.0 ** 40
    table = torch.zeros(1, pages, dtype=torch.int32)
    table[0, :5] = torch.arange(5)
    q_nope, q_pe, out, lse = unit_queries(3, 16, cuda_device)
    quant.attend(q_nope, q_pe, torch.cat([cache, more]).to(cuda_device), torch.tensor([N + 2], device=cuda_device),
                 table.to(cuda_device), torch.tensor([0, 3], device=cuda_device), SCALE, out, lse)
    want, bound = wanted(scales, x)
    assert ((out[0].cpu().double() - want).abs() <= bound).all()
    assert (out[1:] > 2.0 ** 40).all()


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [-125, -118, -60, 60, 115])
@pytest.mark.parametrize("pages", [5, 900])
def test_scales_of_all_sizes(cuda_device, exponent, pages):
    """One scale in all rows, one code in all places: that value, to bf16 and what a quotient near 2^-133 has (15 bits)."""
    cache = torch.zeros(5, quant.PAGE_BYTES, dtype=torch.uint8)
    codes, _, s = oq.pieces(cache)
    codes[:], s[:] = 0x7E, 2.0 ** exponent
    table = torch.zeros(1, pages, dtype=torch.int32)
    table[0, :5] = torch.arange(5)
    q_nope, q_pe, out, lse = unit_queries(1, 16, cuda_device)
    quant.attend(q_nope, q_pe, cache.to(cuda_device), torch.tensor([300], device=cuda_device), table.to(cuda_device), None, SCALE,
                 out, lse)
    want = 448 * 2.0 ** exponent
    assert ((out.cpu().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -13) * want).all()
    assert ((lse.cpu().double() - math.log2(300)).abs() <= 2.0 ** -17).all()


@pytest.mark.gpu
@pytest.mark.parametrize("length,heads", [(3000, 16), (3000, 64), (20000, 16), (20000, 32)])
def test_outputs_are_the_exact_ones_rounded(cuda_device, length, heads):
    """Against the exact outputs in bf16: an error e of an output moves it to a neighbour, a step of at most 2^-7 of itself away,
    once in step / e times, so that the mean square of the differences is e times the step.  With e at most 2^-14 of the
    outputs (the weights' parts; what logits and sums add is far below that of most tokens) that is the square of 2^-10.5."""
    g = torch.Generator().manual_seed(length)
    pages = (length + 63) // 64
    cache = torch.zeros(pages, quant.PAGE_BYTES, dtype=torch.uint8)
    codes, kpe, scales = oq.pieces(cache)
    codes[:] = (torch.randn(codes.shape, generator=g) * 140).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    kpe[:] = torch.randn(kpe.shape, generator=g).bfloat16()
    scales[:] = torch.exp(torch.randn(scales.shape, generator=g) * 0.3) / 140
    qn, qp = torch.randn(1, heads, 512, generator=g).bfloat16(), torch.randn(1, heads, 64, generator=g).bfloat16()
    table, seq = torch.arange(pages, dtype=torch.int32)[None], torch.tensor([length], dtype=torch.int32)
    out, lse = torch.zeros(1, heads, 512, dtype=torch.bfloat16, device=cuda_device), torch.zeros(1, heads, device=cuda_device)
    quant.attend(qn.to(cuda_device), qp.to(cuda_device), cache.to(cuda_device), seq.to(cuda_device), table.to(cuda_device), None,
                 SCALE, out, lse)
    want, _, _, _ = oq.attend_reference(qn, qp, cache, seq, table, None, SCALE)
    off = out.cpu().double() - want.bfloat16().double()
    assert float(off.square().sum().sqrt() / want.square().sum().sqrt()) <= 2.0 ** -10.5
