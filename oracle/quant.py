"""The latent cache in 8 bits, in 64 bits and byte by byte from the layout of a
page (TEST INFRASTRUCTURE ONLY): written, read, and attention over it.

A page of 64 tokens is 41216 bytes: 64 x 512 e4m3 codes, 64 x 64 bf16, 64 fp32
scales.  ``write`` gives the codes that exact arithmetic gives (the quotients are
of integers of at most 19 and 16 bits, so float64 rounds none of them across a
border of e4m3) and scales and rotated values in 64 bits.
"""

from __future__ import annotations

import math

import torch

PAGE, CKV, KPE = 64, 512, 64
PAGE_BYTES = 41216
LOG2E = 1.4426950408889634


def pieces(cache: torch.Tensor):
    """Codes [pages, 64, 512] (uint8), kpe [pages, 64, 64] (bf16), scales [pages, 64]: views of a uint8 cache."""
    flat = cache.view(torch.uint8).reshape(-1, PAGE_BYTES)
    return (flat[:, :PAGE * CKV].unflatten(1, (PAGE, CKV)),
            flat[:, PAGE * CKV:PAGE * (CKV + 2 * KPE)].view(torch.bfloat16).unflatten(1, (PAGE, KPE)),
            flat[:, PAGE * (CKV + 2 * KPE):].view(torch.float32))


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Bytes of float64 values rounded to nearest even (|x| <= 448; NaN is 0x7F), by their definition."""
    a = x.abs()
    e = torch.floor(torch.log2(torch.where(a > 0, a, 2.0 ** -6))).clamp(min=-6)
    for _ in range(2):  # log2 may be off by one step at a power of two
        e = torch.where(a < 2.0 ** e, e - 1, torch.where(a >= 2.0 ** (e + 1), e + 1, e)).clamp(min=-6)
    steps = torch.round(a / 2.0 ** (e - 3))  # torch rounds halves to even
    code = ((e + 6) * 8 + steps).to(torch.int64)  # the implicit bit is the 8 of the steps; a carry moves the exponent
    code = torch.where(torch.isnan(x), 0x7F, torch.where(torch.signbit(x), code | 0x80, code))
    return code.to(torch.uint8)


def value(code: torch.Tensor) -> torch.Tensor:
    """float64 values of e4m3 bytes."""
    c = code.to(torch.int64)
    e, m = (c >> 3) & 15, c & 7
    v = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e.double() - 10))
    v = torch.where((c & 0x7F) == 0x7F, math.nan, v)
    return torch.where(c >= 128, -v, v)


def write_rows(kv, norm=None, eps=1e-6, positions=None, cos_sin=None, interleaved=False):
    """(codes uint8 [N, 512], scales, kpe), scales and kpe in float64 unrounded, of bf16 rows [N, 576]."""
    c, e = kv[:, :CKV].double(), kv[:, CKV:].double()
    t = c if norm is None else c * norm.double()
    r = torch.ones(len(kv), dtype=torch.float64) if norm is None else 1 / torch.sqrt((c * c).mean(1) + eps)
    top = t.abs().amax(1)
    scale = top * r / 448
    small = ~(scale >= 2.0 ** -126)
    broken = ~torch.isfinite(t).all(1) | (scale > torch.finfo(torch.float32).max)
    code = e4m3(448 * t / torch.where(small | broken, 1.0, top)[:, None].clamp(min=1e-300))
    code[small] = 0
    code[broken] = 0x7F
    scale = torch.where(small | broken, 1.0, scale)
    if positions is not None:
        cos, sin = cos_sin[positions].double().chunk(2, 1)
        a, b = (e[:, 0::2], e[:, 1::2]) if interleaved else e.chunk(2, 1)
        x, y = a * cos - b * sin, b * cos + a * sin
        e = torch.stack([x, y], 2).flatten(1) if interleaved else torch.cat([x, y], 1)
    return code, scale, e


def rows(cache: torch.Tensor, slot: torch.Tensor):
    """(latents, position parts) of slots, float64."""
    codes, kpe, scales = pieces(cache)
    p, t = slot // PAGE, slot % PAGE
    return value(codes[p, t]) * scales[p, t].double()[:, None], kpe[p, t].double()


def bf16(x: torch.Tensor) -> torch.Tensor:
    """A float64 tensor that float32 holds exactly, or nearly: rounded through it to bf16."""
    return x.float().bfloat16()


def scales_of(cache: torch.Tensor, slot: torch.Tensor) -> torch.Tensor:
    return pieces(cache)[2][slot // PAGE, slot % PAGE].double()


def _softmax(q_nope, q_pe, c, e, scales, see, scale):
    """(output, lse and their bounds) of one row's heads over tokens c, e [n, ...] of these scales, of which `see` [n] are
    visible."""
    H = q_nope.shape[0]
    c, e, scales = c[see], e[see], scales[see]
    if len(c) == 0:
        z = torch.zeros(H, CKV, dtype=torch.float64)
        return z, torch.full((H,), -math.inf, dtype=torch.float64), z, torch.zeros(H, dtype=torch.float64)
    q, r = q_nope.double(), q_pe.double()
    x = (q @ c.T + r @ e.T) * (scale * LOG2E)
    off = (q.abs() @ c.abs().T + r.abs() @ e.abs().T) * (600 * 2.0 ** -23 * abs(scale) * LOG2E)
    lse = torch.logsumexp(x / LOG2E, 1) * LOG2E
    move = off.amax(1)
    w = torch.exp2(x - lse[:, None])
    out = w @ c
    err = (2 * math.log(2) * (off + move[:, None]) + 2.0 ** -14 + 2.0 ** -17) * w
    codes = torch.where(scales[:, None] == 0, 0.0, c.abs() / scales[:, None])
    largest = torch.where(codes.any(1) | (scales != 1), w * scales, 0.0).amax(1, keepdim=True)
    bound = err @ c.abs() + 2.0 ** -28 * largest * codes.sum(0) + 2.0 ** -8 * out.abs() + 2.0 ** -20 * c.abs().amax()
    return out, lse, bound, move + 2.0 ** -18 + 2.0 ** -23 * lse.abs()


def attend_reference(q_nope, q_pe, cache, seq_lens, table, cu, scale):
    """(output, lse, output bound, lse bound), float64; rows of no request are NaN.

    * A logit is a sum of 512 products, scaled, and of 64 more, accumulated in fp32 in an order that is not known, in two
      parts of the query, with the scale's and the parts' own roundings: off by at most 600 * 2^-23 of the sum of the
      magnitudes (2^-23, not 2^-24, for accumulators that truncate).
    * The lse moves by at most the largest of these, the exponential's and the sum's errors (2^-18 is far above both) and
      one rounding; a weight by ln 2 times its logit's and the lse's error.
    * A weight is split into four parts of 3 bits each, the last two of what its upper 11 bits leave with its lower ones.
      Each is half a step off what the one before leaves, which may pass a power of two by an eighth: within 2^-14, and
      2^-18 for the lower bits' rounding, 2^-22 for its products.  Where it is far below the largest, it is within half the
      smallest step of the last part, 2^-17 / 128, and 2^-24 of half precision's: in units of which the largest weight times
      its scale is 2^5 or more (rows of zeros that have the scale 1 apart).  Each token's code may so count 2^-28 times that
      product too much or too little.  The output is rounded to bf16, 2^-8 of itself.
    """
    T, H = q_nope.shape[:2]
    out = torch.full((T, H, CKV), math.nan, dtype=torch.float64)
    lse = torch.full((T, H), math.nan, dtype=torch.float64)
    bo, bl = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(len(seq_lens)):
        lo, hi = (b, b + 1) if cu is None else (int(cu[b]), int(cu[b + 1]))
        L = int(seq_lens[b])
        pos = torch.arange(L)
        slot = table[b].long()[pos // PAGE] * PAGE + pos % PAGE
        c, e = rows(cache, slot)
        for i in range(lo, hi):
            out[i], lse[i], bo[i], bl[i] = _softmax(q_nope[i], q_pe[i], c, e, scales_of(cache, slot), pos < L - (hi - 1 - i), scale)
    return out, lse, bo, bl


def sparse_reference(q_nope, q_pe, cache, picked, scale):
    """The same for rows of slots, -1: none."""
    T, H = q_nope.shape[:2]
    out, lse = torch.zeros(T, H, CKV, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    bo, bl = torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(T):
        slot = picked[i].long().clamp(min=0)
        c, e = rows(cache, slot)
        out[i], lse[i], bo[i], bl[i] = _softmax(q_nope[i], q_pe[i], c, e, scales_of(cache, slot), picked[i] >= 0, scale)
    return out, lse, bo, bl
