"""Operators of serving over a latent cache held in 8 bits, and of verifying drafts: cases, plain forms and work.

* ``write``: new tokens' latents normalised, their position part rotated, both stored in the paged cache, the
  latent in 8 bits with a scale for each token (``dsa_b200.quant.write``).
* ``read``: ranges of cached tokens back as bf16 rows (``dsa_b200.quant.read``).
* ``attend``: attention of single tokens, or of chains of drafts, over everything a request has cached
  (``dsa_b200.quant.attend``).
* ``sparse``: attention over the 2048 slots that the indexer selected (``dsa_b200.quant.attend_sparse``).
* ``verify``: drafted tokens accepted or rejected against the target's probabilities, and the token that
  follows drawn, from given random numbers (``dsa_b200.verify.run``).
"""

import math
import os
import random
import sys

import torch

sys.path.append(os.path.abspath("flashinfer-bench-starter-kit_b200"))  # where the package lies

own = False

PAGE, CKV, KPE, TOPK = 64, 512, 64, 2048
PAGE_BYTES = PAGE * (CKV + 2 * KPE + 4)
LOG2E = 1.4426950408889634
SCALE = 1.0 / math.sqrt(192.0)
EPS = 1e-6
MOST_E4M3 = 448.0


# ------------------------------------------------------------------ cases
def listed():
    return [
        # The new tokens of one decode step of 64 requests, where latency counts.
        write_case("write_step", 64, 65536, False, 1),
        # A batch of long prompts.
        write_case("write_prompts", 200003, 131072, True, 2),
        # The cached part of one prompt, read back for its next chunk.
        read_case("read_chunk", 1, 1500, 5000, 3),
        # Long contexts of a batch.
        read_case("read_long", 9, 30000, 65536, 4),
        # One request, one token: plain decoding of a short context.
        attend_case("attend_one", 1, 1, 1, 16, 1000, 1000, 5),
        # An ordinary verification step: 16 requests, chains of up to 4 drafts, ragged contexts.
        attend_case("attend_ordinary", 16, 1, 4, 16, 4096, 16384, 6),
        # The decode batch of the framework's benchmark (64 requests, 65536 tokens each).
        attend_case("attend_long", 64, 1, 1, 16, 65536, 65536, 7),
        # All 128 heads of a layer on one GPU, where the products bound it.
        attend_case("attend_heads", 5, 1, 2, 128, 8000, 30001, 8),
        # A few tokens behind the indexer, some of them with contexts below its selection.
        sparse_case("sparse_small", 5, 16, 500, 20000, 9),
        # The framework's sparse decode batch several times over.
        sparse_case("sparse_large", 300, 16, 3500, 65536, 10),
        # Chains of a few drafts of a small vocabulary.
        verify_case("verify_chains", 4, 3, 6, 1, 32000, False, 11),
        # Trees of a large batch and vocabulary.
        verify_case("verify_trees", 48, 6, 12, 3, 131072, False, 12),
    ]


def write_case(name, tokens, positions, interleaved, mix):
    return {"name": name, "op": "write", "tokens": tokens, "positions": positions, "interleaved": interleaved, "mix": mix}


def read_case(name, batch, len_lo, len_hi, mix):
    return {"name": name, "op": "read", "batch": batch, "len_lo": len_lo, "len_hi": len_hi, "mix": mix}


def attend_case(name, batch, row_lo, row_hi, heads, len_lo, len_hi, mix):
    return {"name": name, "op": "attend", "batch": batch, "row_lo": row_lo, "row_hi": row_hi, "heads": heads,
            "len_lo": len_lo, "len_hi": len_hi, "mix": mix}


def sparse_case(name, batch, heads, len_lo, len_hi, mix):
    return {"name": name, "op": "sparse", "batch": batch, "heads": heads, "len_lo": len_lo, "len_hi": len_hi, "mix": mix}


def verify_case(name, batch, row_lo, row_hi, branch, vocab, certain, mix):
    """`branch`: most children of a node; `certain`: drafts without a distribution of their own."""
    return {"name": name, "op": "verify", "batch": batch, "row_lo": row_lo, "row_hi": row_hi, "branch": branch,
            "vocab": vocab, "certain": certain, "mix": mix}


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "sparse", "verify"])
    mix = rng.randrange(1 << 30)
    if op == "write":
        case = write_case("", log_int(rng, 1, 200000), log_int(rng, 64, 131072), rng.random() < 0.5, mix)
    elif op == "read":
        batch = log_int(rng, 1, 64)
        len_hi = min(log_int(rng, 1, 131072), 400_000 // batch)
        case = read_case("", batch, max(1, int(len_hi * rng.uniform(0.05, 1.0))), len_hi, mix)
    elif op == "attend":
        batch, heads = log_int(rng, 1, 64), rng.choice([16, 16, 16, 8, 24, 32, 64, 128])
        len_hi = min(log_int(rng, 1, 131072), 4_000_000 // batch)
        len_lo = max(1, int(len_hi * rng.uniform(0.1, 1.0)))
        most = min(8, max(1, 60_000_000 // (heads * batch * len_hi)))
        row_hi = rng.randint(1, most)
        case = attend_case("", batch, rng.randint(1, row_hi), row_hi, heads, max(len_lo, row_hi), max(len_hi, row_hi), mix)
    elif op == "sparse":
        len_hi = log_int(rng, 10, 131072)
        case = sparse_case("", log_int(rng, 1, 250), rng.choice([16, 16, 16, 8, 32, 64]), max(1, int(len_hi * rng.uniform(0.05, 1))),
                           len_hi, mix)
    else:
        vocab, batch = log_int(rng, 1000, 131072), log_int(rng, 1, 64)
        row_hi = min(log_int(rng, 1, 32), max(1, 75_000_000 // (vocab * batch)))
        case = verify_case("", batch, rng.randint(1, row_hi), row_hi, rng.randint(1, 4), vocab, rng.random() < 0.25, mix)
    del case["name"]
    return case


# ------------------------------------------------------------------ shapes
def lengths(case):
    """Context length of each request, spread over the logarithm of the case's range, odd ones among them."""
    rng = random.Random(case["mix"])
    return [log_int(rng, case["len_lo"], case["len_hi"]) for _ in range(case["batch"])]


def counts(case):
    rng = random.Random(case["mix"] + 1)
    return [rng.randint(case["row_lo"], case["row_hi"]) for _ in range(case["batch"])]


def starts_of(case):
    """Where each request's range begins: at its first token, or somewhere in its first half."""
    rng = random.Random(case["mix"] + 2)
    return [rng.randrange(n // 2 + 1) if rng.random() < 0.5 else 0 for n in lengths(case)]


def trees(case):
    """Per request the parent of every row (row 0, the token that is certain: -1), at most `branch` children each."""
    rng = random.Random(case["mix"] + 3)
    all_parents = []
    for n in counts(case):
        parents, left = [-1], [case["branch"]]
        for j in range(1, n):
            free = [i for i in range(j) if left[i]]
            par = free[-1] if rng.random() < 0.6 else rng.choice(free)
            left[par] -= 1
            parents.append(par)
            left.append(case["branch"])
        all_parents.append(parents)
    return all_parents


def pages_of(tokens):
    return -(-tokens // PAGE)


def page_table(need, gen):
    """Disjoint random pages of a pool, rows padded with -1; and the pages used."""
    perm = torch.randperm(sum(need), generator=gen)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n].int()
        at += n
    return table, at


# ------------------------------------------------------------------ states
def prepare(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    return {"write": prepare_write, "read": prepare_read, "attend": prepare_attend, "sparse": prepare_sparse,
            "verify": prepare_verify}[case["op"]](case, cpu, gpu)


def normal(gpu, *shape):
    return torch.randn(*shape, generator=gpu, device="cuda", dtype=torch.bfloat16)


def parts(cache):
    """The pieces of a cache [pages, PAGE_BYTES] as tensors of what they hold: latents' codes, position parts, scales."""
    codes = cache[:, :PAGE * CKV].view(torch.float8_e4m3fn).unflatten(1, (PAGE, CKV))
    kpe = cache[:, PAGE * CKV:PAGE * (CKV + 2 * KPE)].view(torch.bfloat16).unflatten(1, (PAGE, KPE))
    return codes, kpe, cache[:, PAGE * (CKV + 2 * KPE):].view(torch.float32)


def full_cache(pool, gpu):
    """A cache as normalised latents leave it: the largest code of a row is 448, scales differ from token to token."""
    cache = torch.empty(pool, PAGE_BYTES, dtype=torch.uint8, device="cuda")
    codes, kpe, scales = parts(cache)
    at = 4096  # pages at a time
    for lo in range(0, pool, at):
        n = min(at, pool - lo)
        x = normal(gpu, n, PAGE, CKV).mul_(140).clamp_(-448, 448)
        codes[lo:lo + n] = x.to(torch.float8_e4m3fn)
        kpe[lo:lo + n] = normal(gpu, n, PAGE, KPE)
    scales[:] = torch.randn(pool, PAGE, generator=gpu, device="cuda").mul_(0.3).exp_().div_(140)
    return cache


def prepare_write(case, cpu, gpu):
    """Rows of the projection before the cache, slots of whole pages and a last, partly filled one, some rows padding."""
    n = case["tokens"]
    pool = pages_of(n) + 1
    slots = (torch.randperm(pool, generator=cpu)[:, None] * PAGE + torch.arange(PAGE)).flatten()[:n].clone()
    slots[torch.rand(n, generator=cpu) < 0.01] = -1
    angle = torch.arange(case["positions"], device="cuda").double()[:, None] * 10000.0 ** (
        -torch.arange(KPE // 2, device="cuda").double() / (KPE // 2))
    return {"op": "write", "kv": normal(gpu, n, CKV + KPE), "slots": slots.cuda(), "interleaved": case["interleaved"],
            "norm": (1 + 0.2 * torch.randn(CKV, generator=gpu, device="cuda")).bfloat16(),
            "positions": torch.randint(0, case["positions"], (n,), generator=cpu).cuda(),
            "table": torch.cat([angle.cos(), angle.sin()], 1).float(),
            "cache": torch.zeros(pool, PAGE_BYTES, dtype=torch.uint8, device="cuda")}


def prepare_read(case, cpu, gpu):
    seq, starts = lengths(case), starts_of(case)
    table, pool = page_table([pages_of(n) for n in seq], cpu)
    cu = torch.tensor([0] + [n - s for n, s in zip(seq, starts)]).cumsum(0)
    total = int(cu[-1])
    return {"op": "read", "cache": full_cache(pool, gpu), "table": table.cuda(), "cu": cu.int().cuda(),
            "starts": torch.tensor(starts, dtype=torch.int32).cuda(),
            "ckv": torch.empty(total, CKV, device="cuda", dtype=torch.bfloat16),
            "kpe": torch.empty(total, KPE, device="cuda", dtype=torch.bfloat16)}


def outputs(rows, heads):
    return {"out": torch.empty(rows, heads, CKV, device="cuda", dtype=torch.bfloat16),
            "lse": torch.empty(rows, heads, device="cuda")}


def prepare_attend(case, cpu, gpu):
    """A decode batch: queries, page tables, a cache that holds contexts and the rows themselves."""
    seq, count, heads = lengths(case), counts(case), case["heads"]
    table, pool = page_table([pages_of(n) for n in seq], cpu)
    total = sum(count)
    return {"op": "attend", "heads": heads, "longest": max(seq), "most": max(count), "chains": case["row_hi"] > 1,
            "q_nope": normal(gpu, total, heads, CKV), "q_pe": normal(gpu, total, heads, KPE),
            "cache": full_cache(pool, gpu), "seq": torch.tensor(seq, dtype=torch.int32).cuda(), "table": table.cuda(),
            "cu": torch.tensor([0] + count).cumsum(0).int().cuda(), **outputs(total, heads)}


def prepare_sparse(case, cpu, gpu):
    """What the indexer selects of each token's context: 2048 slots of it in no order, all of it and -1 where it is shorter."""
    seq, heads = lengths(case), case["heads"]
    table, pool = page_table([pages_of(n) for n in seq], cpu)
    picked = torch.full((len(seq), TOPK), -1, dtype=torch.int32)
    for b, n in enumerate(seq):
        pos = torch.randperm(n, generator=cpu)[:TOPK]
        picked[b, :len(pos)] = table[b, pos // PAGE] * PAGE + (pos % PAGE).int()
    return {"op": "sparse", "heads": heads, "q_nope": normal(gpu, len(seq), heads, CKV), "q_pe": normal(gpu, len(seq), heads, KPE),
            "cache": full_cache(pool, gpu), "picked": picked.cuda(), **outputs(len(seq), heads)}


def prepare_verify(case, cpu, gpu):
    """Target and draft distributions that are near each other, drafts drawn from the draft's (or its likeliest tokens)."""
    parents, count, vocab = trees(case), counts(case), case["vocab"]
    total = sum(count)
    cu = torch.tensor([0] + count).cumsum(0)
    x = torch.randn(total, vocab, generator=gpu, device="cuda").mul_(2.5)
    target = torch.softmax(x, 1)
    draft = torch.softmax(x.add_(torch.randn(total, vocab, generator=gpu, device="cuda").mul_(0.7)), 1)
    del x
    flat = torch.tensor([p for tree in parents for p in tree])
    row = torch.repeat_interleave(cu[:-1], torch.tensor(count)) + flat.clamp(min=0)
    if case["certain"]:  # a node's children are its likeliest tokens
        nth = [sum(q == p for q in tree[:j]) for tree in parents for j, p in enumerate(tree)]
        best = draft.topk(4, 1).indices
        tokens = best[row.cuda(), torch.tensor(nth).clamp(max=3).cuda()]
        draft = None
    else:
        u = torch.rand(total, 1, generator=gpu, device="cuda", dtype=torch.float64)
        tokens = torch.cat([torch.searchsorted(draft[r:r + 1].double().cumsum(1), u[i:i + 1]) for i, r in enumerate(row.tolist())])
        tokens = tokens[:, 0].clamp(max=vocab - 1)
    batch, width = len(count), max(1, max(count) - 1)
    whole = lambda *shape: torch.empty(*shape, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"op": "verify", "most": max(count), "target": target, "draft": draft, "tokens": tokens.int(),
            "parents": flat.int().cuda(), "cu": cu.int().cuda(),
            "accept": torch.rand(total, generator=gpu, device="cuda"), "sample": torch.rand(batch, generator=gpu, device="cuda"),
            "path": whole(batch, width), "accepted": whole(batch), "next": whole(batch)}


# ------------------------------------------------------------------ passes
def run(s):
    if own:
        return run_own(s)
    return {"write": plain_write, "read": plain_read, "attend": plain_attend, "sparse": plain_sparse,
            "verify": plain_verify}[s["op"]](s)


def run_own(s):
    if s["op"] == "verify":
        from dsa_b200 import verify
        verify.run(s["target"], s["draft"], s["tokens"], s["parents"], s["cu"], s["accept"], s["sample"], s["path"],
                   s["accepted"], s["next"])
        return {"path": s["path"], "accepted": s["accepted"], "next": s["next"]}
    from dsa_b200 import quant
    if s["op"] == "write":
        quant.write(s["kv"], s["slots"], s["cache"], s["norm"], EPS, s["positions"], s["table"], s["interleaved"])
        codes, kpe, scales = parts(s["cache"])
        return {"codes": codes, "kpe": kpe, "scales": scales}
    if s["op"] == "read":
        quant.read(s["cache"], s["table"], s["starts"], s["cu"], s["ckv"], s["kpe"])
        return {"ckv": s["ckv"], "kpe": s["kpe"]}
    if s["op"] == "attend":
        quant.attend(s["q_nope"], s["q_pe"], s["cache"], s["seq"], s["table"], s["cu"] if s["chains"] else None, SCALE,
                     s["out"], s["lse"])
    else:
        quant.attend_sparse(s["q_nope"], s["q_pe"], s["cache"], s["picked"], SCALE, s["out"], s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def plain_write(s):
    """y = c / rms(c) * norm as codes 448 y / max|y| and scale max|y| / 448, the rms left to the scale; e rotated."""
    c, e = s["kv"][:, :CKV].float(), s["kv"][:, CKV:].float()
    t = c * s["norm"].float()
    top = t.abs().amax(1)
    r = (c.square().mean(1) + EPS).rsqrt()
    codes = (MOST_E4M3 * t / top[:, None]).to(torch.float8_e4m3fn)
    cos, sin = s["table"][s["positions"]].chunk(2, 1)
    if s["interleaved"]:
        a, b = e[:, 0::2], e[:, 1::2]
        e = torch.stack([a * cos - b * sin, b * cos + a * sin], 2).flatten(1)
    else:
        a, b = e.chunk(2, 1)
        e = torch.cat([a * cos - b * sin, b * cos + a * sin], 1)
    real = s["slots"] >= 0
    at = (s["slots"][real] // PAGE, s["slots"][real] % PAGE)
    to_codes, to_kpe, to_scales = parts(s["cache"])
    to_codes.view(torch.uint8)[at] = codes[real].view(torch.uint8)
    to_kpe[at] = e[real].bfloat16()
    to_scales[at] = (top * r / MOST_E4M3)[real]
    return {"codes": to_codes, "kpe": to_kpe, "scales": to_scales}


def gathered(cache, slot):
    """Latents (32 bits) and position parts of slots of any shape."""
    codes, kpe, scales = parts(cache)
    at = (slot // PAGE, slot % PAGE)
    return codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scales[at][..., None], kpe[at]


def plain_read(s):
    cu = s["cu"].long()
    total = s["ckv"].shape[0]
    req = torch.repeat_interleave(torch.arange(len(cu) - 1, device="cuda"), cu[1:] - cu[:-1], output_size=total)
    pos = torch.arange(total, device="cuda") - cu[req] + s["starts"][req]
    c, e = gathered(s["cache"], s["table"][req, pos // PAGE].long() * PAGE + pos % PAGE)
    return {"ckv": c.bfloat16(), "kpe": e}


def softmax_rows(x, c):
    """Weighted latents and base-2 lse of base-2 logits x [B, rows, tokens], -inf where masked; x is used up."""
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = x.sub_(top).exp2_()
    total = e.sum(-1, keepdim=True)
    return torch.bmm(e, c) / torch.where(total == 0, 1.0, total), (top + total.log2())[..., 0]


def plain_attend(s):
    table, seq, cu = s["table"].long(), s["seq"].long(), s["cu"].long()
    B, longest, most, heads = table.shape[0], s["longest"], s["most"], s["heads"]
    count = cu[1:] - cu[:-1]
    pos = torch.arange(longest, device="cuda")
    c, e = gathered(s["cache"], table[:, pos // PAGE].clamp(min=0) * PAGE + pos % PAGE)
    draft = torch.arange(most, device="cuda")
    row = (cu[:-1, None] + draft).clamp(max=cu[-1] - 1)
    q_nope, q_pe = s["q_nope"][row].float().flatten(1, 2), s["q_pe"][row].float().flatten(1, 2)
    x = torch.bmm(q_nope, c.transpose(1, 2)).add_(torch.bmm(q_pe, e.float().transpose(1, 2))).mul_(SCALE * LOG2E)
    seen = (seq - count + 1)[:, None] + draft
    seen = torch.where(draft < count[:, None], seen, 0)
    x.view(B, most, heads, longest).masked_fill_((pos >= seen[:, :, None])[:, :, None, :], -math.inf)
    out, lse = softmax_rows(x, c)
    total = s["q_nope"].shape[0]
    req = torch.repeat_interleave(torch.arange(B, device="cuda"), count, output_size=total)
    at = (req, torch.arange(total, device="cuda") - cu[req])
    return {"out": out.reshape(B, most, heads, CKV)[at].bfloat16(), "lse": lse.reshape(B, most, heads)[at].contiguous()}


def plain_sparse(s):
    c, e = gathered(s["cache"], s["picked"].long().clamp(min=0))
    x = torch.bmm(s["q_nope"].float(), c.transpose(1, 2)).add_(torch.bmm(s["q_pe"].float(), e.float().transpose(1, 2)))
    x = x.mul_(SCALE * LOG2E).masked_fill_((s["picked"] < 0)[:, None, :], -math.inf)
    out, lse = softmax_rows(x, c)
    return {"out": out.bfloat16(), "lse": lse}


def plain_verify(s):
    """Children in the order of their rows.  With c = 0, R = 1 at a node, child x is accepted if u q(x) R < max(p(x) - c q(x), 0);
    else c += R and R = sum max(p - c q, 0), the residual's weights up to a factor.  A draft without a distribution: q is
    one at x, and a rejected x leaves the residual.  The next token is the first whose running weight exceeds u of all."""
    cu, accept = s["cu"].long(), s["accept"].double()
    B, width, vocab = len(cu) - 1, s["path"].shape[1], s["target"].shape[1]
    new = lambda v, t: torch.full((B,), v, dtype=t, device="cuda")  # noqa: E731
    node, taken, c, R = new(0, torch.long), new(0, torch.long), new(0.0, torch.float64), new(1.0, torch.float64)
    path = torch.full((B, width + 1), -1, dtype=torch.int32, device="cuda")
    count = cu[1:] - cu[:-1]
    out = torch.zeros(B, vocab, dtype=torch.bool, device="cuda")
    for j in range(1, s["most"]):
        row = (cu[:-1] + j).clamp(max=cu[-1] - 1)
        test = (j < count) & (s["parents"][row] == node) & (taken < width)
        at = cu[:-1] + node
        p, x, u = s["target"][at].double(), s["tokens"][row].long()[:, None], accept[row]
        if s["draft"] is None:
            w = p.masked_fill_(out, 0.0).gather(1, x)[:, 0]
            ok = test & (u * R < w)
            no = test & ~ok
            R = torch.where(no, R - w, R)
            out.scatter_(1, x, out.gather(1, x) | no[:, None])
        else:
            q = s["draft"][at].double()
            w = (p.gather(1, x) - c[:, None] * q.gather(1, x)).clamp(min=0)[:, 0]
            ok = test & (u * q.gather(1, x)[:, 0] * R < w)
            no = test & ~ok
            c = torch.where(no, c + R, c)
            R = torch.where(no, p.sub_(q.mul_(c[:, None])).clamp_(min=0).sum(1), R)
        path.scatter_(1, torch.where(ok, taken, width)[:, None], torch.where(ok, j, -1)[:, None].int())
        node, taken = torch.where(ok, j, node), taken + ok
        c, R = torch.where(ok, 0.0, c), torch.where(ok, 1.0, R)
        out &= ~ok[:, None]
    path = path[:, :width].contiguous()
    p = s["target"][cu[:-1] + node].double()
    if s["draft"] is None:
        w = p.masked_fill(out, 0.0)
    else:
        w = torch.where(c[:, None] == 0, p, (p - c[:, None] * s["draft"][cu[:-1] + node].double()).clamp(min=0))
    w = torch.where(w.sum(1, keepdim=True) == 0, p, w).cumsum(1)
    above = w > s["sample"].double()[:, None] * w[:, -1:]
    first = torch.where(above.any(1), above.int().argmax(1), -1)
    return {"path": path, "accepted": taken.int(), "next": first.int()}


# ------------------------------------------------------------------ work
def work(case):
    row = CKV + 2 * KPE + 4  # a cached token's bytes
    if case["op"] == "write":
        n = case["tokens"]
        return {"bytes": n * (2 * (CKV + KPE) + row + 16) + 4 * KPE * min(n, case["positions"]), "flops": 0}
    if case["op"] == "read":
        n = sum(a - b for a, b in zip(lengths(case), starts_of(case)))
        return {"bytes": n * (row + 2 * (CKV + KPE)), "flops": 0}
    if case["op"] == "verify":
        # Of each request at least one row of each kind has to be read for the next token.
        return {"bytes": 4 * case["batch"] * case["vocab"] * (1 if case["certain"] else 2) + 16 * sum(counts(case)), "flops": 0}
    heads, seq = case["heads"], lengths(case)
    if case["op"] == "sparse":
        rows = len(seq) * heads
        tokens = sum(min(n, TOPK) for n in seq)
        pairs = heads * tokens
    else:
        count = counts(case)
        rows, tokens = heads * sum(count), sum(seq)
        pairs = heads * sum(n * L - n * (n - 1) // 2 for n, L in zip(count, seq))
    return {"bytes": row * tokens + rows * (2 * (CKV + KPE) + 2 * CKV + 4), "flops": 2 * pairs * (2 * CKV + KPE)}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"write": exact_write, "read": exact_read, "attend": exact_attend, "sparse": exact_sparse,
            "verify": exact_verify}[case["op"]](s)


def exact_write(s):
    kv, norm, slots = s["kv"].double(), s["norm"].double(), s["slots"]
    pool = s["cache"].shape[0]
    c, e = kv[:, :CKV], kv[:, CKV:]
    y = c / torch.sqrt((c * c).sum(1, keepdim=True) / CKV + EPS) * norm
    scale = y.abs().max(1).values / MOST_E4M3
    # What the codes stand for: y / scale, to half a step of their type.  Free of the rms, the quotient is exact enough to round.
    t = c * norm
    codes = (t * MOST_E4M3 / t.abs().max(1, keepdim=True).values).to(torch.float8_e4m3fn).double()
    turn = torch.complex(s["table"][:, :KPE // 2].double(), s["table"][:, KPE // 2:].double())[s["positions"]]
    if s["interleaved"]:
        e = torch.view_as_real(torch.view_as_complex(e.reshape(-1, KPE // 2, 2).contiguous()) * turn).flatten(1)
    else:
        z = torch.complex(e[:, :KPE // 2], e[:, KPE // 2:]) * turn
        e = torch.cat([z.real, z.imag], 1)
    keep = torch.nonzero(slots >= 0)[:, 0]
    put = lambda v, *shape: torch.zeros(pool * PAGE, *shape, dtype=torch.float64, device="cuda").index_copy_(  # noqa: E731
        0, slots[keep], v[keep]).reshape(pool, PAGE, *shape)
    return {"codes": put(codes, CKV), "kpe": put(e, KPE), "scales": put(scale)}


def rows_64(cache, slot):
    """[latent, position part] of a list of slots in 64 bits, byte by byte from the layout of a page."""
    flat = cache.reshape(-1)
    base = (slot // PAGE * PAGE_BYTES)[:, None]
    t = (slot % PAGE)[:, None]
    byte = lambda at, n, w: flat[base + at + t * w + torch.arange(n, device="cuda")].contiguous()  # noqa: E731
    c = byte(0, CKV, CKV).view(torch.float8_e4m3fn).double()
    e = byte(PAGE * CKV, 2 * KPE, 2 * KPE).view(torch.bfloat16).double()
    return c * byte(PAGE * (CKV + 2 * KPE), 4, 4).view(torch.float32).double(), e


def positions_to_slots(s, b, pos):
    return s["table"][b].long()[pos // PAGE] * PAGE + pos % PAGE


def exact_read(s):
    cu, starts = s["cu"].tolist(), s["starts"].tolist()
    got = [rows_64(s["cache"], positions_to_slots(s, b, starts[b] + torch.arange(cu[b + 1] - cu[b], device="cuda")))
           for b in range(len(starts))]
    return {"ckv": torch.cat([c for c, _ in got]), "kpe": torch.cat([e for _, e in got])}


def exact_rows(s, i, slot, hidden):
    """One token's heads over the rows of `slot`, but for the last `hidden`."""
    c, e = rows_64(s["cache"], slot[:len(slot) - hidden])
    x = (s["q_nope"][i].double() @ c.T + s["q_pe"][i].double() @ e.T) * SCALE
    return torch.softmax(x, 1) @ c, torch.logsumexp(x, 1) * LOG2E


def exact_attend(s):
    cu, seq = s["cu"].tolist(), s["seq"].tolist()
    got = []
    for b, L in enumerate(seq):
        slot = positions_to_slots(s, b, torch.arange(L, device="cuda"))
        got += [exact_rows(s, i, slot, cu[b + 1] - 1 - i) for i in range(cu[b], cu[b + 1])]
    return {"out": torch.stack([o for o, _ in got]), "lse": torch.stack([x for _, x in got])}


def exact_sparse(s):
    got = [exact_rows(s, i, p[p >= 0].long(), 0) for i, p in enumerate(s["picked"])]
    return {"out": torch.stack([o for o, _ in got]), "lse": torch.stack([x for _, x in got])}


def exact_verify(s):
    """Request by request: the residual as a distribution, normalised after every rejection."""
    cu, parents, tokens = s["cu"].tolist(), s["parents"].tolist(), s["tokens"].tolist()
    width = s["path"].shape[1]
    paths, accepted, following = [], [], []
    for b in range(len(cu) - 1):
        lo, hi, node, path = cu[b], cu[b + 1], 0, []
        p = s["target"][lo].double()
        for j in range(1, hi - lo):
            if parents[lo + j] != node or len(path) == width:
                continue
            x, u = tokens[lo + j], float(s["accept"][lo + j])
            if s["draft"] is None:
                q = torch.zeros_like(p)
                q[x] = 1
            else:
                q = s["draft"][lo + node].double()
            if u * float(q[x]) < float(p[x]):
                path.append(j)
                node = j
                p = s["target"][lo + node].double()
            else:
                left = (p - q).clamp(min=0)
                if s["draft"] is None:
                    left = p.clone()
                    left[x] = 0
                p = left / left.sum() if float(left.sum()) > 0 else p
        run_up = p.cumsum(0)
        following.append(int(torch.nonzero(run_up > float(s["sample"][b]) * run_up[-1])[0, 0]))
        paths.append(path + [-1] * (width - len(path)))
        accepted.append(len(path))
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"path": whole(paths), "accepted": whole(accepted), "next": whole(following)}
