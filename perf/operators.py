"""Speculative-decoding and cache-eviction operators over the paged caches: cases, plain forms and work.

* ``tree``: attention of a tree of drafted tokens over the paged ckv / kpe cache (``dsa_b200.tree.run``).
* ``weights``: the attention weight each cached token got from such rows, added to its accumulator
  (``dsa_b200.evict.accumulate``).
* ``evict``: the kept tokens of every request and their rows moved to new pages (``dsa_b200.evict.run``).
"""

import math
import os
import random
import sys

import torch

sys.path.append(os.path.abspath("flashinfer-bench-starter-kit_b200"))  # where the package lies

own = False

PAGE, CKV, KPE, IDX = 64, 512, 64, 132
LOG2E = 1.4426950408889634
SCALE = 1.0 / math.sqrt(192.0)


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One request, one token: plain decoding of a short context, where latency counts.
        tree_case("tree_one", 1, 1, 1, 16, 1000, 1000, 1),
        # A few requests with a handful of drafts each, short ragged contexts.
        tree_case("tree_small", 5, 2, 5, 16, 200, 4100, 2),
        # An ordinary verification step: 16 requests, up to 8 drafts, ragged contexts.
        tree_case("tree_ordinary", 16, 3, 8, 16, 4096, 16384, 3),
        # The decode batch of the framework's benchmark (64 requests, 65536 tokens each), 4 drafts each.
        tree_case("tree_long", 64, 4, 4, 16, 65536, 65536, 4),
        # Wide trees: 64 drafts per request, where the products bound it.
        tree_case("tree_wide", 4, 64, 64, 16, 30000, 32768, 5),
        # All 128 heads of a layer on one GPU, an odd number of drafts.
        tree_case("tree_heads", 3, 5, 7, 128, 2000, 20001, 6),
        # Accumulating weights after single-token steps of short contexts.
        weights_case("weights_small", 2, 1, 1, 16, 300, 2900, 7),
        # After a verification step of a long-context batch.
        weights_case("weights_long", 32, 4, 4, 16, 8192, 65536, 8),
        # After wide trees.
        weights_case("weights_wide", 4, 32, 40, 16, 12000, 16384, 9),
        # One request of a few thousand tokens brought down to 1024.
        evict_case("evict_small", 1, 5001, 5001, 1024, 4, 64, 10),
        # A batch of ragged contexts, some within the budget.
        evict_case("evict_ordinary", 16, 1500, 16384, 2048, 4, 128, 11),
        # Long contexts brought down to 8192 tokens each.
        evict_case("evict_long", 32, 32768, 65536, 8192, 16, 1000, 12),
    ]


def tree_case(name, batch, draft_lo, draft_hi, heads, len_lo, len_hi, mix):
    return {"name": name, "op": "tree", "batch": batch, "draft_lo": draft_lo, "draft_hi": draft_hi, "heads": heads,
            "len_lo": len_lo, "len_hi": len_hi, "mix": mix}


def weights_case(name, *sizes):
    return {**tree_case(name, *sizes), "op": "weights"}


def evict_case(name, batch, len_lo, len_hi, budget, sink, recent, mix):
    return {"name": name, "op": "evict", "batch": batch, "len_lo": len_lo, "len_hi": len_hi, "budget": budget,
            "sink": sink, "recent": recent, "mix": mix}


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "weights", "evict"])
    batch = log_int(rng, 1, 64)
    len_hi = min(log_int(rng, 64, 131072), 2_000_000 // batch)
    len_lo = max(1, int(len_hi * rng.uniform(0.1, 1.0)))
    mix = rng.randrange(1 << 30)
    if op == "evict":
        budget = log_int(rng, 32, 16384)
        sink = rng.randrange(0, budget // 4 + 1)
        recent = rng.randrange(0, budget // 2 + 1)
        case = evict_case("", batch, len_lo, len_hi, budget, sink, recent, mix)
    else:
        heads = rng.choice([16, 16, 16, 8, 24, 32, 64, 128])
        most = min(64, max(1, 120_000_000 // (heads * batch * len_hi)))  # rows x tokens within the largest listed case's
        draft_hi = log_int(rng, 1, most)
        draft_lo = rng.randint(1, draft_hi)
        make = tree_case if op == "tree" else weights_case
        case = make("", batch, draft_lo, draft_hi, heads, len_lo, len_hi, mix)
    del case["name"]
    return case


# ------------------------------------------------------------------ shapes
def lengths(case):
    """Prefix (or context) length per request, spread over the logarithm of the case's range, odd ones among them."""
    rng = random.Random(case["mix"])
    return [log_int(rng, case["len_lo"], case["len_hi"]) for _ in range(case["batch"])]


def trees(case):
    """Per request the parent of every draft (-1: the prefix), parents before children."""
    rng = random.Random(case["mix"] + 1)
    return [[rng.randrange(-1, j) if rng.random() < 0.5 else j - 1 for j in range(rng.randint(case["draft_lo"], case["draft_hi"]))]
            for _ in range(case["batch"])]


def masks_of(parents):
    """Bit j of a draft's mask: it sees draft j (its ancestors and itself)."""
    masks = []
    for j, par in enumerate(parents):
        masks.append((1 << j) | (masks[par] if par >= 0 else 0))
    return masks


def pages_of(tokens):
    return -(-tokens // PAGE)


def page_table(need, width, offset, gen):
    """Disjoint random pages of a pool, rows padded with -1; and the pages used."""
    perm = torch.randperm(sum(need), generator=gen) + offset
    table = torch.full((len(need), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n].int()
        at += n
    return table, at


# ------------------------------------------------------------------ states
def prepare(case, seed):
    return prepare_evict(case, seed) if case["op"] == "evict" else prepare_tree(case, seed)


def prepare_tree(case, seed):
    """A decode batch: queries of the drafts, caches that hold prefix and drafts, page tables, trees."""
    cpu = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gpu, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    prefix, parents = lengths(case), trees(case)
    count = [len(p) for p in parents]
    need = [pages_of(p + n) for p, n in zip(prefix, count)]
    table, pool = page_table(need, max(need), 0, cpu)
    total, heads = sum(count), case["heads"]
    bits = [m - (1 << 64) if m >= 1 << 63 else m for p in parents for m in masks_of(p)]
    cu = torch.tensor([0] + count).cumsum(0).int()
    s = {"op": case["op"], "heads": heads, "longest": max(p + n for p, n in zip(prefix, count)), "most": max(count),
         "q_nope": normal(total, heads, CKV), "q_pe": normal(total, heads, KPE),
         "ckv": normal(pool, PAGE, CKV), "kpe": normal(pool, PAGE, KPE),
         "prefix": torch.tensor(prefix, dtype=torch.int32).cuda(), "table": table.cuda(), "cu": cu.cuda(),
         "mask": torch.tensor(bits, dtype=torch.int64).reshape(-1, 1).cuda()}
    if case["op"] == "tree":
        s["out"] = torch.empty(total, heads, CKV, device="cuda", dtype=torch.bfloat16)
        s["lse"] = torch.empty(total, heads, device="cuda")
    else:
        s["lse"] = plain_tree(s)[1]
        s["acc"] = torch.rand(len(prefix), table.shape[1] * PAGE, generator=gpu, device="cuda")
        s["new"] = torch.empty_like(s["acc"])
    return s


def prepare_evict(case, seed):
    """Caches of a batch with heavy-tailed accumulated weights, many of them equal, and free pages for what is kept."""
    cpu = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device="cuda").manual_seed(seed)
    seq = lengths(case)
    need = [pages_of(n) for n in seq]
    table, used = page_table(need, max(need), 0, cpu)
    fresh = [pages_of(min(n, case["budget"])) for n in seq]
    new_table, more = page_table(fresh, pages_of(case["budget"]), used, cpu)
    pool, wide = used + more, table.shape[1] * PAGE
    acc = torch.randn(len(seq), wide, generator=gpu, device="cuda").mul_(2).exp_()
    acc[torch.rand(len(seq), wide, generator=gpu, device="cuda") < 0.3] = 0
    return {"op": "evict", "budget": case["budget"], "sink": case["sink"], "recent": case["recent"], "acc": acc,
            "seq": torch.tensor(seq, dtype=torch.int32).cuda(), "table": table.cuda(), "new_table": new_table.cuda(),
            "ckv": torch.randn(pool, PAGE, CKV, generator=gpu, device="cuda", dtype=torch.bfloat16),
            "kpe": torch.randn(pool, PAGE, KPE, generator=gpu, device="cuda", dtype=torch.bfloat16),
            "index": torch.randint(0, 256, (pool, PAGE, 1, IDX), generator=gpu, device="cuda", dtype=torch.uint8),
            "keep": torch.empty(len(seq), case["budget"], dtype=torch.int32, device="cuda"),
            "new_seq": torch.empty(len(seq), dtype=torch.int32, device="cuda"),
            "new_acc": torch.empty(len(seq), new_table.shape[1] * PAGE, device="cuda")}


# ------------------------------------------------------------------ passes
def run(s):
    if s["op"] == "tree":
        if own:
            from dsa_b200 import tree
            tree.run(s["q_nope"], s["q_pe"], s["ckv"], s["kpe"], s["prefix"], s["table"], s["cu"], s["mask"], SCALE,
                     s["out"], s["lse"])
            return {"out": s["out"], "lse": s["lse"]}
        out, lse = plain_tree(s)
        return {"out": out, "lse": lse}
    if s["op"] == "weights":
        if own:
            from dsa_b200 import evict
            evict.accumulate(s["q_nope"], s["q_pe"], s["ckv"], s["kpe"], s["prefix"], s["table"], s["cu"], s["mask"],
                             SCALE, s["lse"], s["acc"], s["new"])
            return {"acc": s["new"]}
        return {"acc": plain_weights(s)}
    if own:
        from dsa_b200 import evict
        evict.run(s["acc"], s["seq"], s["table"], s["new_table"], s["ckv"], s["kpe"], s["index"], s["sink"], s["recent"],
                  s["keep"], s["new_seq"], s["new_acc"])
        return {"keep": s["keep"], "new_seq": s["new_seq"], "new_acc": s["new_acc"], "ckv": s["ckv"], "kpe": s["kpe"],
                "index": s["index"]}
    return plain_evict(s)


def plain_logits(s):
    """(keys [B, longest, 576], base-2 logits [B, most * heads, longest] with -inf where masked, row map)."""
    table, prefix, cu = s["table"].long(), s["prefix"].long(), s["cu"].long()
    B, longest, most, heads = table.shape[0], s["longest"], s["most"], s["heads"]
    count = cu[1:] - cu[:-1]
    pos = torch.arange(longest, device="cuda")
    slot = table[:, pos // PAGE].clamp(min=0) * PAGE + pos % PAGE
    keys = torch.cat([s["ckv"].reshape(-1, CKV)[slot], s["kpe"].reshape(-1, KPE)[slot]], -1).float()
    draft = torch.arange(most, device="cuda")
    row = (cu[:-1, None] + draft).clamp(max=cu[-1] - 1)
    real = draft < count[:, None]
    q = torch.cat([s["q_nope"], s["q_pe"]], -1)[row].float().reshape(B, most * heads, CKV + KPE)
    x = torch.bmm(q, keys.transpose(1, 2)).mul_(SCALE * LOG2E)
    j = pos - prefix[:, None]
    bit = (s["mask"][row, 0][:, :, None] >> j.clamp(0, 63)[:, None, :]) & 1
    seen = (j[:, None, :] < 0) | ((j[:, None, :] < count[:, None, None]) & (bit != 0))
    seen &= real[:, :, None]
    x.view(B, most, heads, longest).masked_fill_(~seen[:, :, None, :], -math.inf)
    back = torch.repeat_interleave(torch.arange(B, device="cuda"), count, output_size=s["q_nope"].shape[0])
    return keys, x, (back, torch.arange(s["q_nope"].shape[0], device="cuda") - cu[back])


def plain_tree(s):
    keys, x, (req, draft) = plain_logits(s)
    B, longest, most, heads = x.shape[0], s["longest"], s["most"], s["heads"]
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = x.sub_(top).exp2_()
    total = e.sum(-1, keepdim=True)
    out = torch.bmm(e, keys[:, :, :CKV]) / torch.where(total == 0, 1.0, total)
    lse = (top + total.log2()).reshape(B, most, heads)
    return out.reshape(B, most, heads, CKV)[req, draft].bfloat16(), lse[req, draft].contiguous()


def plain_weights(s):
    keys, x, (req, draft) = plain_logits(s)
    B, longest, most, heads = x.shape[0], s["longest"], s["most"], s["heads"]
    lse = torch.zeros(B, most, heads, device="cuda")
    lse[req, draft] = s["lse"]
    lse = lse.reshape(B, most * heads, 1)
    w = x.sub_(torch.where(lse == -math.inf, 0.0, lse)).exp2_()
    new = s["acc"].clone()
    new[:, :longest] += w.sum(1)
    return new


def plain_evict(s):
    acc, seq, budget = s["acc"], s["seq"].long()[:, None], s["budget"]
    pos = torch.arange(acc.shape[1], device="cuda")
    rank = torch.where((pos < s["sink"]) | (pos >= seq - s["recent"]), math.inf, acc)
    rank = torch.where(pos < seq, rank, -math.inf)
    best = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :budget]
    if best.shape[1] < budget:
        best = torch.cat([best, best.new_full((best.shape[0], budget - best.shape[1]), 1 << 30)], 1)
    best = torch.where(best < seq, best, 1 << 30).sort(dim=1).values
    kept = best < (1 << 30)
    keep = torch.where(kept, best, -1)
    new_acc = torch.zeros_like(s["new_acc"])
    new_acc[:, :budget] = torch.where(kept, acc.gather(1, keep.clamp(min=0)), 0.0)
    to = torch.arange(budget, device="cuda")
    src = (s["table"].long().gather(1, keep.clamp(min=0) // PAGE) * PAGE + keep.clamp(min=0) % PAGE)[kept]
    dst = (s["new_table"].long()[:, to // PAGE] * PAGE + to % PAGE)[kept]
    ckv, kpe = s["ckv"].view(-1, CKV), s["kpe"].view(-1, KPE)
    ckv[dst] = ckv[src]
    kpe[dst] = kpe[src]
    index = s["index"].view(s["index"].shape[0], PAGE * IDX)
    keys = index[:, :PAGE * 128].unflatten(1, (PAGE, 128))
    keys[dst // PAGE, dst % PAGE] = keys[src // PAGE, src % PAGE]
    scales = index[:, PAGE * 128:].unflatten(1, (PAGE, 4))
    scales[dst // PAGE, dst % PAGE] = scales[src // PAGE, src % PAGE]
    return {"keep": keep.int(), "new_seq": kept.sum(1).int(), "new_acc": new_acc, "ckv": s["ckv"], "kpe": s["kpe"],
            "index": s["index"]}


# ------------------------------------------------------------------ work
def work(case):
    if case["op"] == "evict":
        seq = lengths(case)
        kept = sum(min(n, case["budget"]) for n in seq)
        judged = sum(n for n in seq if n > case["budget"])  # a request within its budget is kept whole
        rows = len(seq) * (4 * case["budget"] + 4 * PAGE * pages_of(case["budget"]))
        return {"bytes": kept * (2 * (2 * (CKV + KPE) + IDX) + 4) + 4 * judged + rows, "flops": 0}
    heads = case["heads"]
    tokens = rows = pairs = 0
    for p, parents in zip(lengths(case), trees(case)):
        tokens += p + len(parents)
        rows += len(parents) * heads
        pairs += heads * sum(p + bin(m).count("1") for m in masks_of(parents))
    if case["op"] == "tree":
        return {"bytes": 2 * (CKV + KPE) * (tokens + rows) + rows * (2 * CKV + 4), "flops": 2 * pairs * (2 * CKV + KPE)}
    return {"bytes": 2 * (CKV + KPE) * (tokens + rows) + rows * 4 + 8 * tokens, "flops": 2 * pairs * (CKV + KPE)}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] == "evict":
        return exact_evict(prepare(case, seed))
    s = prepare(case, seed)
    cu, prefix, table = s["cu"].tolist(), s["prefix"].tolist(), s["table"]
    flat = torch.cat([s["ckv"].reshape(-1, CKV), s["kpe"].reshape(-1, KPE)], 1)
    outs, lses, new = [], [], None
    if case["op"] == "weights":
        new = s["acc"].double()
    for b in range(len(prefix)):
        n, p, H = cu[b + 1] - cu[b], prefix[b], s["heads"]
        where = torch.arange(p + n, device="cuda")
        k = flat[table[b].long()[where // PAGE] * PAGE + where % PAGE].double()
        q = torch.cat([s["q_nope"][cu[b]:cu[b + 1]], s["q_pe"][cu[b]:cu[b + 1]]], -1).double().flatten(0, 1)
        see = torch.ones(n, p + n, dtype=torch.bool)
        for i, m in enumerate(s["mask"][cu[b]:cu[b + 1], 0].tolist()):
            see[i, p:] = torch.tensor([bool((m >> j) & 1) for j in range(n)])
        see = see.cuda().repeat_interleave(H, 0)
        for lo in range(0, n * H, 64):
            x = (q[lo:lo + 64] @ k.T) * SCALE
            x = x.masked_fill(~see[lo:lo + 64], -math.inf)
            if new is None:
                lses.append(torch.logsumexp(x, 1) * LOG2E)
                outs.append(torch.softmax(x, 1) @ k[:, :CKV])
            else:
                given = s["lse"][cu[b]:cu[b + 1]].reshape(-1, 1)[lo:lo + 64].double()
                new[b, :p + n] += torch.exp(x - given / LOG2E).sum(0)
    if new is not None:
        return {"acc": new}
    return {"out": torch.cat(outs).reshape(-1, s["heads"], CKV), "lse": torch.cat(lses).reshape(-1, s["heads"])}


def exact_evict(s):
    """Request by request: the positions ordered by (protected, weight, earlier first), then rows moved one gather each."""
    acc, budget = s["acc"].double().cpu(), s["budget"]
    new_acc = torch.zeros(s["new_acc"].shape, dtype=torch.float64)
    ckv, kpe = s["ckv"].view(-1, CKV).double(), s["kpe"].view(-1, KPE).double()
    for b, n in enumerate(s["seq"].tolist()):
        keep = list(range(n))
        if n > budget:
            weight = acc[b, :n].tolist()
            middle = sorted(range(s["sink"], n - s["recent"]), key=lambda i: (-weight[i], i))
            keep = sorted([*range(s["sink"]), *middle[:budget - s["sink"] - s["recent"]], *range(n - s["recent"], n)])
        keep = torch.tensor(keep)
        new_acc[b, :len(keep)] = acc[b, keep]
        to = torch.arange(len(keep))
        src = (s["table"][b].cpu().long()[keep // PAGE] * PAGE + keep % PAGE).cuda()
        dst = (s["new_table"][b].cpu().long()[to // PAGE] * PAGE + to % PAGE).cuda()
        ckv[dst] = ckv[src]
        kpe[dst] = kpe[src]
    return {"keep": None, "new_seq": None, "new_acc": new_acc.cuda(), "ckv": ckv.view(s["ckv"].shape),
            "kpe": kpe.view(s["kpe"].shape), "index": None}
