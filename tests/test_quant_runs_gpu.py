"""The 8-bit latent cache's operators together, as a serving loop calls them:
prompts written and read back, decode steps of drafts with their verification,
the indexer's selection; and where single calls rarely go: pages behind 4 GB,
threads, streams and graphs at once."""

import math
import threading

import pytest
import torch

from dsa_b200 import attention, cache, indexer, quant, tree, verify, workloads
from oracle import quant as oq
from oracle import verify as ov
from test_quant import angles, kv_rows
from test_quant_attention_gpu import Dense, cache_of, compare, run, sparse_case

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(192.0)


def test_a_serving_loop(cuda_device):
    """Two requests: prompts written, read back in part for the next chunk, then steps of a chain of drafts: written, attended
    to, verified; what the path says stays in the cache."""
    g = torch.Generator().manual_seed(5)
    lens, heads, vocab = [150, 321], 16, 500
    table = torch.tensor([[7, 3, 0, 10, -1, -1], [1, 9, 4, 2, 8, 6]], dtype=torch.int32)
    w, cos_sin = (1 + 0.2 * torch.randn(512, generator=g)).bfloat16(), angles(400)
    store = torch.zeros(11, quant.PAGE_BYTES, dtype=torch.uint8, device=cuda_device)
    host = store.cpu().clone()
    slot = lambda b, pos: table[b].long()[pos // 64] * 64 + pos % 64  # noqa: E731

    def write(b, first, n, seed):
        kv, pos = kv_rows(n, seed, spread=1), torch.arange(first, first + n)
        quant.write(kv.to(cuda_device), slot(b, pos).to(cuda_device), store, w.to(cuda_device), 1e-6, pos.to(cuda_device),
                    cos_sin.to(cuda_device))
        code, scale, e = oq.write_rows(kv, w, 1e-6, pos, cos_sin)
        codes, kpe, scales = oq.pieces(host)
        codes[slot(b, pos) // 64, slot(b, pos) % 64] = code
        kpe[slot(b, pos) // 64, slot(b, pos) % 64] = e.float().bfloat16()
        scales[slot(b, pos) // 64, slot(b, pos) % 64] = scale.float()

    for b, n in enumerate(lens):
        write(b, 0, n, 10 + b)
    back = torch.zeros(40, 576, dtype=torch.bfloat16, device=cuda_device)
    quant.read(store, table.to(cuda_device), torch.tensor([100, 0], device=cuda_device), torch.tensor([0, 40, 40], device=cuda_device),
               back[:, :512], back[:, 512:])
    c, e = oq.rows(host, slot(0, 100 + torch.arange(40)))
    assert ((back[:, :512].cpu().double() - c).abs() <= 2.0 ** -7 * c.abs() + 1e-6).all()
    for step in range(3):
        count = [3, 4]
        for b in range(2):
            write(b, lens[b], count[b], 100 + 10 * step + b)
        seq = torch.tensor([n + k for n, k in zip(lens, count)], dtype=torch.int32)
        cu = torch.tensor([0, 3, 7], dtype=torch.int32)
        qn, qp = torch.randn(7, heads, 512, generator=g).bfloat16(), torch.randn(7, heads, 64, generator=g).bfloat16()
        out, lse = torch.zeros(7, heads, 512, dtype=torch.bfloat16, device=cuda_device), torch.zeros(7, heads, device=cuda_device)
        quant.attend(*[t.to(cuda_device) for t in (qn, qp)], store, seq.to(cuda_device), table.to(cuda_device), cu.to(cuda_device), SCALE,
                     out, lse)
        ro, rl, bo, bl = oq.attend_reference(qn, qp, store.cpu(), seq, table, cu, SCALE)
        compare(out, lse, ro, rl, bo, bl)
        # a model of one layer: its logits are a fixed projection of the outputs
        head = torch.randn(heads * 512, vocab, generator=torch.Generator().manual_seed(3)).to(cuda_device) * 0.02
        target = torch.softmax(out.float().flatten(1) @ head, 1)
        draft = torch.softmax(target.log() + 0.3 * torch.randn(7, vocab, generator=g).to(cuda_device), 1)
        tokens = torch.multinomial(draft.cpu(), 1, generator=g)[:, 0].roll(1)
        parents = torch.tensor([-1, 0, 1, -1, 0, 1, 2])
        u, s = torch.rand(7, generator=g), torch.rand(2, generator=g)
        got = [torch.zeros(2, 3, dtype=torch.int32, device=cuda_device), torch.zeros(2, dtype=torch.int32, device=cuda_device),
               torch.zeros(2, dtype=torch.int32, device=cuda_device)]
        verify.run(target, draft, *[t.to(cuda_device) for t in (tokens, parents, cu, u, s)], *got)
        want = ov.verify_reference(target.cpu(), draft.cpu(), tokens, parents, cu, u, s, 3)
        assert [x.tolist() for x in got] == list(want)
        lens = [n + 1 + a for n, a in zip(lens, want[1])]  # the certain token and the accepted drafts
    same = store.cpu()
    for a, b in zip(oq.pieces(same), oq.pieces(host)):
        assert torch.allclose(a.double(), b.double(), rtol=2.0 ** -7, atol=1e-6)
    assert torch.equal(oq.pieces(same)[0], oq.pieces(host)[0])


def test_indexer_selects_and_attention_reads(cuda_device):
    """One graph: new tokens into both caches, the indexer's selection, attention over it; against the bf16 attention of the
    rows read back, and the oracle."""
    lens = [3000, 700, 65]
    dec = workloads.make_decode_inputs(lens, seed=81, device=cuda_device)
    ix, bt = dec.indexer, dec.indexer.block_table
    pool = dec.ckv_cache.shape[0]
    store = torch.zeros(pool, quant.PAGE_BYTES, dtype=torch.uint8, device=cuda_device)
    every = torch.arange(pool * 64, device=cuda_device)
    quant.write(torch.cat([dec.ckv_cache.reshape(-1, 512), dec.kpe_cache.reshape(-1, 64)], 1), every, store)
    topk = torch.zeros(3, 2048, dtype=torch.int32, device=cuda_device)
    out, lse = torch.zeros(3, 16, 512, dtype=torch.bfloat16, device=cuda_device), torch.zeros(3, 16, device=cuda_device)
    new, keys = kv_rows(3, 9, spread=1).to(cuda_device), torch.randn(3, 128, device=cuda_device).bfloat16()
    slots = torch.tensor([int(bt[b, (n - 1) // 64]) * 64 + (n - 1) % 64 for b, n in enumerate(lens)], device=cuda_device)

    def step():
        cache.write_index_k(keys, slots, ix.k_index_cache_fp8)
        quant.write(new, slots, store)
        indexer.run(ix.q_index_fp8, ix.k_index_cache_fp8, ix.weights, ix.seq_lens, bt, topk)
        quant.attend_sparse(dec.q_nope, dec.q_pe, store, topk, dec.sm_scale, out, lse)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        out.zero_()
        graph.replay()
    torch.cuda.synchronize()
    compare(out, lse, *oq.sparse_reference(dec.q_nope.cpu(), dec.q_pe.cpu(), store.cpu(), topk.cpu(), dec.sm_scale))
    ckv = torch.zeros(pool * 64, 512, dtype=torch.bfloat16, device=cuda_device)
    kpe = torch.zeros(pool * 64, 64, dtype=torch.bfloat16, device=cuda_device)
    quant.read(store, torch.arange(pool, device=cuda_device)[None], torch.zeros(1, device=cuda_device).int(),
               torch.tensor([0, pool * 64], device=cuda_device), ckv, kpe)
    o2, l2 = torch.zeros_like(out), torch.zeros_like(lse)
    attention.run(dec.q_nope, dec.q_pe, ckv.view(pool, 64, 512), kpe.view(pool, 64, 64), topk, dec.sm_scale, o2, l2)
    assert torch.allclose(lse, l2, atol=2e-2, rtol=0) and torch.allclose(out.float(), o2.float(), atol=2e-2, rtol=2e-2)
    # a context within the selection: dense attention is the same function
    o3, l3 = torch.zeros_like(out), torch.zeros_like(lse)
    quant.attend(dec.q_nope, dec.q_pe, store, ix.seq_lens, bt, None, dec.sm_scale, o3, l3)
    assert torch.allclose(lse[1:], l3[1:], atol=1e-4, rtol=0) and torch.allclose(out[1:].float(), o3[1:].float(), atol=1e-2, rtol=1e-2)


def test_pages_behind_4_gb(cuda_device):
    """Offsets that pass 32 bits: a pool of 110000 pages (4.5 GB), written, read and attended to at its end."""
    pages = 110000
    store = torch.zeros(pages, quant.PAGE_BYTES, dtype=torch.uint8, device=cuda_device)
    n = 300
    table = torch.tensor([[pages - 1, 3, pages - 7, pages // 2, pages - 2]], dtype=torch.int32)
    pos = torch.arange(n)
    slots = table[0].long()[pos // 64] * 64 + pos % 64
    kv = kv_rows(n, 4, spread=1)
    quant.write(kv.to(cuda_device), slots.to(cuda_device), store)
    # the same tokens in a small pool
    small = torch.zeros(5, quant.PAGE_BYTES, dtype=torch.uint8, device=cuda_device)
    near = torch.arange(5, dtype=torch.int32)[None]
    quant.write(kv.to(cuda_device), pos.to(cuda_device), small)
    for far_page, page in zip(table[0].tolist(), range(5)):
        assert torch.equal(store[far_page], small[page])
    g = torch.Generator().manual_seed(6)
    qn, qp = torch.randn(1, 16, 512, generator=g).bfloat16().cuda(), torch.randn(1, 16, 64, generator=g).bfloat16().cuda()
    seq = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    results = []
    for cache_, t, s in ((store, table, slots), (small, near, pos)):
        t = t.to(cuda_device)
        ckv, kpe = torch.zeros(n, 512, dtype=torch.bfloat16, device=cuda_device), torch.zeros(n, 64, dtype=torch.bfloat16, device=cuda_device)
        quant.read(cache_, t, torch.zeros(1, dtype=torch.int32, device=cuda_device), torch.tensor([0, n], device=cuda_device), ckv, kpe)
        outs = [ckv, kpe]
        for call in (lambda o, l: quant.attend(qn, qp, cache_, seq, t, None, SCALE, o, l),  # noqa: B023
                     lambda o, l: quant.attend_sparse(qn, qp, cache_, s[None].to(cuda_device), SCALE, o, l)):  # noqa: B023
            o, l = torch.zeros(1, 16, 512, dtype=torch.bfloat16, device=cuda_device), torch.zeros(1, 16, device=cuda_device)
            call(o, l)
            outs += [o, l]
        results.append(outs)
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_probabilities_behind_4_gb(cuda_device):
    vocab, rows = 1 << 20, 1100  # 4.6 GB each
    target = torch.zeros(rows, vocab, device=cuda_device)
    target[-3:] = torch.softmax(torch.randn(3, vocab, generator=torch.Generator().manual_seed(1)), 1).cuda()
    cu = torch.tensor([0, rows - 3, rows], dtype=torch.int32)
    tokens, parents = torch.zeros(rows, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
    parents[rows - 3:] = torch.tensor([-1, 0, 1])
    parents[:rows - 3] = -1
    tokens[rows - 2] = int(target[-3].argmax())
    u, s = torch.full((rows,), 0.9), torch.tensor([0.5, 0.37])
    got = [torch.zeros(2, 3, dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda()]
    verify.run(target, None, *[t.cuda() for t in (tokens, parents, cu, u, s)], *got)
    want = ov.verify_reference(target[-3:].cpu(), None, tokens[-3:], parents[-3:], [0, 3], u[-3:], s[1:], 3)
    assert [x.tolist()[1] for x in got] == [w[0] for w in want] and int(got[2][0]) == -1


@pytest.mark.parametrize("seed", [0, 1])
def test_calls_back_to_back_on_two_streams(cuda_device, seed):
    """Dense and sparse calls of changing sizes one behind the other, without waits, on two streams: each as alone."""
    dense = [Dense([3000, 64, 700], [2, 1, 3], 16, seed=41), Dense([20], None, 16, seed=42), Dense([300] * 90, None, 32, seed=43)]
    sparse = [sparse_case(5, 16, 300, 9, 44), sparse_case(200, 16, 64, 9, 45)]
    want = [run(c) for c in dense]
    args = [c.args() for c in dense]
    picked = [[t.cuda() for t in c] for c in sparse]
    blank = lambda c: (torch.zeros(*c[0].shape, dtype=torch.bfloat16, device="cuda"), torch.zeros(*c[0].shape[:2], device="cuda"))  # noqa: E731
    for c in picked:
        o, l = blank(c)
        quant.attend_sparse(*c, SCALE, o, l)
        want.append((o, l))
    torch.cuda.synchronize()
    g = torch.Generator().manual_seed(seed)
    order = torch.randint(0, 5, (60,), generator=g).tolist()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for n, k in enumerate(order):
        with torch.cuda.stream(streams[n % 2]):
            o, l = dense[k].outs() if k < 3 else blank(picked[k - 3])
            if k < 3:
                quant.attend(*args[k], SCALE, o, l)
            else:
                quant.attend_sparse(*picked[k - 3], SCALE, o, l)
            got.append((k, o, l))
    torch.cuda.synchronize()
    for k, o, l in got:
        assert torch.equal(o, want[k][0]) and torch.equal(l, want[k][1])


def test_threads(cuda_device, monkeypatch):
    """Each operator first thing from a new host thread, and four threads on one stream: as from the main thread."""
    for module in (quant, verify, tree):
        monkeypatch.setattr(module, "_CHECK", False)
    c = Dense([3000, 64, 700], [2, 1, 3], 16, seed=51)
    args, (want, want_lse) = c.args(), run(c)
    case = [None if t is None else t.cuda() for t in ov.random_case(4, 8, 300, 2, False, 5)]
    kv, slots, store = kv_rows(90, 3).cuda(), torch.randperm(128)[:90].cuda(), torch.zeros(2, quant.PAGE_BYTES, dtype=torch.uint8).cuda()
    quant.write(kv, slots, store)
    first = [torch.zeros(4, 7, dtype=torch.int32).cuda(), *(torch.zeros(4, dtype=torch.int32).cuda() for _ in range(2))]
    verify.run(*case, *first)
    torch.cuda.synchronize()
    errors = []

    def body(times):
        try:
            for _ in range(times):
                o, l = c.outs()
                quant.attend(*args, SCALE, o, l)
                other, v = torch.zeros_like(store), [torch.zeros_like(t) for t in first]
                quant.write(kv, slots, other)
                verify.run(*case, *v)
                results.append((o, l, other, v))
        except Exception as e:  # noqa: BLE001  raised below
            errors.append(e)

    results = []
    for count, times in ((1, 1), (4, 25)):
        threads = [threading.Thread(target=body, args=(times,)) for _ in range(count)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
    assert not errors, errors
    for o, l, other, v in results:
        assert torch.equal(o, want) and torch.equal(l, want_lse) and torch.equal(other, store)
        assert all(torch.equal(a, b) for a, b in zip(v, first))


def test_largest_batches(cuda_device):
    """Thousands of requests of a token or two, and single rows whose groups outnumber the records."""
    c = Dense([1, 2, 0] * 1400, None, 1, seed=61)
    c.check(*run(c))
    c = Dense([65, 200] * 300, [1, 2] * 300, 16, seed=62)
    c.check(*run(c))


def test_all_pages_in_any_order_and_shared(cuda_device):
    """Requests that share pages, a page given twice in one context."""
    c = Dense([500, 500, 130], [2, 1, 1], 16, seed=63, hidden="")
    c.table[1, :8] = c.table[0, :8]
    c.table[2, :3] = c.table[2, 0]
    c.check(*run(c))
    many = cache_of(4, 3)
    assert many.shape[0] == 4
