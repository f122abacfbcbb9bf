"""Every operator called first thing from a host thread that has made no CUDA
call yet: the same results as from the main thread."""

import threading

import pytest
import torch

from dsa_b200 import attention, evict, indexer, tree, workloads

pytestmark = pytest.mark.gpu


def in_new_thread(call):
    errors = []

    def body():
        try:
            call()
        except Exception as e:  # noqa: BLE001  raised below, in the test's own thread
            errors.append(e)

    t = threading.Thread(target=body)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not errors, errors


@pytest.fixture(autouse=True)
def no_waits(monkeypatch):
    # The check after a call is the runtime's; the operator itself has to be the thread's first call.
    for module in (attention, indexer, tree):
        monkeypatch.setattr(module, "_CHECK", False)


def twice(call, outs):
    call()
    torch.cuda.synchronize()
    want = [t.clone() for t in outs]
    for t in outs:
        t.zero_()
    torch.cuda.synchronize()
    in_new_thread(call)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_indexer_and_attention(cuda_device):
    dec = workloads.make_decode_inputs([3000, 700, 65], seed=81, device=cuda_device)
    ix = dec.indexer
    topk = torch.full((3, 2048), 7, dtype=torch.int32, device=cuda_device)
    twice(lambda: indexer.run(ix.q_index_fp8, ix.k_index_cache_fp8, ix.weights, ix.seq_lens, ix.block_table, topk), [topk])
    out, lse = torch.zeros(3, 16, 512, dtype=torch.bfloat16, device=cuda_device), torch.zeros(3, 16, device=cuda_device)
    twice(lambda: attention.run(dec.q_nope, dec.q_pe, dec.ckv_cache, dec.kpe_cache, topk, dec.sm_scale, out, lse), [out, lse])


def test_prefill_indexer(cuda_device):
    pf = workloads.make_prefill_inputs([2500, 40], [4, 2], seed=82, device=cuda_device)
    topk = torch.zeros(6, 2048, dtype=torch.int32, device=cuda_device)
    twice(lambda: indexer.run_prefill(pf.q_index_fp8, pf.k_index_cache_fp8, pf.weights, pf.seq_lens, pf.block_table,
                                      pf.cu_seqlens_q, topk), [topk])


def test_tree_weights_and_eviction(cuda_device):
    dec = workloads.make_decode_inputs([900, 1300], seed=83, device=cuda_device, pool_pages=64)
    bt = dec.indexer.block_table
    prefix = torch.tensor([890, 1290], dtype=torch.int32, device=cuda_device)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device)
    mask = torch.ones(2, 1, dtype=torch.int64, device=cuda_device)
    out, lse = torch.zeros(2, 16, 512, dtype=torch.bfloat16, device=cuda_device), torch.zeros(2, 16, device=cuda_device)
    rows = (dec.q_nope, dec.q_pe, dec.ckv_cache, dec.kpe_cache, prefix, bt, cu, mask, dec.sm_scale)
    twice(lambda: tree.run(*rows, out, lse), [out, lse])
    acc = torch.zeros(2, bt.shape[1] * 64, device=cuda_device)
    new = torch.zeros_like(acc)
    twice(lambda: evict.accumulate(*rows, lse, acc, new), [new])
    used = {int(x) for x in bt.flatten() if x >= 0}
    fresh = torch.tensor([x for x in range(64) if x not in used][:10], dtype=torch.int32, device=cuda_device).reshape(2, 5)
    keep, lens = torch.zeros(2, 300, dtype=torch.int32, device=cuda_device), torch.zeros(2, dtype=torch.int32, device=cuda_device)
    new2, seq = torch.zeros(2, 320, device=cuda_device), prefix + 1
    twice(lambda: evict.run(new, seq, bt, fresh, dec.ckv_cache, dec.kpe_cache, None, 4, 32, keep, lens, new2),
          [keep, lens, new2])


def test_two_threads_of_indexer_calls_on_one_stream(cuda_device):
    """A call's launches hand histograms and scores on through the stream's
    workspace: another thread's must not come between them."""
    ix = [workloads.make_indexer_inputs(lens, pool_pages=256, seed=84 + k, device=cuda_device)
          for k, lens in enumerate(([5000, 2500, 70], [3000, 9000, 2049]))]
    pf = [workloads.make_prefill_inputs([2500 + 300 * k, 40], [4, 2], seed=86 + k, device=cuda_device) for k in range(2)]
    topk = [[torch.zeros(n, 2048, dtype=torch.int32, device=cuda_device) for _ in range(101)] for n in (3, 3, 6, 6)]

    def decode(k, out):
        i = ix[k]
        indexer.run(i.q_index_fp8, i.k_index_cache_fp8, i.weights, i.seq_lens, i.block_table, out)

    def prefill(k, out):
        p = pf[k]
        indexer.run_prefill(p.q_index_fp8, p.k_index_cache_fp8, p.weights, p.seq_lens, p.block_table, p.cu_seqlens_q, out)

    for k in range(2):
        decode(k, topk[k][0])
        prefill(k, topk[2 + k][0])
    torch.cuda.synchronize()
    start, errors = threading.Barrier(2), []

    def calls(k):
        try:
            start.wait()
            for n in range(1, 101):
                decode(k, topk[k][n])
                prefill(k, topk[2 + k][n])
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=calls, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert indexer.device_status(cuda_device) == 0
    for rows in topk:
        assert all(torch.equal(t, rows[0]) for t in rows[1:])
