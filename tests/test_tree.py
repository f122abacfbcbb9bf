"""CPU tests of tree attention and weight accumulation: the C ABI's and the
Python entry points' refusals, and the mask helper."""

import ctypes

import pytest
import torch

from dsa_b200 import _native, evict, tree

P = ctypes.c_void_p


def call(lib, requests=1, drafts=2, heads=16, max_pages=4, words=1, pages=3, q=16, ckv=16, ckv_page=65536, ckv_row=1024,
         kpe_page=8192, kpe_row=128, mask=16, ws=16, nbytes=1 << 30, out=16):
    return lib.dsa_tree_attention_run(P(q), P(16), P(ckv), ckv_page, ckv_row, P(16), kpe_page, kpe_row, pages, P(16), P(16),
                                      P(16), P(mask), requests, drafts, heads, max_pages, words, 0.1, P(out), P(16), P(ws),
                                      nbytes, None)


@pytest.mark.parametrize("change,status", [
    (dict(requests=-1), 1), (dict(drafts=-1), 1), (dict(heads=0), 1), (dict(heads=129), 1), (dict(requests=65537), 1),
    (dict(drafts=0), 0), (dict(requests=0), 0), (dict(q=None), 1), (dict(ws=None), 1), (dict(out=None), 1),
    (dict(pages=0), 1), (dict(max_pages=0), 1), (dict(words=0), 1), (dict(words=65), 1), (dict(ckv_row=512), 1),
    (dict(ckv=8), 2), (dict(ckv_page=65528), 2), (dict(kpe_row=136), 2), (dict(mask=20), 2), (dict(out=8), 2),
    (dict(max_pages=1 << 24, drafts=1 << 16), 1), (dict(drafts=(1 << 20) + 1), 1), (dict(max_pages=(1 << 24) + 1), 1),
])
def test_c_abi_refuses_bad_arguments(change, status):
    assert call(_native.lib(), **change) == status


def test_workspace_is_the_same_for_every_call():
    # without a GPU: two records of 64 rows for each of 160 SMs, and the groups of the largest call
    records, groups = 2 * 160 * 64 * (512 + 4) * 4, 2 * (2 ** 24 // 64 + 65536) * 4
    assert _native.lib().dsa_tree_attention_workspace_bytes() >= 256 + records * 148 // 160 + groups


def test_masks_from_parents():
    rows = tree.masks_from_parents([-1, 0, 0, 2, -1])
    assert rows == [[0b1], [0b11], [0b101], [0b1101], [0b10000]]
    chain = tree.masks_from_parents(list(range(-1, 69)))
    assert len(chain[0]) == 2 and chain[63] == [-1, 0] and chain[69] == [-1, 63]
    with pytest.raises(ValueError):
        tree.masks_from_parents([-1, 1])
    assert tree.masks_from_parents([]) == []


def test_entry_points_refuse_cpu_tensors():
    a = dict(q_nope=torch.zeros(1, 16, 512), q_pe=torch.zeros(1, 16, 64), ckv_cache=torch.zeros(1, 64, 512),
             kpe_cache=torch.zeros(1, 64, 64), prefix_lens=torch.zeros(1), block_table=torch.zeros(1, 1),
             cu_drafts=torch.zeros(2), tree_mask=torch.zeros(1, 1), sm_scale=0.1)
    with pytest.raises(ValueError, match="CUDA"):
        tree.run(**a, output=torch.zeros(1), lse=torch.zeros(1))
    with pytest.raises(ValueError, match="CUDA"):
        evict.accumulate(**a, lse=torch.zeros(1), acc=torch.zeros(1), out=torch.zeros(1))


def test_cache_strides():
    def fail(msg):
        raise ValueError(msg)

    both = torch.zeros(3, 64, 576, dtype=torch.bfloat16)
    assert tree._strides("ckv", both[:, :, :512], 512, fail) == (3, 2 * 64 * 576, 2 * 576)
    assert tree._strides("kpe", both[:, :, 512:], 64, fail) == (3, 2 * 64 * 576, 2 * 576)
    assert tree._strides("ckv", both[:1, :, :512], 512, fail) == (1, 2 * 64 * 576, 2 * 576)
    for bad in (both[:, :, 4:516], both[:, :, :511], torch.zeros(3, 64, 580, dtype=torch.bfloat16)[:, :, :512],
                both[:, :, :512].transpose(0, 1), both[:0, :, :512], both[:1, :, :512].expand(3, 64, 512),
                both.flatten(0, 1)[:, :512]):
        with pytest.raises(ValueError):
            tree._strides("ckv", bad, 512, fail)


def evict_call(lib, requests=1, max_pages=4, new_pages=2, pages=9, budget=100, sink=4, recent=8, acc=16, acc_stride=256,
               new_stride=128, ckv=16, ckv_row=1024, index=16, keep=16, nbytes=256):
    return lib.dsa_cache_evict_run(P(acc), acc_stride, P(16), P(16), P(16), requests, max_pages, new_pages, P(ckv), 65536,
                                   ckv_row, P(16), 8192, 128, P(index), pages, budget, sink, recent, P(keep), P(16), P(16),
                                   new_stride, P(16), nbytes, None)


@pytest.mark.parametrize("change,status", [
    (dict(requests=-1), 1), (dict(requests=0), 0), (dict(requests=65537), 1), (dict(acc=None), 1), (dict(keep=None), 1),
    (dict(budget=0), 1), (dict(budget=129), 1), (dict(sink=-1), 1), (dict(sink=60, recent=41), 1), (dict(pages=0), 1),
    (dict(max_pages=0), 1), (dict(acc_stride=255), 1), (dict(new_stride=127), 1), (dict(ckv_row=1000), 1),
    (dict(ckv_row=1032), 2), (dict(ckv=8), 2), (dict(index=8), 2), (dict(acc=18), 2), (dict(nbytes=255), 3),
])
def test_evict_c_abi_refuses_bad_arguments(change, status):
    assert evict_call(_native.lib(), **change) == status


@pytest.mark.parametrize("change,status", [
    (dict(lse=None), 1), (dict(acc=18), 2), (dict(stride=100), 1), (dict(out=16, out_stride=300), 1), (dict(requests=0), 0),
])
def test_weights_c_abi_refuses_bad_arguments(change, status):
    a = dict(lse=16, acc=16, stride=256, out=32, out_stride=256, requests=1) | change
    assert _native.lib().dsa_tree_weights_run(
        P(16), P(16), P(16), 65536, 1024, P(16), 8192, 128, 3, P(16), P(16), P(16), P(16), a["requests"], 2, 16, 4, 1, 0.1,
        P(a["lse"]), P(a["acc"]), a["stride"], P(a["out"]), a["out_stride"], P(16), 256, None) == status


def test_overlapping_accumulators():
    buf = torch.zeros(1000)
    rows = lambda at, n, width, pitch: buf[at:].as_strided((n, width), (pitch, 1))  # noqa: E731
    a = rows(0, 4, 64, 150)
    assert not evict._overlap(a, rows(64, 4, 64, 150)) and not evict._overlap(rows(64, 4, 64, 150), a)
    assert not evict._overlap(a, rows(514, 2, 64, 64))       # behind the last row
    assert evict._overlap(a, rows(1, 4, 64, 150))
    assert evict._overlap(a, rows(100, 4, 64, 150))          # wraps into the next row
    assert evict._overlap(a, rows(64, 4, 64, 151))
    assert evict._overlap(a, rows(513, 2, 64, 64))
    assert not evict._overlap(rows(0, 1, 64, 7), rows(64, 1, 64, 7))


def test_evict_oracle():
    from oracle import tree as otree
    acc = torch.tensor([[3.0, 1.0, 2.0, 2.0, 0.0, 9.0], [float("nan"), 1, 5, 5, 5, 0]])
    assert otree.evict_reference(acc, torch.tensor([6, 5]), 3, 1, 1) == [[0, 2, 5], [0, 2, 4]]
    assert otree.evict_reference(acc, torch.tensor([6, 3]), 3, 0, 0) == [[0, 2, 5], [0, 1, 2]]
