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


def test_cache_layout():
    def fail(msg):
        raise ValueError(msg)

    both = torch.zeros(3, 64, 576, dtype=torch.bfloat16)
    ckv, kpe = both[:, :, :512], both[:, :, 512:]
    at = both.data_ptr()
    assert tree.cache_layout(fail, ckv, kpe) == (at, 2 * 64 * 576, 2 * 576, at + 1024, 2 * 64 * 576, 2 * 576, 3)
    one = tree.cache_layout(fail, ckv[:1], kpe[:1].contiguous())
    assert one[1:3] == (2 * 64 * 576, 2 * 576) and one[4:] == (2 * 64 * 64, 128, 1)
    wide = torch.zeros(3, 64, 580, dtype=torch.bfloat16)
    for bad in ((both[:, :, 4:516], kpe), (both[:, :, :511], kpe), (wide[:, :, :512], kpe), (ckv.transpose(0, 1), kpe),
                (ckv[:0], kpe[:0]), (ckv[:1].expand(3, 64, 512), kpe), (ckv.flatten(0, 1), kpe), (ckv, kpe[1:]),
                (ckv, kpe.half()), (ckv.float(), kpe), (ckv, both[:, :, 8:72]), (torch.zeros(()), kpe)):
        if bad[1].data_ptr() == at + 16:  # aligned, and allowed to lie within the other
            tree.cache_layout(fail, *bad)
            continue
        with pytest.raises(ValueError):
            tree.cache_layout(fail, *bad)


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
    o = lambda at, n, width, pitch, at2, width2, pitch2: evict._overlap(  # noqa: E731
        n, 4096 + 4 * at, pitch, width, 4096 + 4 * at2, pitch2, width2)
    assert not o(0, 4, 64, 150, 64, 64, 150) and not o(64, 4, 64, 150, 0, 64, 150)
    assert not o(0, 4, 64, 150, 514, 64, 64)       # behind the last row
    assert o(0, 4, 64, 150, 513, 64, 64)
    assert o(0, 4, 64, 150, 1, 64, 150)
    assert o(0, 4, 64, 150, 100, 64, 150)          # wraps into the next row
    assert o(0, 4, 64, 150, 64, 64, 151)
    assert o(0, 4, 64, 150, 64, 87, 150) and not o(0, 4, 64, 150, 64, 86, 150)
    assert not o(0, 1, 64, 64, 64, 64, 64) and o(0, 1, 64, 64, 63, 64, 64) and o(5, 2, 64, 64, 5, 64, 64)


def test_evict_oracle():
    from oracle import tree as otree
    acc = torch.tensor([[3.0, 1.0, 2.0, 2.0, 0.0, 9.0], [float("nan"), 1, 5, 5, 5, 0]])
    assert otree.evict_reference(acc, torch.tensor([6, 5]), 3, 1, 1) == [[0, 2, 5], [0, 2, 4]]
    assert otree.evict_reference(acc, torch.tensor([6, 3]), 3, 0, 0) == [[0, 2, 5], [0, 1, 2]]


def test_weights_of_accepted_drafts_alone():
    """Rows of rejected drafts are kept out by an lse of -inf; rows that are
    left out instead move the drafts behind them to other positions."""
    import math

    from oracle import tree as otree
    g = torch.Generator().manual_seed(1)
    normal = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    qn, qp, ckv, kpe = normal(4, 2, 512), normal(4, 2, 64), normal(2, 64, 512), normal(2, 64, 64)
    table = torch.tensor([[1, 0]])
    mask = torch.tensor(tree.masks_from_parents([-1, 0, 0, 0]))
    rest = (ckv, kpe, torch.tensor([70]), table)
    lse = otree.tree_reference(qn, qp, *rest, torch.tensor([0, 4]), mask, 0.05)[1]
    acc, accepted = torch.zeros(1, 128), torch.tensor([True, False, False, True])
    kept_out = torch.where(accepted[:, None], lse, -math.inf)
    new = otree.weights_reference(qn, qp, *rest, torch.tensor([0, 4]), mask, 0.05, kept_out, acc)[0]
    assert abs(float(new.sum()) - 4) < 1e-9 and float(new[0, 73]) > 0 and (new[0, 71:73] == 0).all()
    alone = otree.weights_reference(qn[accepted], qp[accepted], *rest, torch.tensor([0, 2]), mask[accepted], 0.05,
                                    lse[accepted], acc)[0]
    assert float(alone.sum()) < 4 - 1e-3


def test_masks_of_a_batch_have_the_words_of_its_largest_tree():
    small, large = [-1, 0, 0], list(range(-1, 69))
    rows = tree.masks_from_parents(small, words=2) + tree.masks_from_parents(large, words=2)
    assert torch.tensor(rows).shape == (73, 2)
    assert rows[:3] == [[1, 0], [3, 0], [5, 0]] and rows[3:] == tree.masks_from_parents(large)
    with pytest.raises(ValueError, match="2 words"):
        tree.masks_from_parents(large, words=1)


# name -> bytes, one behind the other: 3 requests of 4 pages, 5 drafts of 16 heads, one word of mask, 9 pages of cache
SIZES = {"q_nope": 5 * 16 * 1024, "q_pe": 5 * 16 * 128, "ckv": 9 * 65536, "kpe": 9 * 8192, "prefix": 12, "table": 48, "cu": 16,
         "pad": 4, "mask": 40, "lse": 5 * 16 * 4, "pad2": 8, "out": 5 * 16 * 1024, "acc": 3 * 4 * 256, "new": 3 * 4 * 256}
AT, _end = {}, 1 << 20
for _name, _bytes in SIZES.items():
    AT[_name] = _end
    _end += _bytes


def placed(entry, **where):
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up: no launch may follow")
    at = {k: P(v) for k, v in (AT | where).items()}
    rows = (at["q_nope"], at["q_pe"], at["ckv"], 65536, 1024, at["kpe"], 8192, 128, 9, at["prefix"], at["table"], at["cu"],
            at["mask"], 3, 5, 16, 4, 1, 0.1)
    if entry == "attention":
        return _native.lib().dsa_tree_attention_run(*rows, at["out"], at["lse"], P(16), 1 << 30, None)
    return _native.lib().dsa_tree_weights_run(*rows, at["lse"], at["acc"], 256, at["new"], 256, P(16), 256, None)


def test_outputs_beside_the_inputs_and_in_place_are_taken():
    known = (1, 2, 3, _native.DSA_ERR_OVERLAP)  # only the device is missing
    assert placed("attention") not in known and placed("attention", out=AT["q_nope"]) not in known
    assert placed("weights") not in known and placed("weights", new=AT["acc"]) not in known


@pytest.mark.parametrize("entry,out", [("attention", "out"), ("attention", "lse"), ("weights", "new")])
@pytest.mark.parametrize("other", ["q_nope", "q_pe", "ckv", "kpe", "prefix", "table", "cu", "mask", "lse", "acc"])
def test_outputs_over_inputs_are_refused(entry, out, other):
    if other == out or (other, entry) == ("acc", "attention"):
        pytest.skip("not an input of this call")
    step = 16 if out == "out" else 4  # outputs keep their alignment
    last = (AT[other] + SIZES[other] - 1) // step * step
    first = -(-(AT[other] - SIZES[out] + 1) // step) * step
    assert placed(entry, **{out: last}) == _native.DSA_ERR_OVERLAP
    assert placed(entry, **{out: first}) == _native.DSA_ERR_OVERLAP
