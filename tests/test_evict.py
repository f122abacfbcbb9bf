"""CPU tests of the eviction's C ABI: outputs that share memory with an input or
with each other are refused on the host, before a device is looked for."""

import ctypes

import pytest

from dsa_b200 import _native

P = ctypes.c_void_p
OVERLAP = _native.DSA_ERR_OVERLAP
REQUESTS, PAGES, NEW_PAGES, BUDGET = 3, 4, 2, 100
# name -> (address, bytes): one after the other
SIZES = {"acc": REQUESTS * PAGES * 256, "seq_lens": REQUESTS * 4, "block_table": REQUESTS * PAGES * 4,
         "new_block_table": REQUESTS * NEW_PAGES * 4, "keep": REQUESTS * BUDGET * 4, "new_seq_lens": REQUESTS * 4,
         "new_acc": REQUESTS * NEW_PAGES * 256}
AT, _end = {}, 1 << 20
for _name, _bytes in SIZES.items():
    AT[_name] = _end
    _end += _bytes


def call(acc_stride=PAGES * 64, new_stride=NEW_PAGES * 64, **where):
    at = AT | where
    return _native.lib().dsa_cache_evict_run(
        P(at["acc"]), acc_stride, P(at["seq_lens"]), P(at["block_table"]), P(at["new_block_table"]), REQUESTS, PAGES, NEW_PAGES,
        P(1 << 30), 65536, 1024, P(1 << 31), 8192, 128, None, 9, BUDGET, 4, 8, P(at["keep"]), P(at["new_seq_lens"]),
        P(at["new_acc"]), new_stride, P(16), 256, None)


@pytest.fixture(autouse=True)
def no_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up: no launch may follow")


def test_neighbours_and_lengths_in_place_are_taken():
    assert call() not in (1, 2, 3, OVERLAP)  # only the device is missing
    assert call(new_seq_lens=AT["seq_lens"]) not in (1, 2, 3, OVERLAP)


@pytest.mark.parametrize("out", ["keep", "new_seq_lens", "new_acc"])
@pytest.mark.parametrize("other", [n for n in SIZES])
def test_outputs_that_share_memory_are_refused(out, other):
    if other == out:
        pytest.skip("itself")
    last = AT[other] + SIZES[other] - 4       # begins in the other's last element
    first = AT[other] - SIZES[out] + 4        # ends in the other's first
    assert call(**{out: last}) == OVERLAP
    assert call(**{out: first}) == OVERLAP
    if (out, other) != ("new_seq_lens", "seq_lens"):
        assert call(**{out: AT[other]}) == OVERLAP


def test_interleaved_accumulators():
    # the new ones as columns of the buffer that holds the old ones
    pitch, far = (PAGES + NEW_PAGES) * 64, 1 << 28
    put = lambda shift, p=pitch: call(acc_stride=pitch, new_stride=p, acc=far, new_acc=far + 4 * shift)  # noqa: E731
    assert put(PAGES * 64) not in (1, 2, 3, OVERLAP)
    assert put(PAGES * 64 - 1) == OVERLAP and put(PAGES * 64 + 1) == OVERLAP and put(0) == OVERLAP
    assert put(PAGES * 64, pitch + 1) == OVERLAP
