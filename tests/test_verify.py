"""CPU tests of the verification of drafts: the oracle's distribution, and the
refusals of the C ABI and the Python entry point."""

import ctypes
import itertools
import math
from fractions import Fraction

import pytest
import torch

from dsa_b200 import _native, verify
from oracle import verify as ov

P = ctypes.c_void_p


@pytest.mark.parametrize("certain", [False, True])
def test_oracle_draws_as_the_target_would(certain):
    """The first token that comes out of a root with two drafted children has the target's distribution: over a fine
    grid of all random numbers (or, for drawn drafts, over the drafts as well) its frequencies are the target's."""
    p, q = [0.5, 0.125, 0.25, 0.125], [0.25, 0.25, 0.5, 0.0]
    target = torch.tensor([p] * 3)
    grid = [(2 * i + 1) / 16 for i in range(8)]
    got = [0.0] * 4
    for x in range(4):
        for y in range(4):
            chance = q[x] * q[y] if not certain else float((x, y) == (2, 0))
            if chance == 0:
                continue
            for u in grid:
                for v in grid:
                    us = [(2 * i + 1) / 64 for i in range(32)]
                    for s in us:
                        path, n, nxt = ov.verify_reference(target, None if certain else torch.tensor([q] * 3), [0, x, y], [-1, 0, 0],
                                                           [0, 3], [0.0, u, v], [s], 2, exact=True)
                        first = [0, x, y][path[0][0]] if n[0] else nxt[0]
                        got[first] += chance / (64 * len(us))
    # A grid of n midpoints gives a probability to 1 / (2 n).  A token comes out by the first test, the second or the draw
    # (two borders): off by at most 1/16 + 1/16 + 2/64.
    assert all(abs(a - b) <= 1 / 16 + 1 / 16 + 2 / 64 for a, b in zip(got, p)), got


def first_token(p, q, drafts, accept, draw):
    """The distribution of the first token that comes out of a root, exactly: `drafts` are its children (or, with q, their
    number, each drawn from q), `accept` the cells of each child's random number and `draw` those of the last one, whose borders
    lie at multiples of one over their number."""
    got = [Fraction(0)] * len(p)
    children = drafts if q is None else list(itertools.product(*[[x for x in range(len(q)) if q[x]] for _ in range(drafts)]))
    rows = 1 + len(children[0])
    target, draft = torch.tensor([p] * rows), None if q is None else torch.tensor([q] * rows)
    middle = lambda i, n: (2 * i + 1) / (2 * n)  # noqa: E731
    for kids in children:
        chance = math.prod([Fraction(q[x]) for x in kids]) if q is not None else Fraction(1)
        for cells in itertools.product(*[range(n) for n in accept]):
            us = [0.0, *(middle(i, n) for i, n in zip(cells, accept))]
            each = chance / math.prod(accept)
            for i in range(draw):
                path, n, following = ov.verify_reference(target, draft, [0, *kids], [-1] + [0] * len(kids), [0, rows], us,
                                                         [middle(i, draw)], 1, exact=True)
                if n[0]:  # whatever the draw
                    got[kids[path[0][0] - 1]] += each
                    break
                got[following[0]] += each / draw
    return got


@pytest.mark.parametrize("p,q,drafts,accept,draw", [
    # p / q of the children 2, 1/2 and 1/2; left are 2/3 and 1/3, then 5/9 and 4/9, then 11/27 and 16/27
    ([0.5, 0.125, 0.25, 0.125], [0.25, 0.25, 0.5, 0.0], 1, [2], 3),
    ([0.5, 0.125, 0.25, 0.125], [0.25, 0.25, 0.5, 0.0], 2, [2, 2], 9),
    ([0.5, 0.125, 0.25, 0.125], [0.25, 0.25, 0.5, 0.0], 3, [2, 2, 2], 27),
    # left are 1/4, 1/2 and 1/4, of which the first is accepted in 2 of 3; then 4/5 and 1/5; then 32/35 and 3/35
    ([0.5, 0.25, 0.25, 0.0], [0.375, 0.0, 0.125, 0.5], 2, [3, 3], 20),
    ([0.5, 0.25, 0.25, 0.0], [0.375, 0.0, 0.125, 0.5], 3, [3, 3, 3], 140),
    # drafts without a distribution: accepted in 1/4; of 2/3, 1/6, 1/6 in 2/3; of 1/2, 1/2 in 1/2; a draft given twice never again
    ([0.5, 0.125, 0.25, 0.125], None, [(2,)], [4], 6),
    ([0.5, 0.125, 0.25, 0.125], None, [(2, 0)], [4, 3], 2),
    ([0.5, 0.125, 0.25, 0.125], None, [(2, 0, 1)], [4, 3, 2], 1),
    ([0.5, 0.125, 0.25, 0.125], None, [(2, 2, 0)], [4, 1, 3], 2),
])
def test_oracle_draws_exactly_as_the_target(p, q, drafts, accept, draw):
    assert first_token(p, q, drafts, accept, draw) == [Fraction(x) for x in p]


def call(lib, target=4096, stride=8, draft=8192, draft_stride=8, tokens=16, parents=64, cu=128, au=192, su=256, requests=2,
         rows=5, vocab=8, width=3, path=16384, accepted=17000, following=18000, status=320):
    return lib.dsa_verify_run(P(target), stride, P(draft), draft_stride, P(tokens), P(parents), P(cu), P(au), P(su), requests,
                              rows, vocab, width, P(path), P(accepted), P(following), P(status), None)


@pytest.mark.parametrize("change,status", [
    (dict(requests=-1), 1), (dict(rows=-1), 1), (dict(requests=0), 0), (dict(requests=65537), 1), (dict(vocab=0), 1),
    (dict(stride=7), 1), (dict(draft_stride=7), 1), (dict(width=0), 1), (dict(width=65537), 1), (dict(target=None), 1),
    (dict(tokens=None), 1), (dict(status=None), 1), (dict(following=None), 1), (dict(rows=(1 << 24) + 1), 1),
    (dict(target=4098), 2), (dict(path=16386), 2), (dict(cu=130), 2), (dict(path=4096 + 156), 7), (dict(path=8192 - 20), 7),
    (dict(accepted=16384 + 20), 7), (dict(following=17004), 7), (dict(accepted=64 + 16), 7), (dict(following=256), 7),
])
def test_c_abi_refuses_bad_arguments(change, status):
    assert call(_native.lib(), **change) == status


def test_entry_point_refuses_cpu_tensors():
    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        verify.run(z(1, 4), None, z(1).int(), z(1).int(), z(2).int(), z(1), z(1), z(1, 1).int(), z(1).int(), z(1).int())
