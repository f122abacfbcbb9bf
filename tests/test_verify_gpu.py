"""GPU parity of the verification of drafts (dsa_b200.verify.run) with the oracle:
whole numbers, equal in every case."""

import pytest
import torch

from dsa_b200 import DsaError, verify
from oracle import verify as ov

pytestmark = pytest.mark.gpu


def outs(batch, width, device):
    return (torch.full((batch, width), 7, dtype=torch.int32, device=device), torch.full((batch,), 7, dtype=torch.int32, device=device),
            torch.full((batch,), 7, dtype=torch.int32, device=device))


def on(case, device):
    return [None if t is None else t.to(device) for t in case]


def check(case, device, width, exact=False):
    got = outs(len(case[4]) - 1, width, device)
    verify.run(*on(case, device), *got)
    want = ov.verify_reference(*case, width, exact)
    assert [g.tolist() for g in got] == list(want)


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("batch,most,vocab,branch", [(1, 1, 1, 1), (1, 2, 2, 1), (3, 5, 7, 2), (5, 9, 128, 3), (4, 6, 1001, 4), (20, 12, 513, 2),
                                                     (3, 40, 5000, 8), (2, 70, 64, 70)])
def test_random_trees(cuda_device, batch, most, vocab, branch, certain):
    for seed in range(4):
        check(ov.random_case(batch, most, vocab, branch, certain, seed), cuda_device, max(1, most - 1))


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("vocab,most,branch", [(3, 6, 3), (9, 12, 4), (140, 10, 2)])
def test_ties_zeros_and_borders(cuda_device, vocab, most, branch, certain):
    """Probabilities and random numbers on a coarse grid: equal values, zeros, random numbers at the borders of running sums,
    and residuals with nothing left; against exact fractions."""
    for seed in range(12):
        check(ov.random_case(6, most, vocab, branch, certain, seed, dyadic=True), cuda_device, most, exact=True)


@pytest.mark.parametrize("certain", [False, True])
def test_large_vocabulary(cuda_device, certain):
    case = ov.random_case(3, 6, 50003, 3, certain, 1)
    check(case, cuda_device, 5)
    wide = [None if t is None else torch.cat([t, torch.full((len(t), 13), 5.0)], 1)[:, :50003] for t in case[:2]]  # rows at odd places
    check((*wide, *case[2:]), cuda_device, 5)


def test_full_paths(cuda_device):
    """A walk ends where its path is full; the next token is then the last accepted row's."""
    case = ov.random_case(8, 9, 50, 1, False, 3)
    case = (*case[:5], torch.zeros_like(case[5]), case[6])  # everything with any probability is accepted
    for width in (1, 2, 20):
        check(case, cuda_device, width)


def test_equal_distributions_and_nothing_left(cuda_device):
    p = torch.tensor([[0.5, 0.5, 0.0, 0.0]] * 4)
    # token 2 has no probability in either: rejected, nothing is left, p is drawn from; so for the siblings behind it
    case = (p, p.clone(), torch.tensor([0, 2, 0, 3]), torch.tensor([-1, 0, 0, 0]), torch.tensor([0, 4]), torch.full((4,), 0.25),
            torch.tensor([0.5]))
    got = outs(1, 3, cuda_device)
    verify.run(*on(case, cuda_device), *got)
    assert [g.tolist() for g in got] == [[[-1, -1, -1]], [0], [1]]
    # struck out until nothing is left
    one = torch.zeros(2, 4)
    one[:, 1] = 1
    got = outs(1, 3, cuda_device)
    verify.run(*on((one, None, torch.tensor([0, 1]), torch.tensor([-1, 0]), torch.tensor([0, 2]), torch.full((2,), 1.0),
                    torch.tensor([0.0])), cuda_device), *got)
    assert [g.tolist() for g in got] == [[[-1, -1, -1]], [0], [1]]
    for bad in (0.0, float("nan")):
        got = outs(1, 3, cuda_device)
        verify.run(*on((torch.full((1, 300), bad), None, torch.tensor([0]), torch.tensor([-1]), torch.tensor([0, 1]),
                        torch.zeros(1), torch.tensor([0.5])), cuda_device), *got)
        assert got[2].tolist() == [-1]


def test_what_does_not_fit_is_reported(cuda_device):
    case = ov.random_case(4, 8, 60, 2, False, 5)
    want = ov.verify_reference(*case, 7)
    lo = int(case[4][3])
    tokens = case[2].clone()
    tokens[lo] = 99  # row 0's token is not read
    for t in (tokens, case[2]):
        got = outs(4, 7, cuda_device)
        verify.run(*on((*case[:2], t, *case[3:]), cuda_device), *got)
        assert [g.tolist() for g in got] == list(want)
    tokens[lo + 1] = 60
    got = outs(4, 7, cuda_device)
    with pytest.raises(DsaError, match="index"):
        verify.run(*on((*case[:2], tokens, *case[3:]), cuda_device), *got)
    assert [g.tolist()[:3] for g in got] == [w[:3] for w in want]
    cu = case[4].clone()
    cu[2] = 1 << 20
    got = outs(4, 7, cuda_device)
    with pytest.raises(DsaError, match="seq_len"):
        verify.run(*on((*case[:4], cu, *case[5:]), cuda_device), *got)
    assert got[2].tolist()[1:3] == [-1, -1] and got[2].tolist()[0] == want[2][0] and got[2].tolist()[3] == want[2][3]


def test_many_rows(cuda_device):
    """Requests of thousands of rows; behind the 4096th they are left out."""
    n, vocab = 5000, 40
    p = torch.softmax(torch.randn(n, vocab, generator=torch.Generator().manual_seed(2)), 1)
    chain = (p, p, torch.zeros(n).long(), torch.arange(-1, n - 1), torch.tensor([0, n]), torch.zeros(n), torch.tensor([0.3]))
    got = outs(1, 5000, cuda_device)
    with pytest.raises(DsaError, match="seq_len"):
        verify.run(*on(chain, cuda_device), *got)
    assert got[1].tolist() == [4095] and got[0][0, :4095].tolist() == list(range(1, 4096))
    star = (p[:3000], None, torch.arange(3000) % 7, torch.tensor([-1] + [0] * 2999), torch.tensor([0, 3000]),
            torch.full((3000,), 1.0), torch.tensor([0.9]))
    check(star, cuda_device, 4)


def test_refusals(cuda_device):
    case = on(ov.random_case(4, 6, 60, 2, False, 7), cuda_device)
    got = list(outs(4, 5, cuda_device))
    verify.run(*case, *got)
    bad = [(0, case[0].half()), (0, case[0][:, :50]), (0, case[0].T), (1, case[1][1:]), (2, case[2][1:]), (2, case[2].float()), (3, case[3][1:]),
           (4, case[4][:, None]), (5, case[5].double()), (6, case[6][1:]), (2, case[2].cpu()), (7, got[0].long()), (7, got[0][:3]),
           (7, got[0].T), (8, got[1][:2]), (9, got[2].cpu()), (9, got[1]), (7, case[5].view(torch.int32)[:4].reshape(4, 1))]
    for k, t in bad:
        args = [*case, *got]
        args[k] = t
        with pytest.raises(ValueError, match="dsa_verify.run"):
            verify.run(*args)


def test_empty_calls(cuda_device):
    got = outs(3, 2, cuda_device)
    z = lambda *s: torch.zeros(*s, device=cuda_device)  # noqa: E731
    verify.run(z(0, 5), None, z(0).int(), z(0).int(), z(4).int(), z(0), z(3), *got)
    assert got[0].tolist() == [[-1, -1]] * 3 and got[1].tolist() == [0] * 3 and got[2].tolist() == [-1] * 3
    verify.run(z(0, 5), None, z(0).int(), z(0).int(), z(1).int(), z(0), z(0), *outs(0, 2, cuda_device))


def test_in_a_graph_with_new_numbers(cuda_device):
    case = ov.random_case(6, 9, 3000, 2, False, 8)
    args, got = on(case, cuda_device), outs(6, 8, cuda_device)
    args[2:5] = [t.int() for t in args[2:5]]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        verify.run(*args, *got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            verify.run(*args, *got)
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        u, s = torch.rand(len(case[5]), generator=g), torch.rand(6, generator=g)
        args[5].copy_(u)
        args[6].copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert [t.tolist() for t in got] == list(ov.verify_reference(*case[:5], u, s, 8))


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("vocab,most,branch", [(9, 12, 4), (140, 10, 3), (5003, 8, 3)])
def test_zeros_of_either_sign(cuda_device, vocab, most, branch, certain):
    """-0.0 is 0 in both distributions, with rejections before siblings and before the draw."""
    for seed in range(8):
        target, draft, tokens, parents, cu, _, s = ov.random_case(5, most, vocab, branch, certain, seed, dyadic=True)
        negative = lambda t: None if t is None else torch.where(t == 0, -0.0, t)  # noqa: E731
        u = torch.full((len(tokens),), 1 - 2.0 ** -6) - (torch.arange(len(tokens)) % 3) / 4
        for case in ((negative(target), negative(draft)), (target, negative(draft))):
            check((*case, tokens, parents, cu, u, s), cuda_device, most, exact=vocab < 1000)


@pytest.mark.parametrize("vocab", [4, 300, 3001])
def test_subnormal_probabilities_count(cuda_device, vocab):
    """What is left after a rejection is one token of 2^-130, where the draft has 0, and beside it 2^-140 of one of 2^-139."""
    p, q = torch.zeros(2, vocab), torch.zeros(2, vocab)
    p[:, 0], p[:, 1], p[:, 2] = 0.5, 0.5, 2.0 ** -130
    q[:, 0], q[:, 1], q[:, 3] = 0.5, 0.5, 2.0 ** -149
    for u, token in ((0.0, 2), (0.9, 2)):
        got = outs(1, 1, cuda_device)
        verify.run(*on((p, q, torch.tensor([0, 3]), torch.tensor([-1, 0]), torch.tensor([0, 2]), torch.zeros(2), torch.tensor([u])),
                       cuda_device), *got)
        assert [g.tolist() for g in got] == [[[-1]], [0], [token]]
    p[:, 2], p[:, vocab - 2], q[:, vocab - 2] = 2.0 ** -140, 2.0 ** -139, 2.0 ** -140
    if vocab > 4:  # two tokens of 2^-140 each are left
        for u, token in ((0.49, 2), (0.51, vocab - 2)):
            got = outs(1, 1, cuda_device)
            verify.run(*on((p, q, torch.tensor([0, 3]), torch.tensor([-1, 0]), torch.tensor([0, 2]), torch.zeros(2), torch.tensor([u])),
                           cuda_device), *got)
            assert [g.tolist() for g in got] == [[[-1]], [0], [token]]


@pytest.mark.parametrize("vocab", [5, 700, 20001])
def test_nan_in_the_draft_is_not_drawn_from(cuda_device, vocab):
    """A rejection takes q away from p: with NaN in it nothing can be drawn, and no sibling accepted.  Where no child is
    rejected q is not read."""
    p = torch.softmax(torch.randn(3, vocab, generator=torch.Generator().manual_seed(vocab)), 1)
    q = p.clone()
    q[0, vocab // 2] = float("nan")
    for u, want in (([0.0, 1.0, 0.5], [[[-1, -1]], [0], [-1]]), ([0.0, 0.0, 0.0], [[[1, -1]], [1], None])):
        got = outs(1, 2, cuda_device)
        verify.run(*on((p, q, torch.tensor([0, 0, 1]), torch.tensor([-1, 0, 0]), torch.tensor([0, 3]), torch.tensor(u),
                        torch.tensor([0.5])), cuda_device), *got)
        assert [g.tolist() for g in got[:2]] == want[:2]
        assert got[2].tolist() == want[2] if want[2] else got[2].item() >= 0
