"""titan_spec.verify_drafts against the definition in whole numbers (exact)."""
import math

import pytest
import torch

import chunk_oracle as O
from conftest import log_case

pytestmark = pytest.mark.gpu


def make(dev, seed, counts, vocab, probs, ids64, sharp=3.0, near=0.7):
    g = torch.Generator(device="cpu").manual_seed(seed)
    D, rows = sum(counts), sum(counts) + len(counts)
    cu = torch.tensor([0] + [n + 1 for n in counts]).cumsum(0)
    req = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    logits = torch.randn(rows, vocab, generator=g) * sharp
    close = logits[torch.arange(D) + req] + near * torch.randn(D, vocab, generator=g)
    draft = torch.softmax(close, dim=1)
    ids = torch.multinomial(draft, 1, generator=g)[:, 0] if D else torch.zeros(0, dtype=torch.int64)
    return [torch.softmax(logits, dim=1).to(dev), (ids if ids64 else ids.to(torch.int32)).to(dev),
            draft.to(dev) if probs else None, cu.to(torch.int32).to(dev), torch.rand(D, generator=g).to(dev),
            torch.rand(len(counts), generator=g, dtype=torch.float64).to(dev)]


def check(a, most):
    from titan_spec import verify_drafts
    tokens, accepted = verify_drafts(*a, most)
    want, count = O.verify(*a, most)
    assert tokens.dtype == torch.int32 and accepted.dtype == torch.int32
    assert torch.equal(accepted.cpu(), count)
    assert torch.equal(tokens.cpu(), want)
    return tokens, accepted


@pytest.mark.parametrize("probs", [True, False], ids=["probs", "lookup"])
@pytest.mark.parametrize("counts,vocab,most", [
    ([3], 32000, 3), ([0], 512, 3), ([1], 1, 1), ([7, 0, 3, 7, 1, 2], 4096, 7), ([5, 5, 5], 4097, 5),
    ([2, 4, 0, 1], 50257, 4), ([70, 3, 130], 999, 130), ([6, 2, 9], 8192, 4), ([0, 0], 300, 0), ([3] * 40, 2000, 3)])
def test_exact(cuda, counts, vocab, most, probs):
    a = make(cuda, vocab + most, counts, vocab, probs, ids64=most % 2 == 0)
    log_case("verify_drafts", counts, vocab, most, probs)
    check(a, most)


@pytest.mark.parametrize("probs", [True, False], ids=["probs", "lookup"])
def test_all_taken_none_taken_and_the_ends_of_the_draw(cuda, probs):
    a = make(cuda, 5, [4, 4, 0, 2], 9000, probs, True)
    for u in (0.0, 1.0):
        a[4].fill_(u)
        for s in (0.0, 0.5, 1.0 - 2.0 ** -53, 1.0):
            a[5].fill_(s)
            log_case("verify_drafts ends", probs, u, s)
            tokens, accepted = check(a, 4)
            if u == 0.0:
                assert accepted.tolist() == [4, 4, 0, 2]
            elif not probs:
                assert accepted.tolist() == [0, 0, 0, 0]


def test_greedy_rows(cuda):
    """One-hot target rows: the draft stands where it is the target's token."""
    a = make(cuda, 6, [3, 3], 5000, False, False)
    best = a[0].argmax(dim=1)
    a[0] = torch.zeros_like(a[0]).scatter_(1, best[:, None], 1.0)
    a[1][:] = best[torch.tensor([0, 1, 2, 4, 5, 6], device=cuda)]
    a[1][4] = (a[1][4] + 1) % 5000
    log_case("verify_drafts greedy")
    tokens, accepted = check(a, 3)
    assert accepted.tolist() == [3, 1]
    assert tokens[0].tolist() == best[:4].tolist() and tokens[1].tolist() == [int(best[4]), int(best[5]), -1, -1]


def test_rows_without_weight_and_values_that_are_no_probabilities(cuda):
    a = make(cuda, 7, [2, 2, 2, 2, 2], 6000, True, True)
    a[2][0:2] = a[0][0:2]          # p = q: nothing left where rejected
    a[4][0] = 2.0                  # (rejects)
    a[0][3:6] = 0                  # an empty target
    a[0][6, 100:3000] = math.nan
    a[0][9, 5] = math.inf
    a[0][12, :4000] = -1.0
    a[4][6:] = 0.999
    log_case("verify_drafts odd values")
    tokens, accepted = check(a, 2)
    assert int(tokens[1, 0]) == -1 and int(tokens[0, 0]) >= 0
    a[4][8] = math.nan             # no number takes no draft
    a[5][2:] = math.nan            # and draws the first token with weight
    tokens, accepted = check_nan(a, 2)
    assert int(accepted[4]) == 0


def check_nan(a, most):
    from titan_spec import verify_drafts
    b = list(a)
    b[5] = torch.nan_to_num(a[5], nan=0.0)
    want, count = O.verify(*b, most)
    tokens, accepted = verify_drafts(*a, most)
    assert torch.equal(accepted.cpu(), count) and torch.equal(tokens.cpu(), want)
    return tokens, accepted


def test_ids_and_rows_outside(cuda):
    from titan_spec import verify_drafts
    for probs in (True, False):
        a = make(cuda, 8, [3, 3, 3], 3000, probs, True)
        a[4].fill_(0.0)
        a[1][1], a[1][3], a[1][8] = 3000, -1, 2 ** 40
        log_case("verify_drafts outside", probs)
        tokens, accepted = check(a, 3)
        assert accepted.tolist() == [1, 0, 2]
    a = make(cuda, 8, [3, 3, 3], 3000, True, False)
    for bad in ([0, 4, 8, 13], [0, 4, 4, 8], [-1, 4, 8, 12], [0, 8, 4, 12], [4, 4, 4, 4]):
        a[3] = torch.tensor(bad, dtype=torch.int32, device=cuda)
        log_case("verify_drafts rows", bad)
        check(a, 3)
    none = verify_drafts(a[0], a[1], a[2], a[3][:1], a[4], a[5][:0], 3)
    assert none[0].shape == (0, 4) and none[1].shape == (0,)


def test_strides(cuda):
    a = make(cuda, 9, [3, 1, 5], 4100, True, False)
    wide = torch.full((a[0].shape[0], 4111), math.nan, device=cuda)
    wide[:, 7:4107] = a[0]
    wd = torch.full((a[2].shape[0], 4200), math.nan, device=cuda)
    wd[:, 3:4103] = a[2]
    want = check(a, 5)
    log_case("verify_drafts strides")
    got = check([wide[:, 7:4107], a[1], wd[:, 3:4103]] + a[3:], 5)
    assert torch.equal(got[0], want[0])
    got = check([a[0].t().contiguous().t(), a[1], a[2].t().contiguous().t()] + a[3:], 5)
    assert torch.equal(got[0], want[0])


def test_distribution(cuda):
    """Over a grid of draws the kept token is distributed as the target: for a
    fixed draft and accept number the drawn tokens' shares are the weights'."""
    from titan_spec import verify_drafts
    p = torch.tensor([0.5, 0.25, 0.125, 0.125], device=cuda)
    q = torch.tensor([0.125, 0.25, 0.5, 0.125], device=cuda)
    n = 4096
    target = p.expand(2 * n, 4).contiguous()
    cu = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=cuda)
    ids = torch.full((n,), 2, dtype=torch.int32, device=cuda)
    u = (torch.arange(n, device=cuda, dtype=torch.float32) + 0.5) / n
    s = (torch.arange(n, device=cuda, dtype=torch.float64) * 1237 % n + 0.5) / n
    log_case("verify_drafts distribution")
    tokens, accepted = verify_drafts(target, ids, q.expand(n, 4).contiguous(), cu, u, s, 1)
    assert int(accepted.sum()) == n // 4           # p / q = 1/4 of the accept numbers
    drawn = tokens[accepted == 0, 0]
    assert bool((drawn == 0).all())                # only token 0 has p > q


def test_captured_and_replayed(cuda):
    from titan_spec import verify_drafts
    a = make(cuda, 10, [4, 2, 7, 0], 20000, True, False)
    verify_drafts(*a, 7)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, accepted = verify_drafts(*a, 7)
    for k in range(4):
        a[4].copy_(torch.rand_like(a[4]))
        a[5].copy_(torch.rand_like(a[5]))
        log_case("verify_drafts replay", k)
        graph.replay()
        torch.cuda.synchronize()
        want, count = O.verify(*a, 7)
        assert torch.equal(tokens.cpu(), want) and torch.equal(accepted.cpu(), count)
