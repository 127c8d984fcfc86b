"""The beam search's step on the CPU against its definition, and the calls that are refused."""
import math

import pytest
import torch

from beam_cases import check_reorder, check_select, pages_case, state
from beam_tails import TAILS, check_shared_tails
from coeus_b200.ops import beam


@pytest.mark.parametrize("K,V,ended,eos", [(1, 7, 0, None), (4, 50, 1, 3), (5, 3, 2, 0), (3, 33, 3, 2),
                                           (4, 2, 0, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select(K, V, ended, eos, dtype):
    check_select(*state(3, K, V, dtype, "cpu", ended=ended), eos)


def test_select_first_step_and_nothing_left():
    logits, scores, done = state(2, 4, 3, torch.float32, "cpu")
    scores[:, 1:], scores[:, 0] = -math.inf, 0.0
    s, p, t, d = check_select(logits, scores, done, 1)
    assert p[0].tolist() == [0, 0, 0, 3] and bool(d[0, 3]) and float(s[0, 3]) == -math.inf
    # equal logits: the lowest token of the lowest beam
    s, p, t, d = check_select(torch.zeros(8, 5), torch.zeros(2, 4), torch.zeros(2, 4).bool(), None)
    assert p[0].tolist() == [0] * 4 and t[0].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("lens", [[1, 63, 64], [65, 128, 200], [640, 7, 130]])
@pytest.mark.parametrize("K", [1, 4])
def test_reorder(lens, K):
    g = torch.Generator().manual_seed(5)
    table, pool, total = pages_case(3, K, lens, 2, "cpu")
    caches = [torch.randn(total, 4, 3, generator=g), torch.randint(0, 99, (total, 8)).to(torch.int8)]
    parent = torch.randint(0, K, (3, K), generator=g)
    table = check_reorder(table, parent, lens, pool, caches)
    check_reorder(table, parent, lens, pool, caches)       # and on from there


def test_copies_of_pages_that_are_not_there():
    c = torch.arange(8).view(4, 2)
    for s, d in ((4, 1), (1, 4)):
        with pytest.raises(ValueError):
            beam.copy_pages([c], torch.tensor([s], dtype=torch.int32), torch.tensor([d], dtype=torch.int32))
    beam.copy_pages([c], torch.tensor([-1, 0], dtype=torch.int32), torch.tensor([9, 1], dtype=torch.int32))
    assert c.tolist() == [[0, 1], [0, 1], [4, 5], [6, 7]]


def test_refusals():
    logits, scores, done = state(2, 3, 9, torch.float32, "cpu")
    for args in ((logits[:5], scores, done, 1), (logits, scores.double(), done, 1),
                 (logits, scores, done.int(), 1), (logits, scores, done, 9), (logits, scores, done, -1),
                 (logits, scores[0], done, 1), (logits, scores, done[:1], 1),
                 (torch.zeros(66, 5), torch.zeros(2, 33), torch.zeros(2, 33).bool(), 1)):
        with pytest.raises(ValueError):
            beam.beam_select(*args)
    table, pool, total = pages_case(2, 3, [70, 20], 2, "cpu")
    parent = torch.zeros(2, 3, dtype=torch.int64)
    n = torch.tensor([70, 20], dtype=torch.int32)
    cache = [torch.zeros(total, 4)]
    good = [table, parent, n, pool, cache]
    for i, bad in ((0, table.long()), (0, table[:5]), (1, parent.int()), (1, parent + 3), (2, n.long()),
                   (2, n[:1]), (2, n + 10 ** 6), (3, pool.long()), (3, pool[:, :1]), (4, []),
                   (4, [cache[0].t()]), (4, [cache[0], torch.zeros(total + 1, 4)])):
        with pytest.raises(ValueError):
            beam.beam_reorder(*[bad if j == i else x for j, x in enumerate(good)])


def test_pool_that_names_a_page_twice():
    table, pool, total = pages_case(2, 4, [70, 20], 2, "cpu")
    n, parent = torch.tensor([70, 20], dtype=torch.int32), torch.tensor([[0, 0, 0, 2], [1, 1, 1, 1]])
    want, src, dst = beam.beam_pages(table, parent, n, pool, total)
    twice = torch.cat([pool[:, :1], pool.repeat_interleave(3, 1), pool], 1)
    got, s, d = beam.beam_pages(table, parent, n, twice, total)
    assert torch.equal(got, want) and torch.equal(s, src) and torch.equal(d, dst)
    for b, lp in ((0, 1), (1, 0)):
        assert len(set(got.view(2, 4, -1)[b, :, lp].tolist())) == 4


@pytest.mark.parametrize("length", [1, 70, 191])
@pytest.mark.parametrize("rows,parent", TAILS)
def test_reorder_shared_tails(length, rows, parent):
    check_shared_tails("cpu", length, rows, parent)
