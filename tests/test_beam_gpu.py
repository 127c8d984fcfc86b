"""The kernels of the beam search's step against its definition."""
import math
import threading

import pytest
import torch

from beam_cases import check_reorder, check_select, pages_case, state
from beam_tails import TAILS, check_shared_tails
from coeus_b200.ops import _lib, beam

pytestmark = pytest.mark.gpu
DEV = "cuda"


def status():
    torch.cuda.synchronize()
    s = _lib.status_buffer(torch.device("cuda", 0))
    code = int(s[0])
    s.zero_()
    return code


@pytest.mark.parametrize("B,K,V,ended,eos", [(1, 1, 1, 0, 0), (2, 4, 5, 1, 3), (3, 3, 1023, 0, None),
                                             (2, 5, 1025, 2, 0), (2, 8, 5003, 3, 5002), (1, 32, 9001, 7, 17),
                                             (4, 3, 2048, 3, 2), (2, 16, 7, 0, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select(B, K, V, ended, eos, dtype):
    check_select(*state(B, K, V, dtype, DEV, ended=ended), eos)


@pytest.mark.parametrize("V", [3, 1000, 4099])
def test_select_first_step(V):
    logits, scores, done = state(3, 4, V, torch.bfloat16, DEV)
    scores[:, 1:], scores[:, 0] = -math.inf, 0.0
    s, p, t, d = check_select(logits, scores, done, 1)
    if V == 3:
        assert p[0].tolist() == [0, 0, 0, 3] and bool(d[0, 3])


def test_select_equal_values_go_to_the_lowest():
    for K, V in ((4, 5000), (7, 300), (2, 1)):
        done = torch.zeros(2, K, dtype=torch.bool, device=DEV)
        check_select(torch.zeros(2 * K, V, device=DEV), torch.zeros(2, K, device=DEV), done, None)
        done[:, 0] = True
        check_select(torch.zeros(2 * K, V, device=DEV), torch.zeros(2, K, device=DEV), done, V - 1)
    # a few levels only: many equal values, in every block
    g = torch.Generator().manual_seed(3)
    x = torch.randint(0, 3, (8, 6000), generator=g).float().to(DEV)
    check_select(x, torch.zeros(2, 4, device=DEV), torch.zeros(2, 4, dtype=torch.bool, device=DEV), 0)


def test_select_infinities_and_nan():
    """A masked logit is no continuation, a row with NaN or +inf has none, all masked is the end."""
    logits, scores, done = state(4, 3, 2500, torch.float32, DEV)
    logits[0, 5:] = -math.inf                 # five tokens left
    logits[1] = -math.inf
    logits[2, 77] = math.nan
    logits[3:6] = -math.inf                   # request 1: one token in one beam
    logits[4, 1234] = 2.0
    logits[6:9] = -math.inf                   # request 2: none at all
    logits[9, 3] = math.inf                   # request 3
    scores[3, 1] = math.nan
    s, p, t, d = (x.cpu() for x in beam.beam_select(logits, scores, done, 1))
    assert p[0].tolist() == [0, 0, 0] and max(t[0].tolist()) < 5
    assert p[1].tolist() == [1, 1, 2] and t[1].tolist() == [1234, 1, 1]
    assert s[1].tolist() == [float(scores[1, 1]), -math.inf, -math.inf] and d[1].tolist() == [False, True, True]
    assert (s[2] == -math.inf).all() and p[2].tolist() == [0, 1, 2] and d[2].all()
    assert p[3].tolist() == [2, 2, 2]


def test_select_views_and_graph():
    logits, scores, done = state(2, 4, 3001, torch.bfloat16, DEV)
    wide = torch.randn(8, 4000, device=DEV).bfloat16()
    wide[:, 7:3008] = logits
    a = check_select(wide[:, 7:3008], scores, done, 2)
    b = beam.beam_select(logits.t().contiguous().t(), scores.t().contiguous().t(), done, 2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = beam.beam_select(logits, scores, done, 2)
    logits.copy_(torch.randn_like(logits))
    g.replay()
    for x, y in zip(c, check_select(logits, scores, done, 2)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("lens", [[1, 63, 64], [65, 128, 200], [640, 7, 1300]])
@pytest.mark.parametrize("K", [1, 4, 11])
def test_reorder(lens, K):
    g = torch.Generator().manual_seed(5)
    table, pool, total = pages_case(3, K, lens, 3, DEV)
    caches = [torch.randn(total, 64, 2, 8, generator=g).bfloat16().to(DEV),
              torch.randint(-99, 99, (total, 2, 1, 64, 64), generator=g).to(torch.int8).to(DEV),
              torch.rand(total, 3, generator=g).to(DEV)]
    for i in range(4):
        parent = torch.randint(0, K, (3, K), generator=g).to(DEV)
        table = check_reorder(table, parent, lens, pool, caches)
    assert status() == 0


def test_reorder_many_tensors_and_graph():
    g = torch.Generator().manual_seed(6)
    table, pool, total = pages_case(2, 3, [70, 130], 2, DEV)
    caches = [torch.rand(total, 4, generator=g).to(DEV) for _ in range(400)]
    parent = torch.tensor([[1, 1, 0], [2, 2, 2]], device=DEV)
    want = check_reorder(table, parent, [70, 130], pool, [c.clone() for c in caches])
    n = torch.tensor([70, 130], dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beam.beam_reorder(table, parent, n, pool, caches)
    graph.replay()
    assert torch.equal(out, want) and status() == 0


def test_copies_of_pages_that_are_not_there():
    """Only the copies that the tensors have are made; the others are reported."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    caches = [torch.arange(5 * 48, device=DEV, dtype=torch.int32).view(5, 48), torch.rand(5, 7, device=DEV)]
    before = [c.clone() for c in caches]
    beam.copy_pages(caches, i32([0, 2, 5, 2 ** 31 - 1]), i32([1, 2 ** 31 - 1, 3, 4]))
    assert status() == 2
    for c, b in zip(caches, before):
        b[1] = b[0]
        assert torch.equal(c, b)
    beam.copy_pages(caches, i32([-1, 3]), i32([2, -5]))
    assert status() == 0 and all(torch.equal(c, b) for c, b in zip(caches, before))


def test_reorder_reports_what_it_cannot_do():
    table, pool, total = pages_case(2, 3, [70, 20], 2, DEV)
    cache = [torch.arange(total * 4, device=DEV, dtype=torch.float32).view(total, 4)]
    n = torch.tensor([70, 20], dtype=torch.int32, device=DEV)
    parent = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    before = cache[0].clone()
    out = beam.beam_reorder(table, parent, n, pool[:, :1].contiguous(), cache)      # no free pages
    assert status() == 2 and int(out[0, 1]) >= 0 and (out.view(2, 3, -1)[0, 1:, 1] == -1).all()
    assert torch.equal(cache[0], before)
    beam.beam_reorder(table, parent + 7, n, pool, cache)
    assert status() == 2
    out = beam.beam_reorder(table, parent, n + 10 ** 6, pool, cache)
    assert status() == 2 and torch.equal(out, table)
    with pytest.raises(ValueError):
        beam.copy_pages([torch.zeros(4, 3, dtype=torch.int8, device=DEV)], n, n)
    with pytest.raises(ValueError):
        beam.beam_reorder(table, parent.cpu(), n, pool, cache)


def test_pool_that_names_a_page_twice():
    table, pool, total = pages_case(2, 4, [70, 20], 2, DEV)
    n, parent = torch.tensor([70, 20], dtype=torch.int32, device=DEV), torch.tensor([[0, 0, 0, 2], [1, 1, 1, 1]], device=DEV)
    want, src, dst = beam.beam_pages(table, parent, n, pool, total)
    twice = torch.cat([pool[:, :1], pool.repeat_interleave(3, 1), pool], 1)
    got, s, d = beam.beam_pages(table, parent, n, twice, total)
    assert torch.equal(got, want) and torch.equal(s, src) and torch.equal(d, dst)
    for b, lp in ((0, 1), (1, 0)):
        assert len(set(got.view(2, 4, -1)[b, :, lp].tolist())) == 4
    assert status() == 0


@pytest.mark.parametrize("length", [1, 70, 191])
@pytest.mark.parametrize("rows,parent", TAILS)
def test_reorder_shared_tails(length, rows, parent):
    check_shared_tails(DEV, length, rows, parent)
    assert status() == 0


@pytest.mark.parametrize("V", [37, 5003, 20001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_equal_rows(V, dtype):
    """Beams with the same logits and scores tie in every continuation, wherever their rows begin in memory."""
    logits, _, done = state(3, 8, V, dtype, DEV)
    logits[:] = logits[::8].repeat_interleave(8, 0)
    for wide in (V, V + 1, V + 3, V + 64):
        rows = torch.zeros(24, wide, dtype=dtype, device=DEV)
        for skip in sorted({0, min(3, wide - V)}):
            rows[:, skip:skip + V] = logits
            check_select(rows[:, skip:skip + V], torch.zeros(3, 8, device=DEV), done, 1)


def test_large_caches_in_two_threads():
    """Threads whose caches differ in size, both beyond what a launch may use without asking: every launch is
    accepted, whichever thread asked last."""
    table, pool, total = pages_case(2, 4, [70, 20], 2, DEV)
    n, parent = torch.tensor([70, 20], dtype=torch.int32, device=DEV), torch.tensor([[0, 0, 0, 2], [1, 1, 1, 1]], device=DEV)
    want = beam.beam_pages(table, parent, n, pool, total)
    state, stream = _lib.status_buffer(table.device), _lib.stream_int()
    call, refused, wrong = _lib.entry("cb_beam_pages", "piiipppiippppp"), [], []

    def work(pages):
        got = [torch.empty_like(t) for t in want]
        for _ in range(10000):             # the library's entry itself: the interpreter's lock would keep the calls apart
            rc = call(table.data_ptr(), table.shape[1], 2, 4, parent.data_ptr(), n.data_ptr(), pool.data_ptr(),
                      pool.shape[1], pages, *[t.data_ptr() for t in got], state.data_ptr(), stream)
            if rc:
                refused.append((pages, rc))
        torch.cuda.synchronize()
        wrong.extend(pages for a, b in zip(got, want) if not torch.equal(a, b))
    threads = [threading.Thread(target=work, args=(p,)) for p in (350_000, 200 * 1024 * 8) * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not refused and not wrong, (len(refused), refused[:3], wrong)
    assert status() == 0
