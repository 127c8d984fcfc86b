"""Beams whose rows name the same page that is not full, shared by the CPU and the GPU tests."""
import torch

from coeus_b200.ops import beam
from plain_kv8 import PAGE


def check_shared_tails(dev, length, rows, parent):
    """Request 1 of two: ``rows`` says which of the beams hold the same pages before the step.  Every beam has
    a last page of its own afterwards, with what its parent's held."""
    K, lp = len(rows), length // PAGE
    g = torch.Generator().manual_seed(length)
    kinds = max(rows) + 1
    pool = torch.randperm(60, generator=g).int()[:4 * K]
    table = torch.full((2 * K, lp + 2), -1, dtype=torch.int32)
    for j in range(K):
        table[j, :lp + 1] = 60 + j
        table[K + j, :lp] = 40 + torch.arange(lp).int() + 80
        table[K + j, lp] = 80 + rows[j]
    cache = torch.randint(-99, 99, (140, 16), generator=g).to(torch.int8).to(dev)
    before = cache.clone()
    pools = torch.stack([pool, pool.flip(0)]).contiguous()
    parents = torch.tensor([list(range(K)), parent])
    got = beam.beam_reorder(table.to(dev), parents.to(dev), torch.tensor([length, length], dtype=torch.int32, device=dev),
                            pools.to(dev), [cache])
    mine = got[K:, lp].tolist()
    assert torch.equal(got[:K].cpu(), table[:K])           # beams with pages of their own stay
    assert len(set(mine)) == K, mine
    seen = []
    for j, p in enumerate(parent):
        tail = 80 + rows[p]
        if tail in seen:
            assert mine[j] in pools[1].tolist() and torch.equal(cache[mine[j]], before[tail])
        else:
            assert mine[j] == tail
        seen.append(tail)
        assert got[K + j, :lp].tolist() == table[K + p, :lp].tolist()
    changed = (cache != before).any(1).nonzero()[:, 0].tolist()
    assert set(changed) <= set(mine) - set(seen)
    assert kinds == len(set(rows))


TAILS = [([0, 0, 0, 0], [0, 1, 2, 3]), ([0, 0, 0, 0], [0, 0, 2, 3]), ([0, 0, 1, 1], [3, 1, 0, 2]),
         ([0, 1, 1, 2], [1, 2, 0, 0]), ([0, 0, 0], [2, 2, 0])]
