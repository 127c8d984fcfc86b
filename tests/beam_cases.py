"""Cases of the beam search's tests, shared by the CPU and the GPU files."""
import math

import torch

from coeus_b200.ops import beam
from plain_kv8 import PAGE, beam_pages, beam_step


def check_select(logits, scores, done, eos):
    B, K = scores.shape
    got = beam.beam_select(logits, scores, done, eos)
    s, p, t, d = (x.cpu() for x in got)
    for b in range(B):
        want = beam_step(logits[b * K:(b + 1) * K].cpu(), scores[b].cpu(), done[b].cpu(), eos)
        assert p[b].tolist() == [w[1] for w in want], (b, p[b], want)
        assert t[b].tolist() == [w[2] for w in want], (b, t[b], want)
        assert d[b].tolist() == [w[3] for w in want]
        for i in range(K):
            # one rounding to fp32, and a logarithm whose argument is summed in fp32 blocks
            if math.isinf(want[i][0]):
                assert float(s[b, i]) == want[i][0]
            else:
                assert abs(float(s[b, i]) - want[i][0]) <= 2.0 ** -23 * (1 + abs(want[i][0]))
    return got


def state(B, K, V, dtype, dev, seed=0, ended=0):
    g = torch.Generator().manual_seed(seed)
    logits = (2.5 * torch.randn(B * K, V, generator=g)).to(dtype)
    scores = -10.0 * torch.rand(B, K, generator=g)
    done = torch.zeros(B, K, dtype=torch.bool)
    for b in range(B):
        done[b, torch.randperm(K, generator=g)[:ended]] = True
    return logits.to(dev), scores.to(dev), done.to(dev)


def pages_case(B, K, lens, own, dev, seed=0, pool=None):
    """Beams that share all but their last ``own`` pages."""
    g = torch.Generator().manual_seed(seed)
    width = max(n // PAGE for n in lens) + 2
    pool = pool or K * (own + 1)
    need = [(n + PAGE - 1) // PAGE for n in lens]
    shared = [max(0, n - own) for n in need]
    total = sum(shared) + B * pool + 1
    perm = torch.randperm(total, generator=g).int()
    table = torch.full((B, K, width), -1, dtype=torch.int32)
    pools, at = [], 0
    for b in range(B):
        table[b, :, :shared[b]] = perm[at:at + shared[b]]
        at += shared[b]
        mine = perm[at:at + pool]
        at += pool
        pools.append(mine)
        c = need[b] - shared[b]
        for j in range(K):
            table[b, j, shared[b]:need[b]] = mine[j * c:(j + 1) * c]
    return table.view(B * K, width).to(dev), torch.stack(pools).to(dev), total


def check_reorder(table, parent, lens, pool, caches):
    B, K = parent.shape
    before = [c.clone() for c in caches]
    n = torch.tensor(lens, dtype=torch.int32, device=table.device)
    got = beam.beam_reorder(table, parent, n, pool, caches)
    rows = got.view(B, K, -1).tolist()
    old = table.view(B, K, -1).tolist()
    copies = {}
    for b in range(B):
        want, moves = beam_pages(old[b], parent[b].tolist(), lens[b], pool[b].tolist())
        assert rows[b] == want, (b, rows[b], want)
        for m in moves:
            if m is not None:
                copies[m[1]] = m[0]
        lp = lens[b] // PAGE
        assert len({r[lp] for r in rows[b]}) == K          # every beam has a page to write to
    for c, was in zip(caches, before):
        want = was.view(torch.uint8).clone()
        for d, s in copies.items():
            want[d] = was.view(torch.uint8)[s]
        assert torch.equal(c.view(torch.uint8), want)
    return got
