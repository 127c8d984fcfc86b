"""Cases of the 8-bit cache's tests, shared by the CPU and the GPU files."""
import torch

from coeus_b200.ops import kv8
from plain_kv8 import PAGE, PlainCache


def starts(rows):
    out = [0]
    for r in rows:
        out.append(out[-1] + r)
    return out


def i32(x, dev="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def tables(need, width, gen, spare=2):
    """Page tables over a shuffled pool; places that no entry needs hold -1."""
    total = sum(need) + spare
    perm = torch.randperm(total, generator=gen).int()
    out = torch.full((len(need), width), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(need):
        out[i, :c] = perm[at:at + c]
        at += c
    return out, total


class Case:
    """A framework cache and a plain one, filled by the same writes."""

    def __init__(self, kind, heads, dh, lens, dev="cpu", seed=0, width=None):
        self.gen = torch.Generator().manual_seed(seed)
        self.kind, self.heads, self.dh, self.dev = kind, heads, dh, dev
        need = [(n + PAGE - 1) // PAGE for n in lens]
        self.table, total = tables(need, width or max(need + [1]) + 1, self.gen)
        self.c = kv8.kv8_alloc(total, heads, dh, kind, dev)
        self.plain = PlainCache(total, heads, dh, kind)

    def rows(self, n, size=1.0):
        x = torch.randn(n, self.heads * self.dh, generator=self.gen) * size
        return x.bfloat16()

    def write(self, pos0, rows, sizes=None, edit=None):
        """Writes ``rows[e]`` new tokens at ``pos0[e]``, of magnitude ``sizes[e]``."""
        sizes = sizes or [1.0] * len(rows)
        k = torch.cat([self.rows(r, s) for r, s in zip(rows, sizes)] or [self.rows(0)])
        v = torch.cat([self.rows(r, 0.3 * s) for r, s in zip(rows, sizes)] or [self.rows(0)])
        if edit is not None:
            edit(k, v)
        one = all(r == 1 for r in rows)
        kv8.kv8_write(k.to(self.dev), v.to(self.dev), *self.c, self.table.to(self.dev),
                      i32(pos0, self.dev), row0=None if one else i32(starts(rows), self.dev),
                      max_rows=max(rows + [1]))
        self.plain.write(k, v, self.table, pos0, rows)

    def read(self, pos0, rows):
        out = kv8.kv8_read(*self.c, self.table.to(self.dev), i32(pos0, self.dev),
                           i32(starts(rows), self.dev), sum(rows), max_rows=max(rows + [1]))
        return tuple(o.double().cpu() for o in out)

    def check_read(self, pos0, rows):
        for got, want in zip(self.read(pos0, rows), self.plain.read(self.table, pos0, rows)):
            assert torch.equal(torch.nan_to_num(got, 1e30), torch.nan_to_num(want, 1e30))

    def attend(self, q, ctx, rows, nh, scale=None, max_rows=None):
        one = all(r == 1 for r in rows)
        return kv8.kv8_attention(q.to(self.dev), *self.c, self.table.to(self.dev),
                                 i32(ctx, self.dev), nh,
                                 row0=None if one else i32(starts(rows), self.dev),
                                 max_rows=max_rows or max(rows + [1]), scale=scale)

    def check_attend(self, ctx, rows, nh, scale=None, size=1.0, max_rows=None):
        q = (torch.randn(sum(rows), nh * self.dh, generator=self.gen) * size).bfloat16()
        got = self.attend(q, ctx, rows, nh, scale, max_rows).double().cpu()
        want, spread = self.plain.attention(q, self.table, ctx, rows, nh, scale or self.dh ** -0.5)
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        err = torch.where(nan, torch.zeros_like(want), (got - want).abs())
        # the result is rounded to bf16 (2^-8 of it), the weights to fp16 (2^-11 each, 2^-36 of the
        # largest where they are that small), their exponents and sums are fp32: scores of size
        # s lose 2^-22 s, and s stays below 2^8 here
        bound = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * spread + 1e-30
        bad = (err > torch.nan_to_num(bound, 0.0)) & ~nan
        assert not bad.any(), (float(err[bad].max()), float((err / bound)[bad].max()))
        return got
