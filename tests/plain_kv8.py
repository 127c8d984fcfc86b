"""The 8-bit cache and the beam search's step from their definitions, in 64 bits and plain Python
loops over entries, pages and heads: what the operators' tests compare against."""
import math

import torch

PAGE = 64
QMAX = {"int8": 127.0, "e4m3": 448.0}


def code(y, kind):
    """Nearest code of ``y`` (float64), ties to even."""
    if kind == "int8":
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def exponent(amax, kind):
    if amax == 0.0:
        return -126
    e = math.frexp(amax)[1] - 10
    while amax > QMAX[kind] * 2.0 ** e:
        e += 1
    return max(e, -126)


class PlainCache:
    """Values of one layer: ``x[side][page, head, token, dh]`` and exponents ``e[side][page, head]``
    (side 0: keys)."""

    def __init__(self, pages, heads, dh, kind):
        self.x = [torch.zeros(pages, heads, PAGE, dh, dtype=torch.float64) for _ in range(2)]
        self.e = [torch.zeros(pages, heads, dtype=torch.float64) for _ in range(2)]
        self.kind, self.heads, self.dh = kind, heads, dh

    def write(self, k, v, table, pos0, rows):
        at = 0
        for entry, (p0, n) in enumerate(zip(pos0, rows)):
            for i in range(p0 // PAGE, (p0 + n - 1) // PAGE + 1 if n else 0):
                page = int(table[entry][i])
                lo, hi = max(0, p0 - i * PAGE), min(PAGE, p0 + n - i * PAGE)
                r = at + i * PAGE + lo - p0
                for side, src in enumerate((k, v)):
                    new = src[r:r + hi - lo].double().view(hi - lo, self.heads, self.dh)
                    for h in range(self.heads):
                        self._page(side, page, h, lo, hi, new[:, h])
            at += n

    def _page(self, side, page, h, lo, hi, new):
        amax = float(new.abs().max())
        x = self.x[side][page, h]
        if not math.isfinite(amax) or (lo and math.isnan(float(self.e[side][page, h]))):
            self.e[side][page, h] = math.nan
            x[:hi] = math.nan
            return
        e = exponent(amax, self.kind)
        if lo:
            e = max(e, int(self.e[side][page, h]))
            x[:lo] = code(x[:lo] * 2.0 ** -e, self.kind) * 2.0 ** e
        x[lo:hi] = code(new * 2.0 ** -e, self.kind) * 2.0 ** e
        self.e[side][page, h] = e

    def read(self, table, pos0, rows):
        out = ([], [])
        for entry, (p0, n) in enumerate(zip(pos0, rows)):
            for t in range(p0, p0 + n):
                for side in range(2):
                    out[side].append(self.x[side][int(table[entry][t // PAGE]), :, t % PAGE].reshape(-1))
        empty = torch.zeros(0, self.heads * self.dh, dtype=torch.float64)
        return tuple(torch.stack(o) if o else empty for o in out)

    def attention(self, q, table, ctx, rows, nh, scale):
        """``(o, a)``: outputs and the sums of weight times |value|, that bound rounding of weights."""
        g = nh // self.heads
        o = torch.zeros(q.shape[0], nh, self.dh, dtype=torch.float64)
        a = torch.zeros_like(o)
        x = q.double().view(q.shape[0], nh, self.dh)
        at = 0
        for entry, (c, n) in enumerate(zip(ctx, rows)):
            pages = [int(table[entry][i]) for i in range((c + PAGE - 1) // PAGE)]
            for h in range(self.heads):
                if c < 1:
                    continue
                k = torch.cat([self.x[0][p, h] for p in pages])
                v = torch.cat([self.x[1][p, h] for p in pages])
                for i in range(n):
                    seen = c - n + i + 1
                    if seen < 1:
                        continue
                    s = x[at + i, h * g:(h + 1) * g] @ k[:seen].T * scale
                    w = torch.softmax(s, -1)
                    o[at + i, h * g:(h + 1) * g] = w @ v[:seen]
                    a[at + i, h * g:(h + 1) * g] = w @ v[:seen].abs()
            at += n
        return o.reshape(q.shape[0], -1), a.reshape(q.shape[0], -1)


def beam_step(logits, scores, done, eos):
    """``(scores, parent, token, done)`` of one request's ``K`` beams, by sorting everything."""
    K, V = logits.shape
    items = []
    for j in range(K):
        s = float(scores[j])
        if bool(done[j]):
            if eos is not None and s > -math.inf:
                items.append((-s, j * V + eos))
            continue
        x = logits[j].double()
        val = (s + (x - torch.logsumexp(x, 0))).tolist()
        items += [(-v, j * V + t) for t, v in enumerate(val) if v > -math.inf]
    items.sort()
    out = []
    for i in range(K):
        if i < len(items):
            v, at = items[i]
            j, t = divmod(at, V)
            out.append((-v, j, t, bool(done[j]) or t == eos))
        else:
            out.append((-math.inf, i, eos or 0, True))
    return out


def beam_pages(table, parent, n, pool):
    """New rows and copies ``[(src, dst), ...]`` (``None``: none) of one request."""
    lp, rest = divmod(n, PAGE)
    new = [list(r) for r in table]
    held = set()
    for j, p in enumerate(parent):
        new[j][:lp] = table[p][:lp]
        held.update(table[p][:lp])
        if rest and p not in parent[:j]:
            new[j][lp] = table[p][lp]
            held.add(table[p][lp])
    moves = []
    for j, p in enumerate(parent):
        if rest and p not in parent[:j]:
            moves.append(None)
            continue
        page = next(x for x in pool if x not in held)
        held.add(page)
        new[j][lp] = page
        moves.append((table[p][lp], page) if rest else None)
    return new, moves
