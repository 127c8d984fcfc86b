"""Workloads of the operators that decode several continuations of a request from a cache in 8 bits.

Four operators: appending keys and values to a paged cache in 8 bits (``write``, followed by the
read that hands the stored values back), attention over that cache (``attend``), the selection of
a beam search (``select``) and the re-parenting of the beams' pages (``reorder``).

A page holds 64 tokens.  Keys are kept as ``[page, head, dh / 64, token, 64]`` codes, values as
``[page, head, dh, token]`` codes, with one power of two per page and head as the scale of each.
"""
import math

import torch

own = False          # False: plain torch operations; True: the framework's kernels

PAGE = 64
QMAX = {"int8": 127.0, "e4m3": 448.0}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One new token per sequence of a batch that is decoding, somewhere inside a page: the
        # page's scale may have to grow.  16 heads of 64: the repository's 250M decoder.
        dict(name="write_tokens", op="write", kind="int8", nkv=16, dh=64, n=64, lo=1, hi=1,
             at_lo=65, at_hi=2000),
        # Prompts of different lengths, from the first position.
        dict(name="write_prompts", op="write", kind="e4m3", nkv=8, dh=128, n=16, lo=37, hi=2049,
             at_lo=0, at_hi=0),
        # One short conversation: latency.
        dict(name="attend_one_short", op="attend", kind="int8", nh=16, nkv=16, dh=64, n=1, lo=1,
             hi=1, ctx_lo=300, ctx_hi=300),
        # A decoding batch of a multi-head model (the 250M decoder's heads), moderate contexts.
        dict(name="attend_heads64", op="attend", kind="int8", nh=16, nkv=16, dh=64, n=64, lo=1,
             hi=1, ctx_lo=17, ctx_hi=2050),
        # A decoding batch with grouped heads and long, unequal contexts.
        dict(name="attend_grouped", op="attend", kind="int8", nh=32, nkv=8, dh=128, n=64, lo=1,
             hi=1, ctx_lo=1000, ctx_hi=8200),
        # One sequence with a very long context: the axis has to be split.
        dict(name="attend_one_long", op="attend", kind="e4m3", nh=32, nkv=8, dh=128, n=1, lo=1,
             hi=1, ctx_lo=131071, ctx_hi=131071),
        # A few new tokens per sequence: drafts that are checked, short turns.
        dict(name="attend_few_rows", op="attend", kind="e4m3", nh=32, nkv=8, dh=128, n=24, lo=1,
             hi=9, ctx_lo=500, ctx_hi=4100),
        # Portions of prompts that continue a cached prefix.
        dict(name="attend_portions", op="attend", kind="int8", nh=32, nkv=8, dh=128, n=4, lo=301,
             hi=700, ctx_lo=2000, ctx_hi=8200),
        # One request, four beams.
        dict(name="select_one", op="select", dtype="bf16", b=1, k=4, v=32000, first=False),
        # A batch of requests with eight beams over a large vocabulary in fp32.
        dict(name="select_batch", op="select", dtype="fp32", b=32, k=8, v=100003, first=False),
        # One request's four beams, two layers in 8 bits.
        dict(name="reorder_one", op="reorder", kind="int8", nkv=8, dh=128, b=1, k=4, moved=2,
             layers=2, lo=700, hi=700, room=3, edge=False),
        # A batch of beams over a cache of eight bf16 tensors.
        dict(name="reorder_batch", op="reorder", kind="bf16", nkv=8, dh=128, b=16, k=8, moved=4,
             layers=4, lo=130, hi=1500, room=5, edge=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["write", "attend", "attend", "attend", "select", "reorder"])
    kind = rng.choice(["int8", "e4m3"])
    dh = rng.choice([64, 128])
    if op == "write":
        nkv = _log(rng, 1, 16)
        n = _log(rng, 1, 64)
        hi = 1 if rng.random() < 0.3 else _log(rng, 2, max(2, 16384 // n))
        at = 0 if rng.random() < 0.3 else _log(rng, 1, 2000)
        return dict(op=op, kind=kind, nkv=nkv, dh=dh, n=n, lo=rng.randint(1, hi), hi=hi,
                    at_lo=at // 3, at_hi=at)
    if op == "attend":
        nkv = _log(rng, 1, 16)
        group = rng.choice([1, 2, 3, 4, 5, 8, 16])
        while nkv * group > 64:
            group = max(1, group // 2)
        shape = rng.choice(["tokens", "tokens", "few", "portions"])
        budget = 2 ** 19 * 8 * 128                    # cached numbers, as in the largest case
        if shape == "tokens":
            n = _log(rng, 1, 96)
            lo = hi = 1
        elif shape == "few":
            n = _log(rng, 1, 48)
            hi = rng.randint(2, 16)
            lo = rng.randint(1, hi)
        else:
            n = _log(rng, 1, 6)
            hi = _log(rng, 17, 700)
            lo = rng.randint(1, hi)
        most = max(2, min(131072 if hi == 1 else 8200, budget // (n * nkv * dh)))
        ctx_hi = max(hi, _log(rng, 1, most))
        return dict(op=op, kind=kind, nh=nkv * group, nkv=nkv, dh=dh, n=n, lo=lo, hi=hi,
                    ctx_lo=max(hi, rng.randint(1, ctx_hi)), ctx_hi=ctx_hi)
    if op == "select":
        k = rng.randint(1, 16)
        b = _log(rng, 1, 64)
        v = _log(rng, 5, max(5, min(131072, 25_000_000 // (b * k))))
        return dict(op=op, dtype=rng.choice(["bf16", "fp32"]), b=b, k=k, v=v,
                    first=rng.random() < 0.25)
    k = rng.randint(1, 12)
    hi = _log(rng, 1, 2000)
    b = _log(rng, 1, 16)
    return dict(op=op, kind=rng.choice(["bf16", "int8", "e4m3"]), nkv=_log(rng, 1, 8), dh=dh, b=b,
                k=k, moved=rng.randint(0, k - 1), layers=rng.randint(1, 4), lo=rng.randint(1, hi),
                hi=hi, room=rng.randint(2, 5), edge=b > 1 and rng.random() < 0.5)


def _spread(lo, hi, n):
    """``n`` whole numbers from ``hi`` down to ``lo``, evenly."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _pages(n):
    return (n + PAGE - 1) // PAGE


def work(case):
    op = case["op"]
    if op == "write":
        rows = sum(_spread(case["lo"], case["hi"], case["n"]))
        kept = sum(a % PAGE for a in _spread(case["at_lo"], case["at_hi"], case["n"]))
        num = case["nkv"] * case["dh"] * 2
        return {"bytes": num * (rows * (2 + 1) + (rows + kept) * (1 + 2)),
                "flops": num * (rows * 3 + (rows + kept))}
    if op == "attend":
        rows = _spread(case["lo"], case["hi"], case["n"])
        ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["n"])
        seen = sum(r * c - r * (r - 1) // 2 for r, c in zip(rows, ctx))
        return {"bytes": sum(ctx) * case["nkv"] * case["dh"] * 2
                + sum(rows) * case["nh"] * case["dh"] * 4,
                "flops": 4 * seen * case["nh"] * case["dh"]}
    if op == "select":
        size = 2 if case["dtype"] == "bf16" else 4
        live = case["b"] * (1 if case["first"] else _live(case["k"]))
        return {"bytes": live * case["v"] * size + case["b"] * case["k"] * 29,
                "flops": live * case["v"] * 3}
    groups = case["b"] - (1 if case["edge"] else 0)
    page = case["nkv"] * PAGE * case["dh"] * (2 if case["kind"] == "bf16" else 1)
    width = _pages(case["hi"]) + case["room"]
    tails = 0 if case["kind"] == "bf16" else \
        case["b"] * case["k"] * PAGE * case["nkv"] * case["dh"] * case["layers"] * 2 * 2
    return {"bytes": 2 * groups * case["moved"] * page * case["layers"] * 2 + tails
            + case["b"] * case["k"] * width * 8, "flops": 0}


def _live(k):
    """Beams of a request that have not ended: all but a quarter."""
    return max(1, k - k // 4)


# ------------------------------------------------------------------------------------ inputs
def _exponent(amax, kind):
    """Smallest e with amax <= QMAX 2^e."""
    m, x = torch.frexp(amax)
    if kind == "int8":
        e = x - 7 + (m > 127.0 / 128.0).to(x.dtype)
    else:
        e = x - 9 + (m > 0.875).to(x.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, -126)).clamp_min(-126)


def _encode(x, e, kind):
    """fp32 values to codes (still as fp32 numbers) under the exponent ``e``."""
    y = torch.ldexp(x, -e)
    return y.round() if kind == "int8" else y.to(torch.float8_e4m3fn).float()


def _dtype(kind):
    return torch.int8 if kind == "int8" else torch.float8_e4m3fn


def _cache(gen, pages, nkv, dh, kind, keys):
    """Random stored content: codes ``[pages, nkv, 64, dh]`` and scales ``[pages, nkv]``; channels
    differ in size, as they do behind a projection."""
    dev = gen.device
    channel = torch.exp(0.5 * torch.randn(nkv, 1, dh, generator=gen, device=dev))
    codes = torch.empty((pages, nkv, PAGE, dh), dtype=torch.int8, device=dev)
    scale = torch.empty((pages, nkv), dtype=torch.float32, device=dev)
    step = max(1, (1 << 26) // (nkv * PAGE * dh))
    for p in range(0, pages, step):
        q = min(pages, p + step)
        x = torch.randn(q - p, nkv, PAGE, dh, generator=gen, device=dev) * channel
        e = _exponent(x.abs().amax((2, 3)), kind)
        c = _encode(x, e[:, :, None, None], kind)
        codes[p:q] = c.to(torch.int8) if kind == "int8" else \
            c.to(torch.float8_e4m3fn).view(torch.int8)
        scale[p:q] = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
    if keys:
        laid = codes.view(pages, nkv, PAGE, dh // 64, 64).transpose(2, 3).contiguous()
    else:
        laid = codes.transpose(2, 3).contiguous()
    return laid.view(_dtype(kind)), scale


def _unlay(codes, keys):
    """Stored codes to fp32 numbers ``[pages, nkv, 64, dh]`` (without their scale)."""
    x = codes.float()
    if keys:
        return x.transpose(2, 3).reshape(x.shape[0], x.shape[1], PAGE, -1)
    return x.transpose(2, 3)


def _pick(codes, index):
    """Pages of an 8-bit tensor (torch does not index its 8-bit floating type)."""
    return codes.view(torch.int8)[index].view(codes.dtype)


def _tables(gen, need, width, spare=3):
    """Page tables ``[n, width]`` over a pool in random order; unused places hold page 0."""
    total = sum(need) + spare
    perm = torch.randperm(total, generator=gen, device=gen.device).to(torch.int32)
    table = torch.zeros((len(need), width), dtype=torch.int32, device=gen.device)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = perm[at:at + c]
        at += c
    return table, total


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _shuffled(values, seed, salt):
    order = torch.randperm(len(values), generator=torch.Generator().manual_seed(seed * 31 + salt))
    return [values[i] for i in order.tolist()]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    return globals()["_prepare_" + case["op"]](case, seed, dev, gen)


def _prepare_write(case, seed, dev, gen):
    kind, nkv, dh, n = case["kind"], case["nkv"], case["dh"], case["n"]
    rows = _shuffled(_spread(case["lo"], case["hi"], n), seed, 1)
    at = _shuffled(_spread(case["at_lo"], case["at_hi"], n), seed, 2)
    need = [_pages(a + r) for a, r in zip(at, rows)]
    table, total = _tables(gen, need, max(need) + 1)
    kc, ks = _cache(gen, total, nkv, dh, kind, True)
    vc, vs = _cache(gen, total, nkv, dh, kind, False)
    row0 = _starts(rows)
    # keys and values are columns of one projection's output, larger for some sequences
    qkv = torch.randn(row0[-1], 3 * nkv * dh, generator=gen, device=dev)
    size = torch.exp(0.7 * torch.randn(n, generator=gen, device=dev))
    qkv = (qkv * size.repeat_interleave(torch.tensor(rows, device=dev))[:, None]).bfloat16()
    begin = [a // PAGE * PAGE for a in at]              # read back from the first page written
    back = [a + r - s for a, r, s in zip(at, rows, begin)]
    # the places of the pages written, for the plain form
    entry, page, first = [], [], []
    for i in range(n):
        for p in range(at[i] // PAGE, need[i]):
            entry.append(i)
            page.append(p)
            first.append(max(0, at[i] - p * PAGE))
    index = torch.tensor([entry, page, first], dtype=torch.int64).to(dev)
    return dict(op="write", kind=kind, nkv=nkv, dh=dh, k=qkv[:, nkv * dh:2 * nkv * dh],
                v=qkv[:, 2 * nkv * dh:], kc=kc, ks=ks, vc=vc, vs=vs, table=table,
                row0=_ints(row0, dev), pos0=_ints(at, dev), most=max(rows),
                tokens=n if max(rows) == 1 else 0, begin=_ints(begin, dev),
                back0=_ints(_starts(back), dev), back=sum(back), back_most=max(back),
                written=index)


def _prepare_attend(case, seed, dev, gen):
    kind, nh, nkv, dh, n = (case[x] for x in ("kind", "nh", "nkv", "dh", "n"))
    both = list(zip(_spread(case["lo"], case["hi"], n), _spread(case["ctx_lo"], case["ctx_hi"], n)))
    both = _shuffled(both, seed, 1)
    rows, ctx = [r for r, _ in both], [c for _, c in both]
    need = [_pages(c) for c in ctx]
    table, total = _tables(gen, need, max(need) + 1)
    kc, ks = _cache(gen, total, nkv, dh, kind, True)
    vc, vs = _cache(gen, total, nkv, dh, kind, False)
    row0 = _starts(rows)
    q = torch.randn(row0[-1], (nh + 2 * nkv) * dh, generator=gen, device=dev).bfloat16()
    return dict(op="attend", nh=nh, nkv=nkv, dh=dh, q=q[:, :nh * dh], kc=kc, ks=ks, vc=vc, vs=vs,
                table=table, ctx=_ints(ctx, dev), row0=_ints(row0, dev), most=max(rows),
                one=max(rows) == 1, host=(rows, ctx))


def _prepare_select(case, seed, dev, gen):
    b, k, v = case["b"], case["k"], case["v"]
    # a few likely tokens above a broad rest
    x = 2.0 * torch.randn(b * k, v, generator=gen, device=dev)
    hot = torch.randint(0, v, (b * k, 12), generator=gen, device=dev)
    x.scatter_add_(1, hot, 6.0 + 4.0 * torch.rand(b * k, 12, generator=gen, device=dev))
    logits = x.bfloat16() if case["dtype"] == "bf16" else x
    done = torch.zeros((b, k), dtype=torch.bool, device=dev)
    if case["first"]:
        scores = torch.full((b, k), -math.inf, device=dev)
        scores[:, 0] = 0.0
    else:
        scores = -4.0 - 3.0 * torch.rand(b, k, generator=gen, device=dev).sort(1).values
        done[:, k - (k - _live(k)):] = True
        done = done[:, torch.randperm(k, generator=gen, device=dev)].contiguous()
    return dict(op="select", logits=logits, scores=scores, done=done, eos=min(2, v - 1))


def _prepare_reorder(case, seed, dev, gen):
    b, k, nkv, dh, kind = (case[x] for x in ("b", "k", "nkv", "dh", "kind"))
    lens = [x + 1 if x % PAGE == 0 else x for x in _spread(case["lo"], case["hi"], b)]
    if case["edge"]:
        lens[0] = max(PAGE, lens[0] // PAGE * PAGE)
    lens = _shuffled(lens, seed, 1)
    width = _pages(max(lens)) + case["room"]
    # every beam's pages: the prompt's are shared, the last `room - 1` and the tail are its own
    shared = [max(0, _pages(x) - (case["room"] - 1)) for x in lens]
    own_pages = [_pages(x) - s for x, s in zip(lens, shared)]
    pool = k * (case["room"] + 1)
    total = sum(shared) + b * pool + 2
    perm = torch.randperm(total, generator=gen, device=dev).to(torch.int32).cpu()
    table = torch.zeros((b, k, width), dtype=torch.int32)
    pools, at = [], 0
    for i in range(b):
        table[i, :, :shared[i]] = perm[at:at + shared[i]]
        at += shared[i]
        mine = perm[at:at + pool]
        at += pool
        pools.append(mine)
        for j in range(k):
            table[i, j, shared[i]:_pages(lens[i])] = mine[j * own_pages[i]:(j + 1) * own_pages[i]]
    table = table.to(dev)
    # `moved` beams of a request go on from a beam that another one goes on from too
    rnd = torch.Generator().manual_seed(seed * 31 + 7)
    parents = []
    for i in range(b):
        kept = torch.randperm(k, generator=rnd)[:k - case["moved"]]
        more = kept[torch.randint(0, len(kept), (case["moved"],), generator=rnd)]
        both = torch.cat([kept, more])
        parents.append(both[torch.randperm(k, generator=rnd)])
    caches = []
    for _ in range(case["layers"]):
        if kind == "bf16":
            caches += [torch.randn(total, PAGE, nkv, dh, generator=gen, device=dev).bfloat16()
                       for _ in range(2)]
        else:
            for keys in (True, False):
                caches += list(_cache(gen, total, nkv, dh, kind, keys))
    first = [x // PAGE * PAGE for x in lens for _ in range(k)]
    tail = [x % PAGE for x in lens for _ in range(k)]
    return dict(op="reorder", kind=kind, table=table.view(b * k, width),
                parent=torch.stack(parents).to(dev), length=_ints(lens, dev),
                pool=torch.stack(pools).to(dev), caches=caches, begin=_ints(first, dev),
                back0=_ints(_starts(tail), dev), back=sum(tail),
                where=torch.tensor([[i, t] for i, c in enumerate(tail) for t in range(c)],
                                   dtype=torch.int64).reshape(-1, 2).to(dev))


# ------------------------------------------------------------------------------------ passes
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["op"]](state)


def _own_write(s):
    from coeus_b200.ops import kv8
    kv8.kv8_write(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["pos0"],
                  row0=None if s["tokens"] else s["row0"], max_rows=s["most"])
    return kv8.kv8_read(s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["begin"], s["back0"],
                        s["back"], max_rows=s["back_most"])


def _plain_write(s):
    kind, nkv, dh = s["kind"], s["nkv"], s["dh"]
    entry, lp, first = s["written"]
    pages = s["table"][entry, lp].long()
    row0, pos0 = s["row0"].long(), s["pos0"].long()
    offset = torch.arange(PAGE, device=pages.device)
    # the row of every place of every written page
    place = lp[:, None] * PAGE + offset[None]
    row = row0[entry][:, None] + place - pos0[entry][:, None]
    new = (place >= pos0[entry][:, None]) & (row < row0[entry + 1][:, None])
    kept = (offset[None] < first[:, None])[:, None, :, None]
    row = row.clamp(0, s["k"].shape[0] - 1)
    for x, codes, scale, keys in ((s["k"], s["kc"], s["ks"], True),
                                  (s["v"], s["vc"], s["vs"], False)):
        y = x.float().view(-1, nkv, dh)[row].transpose(1, 2)        # [written, nkv, 64, dh]
        y = torch.where(new[:, None, :, None], y, torch.zeros_like(y))
        e = _exponent(y.abs().amax((2, 3)), kind)
        before = torch.frexp(scale[pages])[1] - 1
        e = torch.where(first[:, None] > 0, torch.maximum(e, before), e)
        old = _unlay(_pick(codes, pages), keys)
        shifted = _encode(old, (e - before)[:, :, None, None], kind)
        c = torch.where(new[:, None, :, None], _encode(y, e[:, :, None, None], kind),
                        torch.where(kept, shifted, old))
        if keys:
            c = c.view(-1, nkv, PAGE, dh // 64, 64).transpose(2, 3)
        else:
            c = c.transpose(2, 3)
        c = c.to(torch.int8) if kind == "int8" else c.to(torch.float8_e4m3fn).view(torch.int8)
        codes.view(torch.int8)[pages] = c
        scale[pages] = torch.ldexp(torch.ones_like(scale[pages]), e)
    out = []
    begin, back0 = s["begin"].long(), s["back0"].long()
    rows = torch.arange(s["back"], device=pages.device)
    entry = torch.searchsorted(back0, rows, right=True) - 1
    place = begin[entry] + rows - back0[entry]
    page = s["table"][entry, place // PAGE].long()
    for codes, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        values = torch.empty((s["back"], nkv * dh), dtype=torch.bfloat16, device=pages.device)
        for r in range(0, s["back"], 4096):                          # bounds the memory
            cut = slice(r, min(s["back"], r + 4096))
            pg, off = page[cut], place[cut] % PAGE
            raw = codes.view(torch.int8)
            c = raw[pg, :, :, off]         # [rows, nkv, dh / 64, 64] of keys, [rows, nkv, dh]
            c = c.contiguous().view(codes.dtype).float().reshape(pg.numel(), nkv, dh)
            values[cut] = (c * scale[pg][:, :, None]).reshape(pg.numel(), -1).bfloat16()
        out.append(values)
    return tuple(out)


def _own_attend(s):
    from coeus_b200.ops import kv8
    return kv8.kv8_attention(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["ctx"],
                             s["nh"], row0=None if s["one"] else s["row0"], max_rows=s["most"])


def _plain_attend(s):
    nh, nkv, dh = s["nh"], s["nkv"], s["dh"]
    out = torch.empty((s["q"].shape[0], nh * dh), dtype=torch.bfloat16, device=s["q"].device)
    at = 0
    for i, (r, c) in enumerate(zip(*s["host"])):
        pages = s["table"][i, :_pages(c)].long()
        k = _unlay(_pick(s["kc"], pages), True) * s["ks"][pages][:, :, None, None]
        v = _unlay(_pick(s["vc"], pages), False) * s["vs"][pages][:, :, None, None]
        k = k.transpose(0, 1).reshape(nkv, -1, dh)[:, :c]            # [nkv, c, dh]
        v = v.transpose(0, 1).reshape(nkv, -1, dh)[:, :c]
        q = s["q"][at:at + r].float().view(r, nkv, nh // nkv, dh).permute(1, 2, 0, 3)
        x = torch.matmul(q, k[:, None].transpose(-1, -2)) / math.sqrt(dh)
        place = torch.arange(c, device=q.device)
        mine = torch.arange(c - r, c, device=q.device)
        x = x.masked_fill(place[None] > mine[:, None], -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(p, v[:, None]) / p.sum(-1, keepdim=True)
        out[at:at + r] = o.permute(2, 0, 1, 3).reshape(r, nh * dh).bfloat16()
        at += r
    return out


def _own_select(s):
    from coeus_b200.ops import beam
    return beam.beam_select(s["logits"], s["scores"], s["done"], s["eos"])


def _plain_select(s):
    b, k = s["scores"].shape
    x = s["logits"].double().view(b, k, -1)
    v = x.shape[-1]
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    total = s["scores"].double()[:, :, None] + (x - lse)
    token = torch.arange(v, device=x.device)
    ended = torch.where(token == s["eos"], s["scores"].double()[:, :, None],
                        torch.full_like(total, -math.inf))
    total = torch.where(s["done"][:, :, None], ended, total).view(b, k * v)
    best, where = torch.sort(total, dim=-1, descending=True, stable=True)
    best, where = best[:, :k], where[:, :k]
    parent, tok = where // v, where % v
    empty = best == -math.inf
    parent = torch.where(empty, torch.arange(k, device=x.device)[None], parent)
    tok = torch.where(empty, torch.full_like(tok, s["eos"]), tok)
    done = torch.gather(s["done"], 1, parent) | (tok == s["eos"]) | empty
    return best.float(), parent, tok, done


def _own_reorder(s):
    from coeus_b200.ops import beam, kv8
    table = beam.beam_reorder(s["table"], s["parent"], s["length"], s["pool"], s["caches"])
    if s["kind"] == "bf16":
        return [table] + s["caches"]
    out = [table]
    for l in range(0, len(s["caches"]), 4):
        kc, ks, vc, vs = s["caches"][l:l + 4]
        out += kv8.kv8_read(kc, vc, ks, vs, table, s["begin"], s["back0"], s["back"],
                            max_rows=PAGE)
    return out


def _plain_reorder(s):
    b, k = s["parent"].shape
    old = s["table"].view(b, k, -1)
    width = old.shape[-1]
    dev = old.device
    lp = (s["length"] // PAGE).long()[:, None]
    partial = (s["length"] % PAGE != 0)[:, None]
    column = torch.arange(width, device=dev)
    from_parent = torch.gather(old, 1, s["parent"][:, :, None].expand(b, k, width))
    table = torch.where(column[None, None] < lp[:, :, None], from_parent, old)
    tail = torch.gather(from_parent, 2, lp[:, :, None].expand(b, k, 1))[:, :, 0]
    same = s["parent"][:, :, None] == s["parent"][:, None, :]         # [b, child, other child]
    earlier = torch.arange(k, device=dev)[None, :] < torch.arange(k, device=dev)[:, None]
    keeps = ~(same & earlier[None]).any(-1) & partial
    # the pool's pages that no new row holds, in the pool's order
    held = torch.where((column[None, None] < lp[:, :, None]), table, torch.full_like(table, -1))
    held = torch.cat([held, torch.where(keeps, tail, torch.full_like(tail, -1))[:, :, None]], -1)
    used = (s["pool"][:, :, None] == held.view(b, 1, -1)).any(-1)
    rank = torch.cumsum((~used).long(), 1) - 1
    want = torch.cumsum((~keeps).long(), 1) - 1                       # the child's turn
    hit = (~used)[:, None, :] & (rank[:, None, :] == want[:, :, None])
    fresh = torch.gather(s["pool"], 1, hit.long().argmax(-1))
    here = torch.where(keeps, tail, fresh)
    table.scatter_(2, lp[:, :, None].expand(b, k, 1), here[:, :, None])
    src = torch.where(partial, tail, here).long().view(-1)            # nothing to copy: itself
    dst = here.long().view(-1)
    for c in s["caches"]:
        raw = c.view(torch.int8) if c.element_size() == 1 else c
        raw[dst] = raw[src]
    table = table.view(b * k, width)
    if s["kind"] == "bf16":
        return [table] + s["caches"]
    out = [table]
    beam, off = s["where"][:, 0], s["where"][:, 1]
    page = table[beam, (s["begin"].long() // PAGE)[beam]].long()
    for l in range(0, len(s["caches"]), 4):
        for codes, scale in (s["caches"][l:l + 2], s["caches"][l + 2:l + 4]):
            nkv = scale.shape[1]
            c = codes.view(torch.int8)[page, :, :, off].contiguous().view(codes.dtype).float()
            c = c.reshape(page.numel(), nkv, -1) * scale[page][:, :, None]
            out.append(c.reshape(page.numel(), -1).bfloat16())
    return out


# --------------------------------------------------------------------------- definition, 64 bits
def exact(case, seed):
    return globals()["_exact_" + case["op"]](prepare(case, seed))


def _code64(y, kind):
    """Round ``y`` (64 bits) to the code it gets, ties to even."""
    if kind == "int8":
        return torch.round(y)
    a = y.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(y) * torch.round(a / step) * step


def _need64(a, kind):
    if a == 0.0:
        return -126
    e = math.frexp(a)[1] - 10
    while a > QMAX[kind] * 2.0 ** e:
        e += 1
    return max(e, -126)


def _exact_write(s):
    kind, nkv, dh = s["kind"], s["nkv"], s["dh"]
    n = s["pos0"].numel()
    if s["row0"][-1].item() * nkv > 400_000:
        return None
    row0, pos0 = s["row0"].tolist(), s["pos0"].tolist()
    begin = s["begin"].tolist()
    parts = ([], [])
    for i in range(n):
        r = row0[i + 1] - row0[i]
        for side, (x, codes, scale) in enumerate(((s["k"], s["kc"], s["ks"]),
                                                  (s["v"], s["vc"], s["vs"]))):
            x = x[row0[i]:row0[i + 1]].double().view(r, nkv, dh)
            for p in range(begin[i] // PAGE, _pages(pos0[i] + r)):
                page = int(s["table"][i, p])
                lo = max(0, pos0[i] - p * PAGE)
                hi = min(PAGE, pos0[i] + r - p * PAGE)
                new = x[p * PAGE + lo - pos0[i]:p * PAGE + hi - pos0[i]]
                amax = new.abs().amax((0, 2)).tolist()
                e = torch.tensor([_need64(a, kind) for a in amax], dtype=torch.float64)
                if lo:
                    before = torch.log2(scale[page].double().cpu())
                    e = torch.maximum(e, before)
                unit = torch.exp2(e).to(x.device)
                got = [_code64(new / unit[None, :, None], kind) * unit[None, :, None]]
                if lo:
                    c = codes[page].float().double()
                    c = c.transpose(1, 2).reshape(nkv, PAGE, dh) if side == 0 else c.transpose(1, 2)
                    up = torch.exp2(before.to(x.device)) / unit
                    c = _code64(c * up[:, None, None], kind) * unit[:, None, None]
                    got.insert(0, c.transpose(0, 1)[:lo])
                parts[side].append(torch.cat(got).reshape(hi, nkv * dh))
    return tuple(torch.cat(p) for p in parts)


def _exact_attend(s):
    nh, nkv, dh = s["nh"], s["nkv"], s["dh"]
    g = nh // nkv
    out = torch.zeros((s["q"].shape[0], nkv, g, dh), dtype=torch.float64, device=s["q"].device)
    at = 0
    for i, (r, c) in enumerate(zip(*s["host"])):
        pages = s["table"][i, :_pages(c)].long()
        for h in range(nkv):
            k = s["kc"].view(torch.int8)[pages, h].view(s["kc"].dtype).double()
            k = k.permute(0, 2, 1, 3).reshape(-1, PAGE, dh) * s["ks"][pages, h].double()[:, None, None]
            v = s["vc"].view(torch.int8)[pages, h].view(s["vc"].dtype).double()
            v = v * s["vs"][pages, h].double()[:, None, None]
            k = k.reshape(-1, dh)[:c]
            v = v.permute(0, 2, 1).reshape(-1, dh)[:c]
            q = s["q"][at:at + r].double().view(r, nkv, g, dh)[:, h].reshape(r * g, dh)
            x = (q @ k.T) * dh ** -0.5
            last = c - r + torch.arange(r, device=x.device).repeat_interleave(g)
            x[torch.arange(c, device=x.device)[None] > last[:, None]] = -math.inf
            out[at:at + r, h] = (torch.softmax(x, -1) @ v).view(r, g, dh)
        at += r
    return out.view(-1, nh * dh)


def _exact_select(s):
    b, k = s["scores"].shape
    v = s["logits"].shape[-1]
    best = torch.full((b, k), -math.inf, dtype=torch.float64)
    parent = torch.arange(k).repeat(b, 1)
    token = torch.full((b, k), s["eos"], dtype=torch.int64)
    done = torch.ones((b, k), dtype=torch.bool)
    for i in range(b):
        x = s["logits"][i * k:(i + 1) * k].double()
        total = s["scores"][i].double()[:, None] + torch.log_softmax(x, -1)
        for j in s["done"][i].nonzero()[:, 0].tolist():
            total[j] = -math.inf
            total[j, s["eos"]] = s["scores"][i, j].double()
        total = total.view(-1)
        for n in range(k):
            top = total.max()
            if not top > -math.inf:
                break
            at = int((total == top).nonzero()[0, 0])
            total[at] = -math.inf
            best[i, n], parent[i, n], token[i, n] = float(top), at // v, at % v
            done[i, n] = bool(s["done"][i, at // v]) or at % v == s["eos"]
    dev = s["scores"].device
    return best.to(dev), parent.to(dev), token.to(dev), done.to(dev)


def _exact_reorder(s):
    b, k = s["parent"].shape
    old = s["table"].view(b, k, -1).tolist()
    new = [[list(r) for r in rows] for rows in old]
    for i in range(b):
        n = int(s["length"][i])
        lp = n // PAGE
        parent = s["parent"][i].tolist()
        held, wanting = set(), []
        for j, p in enumerate(parent):
            new[i][j][:lp] = old[i][p][:lp]
            held.update(new[i][j][:lp])
            if n % PAGE and p not in parent[:j]:
                new[i][j][lp] = old[i][p][lp]
                held.add(old[i][p][lp])
            else:
                wanting.append(j)
        free = [x for x in s["pool"][i].tolist() if x not in held]
        for j, page in zip(wanting, free):
            new[i][j][lp] = page
    table = torch.tensor(new, dtype=torch.int32, device=s["table"].device).view(b * k, -1)
    return [table] + [None] * (len(s["caches"]) if s["kind"] == "bf16"
                               else len(s["caches"]) // 2)
