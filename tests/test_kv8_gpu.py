"""The kernels of the 8-bit cache against its definition in 64 bits."""
import math

import pytest
import torch

from coeus_b200.ops import _lib, kv8
from kv8_cases import Case, i32, starts

pytestmark = pytest.mark.gpu
DEV = "cuda"


def status():
    torch.cuda.synchronize()
    s = _lib.status_buffer(torch.device("cuda", 0))
    code = int(s[0])
    s.zero_()
    return code


KINDS = ["int8", "e4m3"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dh", [(1, 64), (3, 64), (2, 128)])
def test_write_and_read(kind, heads, dh):
    c = Case(kind, heads, dh, [70, 300, 5, 64], DEV)
    c.write([0] * 4, [64, 130, 0, 64])
    c.write([64, 130, 0, 0], [1, 1, 1, 1])
    c.write([65, 131, 1, 1], [1, 1, 1, 1], sizes=[9.0, 40.0, 0.01, 1e4])
    c.write([66, 132, 2, 2], [4, 168, 3, 62], sizes=[100.0, 1.0, 1.0, 1e-3])
    c.check_read([0] * 4, [70, 300, 5, 64])
    c.check_read([63, 129, 4, 0], [3, 70, 1, 0])
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_write_extremes(kind):
    """Zeros, the smallest and largest magnitudes, values next to where the scale steps."""
    c = Case(kind, 2, 64, [64, 64, 64, 64], DEV)

    def edit(k, v):
        k[0:3] = 0.0
        k[3:6] *= 1e-38
        k[6:9] = k[6:9].float().mul(1e38).clamp(-3e38, 3e38).bfloat16()
        k[9:12] = 0.0
        k[9, 0], k[10, 64], k[11, 70] = 127.0, 127.5, -448.0
        v[9:12] = 0.0
        v[9, 0], v[10, 64], v[11, 70] = 448.0, 450.0, -896.0
    c.write([0] * 4, [3, 3, 3, 3], edit=edit)
    c.check_read([0] * 4, [3, 3, 3, 3])
    c.write([3] * 4, [2, 2, 2, 2])
    c.check_read([0] * 4, [5, 5, 5, 5])
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_not_a_number_makes_its_block_one(kind):
    c = Case(kind, 2, 64, [130], DEV)

    def edit(k, v):
        k[3, 5] = math.inf
        v[70, 64 + 2] = math.nan
    c.write([0], [128], edit=edit)
    c.write([128], [1])
    c.check_read([0], [129])
    # head 0 reads NaN keys, head 1 NaN values, but not with a context that ends before them
    o = c.check_attend([129], [1], 2)
    assert torch.isnan(o).all()
    o = c.check_attend([64], [3], 2)
    assert torch.isnan(o[:, :64]).all() and not torch.isnan(o[:, 64:]).any()
    # a row in front of the block is not touched by it
    o = c.check_attend([66], [4], 2)
    assert not torch.isnan(o[0:2, 64:]).any() and torch.isnan(o[2:, 64:]).all()
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nh,heads,dh", [(2, 2, 64), (16, 16, 64), (6, 2, 64), (7, 1, 128), (8, 1, 128),
                                         (9, 1, 64), (16, 1, 128), (24, 2, 128), (40, 1, 64)])
def test_attention_one_row(kind, nh, heads, dh):
    lens = [1, 63, 64, 65, 333, 3]
    c = Case(kind, heads, dh, lens, DEV)
    c.write([0] * 6, lens)
    c.check_attend(lens, [1] * 6, nh)
    c.check_attend([0, 62, 1, 64, 300, 0], [1] * 6, nh, scale=0.2)
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nh,heads,dh", [(2, 2, 64), (3, 1, 128), (8, 2, 128), (5, 1, 64)])
@pytest.mark.parametrize("rows", [[2, 0, 9, 1, 5], [1, 64, 17, 130, 40], [3, 3, 3, 3, 3]])
def test_attention_several_rows(kind, nh, heads, dh, rows):
    lens = [2, 64, 200, 131, 44]
    c = Case(kind, heads, dh, lens, DEV)
    c.write([0] * 5, lens)
    c.check_attend(lens, rows, nh)
    c.check_attend([1, 64, 199, 129, 0], rows, nh, max_rows=max(rows) + 70)
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_attention_long_context(kind):
    n = 20000
    c = Case(kind, 1, 128, [n, 64], DEV)
    c.write([0, 0], [n, 64])
    c.check_attend([n, 64], [1, 1], 4)
    c.check_attend([n - 63, 10], [3, 2], 4, size=3.0)
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dh,group,rows", [(6, 128, 3, 1), (6, 64, 1, 1), (3, 128, 3, 5), (4, 64, 4, 4)])
def test_attention_many_pages_per_block(kind, heads, dh, group, rows):
    """Enough pages that the ring of every block goes round several times, over several tiles."""
    n = 70
    lens = [1 + (i * 997) % 6000 for i in range(n)]
    c = Case(kind, heads, dh, lens, DEV)
    k = torch.randn(max(lens), heads * dh, generator=c.gen).bfloat16().to(DEV)
    v = torch.randn(max(lens), heads * dh, generator=c.gen).bfloat16().to(DEV)
    table = c.table.to(DEV)
    for e in range(n):
        kv8.kv8_write(k[:lens[e]], v[:lens[e]], *c.c, table[e:e + 1], i32([0], DEV),
                      row0=i32([0, lens[e]], DEV), max_rows=lens[e])
    counts = [1 if rows == 1 else min(1 + e % rows, lens[e]) for e in range(n)]
    q = torch.randn(sum(counts), heads * group * dh, generator=c.gen).bfloat16()
    got = c.attend(q, lens, counts, heads * group).double()
    # what the cache holds of the longest entry's first page differs from entry to entry only by
    # the scale of their last pages: read it back and compare in 64 bits
    at = 0
    for e in range(n):
        kk, vv = kv8.kv8_read(*c.c, table[e:e + 1], i32([0], DEV), i32([0, lens[e]], DEV), lens[e], lens[e])
        kk = kk.double().view(lens[e], heads, dh).transpose(0, 1)
        vv = vv.double().view(lens[e], heads, dh).transpose(0, 1)
        x = q[at:at + counts[e]].to(DEV).double().view(counts[e], heads, group, dh).permute(1, 2, 0, 3)
        s = torch.einsum("hgrd,hcd->hgrc", x, kk) * dh ** -0.5
        seen = torch.arange(lens[e], device=DEV)[None] <= (lens[e] - counts[e] + torch.arange(counts[e], device=DEV))[:, None]
        w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        want = torch.einsum("hgrc,hcd->rhgd", w, vv).reshape(counts[e], -1)
        spread = torch.einsum("hgrc,hcd->rhgd", w, vv.abs()).reshape(counts[e], -1)
        err = (got[at:at + counts[e]] - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * spread + 1e-30).all(), e
        at += counts[e]
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_attention_scales_apart(kind):
    """Pages whose values differ by 2^30, and a row that only listens to the small ones."""
    c = Case(kind, 1, 64, [192], DEV)
    c.write([0], [64], sizes=[3e4])
    c.write([64], [64], sizes=[3e-5])
    c.write([128], [64])
    c.check_attend([192], [1], 2, size=1e-4)
    c.check_attend([128], [3], 2, size=3e-4)
    # keys of the first page far below the others' scores
    c = Case(kind, 1, 64, [128], DEV)

    def edit(k, v):
        k[:64] = -2.0
        k[64:] = 2.0
        v[:64] *= 2.0 ** 15
        v[64:] *= 2.0 ** -15
    c.write([0], [128], edit=edit)
    q = torch.full((1, 64), 2.0, dtype=torch.bfloat16)
    got = c.attend(q, [128], [1], 1).double().cpu()
    want, spread = c.plain.attention(q, c.table, [128], [1], 1, 64 ** -0.5)
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread).all()
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_stale_codes_behind_the_context(kind):
    """What the last page holds behind the context is never used, whatever it is."""
    c = Case(kind, 1, 64, [70], DEV)
    c.write([0], [70])
    page = int(c.table[0, 1])
    c.c[0].view(torch.int8)[page, 0, 0, 6:] = 127         # e4m3: NaN
    c.c[1].view(torch.int8)[page, 0, :, 6:] = 127
    c.check_attend([70], [1], 2)
    c.check_attend([70], [10], 2)
    c.check_attend([70], [40], 2)
    assert status() == 0


def test_layouts_streams_and_graphs():
    c = Case("int8", 2, 64, [100, 130], DEV)
    c.write([0, 0], [99, 129])
    wide = torch.randn(2, 3 * 128 + 3, device=DEV).bfloat16()
    k, v = wide[:, 1:129], wide[:, 129:257]               # neither aligned nor packed
    kv8.kv8_write(k, v, *c.c, c.table.to(DEV), i32([99, 129], DEV))
    c.plain.write(k.cpu(), v.cpu(), c.table, [99, 129], [1, 1])
    c.check_read([60, 60], [40, 70])
    q = wide[:, 200:328]
    table, ctx = c.table.to(DEV), i32([100, 130], DEV)
    want = kv8.kv8_attention(q, *c.c, table, ctx, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(kv8.kv8_attention(q, *c.c, table, ctx, 2), want)
    torch.cuda.current_stream().wait_stream(side)
    # two graphs over the same tensors, replayed in either order with changed inputs
    pos = i32([99, 129], DEV)
    k, v, q = k.contiguous(), v.contiguous(), q.contiguous()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv8.kv8_write(k, v, *c.c, table, pos)
            out = kv8.kv8_attention(q, *c.c, table, ctx, 2)
        graphs.append((g, out))
    for g, out in graphs[::-1] + graphs:
        for t in (k, v, q):
            t.copy_(torch.randn_like(t))
        g.replay()
        c.plain.write(k.cpu(), v.cpu(), c.table, [99, 129], [1, 1])
        want, spread = c.plain.attention(q.cpu(), c.table, [100, 130], [1, 1], 2, 0.125)
        err = (out.double().cpu() - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread).all()
    assert status() == 0


def test_repeated_calls_give_the_same_bits():
    c = Case("e4m3", 2, 128, [5000, 40], DEV)
    c.write([0, 0], [5000, 40])
    q = torch.randn(2, 8 * 128, device=DEV).bfloat16()
    outs = [c.attend(q, [5000, 40], [1, 1], 8) for _ in range(5)]
    assert all(torch.equal(o, outs[0]) for o in outs)
    assert status() == 0


def test_rows_without_entry_and_bad_entries():
    """Rows behind the last entry are zero; an entry out of range is skipped and recorded, the
    others are answered."""
    c = Case("int8", 1, 64, [100, 40, 70], DEV)
    c.write([0] * 3, [100, 40, 70])
    q = torch.randn(9, 128, device=DEV).bfloat16()
    table, ctx = c.table.to(DEV), i32([100, 40, 70], DEV)
    row0 = i32([0, 2, 2, 5], DEV)
    out = kv8.kv8_attention(q, *c.c, table, ctx, 2, row0=row0, max_rows=4)
    assert (out[5:] == 0).all() and status() == 0
    # more rows than max_rows: that entry is refused alone
    bad = kv8.kv8_attention(q, *c.c, table, ctx, 2, row0=row0, max_rows=2)
    assert torch.equal(bad[:2], out[:2]) and (bad[2:] == 0).all() and status() == 2
    # rows past the tensor
    bad = kv8.kv8_attention(q[:4], *c.c, table, ctx, 2, row0=row0, max_rows=4)
    assert torch.equal(bad[:2], out[:2]) and (bad[2:] == 0).all() and status() == 2
    # a page number that the cache does not have
    wrong = table.clone()
    wrong[2, 1] = 10 ** 6
    bad = kv8.kv8_attention(q, *c.c, wrong, ctx, 2, row0=row0, max_rows=4)
    assert torch.equal(bad[:2], out[:2]) and status() == 2
    before = [t.clone() for t in c.c]
    k = torch.randn(3, 64, device=DEV).bfloat16()
    kv8.kv8_write(k, k, *c.c, wrong[2:], i32([70], DEV), row0=i32([0, 3], DEV), max_rows=3)
    assert status() == 2
    kv8.kv8_write(k, k, *c.c, table[2:], i32([-5], DEV), row0=i32([0, 3], DEV), max_rows=3)
    assert status() == 2
    kv8.kv8_write(k, k, *c.c, table[1:2], i32([400], DEV), row0=i32([0, 3], DEV), max_rows=3)
    assert status() == 2
    kv8.kv8_write(k, k, *c.c, table[1:2], i32([0], DEV), row0=i32([0, 9], DEV), max_rows=9)
    assert status() == 2
    for a, b in zip(before, c.c):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_numbers_at_the_edge():
    """Positions next to 2^31, an unbounded max_rows, more entries than one launch takes, an entry
    whose row numbers wrap around."""
    c = Case("int8", 1, 64, [3, 3], DEV)
    k = torch.randn(2, 64, device=DEV).bfloat16()
    table = c.table.to(DEV)
    kv8.kv8_write(k, k, *c.c, table, i32([2 ** 31 - 1, 2 ** 31 - 40], DEV))
    assert status() == 2
    kv8.kv8_write(k, k, *c.c, table, i32([0, 0], DEV), row0=i32([0, 1, 2], DEV), max_rows=2 ** 40)
    out = kv8.kv8_attention(k, *c.c, table, i32([1, 1], DEV), 1, row0=i32([0, 1, 2], DEV), max_rows=2 ** 40)
    assert status() == 0
    got, _ = kv8.kv8_read(*c.c, table, i32([0, 0], DEV), i32([0, 1, 2], DEV), 2, 2 ** 40)
    assert (got.float() - k.float()).abs().max() < 0.1 and (out.float() - k.float()).abs().max() < 0.1
    kv8.kv8_attention(k, *c.c, table, i32([1, 1], DEV), 1, row0=i32([-2 ** 31, 2 ** 31 - 1, 2], DEV), max_rows=2)
    assert status() in (0, 2)
    kv8.kv8_write(k, k, *c.c, table, i32([0, 0], DEV), row0=i32([2, 2 ** 31 - 1, 0], DEV), max_rows=2 ** 31)
    assert status() == 2


@pytest.mark.parametrize("rows", [1, 60])
def test_more_entries_than_a_launch_takes(rows):
    n = 600
    lens = [60 + (i * 37) % 70 for i in range(n)]
    c = Case("e4m3", 1, 64, lens, DEV)
    c.write([0] * n, lens)
    c.check_attend(lens, [rows] * n if rows == 1 else [rows if i % 100 == 3 else i % 3 for i in range(n)], 2)
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_wide_tiles(kind):
    """Many rows: tiles that end inside a page, heads that do not divide them, several tiles of several
    entries in every block, contexts split over blocks, pages without values, and scales apart."""
    c = Case(kind, 3, 128, [700, 2500, 65, 0, 1500], DEV)

    def edit(k, v):
        v[64:128] = 0.0                                    # entry 0, page 1: no values
        k[128:192] = 0.0
        v[700 + 64:700 + 128] *= 2.0 ** 20                 # entry 1, page 1
        v[700 + 640:700 + 704] *= 2.0 ** -25
    c.write([0] * 5, [700, 2500, 65, 0, 1500], edit=edit)
    c.check_attend([700, 2500, 65, 0, 1500], [333, 57, 65, 0, 129], 15)
    c.check_attend([699, 2500, 3, 0, 64], [50, 1, 65, 0, 64], 3)
    got = [c.attend(torch.ones(130, 3 * 128).bfloat16(), [700, 2500, 65, 0, 1500], [60, 1, 2, 0, 67], 3) for _ in range(3)]
    assert all(torch.equal(x, got[0]) for x in got)
    assert status() == 0


@pytest.mark.parametrize("rows", [24, 25, 32, 33, 64])
@pytest.mark.parametrize("width", [6, 5000])
def test_tiles_by_rows_and_work(rows, width):
    """On both sides of the bounds between the two tiles: of the rows, and of the pages that a table can name."""
    lens = [300, 64, 129]
    c = Case("int8", 2, 64, lens, DEV)
    c.write([0] * 3, lens)
    c.table = torch.cat([c.table, torch.full((3, width - c.table.shape[1]), -1, dtype=torch.int32)], 1)
    c.check_attend(lens, [rows, 1, 7], 2)
    assert status() == 0


def test_wide_tiles_not_a_number():
    c = Case("e4m3", 2, 64, [300], DEV)

    def edit(k, v):
        k[70, 3] = math.nan                                # page 1, head 0: keys
        v[140, 64 + 9] = math.inf                          # page 2, head 1: values
    c.write([0], [300], edit=edit)
    o = c.check_attend([300], [280], 2)                    # rows 0 .. 43 do not see page 1
    assert not torch.isnan(o[:44, :64]).any() and torch.isnan(o[44:, :64]).all()
    assert not torch.isnan(o[:108, 64:]).any() and torch.isnan(o[108:, 64:]).all()
    page = int(c.table[0, 4])
    c.c[1].view(torch.int8)[page, :, :, 44:] = 127         # behind the context: NaN codes
    c.c[0].view(torch.int8)[page, :, :, 44:] = 127
    c.check_attend([300], [100], 2)
    assert status() == 0


def test_gpu_refusals():
    c = Case("int8", 1, 64, [3], DEV)
    x = torch.zeros(1, 64, device=DEV)
    with pytest.raises(ValueError):
        kv8.kv8_write(x, x, *c.c, c.table.to(DEV), i32([0], DEV))
    with pytest.raises(ValueError):
        kv8.kv8_write(x.bfloat16(), x.bfloat16(), *c.c, c.table, i32([0], DEV))
    with pytest.raises(ValueError):
        kv8.kv8_attention(x.bfloat16().cpu(), *c.c, c.table.to(DEV), i32([1], DEV), 1)
    with pytest.raises(ValueError):
        kv8.kv8_read(*c.c, c.table.to(DEV), i32([0], DEV), i32([0, 1], DEV), 1, 1,
                     dtype=torch.float32)


@pytest.mark.parametrize("shift", [1, 4])
def test_rows_that_begin_anywhere(shift):
    """Contiguous rows whose first one is not at a multiple of 16 bytes, for every input of rows."""
    c = Case("int8", 2, 64, [70, 3], DEV)
    flat = torch.randn(3, 2 * 128 + 8, generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    k, v, q = (f[shift:shift + 256].view(2, 128) for f in flat)
    assert k.is_contiguous() and k.data_ptr() % 16
    pos, ctx = i32([0, 2], DEV), i32([1, 3], DEV)
    got = []
    for a, b, x in ((k, v, q), (k.clone(), v.clone(), q.clone())):
        for t in c.c:
            t.zero_()
        kv8.kv8_write(a, b, *c.c, c.table.to(DEV), pos)
        got.append([kv8.kv8_attention(x, *c.c, c.table.to(DEV), ctx, 2)] + [t.clone() for t in c.c])
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(*got))
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e-30, 0.03, 50.0])
def test_first_token_inside_a_page_that_nothing_has_written(kind, size):
    """Nothing is kept of such a page, its scale neither."""
    c = kv8.kv8_alloc(2, 2, 64, kind, DEV)
    k = torch.randn(3, 128, generator=torch.Generator().manual_seed(1)).mul(size).bfloat16()
    qmax = {"int8": 127.0, "e4m3": 448.0}[kind]
    for page, row0, pos in ((0, None, [5]), (1, i32([0, 3], DEV), [64 + 9])):
        n = 1 if row0 is None else 3
        kv8.kv8_write(k[:n].to(DEV), 3 * k[:n].to(DEV), *c, i32([[0, 1]], DEV), i32(pos, DEV), row0, n)
        for x, scale in ((k[:n], c[2]), (3 * k[:n], c[3])):
            for h in range(2):
                top = float(x[:, 64 * h:64 * h + 64].abs().max())
                e = max(-126, math.ceil(math.log2(top / qmax)))
                assert float(scale[page, h]) == 2.0 ** e, (page, h, float(scale[page, h]), e)
        got = kv8.kv8_read(*c, i32([[0, 1]], DEV), i32(pos, DEV), i32([0, n], DEV), n, n)
        for x, y in zip((k[:n], 3 * k[:n]), got):
            # one rounding: half a step, 2^(e - 1), is below the largest / 127; of e4m3 half of three bits, or 2^-10 of the
            # scale for its smallest codes, which is below 2^-17 of the largest
            top = x.abs().max().float()
            step = top / 127.0 if kind == "int8" else x.float().abs() * 2.0 ** -4 + top * 2.0 ** -17
            assert ((y.float().cpu() - x.float()).abs() <= step + 2.0 ** -133).all()
        if row0 is not None:                               # what lies in front of the first token is zero
            assert all((t == 0).all() for t in kv8.kv8_read(*c, i32([[0, 1]], DEV), i32([64], DEV), i32([0, 9], DEV), 9, 9))
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("size", [0.3, 1e-5, 1e-6, 1e-20, 1e-36])
def test_wide_tiles_pages_without_values(kind, dh, size):
    """Pages without values, or never written, count for the denominator and for nothing else, wherever they lie and
    however small the other pages' values are."""
    for empty in (0, 1, 3):
        c = Case(kind, 1, dh, [400], DEV)

        def edit(k, v):
            k[:] = k.float().mul(0.5).bfloat16()
            v[:] = v.float().mul(size).bfloat16()
            k[64 * empty:64 * empty + 64] = 1.0            # most rows listen to it more than to the others
            v[64 * empty:64 * empty + 64] = 0.0
        c.write([0], [400], edit=edit)
        q = (torch.randn(90, 2 * dh, generator=c.gen) + 0.25).bfloat16()
        got = c.attend(q, [400], [90], 2).double().cpu()
        want, spread = c.plain.attention(q, c.table, [400], [90], 2, dh ** -0.5)
        # as in check_attend, and what bf16 holds of numbers next to its smallest
        assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * spread + 2.0 ** -133).all()
    c = Case(kind, 1, dh, [400], DEV)
    c.write([64], [336], sizes=[size])
    c.check_attend([400], [90], 2)
    assert status() == 0


def apart(c, low, high, pages, sparse=False):
    """Keys that tell two kinds of pages apart, and values of either kind: ``pages`` says which kind."""
    n = 64 * len(pages)

    def edit(k, v):
        for i, big in enumerate(pages):
            at = slice(64 * i, 64 * i + 64)
            k[at] = -1.0 if big else 1.0
            v[at] = v[at].float().mul(2.0 ** (high if big else low)).bfloat16()
            if big and sparse:
                v[at, ::2] = 0.0
    c.write([0], [n], edit=edit)


def check_apart(c, n, rows, dh, gap, size=1.0):
    """Rows whose scores of the two kinds of pages are ``gap`` units of log2 apart (the small values' ones above)."""
    q = torch.full((rows, dh), gap * math.log(2.0) / (2 * dh ** 0.5))
    q[1::2] *= torch.rand(rows // 2, 1, generator=c.gen)
    q = (q * size).bfloat16()
    got = c.attend(q, [n], [rows], 1).double().cpu()
    want, spread = c.plain.attention(q, c.table, [n], [rows], 1, dh ** -0.5)
    # as in check_attend: scores stay below 2^8 here too.  And what the fp16 weights of a wide tile cannot hold beside the
    # row's largest product of weight and scale: they are 2^10 times what they count against a maximum up to 2^70 under that
    # one's, less than 2^-25 is lost, and a code is below 2^9: 2^(9 - 25 - 10 - 70) of it per key, of less than 2^13 keys.  The
    # largest one's key has a code of one or more in some channel, so the row's largest sum is no smaller than that product.
    deep = 2.0 ** -83 * spread.view(rows, -1).amax(1, keepdim=True)
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * spread + deep + 2.0 ** -133
    bad = (got - want).abs() > bound
    assert not bad.any(), float(((got - want).abs() / bound)[bad].max())


ORDERS = [[1, 0, 0, 0], [0, 1, 0, 0], [1, 1, 0, 1, 0, 0, 1, 0], [0, 0, 0, 1]]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("low,high", [(-30, 20), (-36, 14), (-60, 40), (-110, 100)])
def test_wide_tiles_values_apart(kind, dh, low, high):
    """Rows that listen to one kind of page alone, and to both, however far apart the values' scales are."""
    for pages in ORDERS + [[1] + [0, 0, 1] * 30]:
        c = Case(kind, 1, dh, [64 * len(pages)], DEV)
        apart(c, low, high, pages)
        for gap in (0.0, 20.0, 90.0, 120.0):
            check_apart(c, 64 * len(pages), 100, dh, gap)
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 5, 100])
def test_values_apart_channel_by_channel(kind, rows):
    """Channels that the large values leave free hold the small ones."""
    for pages in ORDERS:
        c = Case(kind, 1, 128, [64 * len(pages)], DEV)
        apart(c, -25, 20, pages, sparse=True)
        for gap in (0.0, 15.0, -15.0):
            check_apart(c, 64 * len(pages), rows, 128, gap)
    assert status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("rows", [1, 7])
def test_small_weights_of_large_values(kind, dh, rows):
    """A page that a row hardly listens to counts all the same if its values are large enough."""
    for pages in ORDERS + [[1] + [0, 0, 1] * 30]:
        c = Case(kind, 1, dh, [64 * len(pages)], DEV)
        apart(c, -30, 30, pages)
        for gap in (20.0, 30.0, 40.0, 60.0, 90.0):
            check_apart(c, 64 * len(pages), rows, dh, gap)
    assert status() == 0


@pytest.mark.parametrize("row0,good", [([0, 2, 1], 0), ([2, 1, 2], 1), ([-1, 0, 2], 1), ([0, 3, 3], None), ([3, 3, 2], None),
                                       ([0, 2 ** 31 - 1, 2], None), ([-2 ** 31, 2 ** 31 - 1, 2], None),
                                       ([0, 2, -2 ** 31], 0)])
@pytest.mark.parametrize("group", [1, 40])
def test_row_numbers_out_of_order(row0, good, group):
    """Entries whose row numbers run backwards or leave the rows are recorded, each alone, and nothing of theirs is
    written; the others are answered."""
    c = Case("int8", 1, 64, [3, 3], DEV)
    c.write([0, 0], [3, 3])
    before = [t.clone() for t in c.c]
    q = torch.randn(2, group * 64, generator=c.gen).bfloat16().to(DEV)
    table, ctx, rows = c.table.to(DEV), i32([3, 3], DEV), i32(row0, DEV)
    out = kv8.kv8_attention(q, *c.c, table, ctx, group, row0=rows, max_rows=2)
    assert status() == 2
    if good is None:
        assert (out == 0).all()
    else:
        a, b = row0[good], row0[good + 1]
        want, spread = c.plain.attention(q[a:b].cpu(), c.table[good:good + 1], [3], [b - a], group, 0.125)
        err = (out[a:b].double().cpu() - want).abs()                     # bounds as in check_attend
        assert (err <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * spread).all()
        assert (out[:a] == 0).all() and (out[b:] == 0).all()
        kv8.kv8_read(*c.c, table, i32([0, 0], DEV), rows, 2, 2)
        assert status() == 2
    if good is None:
        kv8.kv8_write(q[:, :64], q[:, :64], *c.c, table, i32([0, 0], DEV), rows, 2)
        assert status() == 2
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, c.c))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 3, 100])
def test_pages_that_are_not_there(kind, rows):
    """A page that the cache does not have takes no part, a row that sees no other gets NaN, and a context beyond
    the table ends with it; all of it is recorded."""
    n = 400
    c = Case(kind, 1, 64, [n], DEV, width=7)
    c.write([0], [n])
    q = torch.randn(rows, 64, generator=c.gen).bfloat16()
    table, first, most = c.table.to(DEV), None if rows == 1 else i32([0, rows], DEV), rows
    call = lambda t, ctx: kv8.kv8_attention(q.to(DEV), *c.c, t, i32([ctx], DEV), 1, first, most).double().cpu()
    k, v = (x.view(n, 64) for x in c.plain.read(c.table, [0], [n]))
    gone = table.clone()
    gone[0, 0], gone[0, 2], gone[0, 5] = -1, 10 ** 6, 2 ** 31 - 1
    got = call(gone, n)
    assert status() == 2
    here = torch.tensor([p // 64 not in (0, 2, 5) for p in range(n)])
    for i in range(rows):
        mine = here & (torch.arange(n) <= n - rows + i)
        w = torch.softmax(k[mine] @ q[i].double() * 0.125, 0)[:, None]
        want, spread = (w * v[mine]).sum(0), (w * v[mine].abs()).sum(0)
        assert ((got[i] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * spread).all()    # as in check_attend
    assert torch.isnan(call(torch.full_like(gone, -1), n)).all() and status() == 2
    short = table[:, :6].contiguous()                      # 384 tokens
    got = call(short, 500)
    assert status() == 2
    assert torch.equal(got, call(short, 384)) and status() == 0
