"""The 8-bit cache on the CPU (the restatement of its kernels) against its definition in 64 bits,
and the calls that are refused."""
import math

import pytest
import torch

from coeus_b200.ops import kv8
from kv8_cases import Case, i32


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dh", [64, 128])
def test_write_and_read(kind, dh):
    c = Case(kind, 2, dh, [70, 200, 5])
    c.write([0, 0, 0], [64, 130, 0])
    c.write([64, 130, 0], [1, 1, 1])                       # a new page, the inside of one, the start
    c.write([65, 131, 1], [1, 1, 1], sizes=[9.0, 40.0, 0.01])     # scales grow, or do not
    c.write([66, 132, 2], [4, 68, 3], sizes=[100.0, 1.0, 1.0])
    c.check_read([0, 0, 0], [70, 200, 5])
    c.check_read([63, 129, 4], [3, 70, 1])


def test_codes_use_the_range_and_ties_go_to_even():
    c = Case("int8", 1, 64, [1])
    k = torch.zeros(1, 64)
    k[0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])
    kv8.kv8_write(k, k, *c.c, c.table, i32([0]))
    page = int(c.table[0, 0])
    assert float(c.c[2][page, 0]) == 1.0
    assert c.c[0][page, 0, 0, 0, :4].tolist() == [127, 0, 2, -2]
    assert c.c[1][page, 0, :4, 0].tolist() == [127, 0, 2, -2]
    k[0, 0] = 127.5
    kv8.kv8_write(k, k, *c.c, c.table, i32([0]))
    assert float(c.c[2][page, 0]) == 2.0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_not_a_number_makes_its_block_one(kind):
    c = Case(kind, 2, 64, [130])

    def edit(k, v):
        k[3, 5] = math.inf                                 # page 0, head 0, keys
        v[70, 64 + 2] = math.nan                           # page 1, head 1, values
    c.write([0], [130], edit=edit)
    c.check_read([0], [130])
    k, v = c.read([0], [130])
    assert torch.isnan(k[:64, :64]).all() and not torch.isnan(k[64:]).any()
    assert torch.isnan(v[64:128, 64:]).all() and not torch.isnan(v[:64]).any()
    # rows count what they see: the first two of four rows end in front of page 1
    o = c.check_attend([66], [4], 2)
    assert not torch.isnan(o[:2, 64:]).any() and torch.isnan(o[2:, 64:]).all()
    c.write([0], [130])                                    # from its first token on a page is new
    c.check_read([0], [130])


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("nh,heads,dh", [(2, 2, 64), (6, 2, 64), (4, 1, 128)])
def test_attention(kind, nh, heads, dh):
    c = Case(kind, heads, dh, [1, 64, 130, 3])
    c.write([0] * 4, [1, 64, 130, 3])
    c.check_attend([1, 64, 130, 3], [1, 1, 1, 1], nh)
    c.check_attend([1, 64, 130, 3], [1, 0, 70, 5], nh)     # the last entry's first rows see nothing
    c.check_attend([0, 64, 129, 0], [1, 3, 2, 1], nh, scale=0.3)


def test_refusals():
    c = Case("int8", 2, 64, [70, 3])
    k, v, ks, vs = c.c
    x = torch.zeros(2, 128)
    pos = i32([0, 0])
    ok = (x, x, k, v, ks, vs, c.table, pos)

    def refused(**kw):
        names = ["k", "v", "k_cache", "v_cache", "k_scale", "v_scale", "page_table", "pos0"]
        args = dict(zip(names, ok), **kw)
        with pytest.raises(ValueError):
            kv8.kv8_write(**args)
    refused(k=torch.zeros(2, 64))
    refused(k=torch.zeros(3, 128))
    refused(k=torch.zeros(1, 128), v=torch.zeros(1, 128))
    refused(v_cache=v[:, :1])
    refused(v_cache=v.view(torch.float8_e4m3fn))
    refused(k_cache=k.float())
    refused(k_cache=k[:0], v_cache=v[:0], k_scale=ks[:0], v_scale=vs[:0])
    refused(k_cache=k[:, :0], v_cache=v[:, :0], k_scale=ks[:, :0], v_scale=vs[:, :0], k=x[:, :0], v=x[:, :0])
    refused(k_scale=ks.double())
    refused(page_table=c.table.long())
    refused(page_table=c.table.t().contiguous().t())
    refused(pos0=i32([0]))
    refused(pos0=pos.long())
    refused(max_rows=2)
    refused(row0=i32([0, 1]))
    refused(row0=i32([0, 1, 2]), max_rows=0)
    refused(row0=i32([0, 2, 2]), max_rows=1)
    refused(row0=i32([0, 1, 3]), max_rows=2)
    refused(pos0=i32([0, 64]))                             # no second page
    with pytest.raises(ValueError):
        kv8.kv8_attention(torch.zeros(2, 192), k, v, ks, vs, c.table, pos, 3)
    with pytest.raises(ValueError):
        kv8.kv8_attention(torch.zeros(1, 128), k, v, ks, vs, c.table, pos, 2)
    with pytest.raises(ValueError):
        kv8.kv8_alloc(4, 2, 96, "int8", "cpu")
    with pytest.raises(ValueError):
        kv8.kv8_alloc(4, 2, 64, "fp4", "cpu")
    with pytest.raises(ValueError):
        kv8.kv8_read(k, v, ks, vs, c.table, pos, None, 2, 1)


def test_rows_are_laid_out_for_the_kernels():
    """Rows whose address, stride or order the kernels cannot read are copied, others are not."""
    flat = torch.zeros(8 * 128 + 64, dtype=torch.bfloat16)
    off = (-flat.data_ptr() // 2) % 8                      # numbers up to a multiple of 16 bytes
    lay = lambda x: kv8._rows("rows", x, 64, 0 if x.get_device() == 0 else -1)

    class OnDevice:                                        # a view that says it is on a GPU
        def __init__(self, x):
            self.x = x

        def get_device(self):
            return 0

        def __getattr__(self, name):
            return getattr(self.x, name)

    for x, kept in ((flat[off:off + 256].view(4, 64), True), (flat[off + 1:off + 257].view(4, 64), False),
                    (flat[off:off + 512].view(4, 128)[:, :64], True), (flat[off:off + 512].view(4, 128)[:, 4:68], False),
                    (flat[off:off + 4 * 68].view(4, 68)[:, :64], False), (flat[off:off + 256].view(64, 4).t(), False)):
        y = lay(OnDevice(x))
        assert (y.data_ptr() == x.data_ptr()) == kept
        assert y.data_ptr() % 16 == 0 and y.stride(1) == 1 and y.stride(0) % 8 == 0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("size", [1e-30, 0.03, 50.0])
def test_first_token_inside_a_page_that_nothing_has_written(kind, size):
    """Nothing is kept of such a page, its scale neither."""
    DEV = "cpu"
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


@pytest.mark.parametrize("row0", [[0, 2, 1], [2, 1, 2], [-1, 0, 2], [0, 3, 3], [3, 3, 2], [0, 2 ** 31 - 1, 2],
                                  [-2 ** 31, 2 ** 31 - 1, 2], [0, 2, -2 ** 31]])
def test_row_numbers_out_of_order(row0):
    c = Case("int8", 1, 64, [3, 3])
    c.write([0, 0], [3, 3])
    k = torch.zeros(2, 64)
    for call in (lambda r: kv8.kv8_write(k, k, *c.c, c.table, i32([0, 0]), r, 2),
                 lambda r: kv8.kv8_read(*c.c, c.table, i32([0, 0]), r, 2, 2),
                 lambda r: kv8.kv8_attention(k, *c.c, c.table, i32([3, 3]), 1, r, 2)):
        with pytest.raises(ValueError):
            call(i32(row0))
