"""A paged cache in 8 bits (``csrc/kv8.cu``, ``csrc/kv8_attn.cu``): append, read back, attention.

The cache of one layer is four tensors (:func:`kv8_alloc`).  Pages hold 64 tokens; of a page and
head the keys are ``[dh / 64][token][64]`` codes, the values ``[dh][token]`` codes, in ``int8`` or
``float8_e4m3fn``.  A code stands for ``code * scale`` with one scale per page, head and side, the
smallest power of two (not below 2^-126) under which the block's largest magnitude fits the codes.  A
page that gets more tokens keeps its scale or takes a larger one, to which its codes are then rounded
again.  A key or value that is not finite makes its block's scale NaN, so that whatever attends to the
block is NaN.

``int8`` spends its steps evenly (good for values without outliers), ``float8_e4m3fn`` keeps three
bits of every number however small.

The entries of a call are sequences: entry ``e`` has page-table row ``e``.  With ``row0 [n + 1]`` it
owns rows ``row0[e] .. row0[e + 1] - 1`` of the row-wise tensors, at most ``max_rows`` of them
(possibly none); without, row ``e`` alone.  Entries of one :func:`kv8_write` must not write the same page.

What is out of range is refused on the CPU.  The kernels record it in the status word
(:func:`coeus_b200.ops._lib.check_status`) and touch nothing outside the tensors: an entry whose row
numbers run backwards, leave the rows or are more than ``max_rows``, or whose first position is negative or
next to 2^31, is skipped; a page that the table or the cache does not have is left out, so that its
tokens are neither written nor read and its keys take no part in the softmax (a row that sees tokens, but none
that is there, gets NaN); a context that goes beyond the table ends with it.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from .decode import PAGE

KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def kv8_alloc(num_pages: int, heads: int, dh: int, kind: str, device
              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(k_cache, v_cache, k_scale, v_scale)`` of one layer, all zero; ``kind`` is ``"int8"`` or
    ``"e4m3"``."""
    if kind not in KINDS:
        raise ValueError(f"kv8: the codes are int8 or e4m3, not {kind!r}")
    if dh not in (64, 128):
        raise ValueError(f"kv8: heads of 64 or 128, not {dh}")
    k = torch.zeros((num_pages, heads, dh // 64, PAGE, 64), dtype=torch.int8, device=device)
    v = torch.zeros((num_pages, heads, dh, PAGE), dtype=torch.int8, device=device)
    s = torch.zeros((2, num_pages, heads), dtype=torch.float32, device=device)
    return k.view(KINDS[kind]), v.view(KINDS[kind]), s[0], s[1]


def _check(what: str, k_cache, v_cache, k_scale, v_scale, page_table, ints, row0, max_rows):
    """Shapes and types of what every call takes; returns ``(pages, heads, dh, entries, device)``, the
    device as a number (-1: CPU)."""
    shape, dtype = k_cache.shape, k_cache.dtype
    if len(shape) != 5 or shape[3] != PAGE or shape[4] != 64 or dtype not in _QMAX:
        raise ValueError(f"{what}: keys are [pages, heads, dh / 64, {PAGE}, 64] codes, got "
                         f"{tuple(shape)} {dtype}")
    pages, heads, dh = shape[0], shape[1], shape[2] * 64
    if (dh != 64 and dh != 128) or heads < 1 or pages < 1:
        raise ValueError(f"{what}: pages and heads of 64 or 128, not {tuple(shape)}")
    if v_cache.shape != (pages, heads, dh, PAGE) or v_cache.dtype != dtype:
        raise ValueError(f"{what}: values {tuple(v_cache.shape)} {v_cache.dtype} do not go with "
                         f"keys {tuple(shape)} {dtype}")
    if k_scale.shape != (pages, heads) or v_scale.shape != (pages, heads) \
            or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
        raise ValueError(f"{what}: scales are fp32 [{pages}, {heads}]")
    table = page_table.shape
    if len(table) != 2 or table[1] < 1 or page_table.dtype != torch.int32:
        raise ValueError(f"{what}: the page table is int32 [entries, pages]")
    n = table[0]
    if ints.shape != (n,) or ints.dtype != torch.int32:
        raise ValueError(f"{what}: one int32 number per entry, got {tuple(ints.shape)} {ints.dtype}")
    given = (v_cache, k_scale, v_scale, page_table, ints)
    if row0 is not None:
        if row0.shape != (n + 1,) or row0.dtype != torch.int32:
            raise ValueError(f"{what}: row0 is int32 [{n + 1}]")
        given += (row0,)
    if max_rows < 1 or (row0 is None and max_rows != 1):
        raise ValueError(f"{what}: max_rows is the bound on an entry's rows (1 without row0)")
    device = k_cache.get_device()
    ok = k_cache.is_contiguous()
    for t in given:
        ok = ok and t.is_contiguous()
        if t.get_device() != device:
            raise ValueError(f"{what}: tensors on {t.device} and {k_cache.device}")
    if not ok:
        raise ValueError(f"{what}: cache, tables and lengths have to be contiguous")
    if device >= 0 and (k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise ValueError(f"{what}: the cache has to start at a multiple of 16 bytes")
    return pages, heads, dh, n, device


def _rows(what: str, x: torch.Tensor, width: int, device: int) -> torch.Tensor:
    """A row-wise input as the kernels read it: bf16, unit inner stride, 16-byte rows (a copy where
    the caller's view is laid out otherwise)."""
    if x.dim() != 2 or x.shape[1] != width:
        raise ValueError(f"{what}: rows of {width} numbers, got {tuple(x.shape)}")
    if x.get_device() != device:
        raise ValueError(f"{what}: rows on {x.device}, the cache elsewhere")
    if device < 0:
        return x
    if x.dtype != torch.bfloat16:
        raise ValueError(f"{what}: the kernels take bf16 rows, got {x.dtype}")
    step = x.stride(0)
    if x.stride(1) != 1 or step % 8 or x.data_ptr() % 16 or not 0 <= step < 1 << 31:
        x = x.clone(memory_format=torch.contiguous_format)   # contiguous() keeps an odd address
    return x


def _status(device: int) -> int:
    return _lib.status_buffer(torch.device("cuda", device)).data_ptr()


def _spans(n: int, row0, rows: int, max_rows: int):
    """``(entry, first row, rows)`` of the entries that have any, on the host."""
    if row0 is None:
        if n > rows:
            raise ValueError(f"kv8: {n} entries, {rows} rows")
        return [(e, e, 1) for e in range(n)]
    at = row0.tolist()
    out = []
    for e in range(n):
        if not 0 <= at[e] <= at[e + 1] <= min(rows, at[e] + max_rows):
            raise ValueError(f"kv8: entry {e} has rows {at[e]} .. {at[e + 1] - 1}")
        if at[e + 1] > at[e]:
            out.append((e, at[e], at[e + 1] - at[e]))
    return out


def _exponent(amax: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Smallest ``e >= -126`` with ``amax <= QMAX * 2^e``."""
    m, x = torch.frexp(amax)
    e = x - 7 + (m > 127.0 / 128.0).to(x.dtype) if dtype == torch.int8 else \
        x - 9 + (m > 0.875).to(x.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, -126)).clamp_min(-126)


def _encode(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    y = torch.nan_to_num(y, 0.0, 0.0, 0.0)
    return y.round().to(torch.int8) if dtype == torch.int8 else y.to(dtype)


def _block(codes: torch.Tensor, keys: bool) -> torch.Tensor:
    """Codes of one page ``[heads, ...]`` as fp32 ``[heads, 64, dh]``."""
    x = codes.float()
    if keys:
        return x.transpose(1, 2).reshape(x.shape[0], PAGE, -1)
    return x.transpose(1, 2)


def _values(codes: torch.Tensor, scale: torch.Tensor, page: int, keys: bool) -> torch.Tensor:
    """Values of one page, fp32 ``[heads, 64, dh]``."""
    return _block(codes[page], keys) * scale[page][:, None, None]


def _cpu_page(table: torch.Tensor, e: int, lp: int, pages: int) -> int:
    page = int(table[e, lp]) if lp < table.shape[1] else -1
    if not 0 <= page < pages:
        raise ValueError(f"kv8: entry {e} has no page {lp}")
    return page


def kv8_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              k_scale: torch.Tensor, v_scale: torch.Tensor, page_table: torch.Tensor,
              pos0: torch.Tensor, row0: Optional[torch.Tensor] = None, max_rows: int = 1) -> None:
    """Stores the rows of ``k`` / ``v`` (``[rows, heads * dh]`` views) at positions ``pos0[e]`` and on of
    each entry.  Tokens of the first page before ``pos0[e]`` are kept; what the page held from there on
    is not counted on any more.  A page that is written belongs to one entry."""
    pages, heads, dh, n, device = _check("kv8_write", k_cache, v_cache, k_scale, v_scale,
                                         page_table, pos0, row0, max_rows)
    k = _rows("kv8_write", k, heads * dh, device)
    v = _rows("kv8_write", v, heads * dh, device)
    rows = k.shape[0]
    if rows != v.shape[0]:
        raise ValueError(f"kv8_write: {rows} rows of keys, {v.shape[0]} of values")
    if row0 is None and n > rows:
        raise ValueError(f"kv8_write: {n} entries, {rows} rows")
    if n == 0 or rows == 0:
        return
    if device >= 0:
        with _lib.on_device(device):
            rc = _lib.entry("cb_kv8_write", "ppiippppp" + "iiiii" + "ppiiipp")(
                k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), k_cache.data_ptr(),
                v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), page_table.data_ptr(),
                page_table.shape[1], pages, heads, dh, int(k_cache.dtype != torch.int8),
                None if row0 is None else row0.data_ptr(), pos0.data_ptr(), n, rows,
                min(max_rows, rows), _status(device), _lib.stream_int())
        _lib.check_rc(rc, "cb_kv8_write")
        return
    dtype = k_cache.dtype
    for e, r0, cnt in _spans(n, row0, rows, max_rows):
        at = int(pos0[e])
        for lp in range(at // PAGE, (at + cnt - 1) // PAGE + 1):
            page = _cpu_page(page_table, e, lp, pages)
            lo, hi = max(0, at - lp * PAGE), min(PAGE, at + cnt - lp * PAGE)
            r = r0 + lp * PAGE + lo - at
            for x, codes, scale, keys in ((k, k_cache, k_scale, True), (v, v_cache, v_scale, False)):
                new = x[r:r + hi - lo].float().view(hi - lo, heads, dh).transpose(0, 1)
                amax = new.abs().amax((1, 2))
                bad = ~torch.isfinite(amax)
                ex = _exponent(torch.where(bad, torch.zeros_like(amax), amax), dtype)
                old = _block(codes[page], keys)
                if lo:
                    bad = bad | torch.isnan(scale[page])
                    was = torch.frexp(torch.nan_to_num(scale[page], 1.0))[1] - 1
                    was = was.masked_fill(scale[page] == 0, -127)          # nothing written there yet
                    ex = torch.maximum(ex, was)
                    shift = torch.where(bad, torch.zeros_like(ex), was - ex)
                    kept = torch.ldexp(old[:, :lo], shift[:, None, None])
                    old[:, :lo] = _encode(kept, dtype).float()
                y = torch.where(bad[:, None, None], torch.zeros_like(new), torch.ldexp(new, -ex[:, None, None]))
                old[:, lo:hi] = _encode(y, dtype).float()
                c = _encode(old, dtype)
                if keys:
                    codes[page] = c.view(torch.int8).view(heads, PAGE, dh // 64, 64).transpose(1, 2).view(dtype)
                else:
                    codes[page] = c.view(torch.int8).transpose(1, 2).contiguous().view(dtype)
                one = torch.ldexp(torch.ones(heads), ex)
                scale[page] = torch.where(bad, torch.full_like(one, math.nan), one)


def kv8_read(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
             v_scale: torch.Tensor, page_table: torch.Tensor, pos0: torch.Tensor,
             row0: torch.Tensor, rows: int, max_rows: int,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The stored keys and values of positions ``pos0[e]`` and on as ``[rows, heads * dh]`` (``dtype``;
    bf16 on a GPU, where it holds every stored value exactly).  ``rows`` is ``row0[n]``, known on the
    host; rows that no entry owns are not set."""
    pages, heads, dh, n, device = _check("kv8_read", k_cache, v_cache, k_scale, v_scale,
                                         page_table, pos0, row0, max_rows)
    if row0 is None or rows < 0:
        raise ValueError("kv8_read: needs row0 and the number of rows")
    if device >= 0:
        if dtype != torch.bfloat16:
            raise ValueError(f"kv8_read: the kernels give bf16, not {dtype}")
        out = torch.empty((2, rows, heads * dh), dtype=dtype, device=k_cache.device)
        k, v = out.unbind(0)
        if n and rows:
            with _lib.on_device(device):
                rc = _lib.entry("cb_kv8_read", "ppppp" + "iiiii" + "ppiiippipp")(
                    k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                    v_scale.data_ptr(), page_table.data_ptr(), page_table.shape[1], pages, heads,
                    dh, int(k_cache.dtype != torch.int8), row0.data_ptr(), pos0.data_ptr(), n,
                    rows, min(max_rows, rows), k.data_ptr(), v.data_ptr(), heads * dh, _status(device),
                    _lib.stream_int())
            _lib.check_rc(rc, "cb_kv8_read")
        return k, v
    out = torch.zeros((2, rows, heads * dh), dtype=dtype)
    for e, r0, cnt in _spans(n, row0, rows, max_rows):
        at = int(pos0[e])
        for lp in range(at // PAGE, (at + cnt - 1) // PAGE + 1):
            page = _cpu_page(page_table, e, lp, pages)
            lo, hi = max(0, at - lp * PAGE), min(PAGE, at + cnt - lp * PAGE)
            r = r0 + lp * PAGE + lo - at
            for o, codes, scale, keys in ((out[0], k_cache, k_scale, True),
                                          (out[1], v_cache, v_scale, False)):
                x = _values(codes, scale, page, keys)[:, lo:hi]
                o[r:r + hi - lo] = x.transpose(0, 1).reshape(hi - lo, -1).to(dtype)
    return out[0], out[1]


@lru_cache(maxsize=1024)
def _scratch(*shape: int) -> int:
    fn = _lib.lib().cb_kv8_attn_scratch
    fn.restype = ctypes.c_int64
    return fn(*shape)


def kv8_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  k_scale: torch.Tensor, v_scale: torch.Tensor, page_table: torch.Tensor,
                  ctx_len: torch.Tensor, nh: int, row0: Optional[torch.Tensor] = None,
                  max_rows: int = 1, scale: Optional[float] = None) -> torch.Tensor:
    """``q [rows, nh * dh]`` -> ``[rows, nh * dh]``.  Entry ``e`` holds ``ctx_len[e]`` tokens, its rows
    are the last of them and every row sees the tokens up to itself; a row that sees none gets zeros, and
    so do rows that no entry owns.  Query head ``h`` reads cache head ``h // (nh // heads)``; ``scale``
    defaults to ``1 / sqrt(dh)``.

    The kernels hold queries (against the largest number of their row) and weights in fp16 and every sum in
    fp32.  A weight is off by 2^-11 of itself; one below 2^-23 of its row's largest may lose digits, one
    below 2^-34 may count as nothing in a channel where the values beside it are no larger, and so may a value
    that is 2^60 below another one of its row and head.  Which of the two kernels runs, for few rows or for many,
    goes by the rows that share a cache head and by the entries, heads and width of the page table, not by
    the contexts: they agree up to these roundings."""
    pages, heads, dh, n, device = _check("kv8_attention", k_cache, v_cache, k_scale, v_scale,
                                         page_table, ctx_len, row0, max_rows)
    if nh < 1 or nh % heads:
        raise ValueError(f"kv8_attention: {nh} query heads over {heads}")
    q = _rows("kv8_attention", q, nh * dh, device)
    rows = q.shape[0]
    if row0 is None and n > rows:
        raise ValueError(f"kv8_attention: {n} entries, {rows} rows")
    if scale is None:
        scale = 1.0 / math.sqrt(dh)
    elif not 0.0 <= scale < math.inf:
        raise ValueError(f"kv8_attention: scale {scale}")
    if device >= 0:
        whole = row0 is None and n == rows           # every row is written
        out = (torch.empty if whole else torch.zeros)((rows, nh * dh), dtype=torch.bfloat16,
                                                      device=q.device)
        if n == 0 or rows == 0:
            return out
        width, max_rows = page_table.shape[1], min(max_rows, rows)
        if width * PAGE >= 1 << 31:
            raise ValueError(f"kv8_attention: page tables of {width} pages")
        with _lib.on_device(device):
            scratch = torch.empty(_scratch(n, rows, max_rows, nh // heads, width, heads, dh),
                                  dtype=torch.uint8, device=q.device)
            rc = _lib.entry("cb_kv8_attn", "pippppp" + "iiiii" + "ppiiiifpippp")(
                q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(),
                k_scale.data_ptr(), v_scale.data_ptr(), page_table.data_ptr(), width, pages, heads,
                dh, int(k_cache.dtype != torch.int8), ctx_len.data_ptr(),
                None if row0 is None else row0.data_ptr(), n, rows, max_rows, nh, scale,
                out.data_ptr(), nh * dh, scratch.data_ptr(), _status(device), _lib.stream_int())
        _lib.check_rc(rc, "cb_kv8_attn", launches=2 * ((n + 255) // 256))
        return out
    out = torch.zeros((rows, nh * dh), dtype=q.dtype)
    g = nh // heads
    for e, r0, cnt in _spans(n, row0, rows, max_rows):
        c = int(ctx_len[e])
        if c < 1:
            continue
        ids = [_cpu_page(page_table, e, lp, pages) for lp in range((c + PAGE - 1) // PAGE)]
        K = torch.cat([_values(k_cache, k_scale, p, True) for p in ids], 1)[:, :c]
        V = torch.cat([_values(v_cache, v_scale, p, False) for p in ids], 1)[:, :c]
        x = q[r0:r0 + cnt].float().view(cnt, heads, g, dh)
        s = torch.einsum("rhgd,hcd->hgrc", x, K) * scale
        seen = torch.arange(c)[None] <= (c - cnt + torch.arange(cnt))[:, None]       # [rows, c]
        w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        w = torch.where(seen, w, torch.zeros_like(w))
        # a value that is NaN counts for the rows that see it and no others
        none = torch.isnan(V)
        o = torch.einsum("hgrc,hcd->rhgd", w, V.masked_fill(none, 0.0))
        if none.any():
            hit = torch.einsum("rc,hcd->rhd", seen.float(), none.float()) > 0
            o = o.masked_fill(hit[:, :, None], math.nan)
        o = torch.where(seen.any(-1)[:, None, None, None], o, torch.zeros_like(o))
        out[r0:r0 + cnt] = o.reshape(cnt, -1).to(q.dtype)
    return out
