"""Beam search (``csrc/beam.cu``): selecting the continuations of every request's beams, and moving
the beams' cache pages to where their parents' are."""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .decode import PAGE

MAX_BEAMS = 32
BLOCK = 512            # logits that the kernels sum up at a time (csrc/beam.cu)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, done: torch.Tensor,
                eos_id: Optional[int] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """One step of a beam search over ``B`` requests of ``K`` beams: ``logits [B * K, V]`` (bf16 or
    fp32, unit inner stride), ``scores [B, K]`` (fp32: the beams' summed log-probabilities), ``done
    [B, K]`` (bool: the beam has ended).

    Continuation ``t`` of beam ``j`` is worth ``scores[j] + log_softmax(logits[j])[t]``; a beam that has
    ended goes on with ``eos_id`` alone, at its own score.  Returns the ``K`` best of every request, best
    first (equal ones by the lowest beam, then token): ``(scores, parent, token, done)``, ``parent``
    and ``token`` int64, ``done`` true where the parent had ended or the token is ``eos_id``.  A value
    that is ``-inf`` or NaN is no continuation; places that are left get score ``-inf``, their own index as
    parent, ``eos_id`` (0 if None) as token, and are done.  A first step starts from one copy of the
    prompt with scores ``[0, -inf, ...]``."""
    if scores.dim() != 2 or scores.dtype != torch.float32:
        raise ValueError(f"beam_select: scores are fp32 [B, K], got {tuple(scores.shape)} {scores.dtype}")
    B, K = scores.shape
    if not 1 <= K <= MAX_BEAMS:
        raise ValueError(f"beam_select: 1 to {MAX_BEAMS} beams, not {K}")
    if tuple(done.shape) != (B, K) or done.dtype != torch.bool:
        raise ValueError(f"beam_select: done is bool [{B}, {K}]")
    if logits.dim() != 2 or logits.shape[0] != B * K or logits.shape[1] < 1:
        raise ValueError(f"beam_select: logits of {B * K} rows, got {tuple(logits.shape)}")
    V = logits.shape[1]
    if eos_id is not None and not 0 <= eos_id < V:
        raise ValueError(f"beam_select: eos_id {eos_id} is outside the vocabulary of {V}")
    device = logits.get_device()
    if scores.get_device() != device or done.get_device() != device:
        raise ValueError("beam_select: tensors on different devices")
    if device >= 0:
        f32 = logits.dtype == torch.float32
        if not f32 and logits.dtype != torch.bfloat16:
            raise ValueError(f"beam_select: logits in bf16 or fp32, not {logits.dtype}")
        if V > 1 << 26 or B * K > 65535:
            raise ValueError(f"beam_select: {B * K} rows of {V} logits are too many")
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        scores, done = scores.contiguous(), done.contiguous()
        dev = logits.device
        part = torch.empty(B * K * ((V + 7 + BLOCK - 1) // BLOCK) * 2, dtype=torch.float32, device=dev)
        out, parent = torch.empty_like(scores), torch.empty((2, B, K), dtype=torch.int64, device=dev)
        parent, token = parent.unbind(0)
        ended = torch.empty_like(done)
        if B:
            with _lib.on_device(device):
                rc = _lib.entry("cb_beam_select", "pliiiippipppppp")(
                    logits.data_ptr(), logits.stride(0), int(f32), B, K, V, scores.data_ptr(),
                    done.data_ptr(), -1 if eos_id is None else eos_id, part.data_ptr(),
                    out.data_ptr(), parent.data_ptr(), token.data_ptr(), ended.data_ptr(),
                    _lib.stream_int())
            _lib.check_rc(rc, "cb_beam_select", launches=2)
        return out, parent, token, ended
    x = logits.double().view(B, K, V)
    total = scores.double()[:, :, None] + (x - torch.logsumexp(x, -1, keepdim=True))
    ended = torch.full_like(total, -math.inf)
    if eos_id is not None:
        ended[:, :, eos_id] = scores.double()
    total = torch.where(done[:, :, None], ended, total)
    total = torch.where(torch.isnan(total), torch.full_like(total, -math.inf), total).view(B, K * V)
    if V < K:                                       # one place per beam at least
        total = torch.nn.functional.pad(total, (0, K), value=-math.inf)
    best, where = torch.sort(total, dim=-1, descending=True, stable=True)
    best, where = best[:, :K], where[:, :K]
    empty = best == -math.inf
    parent = torch.where(empty, torch.arange(K)[None], where // V)
    token = torch.where(empty, torch.full_like(where, eos_id or 0), where % V)
    over = torch.gather(done, 1, parent) | empty
    if eos_id is not None:
        over = over | (token == eos_id)
    return best.float(), parent, token, over


def beam_pages(page_table: torch.Tensor, parent: torch.Tensor, length: torch.Tensor,
               pool: torch.Tensor, num_pages: int
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The page table ``[B * K, pages]`` (int32) after every beam has become a child of ``parent [B,
    K]`` (int64, within the request), and the copies this takes: ``(table, src, dst)``, ``src`` / ``dst``
    int32 ``[B * K]`` with -1 where there is none.

    A request's beams all hold ``length[b]`` tokens (int32); afterwards every beam has a page of its own
    for the next one.  Full pages are taken over from the parent.  If the last page is not full, the
    first of the beams whose parents hold it (one parent, or several that share it still) keeps it and
    the others copy it to free pages; if it is, every beam gets a free page.  Free pages come from
    ``pool [B, n]`` (int32, the pages that belong to the request), in its order and each once, without
    those that a new row of the request holds; ``K`` times the pages that a beam can have on its own, plus
    ``K``, always suffice.  When they do not, the row's entry is -1 and the status word says so.  Columns
    behind the next token's page keep what the row had."""
    if parent.dim() != 2 or parent.dtype != torch.int64:
        raise ValueError(f"beam_pages: parent is int64 [B, K], got {tuple(parent.shape)} {parent.dtype}")
    B, K = parent.shape
    if not 1 <= K <= MAX_BEAMS:
        raise ValueError(f"beam_pages: 1 to {MAX_BEAMS} beams, not {K}")
    if page_table.dim() != 2 or page_table.shape[0] != B * K or page_table.dtype != torch.int32 \
            or page_table.shape[1] < 1:
        raise ValueError(f"beam_pages: the page table is int32 [{B * K}, pages]")
    if tuple(length.shape) != (B,) or length.dtype != torch.int32:
        raise ValueError(f"beam_pages: length is int32 [{B}]")
    if pool.dim() != 2 or pool.shape[0] != B or pool.dtype != torch.int32:
        raise ValueError(f"beam_pages: the pool is int32 [{B}, pages]")
    device = page_table.get_device()
    if parent.get_device() != device or length.get_device() != device \
            or pool.get_device() != device:
        raise ValueError("beam_pages: tensors on different devices")
    if not 1 <= num_pages <= 200 * 1024 * 8:
        raise ValueError(f"beam_pages: a cache of 1 to {200 * 1024 * 8} pages, not {num_pages}")
    dev, width = page_table.device, page_table.shape[1]
    page_table, parent, length, pool = (t.contiguous() for t in (page_table, parent, length, pool))
    table = torch.empty_like(page_table)
    moves = torch.empty((2, B * K), dtype=torch.int32, device=dev)
    src, dst = moves.unbind(0)
    if B == 0:
        return table, src, dst
    if device >= 0:
        with _lib.on_device(device):
            rc = _lib.entry("cb_beam_pages", "piiipppiippppp")(
                page_table.data_ptr(), width, B, K, parent.data_ptr(), length.data_ptr(),
                pool.data_ptr(), pool.shape[1], num_pages, table.data_ptr(), src.data_ptr(),
                dst.data_ptr(), _lib.status_buffer(dev).data_ptr(), _lib.stream_int())
        _lib.check_rc(rc, "cb_beam_pages")
        return table, src, dst
    moves.fill_(-1)
    table.copy_(page_table)
    for b in range(B):
        n, par = int(length[b]), parent[b].tolist()
        lp, rest = divmod(n, PAGE)
        if n < 0 or lp >= width or any(not 0 <= p < K for p in par):
            raise ValueError(f"beam_pages: request {b} has {n} tokens, parents {par}, {width} pages")
        held = set()
        tails = [int(page_table[b * K + p, lp]) for p in par]
        keeps = [bool(rest) and t not in tails[:j] for j, t in enumerate(tails)]
        for j, p in enumerate(par):
            table[b * K + j, :lp] = page_table[b * K + p, :lp]
            held.update(page_table[b * K + p, :lp].tolist())
            if keeps[j]:
                held.add(tails[j])
        free = iter(dict.fromkeys(p for p in pool[b].tolist() if p not in held))
        for j, tail in enumerate(tails):
            if keeps[j]:
                table[b * K + j, lp] = tail
                continue
            page = next(free, None)
            if page is None:
                raise ValueError(f"beam_pages: the pool of request {b} is too small")
            table[b * K + j, lp] = page
            if rest:
                src[b * K + j], dst[b * K + j] = tail, page
    return table, src, dst


def copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies page ``src[i]`` to page ``dst[i]`` (int32, -1: nothing) in every tensor of ``caches``, whose
    first dimension is the page.  A page that is written is neither read nor written twice.  A page that the
    tensors do not have is not copied, and the status word says so."""
    if src.shape != dst.shape or src.dim() != 1 or src.dtype != torch.int32 \
            or dst.dtype != torch.int32:
        raise ValueError("copy_pages: src and dst are int32 of one length")
    if not caches or src.numel() == 0:
        return
    pages, device, n = caches[0].shape[0], src.get_device(), len(caches)
    if dst.get_device() != device:
        raise ValueError("copy_pages: tensors on different devices")
    base, sizes, odd = [], [], 0
    for c in caches:
        if not c.is_contiguous() or c.dim() < 1 or c.shape[0] != pages:
            raise ValueError("copy_pages: contiguous tensors with one number of pages")
        if c.get_device() != device:
            raise ValueError("copy_pages: tensors on different devices")
        base.append(c.data_ptr())
        sizes.append(c.numel() // max(1, pages) * c.element_size())
        odd |= base[-1] | sizes[-1]
    if device >= 0:
        if odd % 4 or 0 in sizes:
            raise ValueError("copy_pages: a page is a multiple of four bytes")
        if max(sizes) >= 1 << 31:
            raise ValueError("copy_pages: a page of 2 GB or more")
        with _lib.on_device(device):
            src, dst = src.contiguous(), dst.contiguous()
            rc = _lib.entry("cb_beam_copy", "ppippiipp")(
                (ctypes.c_void_p * n)(*base), (ctypes.c_int * n)(*sizes), n, src.data_ptr(),
                dst.data_ptr(), src.numel(), pages,
                _lib.status_buffer(src.device).data_ptr(), _lib.stream_int())
        _lib.check_rc(rc, "cb_beam_copy", launches=(n + 191) // 192)
        return
    for s, d in zip(src.tolist(), dst.tolist()):
        if max(s, d) >= pages and min(s, d) >= 0:
            raise ValueError(f"copy_pages: page {s} to page {d} of {pages}")
        if s >= 0 and d >= 0:
            for c in caches:
                raw = c.view(torch.int8) if c.element_size() == 1 else c
                raw[d] = raw[s]


def beam_reorder(page_table: torch.Tensor, parent: torch.Tensor, length: torch.Tensor,
                 pool: torch.Tensor, caches: List[torch.Tensor]) -> torch.Tensor:
    """:func:`beam_pages` and its copies in every tensor of ``caches``; returns the new page table."""
    if not caches:
        raise ValueError("beam_reorder: no cache")
    table, src, dst = beam_pages(page_table, parent, length, pool, caches[0].shape[0])
    copy_pages(caches, src, dst)
    return table
