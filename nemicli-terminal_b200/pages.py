"""Page tables of a paged cache (kvcache.KVCache), built on the GPU (kernels: csrc/qmv_pages.cu; contracts:
include/nemicli_qmv.h, qmv_page_plan).

* `plan` — a step's slots, positions and row starts from the sequences' lengths, new pages taken from the free ones.
* `release` — the pages of sequences that ended, given back.
* `reorder` — the tables of a beam search's next step: beams part and join, pages that no beam holds become free.

Free pages are a stack in two tensors: `free` int32 (pages of the cache,) and `counts` int32 (2,): counts[0] entries of free
count, the last is taken first; counts[1] is a running number of pages that were asked for in vain, which a caller looks at
now and then (`pool` makes both).  Everything is read on the device on torch's current stream and CUDA-graph safe.  Lengths and counts come back
in new tensors, so that a call may be made again; tables and free are changed in place.  A captured step copies them back itself:

    step = pages.plan(lens, new, tables, free, counts, cache.page, rows)
    q = cache.write(k, v, step.slots, q=q, rope=(cos, sin, step.positions))
    o = cache.attend(q, tables, step.lens, step.starts, max_new=most)
    lens.copy_(step.lens), counts.copy_(step.counts)

The reference has no counterpart (one sequence, one contiguous cache: ggufengine/mmvq.py:139-180).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

MOST_BEAMS = 64


class Plan(NamedTuple):
    slots: torch.Tensor                    # int64 (rows,), -1 behind the last token
    positions: torch.Tensor                # int64 (rows,)
    starts: torch.Tensor                   # int32 (sequences + 1,) first row of each sequence
    lens: torch.Tensor                     # int32 (sequences,) tokens held, the new ones among them
    counts: torch.Tensor                   # int32 (2,)


class Reordered(NamedTuple):
    tables: torch.Tensor                   # int32 (requests * beams, width), -1 behind a beam's pages
    lens: torch.Tensor                     # int32 (requests * beams,)
    counts: torch.Tensor                   # int32 (2,)
    src: torch.Tensor                      # int32 (requests * beams,): KVCache.copy(src, dst, used) of every layer
    dst: torch.Tensor
    used: torch.Tensor


def pool(n_pages: int, device=None):
    """(free, counts) with every page free; page 0 is taken first."""
    free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device="cuda" if device is None else device)
    return free, torch.tensor([n_pages, 0], dtype=torch.int32, device=free.device)


_I32 = torch.int32
_PAGES = (16, 32, 64, 128, 256, 512, 1024)


def _fits(t: torch.Tensor, where: int, shape, dtype=_I32) -> bool:
    return t.dtype is dtype and t.shape == shape and t.get_device() == where and t.is_contiguous()


def _refuse(what: str, t: torch.Tensor, name: str, shape, device, dtype=_I32):
    raise RuntimeError(f"{what} {name}: contiguous {dtype} {tuple(shape)} on {device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _common(what: str, tables, lens, free, counts, page: int):
    """The index of the tables' device, the tables and their width."""
    where = tables.get_device()
    if where < 0 or not tables.is_cuda:
        raise RuntimeError(f"{what}: tables on {tables.device}; the tables live on a CUDA device")
    if tables.dim() != 2 or tables.dtype is not _I32 or not tables.is_contiguous():
        _refuse(what, tables, "tables", ("sequences", "width"), tables.device)
    n, width = tables.shape
    if not _fits(lens, where, (n,)):
        _refuse(what, lens, "lens", (n,), tables.device)
    if free.dim() != 1 or not _fits(free, where, free.shape):
        _refuse(what, free, "free", ("pages",), tables.device)
    if not _fits(counts, where, (2,)):
        _refuse(what, counts, "counts", (2,), tables.device)
    if page not in _PAGES or width == 0 or free.shape[0] == 0 or not 0 < n <= 65535:
        raise RuntimeError(f"{what}: pages of 16 to 1024 tokens (a power of two), 1 to 65535 tables with a page, and a cache with one "
                           f"expected, got pages of {page}, tables {tuple(tables.shape)}, free {tuple(free.shape)}")
    return where, n, width


def plan(lens: torch.Tensor, new: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, counts: torch.Tensor, page: int,
         rows: int) -> Plan:
    """Sequence b holds lens[b] tokens and gets new[b] (int32, 0 or more); the pages it lacks are taken from free and written into its row
    of tables.  rows: the step's rows, at least the new tokens; the ones behind the last token are padding (slot -1).  Tokens beyond a
    table's end are dropped; tokens whose page is missing get slot -1 and a table entry -1, and counts[1] goes up: both set the
    device status.  One launch."""
    where, n, width = _common("pages.plan", tables, lens, free, counts, page)
    if not _fits(new, where, (n,)):
        _refuse("pages.plan", new, "new", (n,), tables.device)
    if not 0 <= rows <= 1 << 30:
        raise RuntimeError(f"pages.plan: {rows} rows")
    device = tables.device
    slots = torch.empty(rows, dtype=torch.int64, device=device)
    out = Plan(slots, torch.empty_like(slots), torch.empty(n + 1, dtype=_I32, device=device), torch.empty_like(lens), torch.empty_like(counts))
    with _lib.on_device(device):
        st = _lib.load().qmv_page_plan(lens.data_ptr(), new.data_ptr(), tables.data_ptr(), n, width, page, free.data_ptr(), free.shape[0],
                                       counts.data_ptr(), rows, slots.data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(),
                                       out[4].data_ptr(), _lib.stream_of(device))
    if st:
        _lib.check(st, "qmv_page_plan")
    return out


def release(done: torch.Tensor, lens: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, counts: torch.Tensor, page: int):
    """The pages of the sequences with done (bool) go back to free; -> lens, 0 for them, and counts.  Their pages must be their own (a
    request's beams share some: `reorder` with parents -1 frees those).  One launch."""
    where, n, width = _common("pages.release", tables, lens, free, counts, page)
    if not _fits(done, where, (n,), torch.bool):
        _refuse("pages.release", done, "done", (n,), tables.device, torch.bool)
    device = tables.device
    lens_out, counts_out = torch.empty_like(lens), torch.empty_like(counts)
    with _lib.on_device(device):
        st = _lib.load().qmv_page_release(done.data_ptr(), lens.data_ptr(), tables.data_ptr(), n, width, page, free.data_ptr(),
                                          free.shape[0], counts.data_ptr(), lens_out.data_ptr(), counts_out.data_ptr(),
                                          _lib.stream_of(device))
    if st:
        _lib.check(st, "qmv_page_release")
    return lens_out, counts_out


def reorder(parents: torch.Tensor, lens: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, counts: torch.Tensor, page: int,
            own: Optional[torch.Tensor] = None) -> Reordered:
    """parents int32 (requests, beams), as beams.select gives them: beam j of request r goes on from beam parents[r, j] (-1: it ends);
    lens (requests * beams,) and tables (requests * beams, width) are its beams'.  Beams of a request share whole pages, at the same
    place of their tables.  Pages that no beam holds any more become free.  Of the beams that would write to one partly filled page the
    first keeps it, the others get a copy: `KVCache.copy(src, dst, used)` makes it, once a layer and before the next write.
    own int32 (requests,): leading places of the tables whose pages belong to others too (a shared prefix), which are neither freed nor
    written to.  Two launches."""
    where, n, width = _common("pages.reorder", tables, lens, free, counts, page)
    if parents.dim() != 2 or not _fits(parents, where, parents.shape):
        _refuse("pages.reorder", parents, "parents", ("requests", "beams"), tables.device)
    n_req, beams = parents.shape
    if not 0 < beams <= MOST_BEAMS or n_req * beams != n:
        raise RuntimeError(f"pages.reorder: parents {tuple(parents.shape)} for {n} tables, up to {MOST_BEAMS} beams")
    if own is not None and not _fits(own, where, (n_req,)):
        _refuse("pages.reorder", own, "own", (n_req,), tables.device)
    device, lib = tables.device, _lib.load()
    out = Reordered(torch.empty_like(tables), torch.empty_like(lens), torch.empty_like(counts), torch.empty_like(lens), torch.empty_like(lens),
                    torch.empty_like(lens))
    nbytes = lib.qmv_page_reorder_workspace_bytes(n_req, beams, width)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    with _lib.on_device(device):
        st = lib.qmv_page_reorder(parents.data_ptr(), lens.data_ptr(), tables.data_ptr(), _lib.addr(own), n_req, beams, width, page,
                                  free.data_ptr(), free.shape[0], counts.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), out[3].data_ptr(),
                                  out[4].data_ptr(), out[5].data_ptr(), out[2].data_ptr(), ws.data_ptr(), nbytes, _lib.stream_of(device))
    if st:
        _lib.check(st, "qmv_page_reorder")
    return out
