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


def _index(t: torch.Tensor, what: str, device, shape, dtype=torch.int32):
    got = t.shape
    ok = t.device == device and t.dtype == dtype and len(got) == len(shape) and t.is_contiguous()
    if ok:
        for n, want in zip(got, shape):
            if want is not None and n != want:
                ok = False
    if not ok:
        raise RuntimeError(f"{what}: contiguous {dtype} {tuple(shape)} on {device} expected, got {t.dtype} {tuple(got)} on {t.device}")


def _common(what: str, tables, lens, free, counts, page: int):
    device = tables.device
    if not _lib.on_gpu(tables):
        raise RuntimeError(f"{what}: tables on {device}; the tables live on a CUDA device")
    _index(tables, f"{what} tables", device, (None, None))
    n, width = tables.shape
    _index(lens, f"{what} lens", device, (n,))
    _index(free, f"{what} free", device, (None,))
    _index(counts, f"{what} counts", device, (2,))
    if page not in (16, 32, 64, 128, 256, 512, 1024) or width == 0 or free.shape[0] == 0 or not 0 < n <= 65535:
        raise RuntimeError(f"{what}: pages of 16 to 1024 tokens (a power of two), 1 to 65535 tables with a page, and a cache with one "
                           f"expected, got pages of {page}, tables {tuple(tables.shape)}, free {tuple(free.shape)}")
    return device, n, width


def plan(lens: torch.Tensor, new: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, counts: torch.Tensor, page: int,
         rows: int) -> Plan:
    """Sequence b holds lens[b] tokens and gets new[b] (int32, 0 or more); the pages it lacks are taken from free and written into its row
    of tables.  rows: the step's rows, at least the new tokens; the ones behind the last token are padding (slot -1).  Tokens beyond a
    table's end are dropped; tokens whose page is missing get slot -1 and a table entry -1, and counts[1] goes up: both set the
    device status.  One launch."""
    device, n, width = _common("pages.plan", tables, lens, free, counts, page)
    _index(new, "pages.plan new", device, (n,))
    if not 0 <= rows <= 1 << 30:
        raise RuntimeError(f"pages.plan: {rows} rows")
    slots, positions = (torch.empty(rows, dtype=torch.int64, device=device) for _ in range(2))
    starts, lens_out, counts_out = (torch.empty(k, dtype=torch.int32, device=device) for k in (n + 1, n, 2))
    with _lib.on_device(device):
        st = _lib.load().qmv_page_plan(lens.data_ptr(), new.data_ptr(), tables.data_ptr(), n, width, page, free.data_ptr(), free.shape[0],
                                       counts.data_ptr(), rows, slots.data_ptr(), positions.data_ptr(), starts.data_ptr(),
                                       lens_out.data_ptr(), counts_out.data_ptr(), _lib.stream_of(device))
    if st:
        _lib.check(st, "qmv_page_plan")
    return Plan(slots, positions, starts, lens_out, counts_out)


def release(done: torch.Tensor, lens: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, counts: torch.Tensor, page: int):
    """The pages of the sequences with done (bool) go back to free; -> lens, 0 for them, and counts.  Their pages must be their own (a
    request's beams share some: `reorder` with parents -1 frees those).  One launch."""
    device, n, width = _common("pages.release", tables, lens, free, counts, page)
    _index(done, "pages.release done", device, (n,), torch.bool)
    lens_out, counts_out = (torch.empty(k, dtype=torch.int32, device=device) for k in (n, 2))
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
    device, n, width = _common("pages.reorder", tables, lens, free, counts, page)
    _index(parents, "pages.reorder parents", device, (None, None))
    n_req, beams = parents.shape
    if not 0 < beams <= MOST_BEAMS or n_req * beams != n:
        raise RuntimeError(f"pages.reorder: parents {tuple(parents.shape)} for {n} tables, up to {MOST_BEAMS} beams")
    if own is not None:
        _index(own, "pages.reorder own", device, (n_req,))
    lib = _lib.load()
    out = torch.empty_like(tables)
    lens_out, src, dst, used = torch.empty((4, n), dtype=torch.int32, device=device).unbind(0)
    counts_out = torch.empty(2, dtype=torch.int32, device=device)
    nbytes = lib.qmv_page_reorder_workspace_bytes(n_req, beams, width)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    with _lib.on_device(device):
        st = lib.qmv_page_reorder(parents.data_ptr(), lens.data_ptr(), tables.data_ptr(), _lib.addr(own), n_req, beams, width, page,
                                  free.data_ptr(), free.shape[0], counts.data_ptr(), out.data_ptr(), lens_out.data_ptr(), src.data_ptr(),
                                  dst.data_ptr(), used.data_ptr(), counts_out.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_of(device))
    if st:
        _lib.check(st, "qmv_page_reorder")
    return Reordered(out, lens_out, counts_out, src, dst, used)
