"""Page tables of a paged cache (kvcache.KVCache), built on the GPU (kernels: csrc/qmv_pages.cu; contracts:
include/nemicli_qmv.h, qmv_page_plan).

* `plan` — a step's slots, positions and row starts from the sequences' lengths, new pages taken from the free ones.
* `release` — the pages of sequences that ended, given back.
* `reorder` — the tables of a beam search's next step: beams part and join, pages that no beam holds become free.

Free pages are a stack in two tensors: `free` int32 (pages of the cache,) and `counts` int32 (2,): counts[0] entries of free
count, the last is taken first; counts[1] is a running number of pages that were asked for in vain, which a caller looks at
now and then, and sets to 0 when the sequences that lacked them have been released (`pool` makes both).  Everything is read on the device on torch's current stream and CUDA-graph safe.  Lengths and counts come back
in new tensors, so that a call may be made again; tables and free are changed in place.  A call's new tensors are parts of one allocation
(one takes 0.6 us): it lives as long as any of them, and none of them is to be resized (`resize_` would grow into the next); clone what is kept
for long.  A captured step copies lengths and counts back itself:

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


def plan(lens: torch.Tensor, new: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, counts: torch.Tensor, page: int,
         rows: int) -> Plan:
    """Sequence b holds lens[b] tokens and gets new[b] (int32, 0 or more); the pages it lacks are taken from free and written into its row
    of tables.  rows: the step's rows, at least the new tokens; the ones behind the last token are padding (slot -1).  Tokens beyond a
    table's end are dropped; tokens whose page is missing get slot -1 and a table entry -1, and counts[1] goes up: both set the
    device status.  Entries of a table behind its sequence's tokens are written over: where drafted tokens are taken back, the pages that only they
    had go back first, by a release of tables that hold those pages alone.  One launch."""
    return Plan._make(_lib.host().plan(lens, tables, free, counts, page, new, rows))


def release(done: torch.Tensor, lens: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, counts: torch.Tensor, page: int):
    """The pages of the sequences with done (bool) go back to free; -> lens, 0 for them, and counts.  Their pages must be their own (a
    request's beams share some: `reorder` with parents -1 frees those).  Entries of -1, pages that were missing, are left out while counts[1]
    is not 0, which takes a look at every entry of the tables (50 us for 1021 sequences of up to 512 pages, else 4.4): set counts[1] to 0 once the
    sequences that lacked pages are released, not before.  One launch."""
    return _lib.host().release(lens, tables, free, counts, page, done)


def reorder(parents: torch.Tensor, lens: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, counts: torch.Tensor, page: int,
            own: Optional[torch.Tensor] = None) -> Reordered:
    """parents int32 (requests, beams), as beams.select gives them: beam j of request r goes on from beam parents[r, j] (-1: it ends);
    lens (requests * beams,) and tables (requests * beams, width) are its beams'.  Beams of a request share whole pages, at the same
    place of their tables.  Pages that no beam holds any more become free.  Of the beams that would write to one partly filled page the
    first keeps it, the others get a copy: `KVCache.copy(src, dst, used)` makes it, once a layer and before the next write.
    own int32 (requests,): leading places of the tables whose pages belong to others too (a shared prefix), which are neither freed nor
    written to.  Where a prefix ends inside a page, own counts that page for the first call only: every beam gets its copy there, which is
    the request's own from then on, so later calls pass the whole pages alone (with the same own that page would be copied at every call
    and its copies be lost to free).  One launch for up to 32 requests of 8 beams with short tables, else two."""
    return Reordered._make(_lib.host().reorder(lens, tables, free, counts, page, parents, own))
