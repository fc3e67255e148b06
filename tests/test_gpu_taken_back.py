"""Drafted tokens that a step takes back: the pages behind the shorter lengths go back with release, as the documents show it."""
import random

import pytest
import torch

from nemicli_terminal_b200 import _lib, pages

from tests import paging_helpers as PH
from tests.test_gpu_pages import I32, ints

pytestmark = pytest.mark.gpu


def take_back(kept, p, tables, free, page, drafts):
    """-> lens, counts: sequence b keeps kept[b] of its p.lens[b] tokens, at most `drafts` fewer."""
    first = (kept + page - 1) // page
    place = first[:, None] + torch.arange((drafts + page - 1) // page, device=kept.device)
    behind = tables.gather(1, place.clamp(max=tables.shape[1] - 1).long())
    tokens = ((p.lens + page - 1) // page - first) * page
    _, counts = pages.release(torch.ones_like(kept, dtype=torch.bool), tokens, behind, free, p.counts, page)
    return kept, counts


@pytest.mark.parametrize("drafts", [4, 16, 41])
def test_no_page_is_lost(cuda, drafts):
    page, seqs, width = 16, 9, 12
    n_pages = seqs * width
    r = random.Random(drafts)
    free, counts = pages.pool(n_pages, cuda)
    tables, lens = torch.full((seqs, width), -1, dtype=I32, device=cuda), ints([0] * seqs, cuda)
    _lib.device_status(device=cuda)
    for step in range(50):
        new = [min(drafts, width * page - n) for n in lens.tolist()]
        p = pages.plan(lens, ints(new, cuda), tables, free, counts, page, seqs * drafts)
        kept = lens + ints([r.randint(0, n) for n in new], cuda)
        lens, counts = take_back(kept, p, tables, free, page, drafts)
        held = [e for t, n in zip(tables.tolist(), lens.tolist()) for e in t[:PH.up(n, page)]]
        assert sorted(held + free[:counts[0].item()].tolist()) == list(range(n_pages)), step
        done = [n > 150 for n in lens.tolist()]
        lens, counts = pages.release(ints(done, cuda, torch.bool), lens, tables, free, counts, page)
    assert counts[1].item() == 0 and _lib.device_status(device=cuda) == 0
