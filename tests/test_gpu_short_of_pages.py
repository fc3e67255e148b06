"""Pages that were missing: what a server does about it, and back to normal."""
import random

import pytest
import torch

from nemicli_terminal_b200 import _lib, pages

from tests import paging_helpers as PH
from tests.test_gpu_pages import I32, ints

pytestmark = pytest.mark.gpu


def test_the_count_set_back(cuda):
    """The sequences that lack pages are ended; then counts[1] is set to 0, and later steps find and lose no page."""
    page, seqs, width, n_pages = 16, 8, 8, 24
    r = random.Random(3)
    free, counts = pages.pool(n_pages, cuda)
    tables, lens = torch.full((seqs, width), -1, dtype=I32, device=cuda), ints([0] * seqs, cuda)
    set_back = plain = 0
    for step in range(120):
        p = pages.plan(lens, ints([r.randint(0, 20) if n < 90 else 0 for n in lens.tolist()], cuda), tables, free, counts, page, 200)
        short = [-1 in t[:PH.up(n, page)] for t, n in zip(tables.tolist(), p.lens.tolist())]
        assert any(short) == (p.counts[1].item() > 0)
        done = [s or r.random() < 0.1 for s in short]
        lens, counts = pages.release(ints(done, cuda, torch.bool), p.lens, tables, free, p.counts, page)
        if any(short):
            counts[1].zero_()
            set_back += 1
        else:
            plain += any(done)
        held = [e for t, n in zip(tables.tolist(), lens.tolist()) for e in t[:PH.up(n, page)]]
        assert sorted(held + free[:counts[0].item()].tolist()) == list(range(n_pages)), step
    assert set_back > 3 and plain > 3
    _lib.device_status(device=cuda)
