"""Beams of requests whose first pages belong to others too (`own` of pages.reorder)."""
import random

import pytest
import torch

from nemicli_terminal_b200 import pages

from tests import paging_helpers as PH
from tests.test_gpu_pages import beams_of, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reqs, beams, page, width, shared", [(2, 3, 16, 5, 2), (40, 3, 16, 5, 2), (3, 16, 32, 4, 1), (1, 64, 16, 9, 4)])
@pytest.mark.parametrize("own", [(1 << 31) - 1, (1 << 31) - 600, 1 << 20, -1, -(1 << 31)])
def test_own_of_any_size(cuda, reqs, beams, page, width, shared, own):
    """More places than a table has are all of it: nothing falls free and every partly filled page is copied; fewer than none are none."""
    r = random.Random(reqs * beams)
    lens, tables, rest, n_pages = beams_of(r, reqs, beams, page, width, shared, reqs * beams)
    parents = [[r.choice([-1, r.randrange(beams)]) for _ in range(beams)] for _ in range(reqs)]
    free, counts = rest + [0] * (n_pages - len(rest)), [len(rest), 0]
    want = PH.reorder(parents, lens, tables, free, counts, page, [own] * reqs)
    f = ints(free, cuda)
    got = pages.reorder(ints(parents, cuda), ints(lens, cuda), ints(tables, cuda), f, ints(counts, cuda), page, ints([own] * reqs, cuda))
    for name, w in zip(("tables", "lens", "counts", "src", "dst", "used"), want):
        assert getattr(got, name).tolist() == w, name
    assert f.tolist() == want[6]
