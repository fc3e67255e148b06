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


@pytest.mark.parametrize("reqs, beams", [(2, 3), (40, 4)])
@pytest.mark.parametrize("tokens", [40, 48])
def test_steps_behind_a_shared_prefix(cuda, reqs, beams, tokens):
    """Requests that go on from one prefix, which ends inside a page or with one: `own` counts the page that it ends in for the first call,
    which gives every beam a copy, and the whole ones from then on.  At every step each page is the prefix's, a beam's or free."""
    r = random.Random(reqs + tokens)
    page, width, n = 16, 9, reqs * beams
    shared, whole = PH.up(tokens, page), tokens // page
    n_pages = shared + n * width
    order = r.sample(range(n_pages), n_pages)
    prefix = order[:shared]
    free, counts = ints(order[shared:] + [0] * shared, cuda), ints([n_pages - shared, 0], cuda)
    tables = ints([prefix + [-1] * (width - shared)] * n, cuda)
    lens = ints([tokens if b % beams == 0 else 0 for b in range(n)], cuda)      # the prompt is the first beam's
    parents = [[0] * beams for _ in range(reqs)]
    for step in range(40):
        s = pages.reorder(ints(parents, cuda), lens, tables, free, counts, page, ints([shared if step == 0 else whole] * reqs, cuda))
        if step == 0:
            assert s.used.tolist() == [tokens % page] * n and (s.src[s.src >= 0] == prefix[-1]).all()
        p = pages.plan(s.lens, torch.ones_like(s.lens), s.tables, free, s.counts, page, n)
        tables, lens, counts = s.tables, p.lens, p.counts
        assert lens.tolist() == [tokens + step + 1] * n and counts[1].item() == 0
        held = set()
        for row, k in zip(tables.tolist(), lens.tolist()):
            assert row[:whole] == prefix[:whole]
            held |= set(row[whole:PH.up(k, page)])
        left = free[:counts[0].item()].tolist()
        assert -1 not in held and not held & set(prefix) and sorted([*prefix, *held, *left]) == list(range(n_pages)), step
        slots = p.slots.tolist()
        assert len(set(slots)) == n and not {x // page for x in slots} & set(prefix)      # no two beams write to one page
        parents = [[r.randrange(beams) for _ in range(beams)] for _ in range(reqs)]
    s = pages.reorder(ints([[-1] * beams] * reqs, cuda), lens, tables, free, counts, page, ints([whole] * reqs, cuda))
    assert s.counts.tolist() == [n_pages - shared, 0]
