"""Page tables on the GPU against plain forms (paging_helpers): every number equal."""
import random

import pytest
import torch

from nemicli_terminal_b200 import _lib, kvcache, pages

from tests import paging_helpers as PH

pytestmark = pytest.mark.gpu
I32 = torch.int32


def ints(x, device, dtype=I32):
    return torch.tensor(x, dtype=dtype, device=device)


def some_tables(r, seqs, width, page, most, spare):
    """(lens, tables, free pages in any order, pages)"""
    lens = [r.choice([0, 1, page, r.randint(0, most), r.randint(0, most)]) for _ in range(seqs)]
    per = [PH.up(n, page) for n in lens]
    total = sum(per) + spare
    order = r.sample(range(total), total)
    tables, at = [], 0
    for n in per:
        tables.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return lens, tables, order[at:], total


@pytest.mark.parametrize("seqs, page, most, prompt, rows", [
    (1, 16, 40, 0, 1), (1, 64, 500, 700, 700), (64, 64, 700, 0, 64), (7, 16, 100, 90, 400), (1025, 16, 60, 5, 5000),
    (300, 1024, 3000, 2000, 9000), (2500, 32, 70, 1, 4000), (33, 128, 0, 3, 256)])
def test_plan(cuda, seqs, page, most, prompt, rows):
    """More sequences than a CTA looks at together, sequences without a new token, empty caches, steps with padding rows."""
    r = random.Random(seqs + page)
    width = PH.up(most + prompt + 1, page) + 2
    lens, tables, rest, total = some_tables(r, seqs, width, page, most, seqs * (PH.up(prompt, page) + 1))
    new, left = [], rows
    for _ in range(seqs):
        n = min(left, r.choice([0, 1, 1, r.randint(0, max(1, prompt))]))
        new.append(n)
        left -= n
    free = rest + [0] * (total - len(rest))
    got_t, counts = ints(tables, cuda), [len(rest), 3]
    _lib.device_status(device=cuda)
    want = PH.plan(lens, new, tables, free, counts, page, rows)
    for _ in range(2):                                           # the same call gives the same again
        p = pages.plan(ints(lens, cuda), ints(new, cuda), got_t, ints(free, cuda), ints(counts, cuda), page, rows)
        assert p.slots.dtype == p.positions.dtype == torch.int64
        for got, w in zip((*p, got_t), (*want[:5], want[5])):
            assert got.tolist() == w
    assert not want[6] and _lib.device_status(device=cuda) == 0


def test_plan_out_of_order(cuda):
    """Tokens beyond a table, negative numbers, more tokens than rows, missing pages, a stack that claims too much, entries and
    free pages outside the cache: cut or left out, and the status says so."""
    page = 16
    cases = [
        dict(lens=[30], new=[5], tables=[[0, 1]], free=[0, 1, 2], counts=[1, 0], rows=8),              # beyond the table
        dict(lens=[-4, 3], new=[2, -1], tables=[[-1, -1], [2, -1]], free=[0, 1, 2], counts=[2, 0], rows=4),
        dict(lens=[0], new=[9], tables=[[-1]], free=[0, 1], counts=[2, 0], rows=5),
        dict(lens=[16, 15, 0], new=[1, 3, 40], tables=[[0, -1, -1], [1, -1, -1], [-1, -1, -1]], free=[2, 3, 0, 0], counts=[2, 7], rows=50),
        dict(lens=[0], new=[1], tables=[[-1]], free=[1, 0], counts=[9, 0], rows=1),
        dict(lens=[5], new=[1], tables=[[99]], free=[0, 1], counts=[2, 0], rows=1),
        dict(lens=[0, 0], new=[1, 1], tables=[[-1], [-1]], free=[5, -3], counts=[2, 0], rows=2),
        dict(lens=[1 << 30], new=[(1 << 31) - 1], tables=[[0, 1]], free=[0, 1], counts=[-5, 0], rows=0)]
    for c in cases:
        want = PH.plan(*[c[k] for k in ("lens", "new", "tables", "free", "counts")], page, c["rows"])
        t = ints(c["tables"], cuda)
        _lib.device_status(device=cuda)
        p = pages.plan(ints(c["lens"], cuda), ints(c["new"], cuda), t, ints(c["free"], cuda), ints(c["counts"], cuda), page, c["rows"])
        for got, w in zip((*p, t), want[:6]):
            assert got.tolist() == w, c
        assert want[6] and _lib.device_status(device=cuda) == 1, c


@pytest.mark.parametrize("seqs, page, most", [(1, 16, 50), (64, 64, 900), (1500, 16, 90)])
def test_release(cuda, seqs, page, most):
    r = random.Random(seqs)
    lens, tables, rest, total = some_tables(r, seqs, PH.up(most, page) + 1, page, most, 5)
    free = rest + [0] * (total - len(rest))
    for chance in (0.0, 0.3, 1.0):
        done = [r.random() < chance for _ in range(seqs)]
        want = PH.release(done, lens, tables, free, [len(rest), 2], page)
        f = ints(free, cuda)
        for _ in range(2):
            got = pages.release(ints(done, cuda, torch.bool), ints(lens, cuda), ints(tables, cuda), f, ints([len(rest), 2], cuda), page)
            assert [g.tolist() for g in got] == [want[0], want[1]] and f.tolist() == want[2]


@pytest.mark.parametrize("seqs, page, most", [(1, 16, 50), (64, 64, 900), (1500, 16, 90)])
def test_release_after_pages_were_missing(cuda, seqs, page, most):
    """Entries of -1 are no pages; without any missing page the entries are not read one by one."""
    r = random.Random(seqs + 1)
    lens, tables, rest, total = some_tables(r, seqs, PH.up(most, page) + 1, page, most, 5)
    free = rest + [0] * (total - len(rest))
    holes = [[-1 if r.random() < 0.2 else e for e in t] for t in tables]
    done = [r.random() < 0.6 for _ in range(seqs)]
    _lib.device_status(device=cuda)
    for t, missing in ((tables, 0), (holes, 9)):
        want = PH.release(done, lens, t, free, [len(rest), missing], page)
        f = ints(free, cuda)
        got = pages.release(ints(done, cuda, torch.bool), ints(lens, cuda), ints(t, cuda), f, ints([len(rest), missing], cuda), page)
        assert [g.tolist() for g in got] == [want[0], want[1]] and f.tolist() == want[2]
    assert _lib.device_status(device=cuda) == 0


def test_short_of_pages_and_on(cuda):
    """Steps that ask for more pages than there are, sequences that end meanwhile: no page is lost and none is there twice."""
    page, seqs, width, n_pages = 16, 6, 8, 20
    r = random.Random(8)
    free, counts = pages.pool(n_pages, cuda)
    tables, lens = torch.full((seqs, width), -1, dtype=I32, device=cuda), ints([0] * seqs, cuda)
    missing = False
    for step in range(60):
        p = pages.plan(lens, ints([r.randint(0, 20) if n < 90 else 0 for n in lens.tolist()], cuda), tables, free, counts, page, 200)
        done = [r.random() < 0.2 for _ in range(seqs)]
        missing |= p.counts[1].item() > 0
        lens, counts = pages.release(ints(done, cuda, torch.bool), p.lens, tables, free, p.counts, page)
        held = [e for t, n in zip(tables.tolist(), lens.tolist()) for e in t[:PH.up(n, page)] if e >= 0]
        assert sorted(held + free[:counts[0].item()].tolist()) == list(range(n_pages)), step
    assert missing
    _lib.device_status(device=cuda)


def test_release_twice_is_noticed(cuda):
    """More pages than the cache has: the rest is dropped."""
    free, counts = pages.pool(4, cuda)
    t = ints([[0, 1, 2]], cuda)
    _lib.device_status(device=cuda)
    lens, counts = pages.release(ints([True], cuda, torch.bool), ints([40], cuda), t, free, counts, 16)
    assert counts.tolist() == [4, 0] and lens.tolist() == [0] and free.tolist() == [3, 2, 1, 0]
    assert _lib.device_status(device=cuda) == 1


def beams_of(r, reqs, beams, page, width, shared, spare):
    """Tables of beams that parted before: whole shared pages, then pages in common by pairs, then their own."""
    lens, tables, at = [], [], 0
    n_pages = reqs * (shared + beams * width) + spare
    order = r.sample(range(n_pages), n_pages)
    for _ in range(reqs):
        tokens = r.choice([shared * page, shared * page + r.randint(1, (width - shared) * page), width * page, shared * page + page])
        base = order[at:at + shared]
        at += shared
        whole = tokens // page
        for k in range(beams):
            row = list(base)
            for i in range(shared, PH.up(tokens, page)):
                if i < whole and k and r.random() < 0.4:
                    row.append(tables[-1][i])                    # the page of the beam before
                else:
                    row.append(order[at])
                    at += 1
            tables.append(row + [-1] * (width - len(row)))
            lens.append(tokens)
    return lens, tables, order[at:], n_pages


@pytest.mark.parametrize("reqs, beams, page, width, shared, spare", [
    (1, 1, 16, 3, 1, 2), (1, 4, 64, 5, 2, 3), (5, 3, 16, 4, 0, 0), (32, 8, 16, 9, 4, 9), (3, 16, 32, 4, 1, 4), (2, 64, 16, 3, 1, 40),
    (1100, 2, 16, 4, 1, 30), (2, 5, 16, 400, 3, 8)])
@pytest.mark.parametrize("kind", ["any", "first", "ends"])
def test_reorder(cuda, reqs, beams, page, width, shared, spare, kind):
    """All beams from one, beams that end, shared pages in the middle, pages of other requests taken over, prefixes of others."""
    r = random.Random(reqs * beams + width)
    lens, tables, rest, n_pages = beams_of(r, reqs, beams, page, width, shared, spare)
    parents = [[{"any": r.randrange(beams), "first": 0, "ends": r.choice([-1, r.randrange(beams)])}[kind] for _ in range(beams)]
               for _ in range(reqs)]
    own = [r.choice([0, 1, shared, shared + 1]) for _ in range(reqs)] if kind == "ends" else None
    left = r.choice([0, min(len(rest), 2), len(rest)])
    free, counts = rest[:left] + [0] * (n_pages - left), [left, 1]
    want = PH.reorder(parents, lens, tables, free, counts, page, own)
    f = ints(free, cuda)
    for _ in range(2):
        got = pages.reorder(ints(parents, cuda), ints(lens, cuda), ints(tables, cuda), f, ints(counts, cuda), page,
                            None if own is None else ints(own, cuda))
        for name, w in zip(("tables", "lens", "counts", "src", "dst", "used"), want):
            assert getattr(got, name).tolist() == w, name
        assert f.tolist() == want[6]
    live = [p for row, n in zip(want[0], want[1]) for p in row[:PH.up(n, page)] if p >= 0]
    assert not set(live) & set(want[6][:want[2][0]])             # no page is both held and free


def test_reorder_out_of_order(cuda):
    """Parents outside the request end their beams; beams that were given one partly filled page part here; lengths are cut."""
    _lib.device_status(device=cuda)
    t = ints([[0, 1], [0, 1], [0, 1]], cuda)
    free, counts = ints([3, 4, 5, 0, 0, 0], cuda), ints([3, 0], cuda)
    got = pages.reorder(ints([[2, 1, 7]], cuda), ints([20, 20, 99], cuda), t, free, counts, 16)
    assert _lib.device_status(device=cuda) == 1
    assert got.lens.tolist() == [32, 20, 0]                       # the third holds whole pages: nothing to copy
    assert got.tables.tolist() == [[0, 1], [0, 1], [-1, -1]]
    got = pages.reorder(ints([[0, 1, 1]], cuda), ints([20, 20, 20], cuda), t, free, counts, 16)
    assert got.tables.tolist() == [[0, 1], [0, 5], [0, 4]] and got.counts.tolist() == [1, 0]
    assert got.src.tolist() == [-1, 1, 1] and got.dst.tolist() == [-1, 5, 4] and got.used.tolist() == [0, 4, 4]
    assert _lib.device_status(device=cuda) == 0


@pytest.mark.parametrize("dim, kf, vf, page", [(64, "Q4_0", "Q8_0", 16), (96, "Q8_0", "Q4_0", 16), (128, "Q4_0", "Q4_0", 64), (256, "Q8_0", "Q8_0", 32)])
def test_copy(cuda, dim, kf, vf, page):
    """The first tokens of a page (two at a time for V), the rest of the target and all other pages stay; -1 and pages outside the
    cache copy nothing."""
    g = torch.Generator(device=cuda).manual_seed(dim)
    c = kvcache.KVCache(12, 3, dim, page, kf, vf, cuda)
    for t in (c.k_codes, c.v_codes):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=cuda, dtype=torch.uint8))
    c.scales.copy_(torch.randn(c.scales.shape, generator=g, device=cuda))
    old = [t.clone() for t in (c.k_codes, c.v_codes, c.scales)]
    src, dst, used = [0, 1, -1, 2, 3, 4, 0], [5, 6, 7, -1, 8, 9, 10], [1, page - 1, 3, 3, page, 0, 6]
    _lib.device_status(device=cuda)
    c.copy(ints(src, cuda), ints(dst, cuda), ints(used, cuda))
    for s, d, u in zip(src, dst, used):
        if s >= 0 and d >= 0:
            old[0][d, :, :u] = old[0][s, :, :u]
            old[1][d, :, :(u + 1) // 2] = old[1][s, :, :(u + 1) // 2]
            old[2][d, :, :u] = old[2][s, :, :u]
    for a, b in zip((c.k_codes, c.v_codes, c.scales), old):
        assert torch.equal(a, b)
    assert _lib.device_status(device=cuda) == 0
    c.copy(ints([[3, 12]], cuda), ints([[11, 1]], cuda))
    assert _lib.device_status(device=cuda) == 1
    for t in old:
        t[11] = t[3]
    for a, b in zip((c.k_codes, c.v_codes, c.scales), old):
        assert torch.equal(a, b)
    c.copy(ints([], cuda), ints([], cuda))


def test_calls_on_streams_and_in_graphs(cuda):
    """A captured decode step of plan and release, replayed as the sequences grow; and the same calls on another stream."""
    page, seqs, width = 16, 5, 6
    free, counts = pages.pool(40, cuda)
    tables = torch.full((seqs, width), -1, dtype=I32, device=cuda)
    lens, new, done = ints([0] * seqs, cuda), ints([7, 1, 16, 0, 3], cuda), torch.zeros(seqs, dtype=torch.bool, device=cuda)
    state = ([0] * seqs, [[-1] * width for _ in range(seqs)], free.tolist(), counts.tolist())
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        pages.plan(lens, new, tables.clone(), free, counts, page, 30)
        pages.release(done, lens, tables, free.clone(), counts, page)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        p = pages.plan(lens, new, tables, free, counts, page, 30)
        l2, c2 = pages.release(done, p.lens, tables, free, p.counts, page)
        lens.copy_(l2), counts.copy_(c2)
    torch.cuda.synchronize()
    r = random.Random(4)
    for _ in range(6):
        n = [r.randint(0, 6) for _ in range(seqs)]
        d = [r.random() < 0.2 for _ in range(seqs)]
        new.copy_(ints(n, cuda)), done.copy_(ints(d, cuda, torch.bool))
        graph.replay()
        want = PH.plan(state[0], n, state[1], state[2], state[3], page, 30)
        assert p.slots.tolist() == want[0] and p.positions.tolist() == want[1] and p.starts.tolist() == want[2]
        assert tables.tolist() == want[5]
        l, c, f = PH.release(d, want[3], want[5], state[2], want[4], page)
        assert lens.tolist() == l and counts.tolist() == c and free.tolist()[:c[0]] == f[:c[0]]
        state = (l, want[5], free.tolist(), c)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one device")
def test_another_device():
    d = torch.device("cuda", 1)
    free, counts = pages.pool(4, d)
    p = pages.plan(ints([0], d), ints([3], d), torch.full((1, 2), -1, dtype=I32, device=d), free, counts, 16, 3)
    assert p.slots.tolist() == [0, 1, 2] and p.slots.device == d
