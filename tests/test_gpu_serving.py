"""The serving loop around the quantised cache on the GPU: page tables, writes with several axes, boxes, chosen pages, beam selection
and the beams' tables run together as a decoder would use them, against one sequence after the other held in plain tensors."""
import pytest
import torch

from nemicli_terminal_b200 import _lib, beams, kvcache, mmvq, pages

from tests.test_gpu_kvcache import gen

pytestmark = pytest.mark.gpu
I32 = torch.int32


def rope_tables(dim, n, cuda):
    a = torch.arange(n, dtype=torch.float64)[:, None] * torch.pow(1e4, -torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
    return a.cos().float().to(cuda), a.sin().float().to(cuda)


@pytest.fixture(params=[False, True], ids=["plain", "pdl"])
def launches(request):
    """The library's programmatic dependent launches off and on."""
    mmvq.pdl(request.param)
    yield
    mmvq.pdl(False)


def test_steps_of_a_batch(cuda, launches):
    """Requests of unequal prompts, then a token each; some end and others take their pages.  What each sequence's table holds is what
    it was given, in order; attention over all its pages equals attention over the chosen ones where these are all."""
    dim, n_kv, heads, page, seqs, width = 64, 2, 6, 16, 6, 8
    c = kvcache.KVCache(40, n_kv, dim, page, "Q8_0", "Q8_0", cuda)
    free, counts = pages.pool(c.n_pages, cuda)
    tables = torch.full((seqs, width), -1, dtype=I32, device=cuda)
    lens = torch.zeros(seqs, dtype=I32, device=cuda)
    box = c.bounds()
    cos, sin = rope_tables(dim, 200, cuda)
    axes = kvcache.rope_axes((8, 12, 12))
    alone = [[] for _ in range(seqs)]                            # (k, v, position) of each token
    g = gen(1, cuda)
    _lib.device_status(device=cuda)
    for step in range(30):
        new = [17, 1, 33, 5, 16, 40] if step == 0 else [1, 1, 0, 1, 1, 1]
        if step == 12:
            done = torch.tensor([False, True, False, False, False, True], device=cuda)
            lens, counts = pages.release(done, lens, tables, free, counts, page)
            alone[1], alone[5] = [], []
            new = [1, 30, 1, 1, 1, 9]
        rows = sum(new) + 2
        p = pages.plan(lens, torch.tensor(new, dtype=I32, device=cuda), tables, free, counts, page, rows)
        k, v = (torch.randn(rows, n_kv, dim, generator=g, device=cuda).bfloat16() for _ in range(2))
        q = torch.randn(rows, heads, dim, generator=g, device=cuda).bfloat16()
        pos = torch.stack((p.positions, p.positions // 2, p.positions % 7))
        q = c.write(k, v, p.slots, q=q, rope=(cos, sin, pos), axes=axes)
        c.summarise(box, tables, p.lens, p.starts, max_new=max(new))
        o = c.attend(q, tables, p.lens, p.starts, max_new=max(new))
        chosen, held = c.choose(q, box, tables, p.lens, width, starts=p.starts)
        few = c.attend_chosen(q, chosen, held)
        at = 0
        for b, n in enumerate(new):
            alone[b] += [(k[at + i], v[at + i], pos[:, at + i]) for i in range(n)]
            at += n
        assert p.lens.tolist() == [len(a) for a in alone]
        live = sum(new)
        # (kernels for few and for many rows may differ by what they round on the way: weights to 2^-11 each, sums and outputs)
        scale = o[:live].float().abs().amax()
        assert (o[:live].float() - few[:live].float()).abs().amax() <= scale * (2 ** -8 + 4 * 2 ** -11)
        assert not few[live:].any()
        lens, counts = p.lens, p.counts
    assert counts[1].item() == 0 and _lib.device_status(device=cuda) == 0
    held_pages = sum(-(-len(a) // page) for a in alone)
    assert counts[0].item() == c.n_pages - held_pages
    for b, a in enumerate(alone):                                # what the tables hold, read back
        n = len(a)
        i = torch.arange(n, device=cuda)
        slots = tables[b, i // page].long() * page + i % page
        one = kvcache.KVCache(width, n_kv, dim, page, "Q8_0", "Q8_0", cuda)
        one.write(torch.stack([x[0] for x in a]), torch.stack([x[1] for x in a]), i, rope=(cos, sin, torch.stack([x[2] for x in a], 1).contiguous()),
                  axes=axes)
        for x, y in zip(c.read(slots), one.read(i)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("page, prompt", [(16, 20), (16, 32), (32, 5)])
def test_beam_search(cuda, launches, page, prompt):
    """A toy model: a token's key and value are its embedding, logits the attention's output times the embeddings.  Beam search with paged
    tables keeps for every beam what a search that copies whole caches keeps, step by step."""
    dim, n_kv, reqs, k, vocab, width, steps = 64, 1, 3, 4, 97, 8, 14
    g = gen(page + prompt, cuda)
    emb = torch.randn(vocab, dim, generator=g, device=cuda)
    # a prompt's partly filled page belongs to one beam before the first step; three pages of each request's beams are shared at most
    c = kvcache.KVCache(reqs * (k + 1) * width, n_kv, dim, page, "Q8_0", "Q8_0", cuda)
    free, counts = pages.pool(c.n_pages, cuda)
    tables = torch.full((reqs * k, width), -1, dtype=I32, device=cuda)
    lens = torch.zeros(reqs * k, dtype=I32, device=cuda)
    text = torch.randint(0, vocab, (reqs, prompt), generator=g, device=cuda)
    first = torch.zeros(reqs * k, dtype=I32, device=cuda)
    first[::k] = prompt                                          # the prompt is beam 0's
    p = pages.plan(lens, first, tables, free, counts, page, reqs * prompt)
    x = emb[text.flatten()][:, None]
    c.write(x, x, p.slots)
    lens, counts = p.lens, p.counts
    scores = torch.full((reqs, k), -torch.inf, device=cuda)
    scores[:, 0] = 0
    seqs = [[text[r].tolist()] + [[] for _ in range(k - 1)] for r in range(reqs)]
    query = emb[text[:, -1]].repeat_interleave(k, 0)[:, None]
    _lib.device_status(device=cuda)
    for _ in range(steps):
        o = c.attend(query, tables, lens)
        logits = (o[:, 0] @ emb.T).view(reqs, k, vocab)
        scores, parents, tokens = beams.select(logits, scores, k)
        r = pages.reorder(parents, lens, tables, free, counts, page)
        c.copy(r.src, r.dst, r.used)
        tables, lens, counts = r.tables, r.lens, r.counts
        p = pages.plan(lens, torch.ones_like(lens), tables, free, counts, page, reqs * k)
        x = emb[tokens.flatten().long()][:, None]
        c.write(x, x, p.slots)
        lens, counts, query = p.lens, p.counts, x
        seqs = [[seqs[i][q] + [t] for q, t in zip(parents[i].tolist(), tokens[i].tolist())] for i in range(reqs)]
        held = {}
        for i in range(reqs):
            for j in range(k):
                n = len(seqs[i][j])
                assert lens[i * k + j].item() == n
                at = torch.arange(n, device=cuda)
                slots = tables[i * k + j, at // page].long() * page + at % page
                one = kvcache.KVCache(width, n_kv, dim, page, "Q8_0", "Q8_0", cuda)
                y = emb[torch.tensor(seqs[i][j], device=cuda)][:, None]
                one.write(y, y, at)
                for a, b in zip(c.read(slots), one.read(at)):
                    assert torch.equal(a, b)
                for place, no in enumerate(tables[i * k + j, :-(-n // page)].tolist()):
                    assert held.setdefault(no, (i, place)) == (i, place)             # shared within a request, at one place, only
        assert counts[0].item() + len(held) == c.n_pages and counts[1].item() == 0
        assert not set(held) & set(free[:counts[0].item()].tolist())
    r = pages.reorder(torch.full((reqs, k), -1, dtype=I32, device=cuda), lens, tables, free, counts, page)
    assert r.counts[0].item() == c.n_pages and sorted(free.tolist()) == list(range(c.n_pages)) and not r.lens.any()
    assert _lib.device_status(device=cuda) == 0
