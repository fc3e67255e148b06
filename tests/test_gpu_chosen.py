"""Boxes of pages, the choice of pages, and attention over chosen pages on the GPU, against plain forms in 64 bits (kv_helpers)."""
import numpy as np
import pytest
import torch

from nemicli_terminal_b200 import _lib, kvcache

from tests import kv_helpers as KH
from tests.test_gpu_kvcache import gen, tables_of

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def filled(cuda, lens, n_kv, dim, page, kf, vf, seed, extra=3, width=None):
    """A cache of quantised random keys and values whose pages differ in their mean, its tables and lengths."""
    t, n_pages = tables_of(lens, page, extra, cuda, seed, width)
    c = kvcache.KVCache(n_pages, n_kv, dim, page, kf, vf, cuda)
    g = gen(seed, cuda)
    mean = torch.randn(n_pages, 1, n_kv, dim, generator=g, device=cuda)
    k = (mean + torch.randn(n_pages, page, n_kv, dim, generator=g, device=cuda)).flatten(0, 1)
    v = torch.randn(n_pages * page, n_kv, dim, generator=g, device=cuda)
    c.write(k, v, torch.arange(n_pages * page, device=cuda))
    return c, t, torch.tensor(lens, dtype=torch.int32, device=cuda)


def held_values(c):
    """Every slot's keys and values fp64 (pages, page, n_kv, dim)."""
    k, v, s = KH.codes_of(c, np.arange(c.n_pages * c.page))
    out = [KH.values(x, s[:, :, i], f).reshape(c.n_pages, c.page, c.n_kv, c.dim) for x, i, f in ((k, 0, c.k_fmt), (v, 1, c.v_fmt))]
    return [torch.from_numpy(x) for x in out]


def outwards(lo, hi):
    """fp64 -> fp16 numpy, lo downwards and hi upwards, inside fp16's range."""
    out = []
    for x, way in ((lo, -np.inf), (hi, np.inf)):
        x = np.clip(x, -65504.0, 65504.0)
        h = x.astype(np.float16)
        past = h.astype(np.float64) < x if way > 0 else h.astype(np.float64) > x
        with np.errstate(over="ignore"):
            out.append(np.where(past, np.nextafter(h, np.float16(way)), h))
    return out


@pytest.mark.parametrize("dim, kf, page", [(64, "Q4_0", 16), (64, "Q8_0", 64), (96, "Q8_0", 32), (96, "Q4_0", 16), (128, "Q4_0", 64),
                                           (128, "Q8_0", 16), (256, "Q4_0", 128), (256, "Q8_0", 32)])
def test_boxes(cuda, dim, kf, page):
    """Every key lies in its page's box, whose sides are the next fp16 values outwards; only completed pages are written."""
    lens, new = [3 * page, 5, 2 * page + 7, page, 4 * page - 1, 0], [3 * page, 5, page + 9, 1, 0, 0]
    c, t, n = filled(cuda, lens, 3, dim, page, kf, "Q4_0", dim)
    starts = torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device=cuda)
    k, _ = held_values(c)
    b = c.bounds()
    b.fill_(7.0)
    c.summarise(b, t, n, starts, max_new=max(new))
    want = np.full(b.shape, 7.0, np.float16)
    for i, (a, m) in enumerate(zip(lens, new)):
        for p in range((a - m) // page, a // page):
            at = int(t[i, p])
            x = k[at].numpy()
            want[at, :, 0], want[at, :, 1] = outwards(x.min(0), x.max(0))
    assert (b.cpu().numpy() == want).all()
    again = b.clone()
    c.summarise(again, t, n, starts)                              # no bound on the new tokens
    assert torch.equal(again, b) and _lib.device_status(device=cuda) == 0
    one = c.bounds()
    c.summarise(one, t, n)                                        # a token each: only full pages
    for i, a in enumerate(lens):
        for p in range(t.shape[1]):
            at = int(t[i, p])
            if at >= 0:
                assert bool(one[at].any()) == (a > 0 and a % page == 0 and p == a // page - 1)


def test_boxes_of_extreme_keys(cuda):
    """Keys at fp16's ends, denormal scales, zeros, negative scales."""
    c = kvcache.KVCache(2, 1, 128, 16, "Q8_0", "Q4_0", cuda)
    k = torch.zeros(16, 1, 128, device=cuda)
    k[3, 0, :32] = torch.linspace(-65504, 65504, 32)
    k[4, 0, 32:64] = torch.linspace(-3e-7, 2.9e-7, 32)
    k[5, 0, 64:96] = -1e-6
    for fmt in kvcache.FORMATE:
        c = kvcache.KVCache(2, 1, 128, 16, fmt, "Q4_0", cuda)
        c.write(k, k, torch.arange(16, device=cuda))
        b = c.bounds()
        t = torch.tensor([[0]], dtype=torch.int32, device=cuda)
        c.summarise(b, t, torch.tensor([16], dtype=torch.int32, device=cuda))
        x = held_values(c)[0][0].numpy()
        lo, hi = outwards(x.min(0), x.max(0))
        assert (b[0, :, 0].cpu().numpy() == lo).all() and (b[0, :, 1].cpu().numpy() == hi).all()
        assert torch.isfinite(b).all()


def test_boxes_out_of_order(cuda):
    """Pages outside the cache and lengths past the table are left and reported; so are more pages than max_new allows."""
    c, t, n = filled(cuda, [64, 64], 1, 64, 16, "Q4_0", "Q4_0", 1)
    b = c.bounds()
    _lib.device_status(device=cuda)
    bad = t.clone()
    bad[0, 3] = c.n_pages
    c.summarise(b, bad, n)
    assert _lib.device_status(device=cuda) == 1 and not b[t[0, 3].long()].any() and b[t[1, 3].long()].any()
    c.summarise(b, t, torch.tensor([65, 64], dtype=torch.int32, device=cuda))
    assert _lib.device_status(device=cuda) == 1
    starts = torch.tensor([0, 64, 128], dtype=torch.int32, device=cuda)
    c.summarise(b, t, n, starts, max_new=16)
    assert _lib.device_status(device=cuda) == 1
    c.summarise(b, t, n, starts, max_new=64)
    assert _lib.device_status(device=cuda) == 0 and b[t.flatten().long()].flatten(1).any(1).all()


def choice(q, bounds, table, pos, page, keep, first, last, n_kv):
    """The pages of one query, by the definition in fp64: logical numbers a key head."""
    n = pos // page + 1
    if n <= keep:
        return [list(range(n)) for _ in range(n_kv)]
    box = bounds[table[:n].long()].double().cpu()                 # (n, n_kv, 2, dim)
    x = q.double().cpu().unflatten(0, (n_kv, -1))
    out = []
    for h in range(n_kv):
        # max(q lo, q hi) by the query's sign: with an infinite query a side of 0 would be NaN in the other product
        s = torch.where(x[h, None] > 0, x[h, None] * box[:, h, None, 1], x[h, None] * box[:, h, None, 0]).sum(-1)
        s = torch.where(s.isnan(), torch.full_like(s, -torch.inf), s).amax(1).tolist()
        must = list(range(first)) + list(range(n - last, n))
        rest = sorted(range(first, n - last), key=lambda i: (-s[i], i))[:keep - first - last]
        out.append(sorted(must + rest))
    return out


def check(c, q, b, t, n, keep, first, last, starts=None, news=None):
    """choose and attend_chosen against the definitions; the choice is equal where scores differ at all (fp64 has room)."""
    rows, heads, dim = q.shape
    chosen, held = c.choose(q, b, t, n, keep, starts=starts, first=first, last=last)
    assert chosen.shape == (rows, c.n_kv, keep) and chosen.dtype == held.dtype == torch.int32
    o = c.attend_chosen(q, chosen, held)
    k, v = held_values(c)
    k, v = k.to(q.device), v.to(q.device)
    row = 0
    for i, m in enumerate(news or [1] * t.shape[0]):
        for p in range(int(n[i]) - m, int(n[i])):
            if p < 0:
                assert int(held[row]) == 0 and (chosen[row] == -1).all() and not o[row].any()
                row += 1
                continue
            want = choice(q[row], b, t[i], p, c.page, keep, first, last, c.n_kv)
            tokens = (len(want[0]) - 1) * c.page + p % c.page + 1
            assert int(held[row]) == tokens
            group = heads // c.n_kv
            for h in range(c.n_kv):
                pages = t[i, torch.tensor(want[h], device=q.device)]
                assert chosen[row, h].tolist() == pages.tolist() + [-1] * (keep - len(pages)), (i, p, h)
                kk, vv = (x[pages.long(), :, h].flatten(0, 1)[:tokens, None] for x in (k, v))
                qq = q[row:row + 1, h * group:(h + 1) * group].double()
                ref, sizes = KH.attention(qq, kk, vv, torch.tensor([tokens], device=q.device), dim ** -0.5, 0)
                assert ((o[row:row + 1, h * group:(h + 1) * group].double() - ref).abs() <= KH.bound(sizes, ref, q.dtype, tokens, False)).all()
            row += 1
    assert (held[row:] == 0).all() and (chosen[row:] == -1).all() and not o[row:].any()
    return chosen, held


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim, heads, n_kv, page, kf, vf", [
    (64, 14, 2, 16, "Q8_0", "Q4_0"), (96, 6, 3, 32, "Q4_0", "Q8_0"), (128, 32, 8, 64, "Q4_0", "Q4_0"), (256, 8, 1, 16, "Q8_0", "Q8_0"),
    (128, 3, 3, 16, "Q4_0", "Q4_0"), (64, 36, 2, 16, "Q4_0", "Q4_0")])
def test_choose_and_attend(cuda, dtype, dim, heads, n_kv, page, kf, vf):
    """One token a sequence, from one token held to many pages; the first and last pages stay; padding rows behind."""
    lens = [1, page, page + 1, 7 * page - 3, 40 * page + 5, 0, 33 * page]
    c, t, n = filled(cuda, lens, n_kv, dim, page, kf, vf, dim + heads)
    b = c.bounds()
    starts = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=cuda)
    c.summarise(b, t, n, starts)
    q = (torch.randn(len(lens) + 2, heads, dim, generator=gen(3, cuda), device=cuda) * 0.7).to(dtype)
    for keep, first, last in ((1, 0, 1), (3, 1, 2), (5, 1, 2), (8, 0, 1), (39, 2, 3), (64, 1, 1)):
        check(c, q, b, t, n, keep, first, last)
    assert _lib.device_status(device=cuda) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_drafted_tokens(cuda, dtype):
    """Several query rows a sequence, each with its own place and pages; a sequence without one, queries before the start, strides."""
    lens, news = [70, 1, 500, 3, 129], [5, 1, 8, 0, 3]
    c, t, n = filled(cuda, lens, 2, 128, 16, "Q4_0", "Q8_0", 5)
    b = c.bounds()
    c.summarise(b, t, n, torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=cuda))
    starts = torch.tensor(np.cumsum([0] + news), dtype=torch.int32, device=cuda)
    fused = torch.randn(sum(news) + 3, 12 * 128, generator=gen(4, cuda), device=cuda).to(dtype)
    q = fused[:, 256:256 + 8 * 128].unflatten(1, (8, 128))
    check(c, q, b, t, n, 6, 1, 1, starts, news)
    short = n.clone()
    short[0] = 2                                                  # five new tokens of two
    check(c, q, b, t, short, 6, 1, 1, starts, news)


def long_cache(cuda, pages, page=16, dim=64, n_kv=1, seed=9):
    c, t, n = filled(cuda, [pages * page], n_kv, dim, page, "Q4_0", "Q4_0", seed)
    b = c.bounds()
    c.summarise(b, t, n, torch.tensor([0, pages * page], dtype=torch.int32, device=cuda))
    return c, t, n, b


@pytest.mark.parametrize("pages", [513, 2049, 9001])
def test_many_pages(cuda, pages):
    """More pages than a thread each, and than the shared memory holds."""
    c, t, n, b = long_cache(cuda, pages)
    q = torch.randn(1, 4, 64, generator=gen(2, cuda), device=cuda)
    for keep, dtype in ((3, F32), (64, BF16), (500, F32)):
        chosen, held = c.choose(q.to(dtype), b, t, n, keep, first=1, last=1)
        want = choice(q[0].to(dtype), b, t[0], pages * 16 - 1, 16, keep, 1, 1, 1)[0]
        assert chosen[0, 0].tolist() == t[0, torch.tensor(want, device=cuda)].tolist() and held.tolist() == [keep * 16]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scores_alike(cuda, dtype):
    """Pages in order where their scores are equal: queries of zeros, pages that repeat, more of them than a list holds; scores that
    differ in the last bits of fp64 only by their pages' boxes are told apart."""
    c, t, n, b = long_cache(cuda, 1500)
    q = torch.zeros(1, 2, 64, dtype=dtype, device=cuda)
    chosen, _ = c.choose(q, b, t, n, 40, first=2, last=3)
    assert chosen[0, 0].tolist() == t[0, :37].tolist() + t[0, -3:].tolist()
    q = torch.randn(1, 2, 64, generator=gen(7, cuda), device=cuda).to(dtype)
    again = b.clone()
    again[t[0].long()] = b[t[0, torch.arange(1500, device=cuda) % 2].long()]              # two boxes in turns
    chosen, _ = c.choose(q, again, t, n, 801, first=1, last=1)
    want = choice(q[0], again, t[0], 1500 * 16 - 1, 16, 801, 1, 1, 1)[0]
    assert chosen[0, 0].tolist() == t[0, torch.tensor(want, device=cuda)].tolist()
    same = b.clone()
    same[:] = b[0]
    step = torch.finfo(F16).eps
    places = torch.randperm(1400, generator=torch.Generator().manual_seed(3))[:30].to(cuda) + 50
    same[t[0, places].long(), :, :, 5] = (same[0, 0, :, 5].float() * (1 + step)).half()
    near = choice(q[0], same, t[0], 1500 * 16 - 1, 16, 60, 1, 1, 1)[0]
    chosen, _ = c.choose(q, same, t, n, 60, first=1, last=1)
    assert chosen[0, 0].tolist() == t[0, torch.tensor(near, device=cuda)].tolist()


def test_scores_far_apart(cuda):
    """One page far above the others, queries near fp32's ends, infinities and NaN among them."""
    c, t, n, b = long_cache(cuda, 300)
    g = gen(8, cuda)
    peak = b.clone()
    peak[t[0, 77].long(), :, 1] = 60000.0
    q = torch.randn(1, 4, 64, generator=g, device=cuda)
    for bounds, x in ((peak, q), (b, q * 1e30), (b, q * 1e-30), (b, q * 1e-42), (peak, q * 1e33)):
        chosen, _ = c.choose(x, bounds, t, n, 20, first=0, last=2)
        want = choice(x[0], bounds, t[0], 300 * 16 - 1, 16, 20, 0, 2, 1)[0]
        assert chosen[0, 0].tolist() == t[0, torch.tensor(want, device=cuda)].tolist()
    for value in (float("nan"), float("inf"), -float("inf")):
        x = q.clone()
        x[0, 1, 3] = value
        chosen, _ = c.choose(x, b, t, n, 20, first=0, last=2)
        want = choice(x[0], b, t[0], 300 * 16 - 1, 16, 20, 0, 2, 1)[0]
        assert chosen[0, 0].tolist() == t[0, torch.tensor(want, device=cuda)].tolist()
        x[:] = value
        chosen, _ = c.choose(x, b, t, n, 20, first=0, last=2)
        got = chosen[0, 0].tolist()
        assert len(set(got)) == 20 and set(got) <= set(t[0].tolist())


@pytest.mark.parametrize("channel", [6, 7])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_boxes_that_are_no_numbers(cuda, channel, value):
    """A side of a box that is NaN or infinite counts for the heads that read that side."""
    c, t, n, b = long_cache(cuda, 300)
    q = torch.randn(1, 4, 64, generator=gen(12, cuda), device=cuda)
    q[0, :2, channel], q[0, 2:, channel] = 0.5, -0.5
    q[0, 0] *= 3
    for side in (0, 1):
        odd = b.clone()
        odd[t[0, 20:290:3].long(), :, side, channel] = value
        chosen, _ = c.choose(q, odd, t, n, 120, first=1, last=2)
        want = choice(q[0], odd, t[0], 300 * 16 - 1, 16, 120, 1, 2, 1)[0]
        assert chosen[0, 0].tolist() == t[0, torch.tensor(want, device=cuda)].tolist()


def test_bad_pages(cuda):
    """A page outside the cache scores least; chosen all the same it counts as masked, and the status says so."""
    c, t, n, b = long_cache(cuda, 40)
    bad = t.clone()
    bad[0, 5], bad[0, 39] = c.n_pages, -7
    q = torch.randn(1, 2, 64, generator=gen(1, cuda), device=cuda)
    _lib.device_status(device=cuda)
    chosen, held = c.choose(q, b, bad, n, 10)
    assert bad[0, 5].item() not in chosen[0, 0].tolist() and chosen[0, 0, -1].item() == -7
    assert _lib.device_status(device=cuda) == 0
    o = c.attend_chosen(q, chosen, held)
    assert _lib.device_status(device=cuda) == 1 and torch.isfinite(o).all()
    c.choose(q, b, t, n + 1, 10)
    assert _lib.device_status(device=cuda) == 1


def test_captured_and_on_another_stream(cuda):
    """A captured choice and attention, replayed with other queries and lengths."""
    lens = [200, 90, 333]
    c, t, n = filled(cuda, lens, 2, 64, 16, "Q4_0", "Q4_0", 11)
    b = c.bounds()
    c.summarise(b, t, n, torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=cuda))
    q = torch.randn(3, 4, 64, generator=gen(5, cuda), device=cuda)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.attend_chosen(q, *c.choose(q, b, t, n, 6))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        chosen, held = c.choose(q, b, t, n, 6)
        o = c.attend_chosen(q, chosen, held)
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=gen(20 + i, cuda), device=cuda))
        n.sub_(17)
        graph.replay()
        x, y = c.choose(q, b, t, n, 6)
        assert torch.equal(x, chosen) and torch.equal(y, held) and torch.equal(c.attend_chosen(q, x, y), o)
