"""Beam selection on the GPU against the definition in 64 bits."""
import pytest
import torch

from nemicli_terminal_b200 import beams

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
MOST = torch.finfo(F32).max


def define(logits, scores):
    """All candidates' scores (requests, beams * vocab) fp64, and what the kernel's scores may be off by: exponentials 2^-22, their
    arguments' two roundings and log2 e's (2^-23 of the distance to the largest, where it counts at all: up to 90), sums of 32 in fp32;
    all relative to the sum, so absolute in its logarithm."""
    x = logits.double()
    x = torch.where(x.isnan(), torch.full_like(x, -torch.inf), x).clamp(max=MOST)
    top = x.amax(-1, keepdim=True).clamp(min=-MOST)
    total = (x - top).exp().sum(-1, keepdim=True)
    far = torch.where(x > -torch.inf, top - x, torch.zeros_like(x)).amax(-1, keepdim=True).clamp(max=90)
    s = (x - top) - total.clamp(min=1e-300).log() + scores.double()[..., None]
    s = torch.where(s.isnan(), torch.full_like(s, -torch.inf), s)
    off = 2.0 ** -22 + 32 * 2.0 ** -24 + far.amax(1) * 2.0 ** -22
    return s.flatten(1), off                                       # off (requests, 1)


def check(logits, scores, n):
    out, parents, tokens = beams.select(logits, scores, n)
    vocab = logits.shape[2]
    s, off = define(logits, scores)
    place = parents.long() * vocab + tokens.long()
    assert ((parents >= 0) & (parents < logits.shape[1]) & (tokens >= 0) & (tokens < vocab)).all()
    assert (place.sort(1)[0].diff(dim=1) > 0).all()               # no candidate twice
    best, index = torch.sort(s, dim=1, descending=True, stable=True)
    best, index = best[:, :n], index[:, :n]
    mine = s.gather(1, place)
    same = (best == mine) | ((best - mine).abs() <= 2 * off)       # order among scores nearer than the error
    assert same.all()
    # candidates that no other comes near are the ones
    s_next = torch.sort(s, dim=1, descending=True)[0][:, :n + 1]
    gap = torch.full_like(best, torch.inf)
    gap[:, 1:] = best[:, :-1] - best[:, 1:]
    if s_next.shape[1] > n:
        gap = torch.minimum(gap, best - s_next[:, 1:])
    else:
        gap[:, :-1] = torch.minimum(gap[:, :-1], best[:, :-1] - best[:, 1:])
    clear = gap > 2 * off
    assert (place == index)[clear].all()
    live = mine > -torch.inf
    assert (out.double()[live] - mine[live]).abs().le(off.expand_as(mine)[live] + mine[live].abs() * 2.0 ** -24).all()
    assert (out[~live] == -torch.inf).all()
    return out, parents, tokens


def gen(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reqs, k, vocab, n", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 21), (1, 4, 1000, 8), (3, 5, 50257, 10), (2, 8, 128256, 16), (40, 4, 32001, 4), (1, 64, 9001, 64),
    (5, 2, 8192, 33), (300, 2, 2049, 4), (1, 1, 262145, 64)])
def test_select(cuda, dtype, reqs, k, vocab, n):
    g = gen(vocab + n, cuda)
    x = (torch.randn(reqs, k, vocab, generator=g, device=cuda) * 3).to(dtype)
    s = -torch.rand(reqs, k, generator=g, device=cuda).mul(4).cumsum(1)
    a = check(x, s, n)
    b = beams.select(x, s, n)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("reqs, k, vocab, dtype, n", [(74, 8, 140001, BF16, 16), (150, 4, 131072, BF16, 64), (2, 2, 400003, F32, 33)])
def test_long_rows_and_many(cuda, reqs, k, vocab, dtype, n):
    """Rows of more steps than a part has, with as many rows as there are CTAs at once."""
    g = gen(vocab, cuda)
    x = torch.empty(reqs, k, vocab, dtype=dtype, device=cuda)
    for r in x:
        r.copy_(torch.randn(k, vocab, generator=g, device=cuda) * 3)
    s = -torch.rand(reqs, k, generator=g, device=cuda).cumsum(1)
    whole = beams.select(x, s, n)
    for r in (0, reqs - 1):                                       # a request's result does not depend on the others
        one = check(x[r:r + 1], s[r:r + 1], n)
        near = (one[0] - whole[0][r:r + 1]).abs() <= 1e-4
        assert near.all()
    check(x[reqs // 2:reqs // 2 + 8], s[reqs // 2:reqs // 2 + 8], n)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_ties_go_to_the_lowest_place(cuda, dtype):
    """Equal logits in a row; equal rows with equal scores, at every alignment a row can have."""
    for vocab in (1, 37, 4099, 30000):
        x = torch.zeros(2, 3, vocab, dtype=dtype, device=cuda)
        n = min(3 * vocab, 10)
        _, parents, tokens = beams.select(x, torch.zeros(2, 3, device=cuda), n)
        want = torch.arange(n, device=cuda)
        assert (parents.long() * vocab + tokens == want).all()
    g = gen(5, cuda)
    for vocab in (8191, 8193, 20001, 20002, 20004):
        row = torch.randint(-40, 40, (vocab,), generator=g, device=cuda).div(4).to(dtype)
        x = row.expand(4, 5, vocab).contiguous()
        _, parents, tokens = beams.select(x, torch.zeros(4, 5, device=cuda), 64)
        # each value of the row is met in all beams before the next: the first beam's places first
        order = torch.sort(row.float(), descending=True, stable=True)
        want = []
        for v in order[0].unique(sorted=True).flip(0).tolist():
            at = (row.float() == v).nonzero()[:, 0].tolist()
            want += [(k, t) for k in range(5) for t in at]
            if len(want) >= 64:
                break
        got = list(zip(parents[0].tolist(), tokens[0].tolist()))
        assert got == want[:64]
        assert (parents == parents[0]).all() and (tokens == tokens[0]).all()


def test_special_values(cuda):
    """NaN, infinities, rows of -inf, beams without a score, one alive."""
    x = torch.randn(6, 3, 9000, generator=gen(1, cuda), device=cuda)
    x[0, :, ::3] = float("nan")
    x[1, 0, 17] = float("inf")
    x[1, 1, 5:8] = float("inf")
    x[2, 0] = -torch.inf
    x[2, 1] = float("nan")
    x[3] = -torch.inf
    x[3, 2, 8000] = 1.0
    x[4] *= 1e4
    x[5] = x[5] * 1e3 + 1e5
    s = torch.zeros(6, 3, device=cuda)
    s[4, 1:] = -torch.inf
    s[5, 2] = float("nan")
    out, parents, tokens = check(x, s, 6)
    assert parents[1].tolist()[0] == 0 and tokens[1].tolist()[0] == 17
    assert tokens[3].tolist() == [8000, 0, 1, 2, 3, 4] and parents[3].tolist() == [2, 0, 0, 0, 0, 0]
    assert (out[3, 1:] == -torch.inf).all() and out[3, 0] == 0
    assert (parents[4] == 0).all() and (parents[5] < 2).all()
    h = x.half()
    check(h, s, 6)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_orders_that_keep_the_bounds_low(cuda, dtype):
    """Ascending and descending rows, one large value at the end, a plateau under a few peaks."""
    v = 60000
    ramp = torch.linspace(-30, 30, v, device=cuda)
    flat = torch.zeros(v, device=cuda)
    flat[[3, 59990, 30000]] = torch.tensor([1.0, 2.0, 1.0], device=cuda)
    last = torch.randn(v, generator=gen(3, cuda), device=cuda)
    last[-1] = 50
    x = torch.stack((ramp, ramp.flip(0), flat, last)).to(dtype)[None]
    check(x, torch.tensor([[0.0, -1.5, -2.25, -3.0]], device=cuda), 40)


def test_two_streams_at_once(cuda):
    """Calls that overlap have workspaces of their own."""
    g = gen(12, cuda)
    x = [torch.randn(4, 6, 40003, generator=g, device=cuda) for _ in range(2)]
    s = [torch.zeros(4, 6, device=cuda) for _ in range(2)]
    want = [beams.select(a, b, 12) for a, b in zip(x, s)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(beams.select(x[i], s[i], 12))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for i in range(2) for o in got[i] for p, q in zip(o, want[i]))


def test_strides_and_streams(cuda):
    """Rows of a padded projection, requests apart, scores of a search's start; a captured call."""
    g = gen(8, cuda)
    wide = torch.randn(3, 4, 5008, generator=g, device=cuda)
    s = torch.full((3, 4), -torch.inf, device=cuda)
    s[:, 0] = 0
    a = beams.select(wide[..., :5001], s, 8)
    b = beams.select(wide[..., :5001].contiguous(), s, 8)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and (a[1] == 0).all()
    c = beams.select(wide[:, ::2, 3:], s[:, ::2].contiguous(), 8)
    d = beams.select(wide[:, ::2, 3:].contiguous(), s[:, ::2].contiguous(), 8)
    assert all(torch.equal(p, q) for p, q in zip(c, d))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        beams.select(wide, s)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        e = beams.select(wide, s, 6)
    wide.copy_(torch.randn(wide.shape, generator=g, device=cuda))
    s.fill_(0.5)
    graph.replay()
    f = beams.select(wide, s, 6)
    assert all(torch.equal(p, q) for p, q in zip(e, f))
    assert beams.select(wide[:0], s[:0], 3)[0].shape == (0, 3)
