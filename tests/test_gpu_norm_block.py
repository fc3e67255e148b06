"""mmvq.norm_block on the GPU against its 64-bit form."""
import pytest
import torch

from nemicli_terminal_b200 import mmvq

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def plain(y, h, w_pre, eps, w_post, gate, rs):
    z, h = y.double(), h.double()
    if w_post is not None:
        z = z / (z.square().mean(-1, keepdim=True) + eps).sqrt() * w_post.double()
    if gate is not None:
        z = z * gate.double()
    new = h + rs * z
    x = None if w_pre is None else new / (new.square().mean(-1, keepdim=True) + eps).sqrt() * w_pre.double()
    return x, new, z


def close(x, new, want, h, rs, dtype, n):
    """new = h + rs z: z carries the sum's error (n additions of fp32, in pairs and strips of at most n / 32 + 16: half of
    that relative error passes the root), rsqrt and three products: (n / 32 + 32) 2^-24 of |rs z|, the sum and the output
    half a step of the result.  x has that of new (in the norm's relative measure) and its own sum, root and products."""
    wx, wn, z = want
    eps = torch.finfo(dtype).eps / 2
    rel = (n / 32 + 32) * 2.0 ** -24
    en = rel * rs * z.abs() + 2.0 ** -23 * (h.double().abs() + wn.abs())
    tiny = 2.0 ** -24 if dtype == F16 else 0.0
    assert ((new.double() - wn).abs() <= en + eps * wn.abs() + tiny).all()
    if wx is not None:
        inv = (wx.abs() / wn.abs().clamp(min=1e-30))
        shift = (en.square().mean(-1, keepdim=True) / wn.square().mean(-1, keepdim=True).clamp(min=1e-30)).sqrt()
        assert ((x.double() - wx).abs() <= inv * en + wx.abs() * (shift + 2 * rel + eps) + tiny).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [1, 31, 64, 100, 1000, 4096, 5120, 8191, 14336, 32768])
@pytest.mark.parametrize("rows", [1, 3, 200])
def test_norm_block(cuda, dtype, n, rows):
    g = torch.Generator(device=cuda).manual_seed(n + rows)
    y = (3 * torch.randn(rows, n, generator=g, device=cuda)).to(dtype)
    h = (9 * torch.randn(rows, n, generator=g, device=cuda)).to(dtype)
    gate = torch.rand(rows, n, generator=g, device=cuda).to(dtype)
    w1, w2 = (torch.rand(n, generator=g, device=cuda) + 0.5 for _ in range(2))
    for kw in (dict(w_post=w1, gate=gate, rs=0.7), dict(w_post=w1), dict(), dict(gate=gate[0].clone(), rs=-2.0)):
        x, e, new = mmvq.norm_block(y, h, w2, 1e-6, **kw)
        assert e is None and x.dtype == new.dtype == dtype
        full = {"w_post": None, "gate": None, "rs": 1.0, **kw}
        close(x, new, plain(y, h, w2, 1e-6, **full), h, abs(full["rs"]), dtype, n)
    x, _, new = mmvq.norm_block(y, h, None, 1e-6, w_post=w1)
    assert x is None
    close(None, new, plain(y, h, None, 1e-6, w1, None, 1.0), h, 1.0, dtype, n)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, n", [(1, 4096), (5, 64), (2, 14336)])
def test_eingang(cuda, dtype, rows, n):
    """The activation input stands for the fp32 x: two stages of 8 bits, off by at most half a step of the second (its scale
    is d / 254, and the remainder's clamp at 127 costs nothing beyond that), and x itself is off as its own rounding."""
    g = torch.Generator(device=cuda).manual_seed(n)
    y, h = (torch.randn(rows, n, generator=g, device=cuda).to(dtype) for _ in range(2))
    w1, w2 = (torch.rand(n, generator=g, device=cuda) + 0.5 for _ in range(2))
    x, e, _ = mmvq.norm_block(y, h, w2, 1e-6, w_post=w1, eingang=True)
    d = e.xd.double().repeat_interleave(32)
    got = ((e.xq.double() + e.xq2.double() / 254) * d).view(rows, n)
    want, _, _ = plain(y, h, w2, 1e-6, w1, None, 1.0)
    tol = d.view(rows, n) * (0.5 / 254 + 2.0 ** -20) + want.abs() * (n / 16 + 64) * 2.0 ** -24
    assert ((got - want).abs() <= tol).all()
    s = want.view(rows, -1, 32).sum(-1).reshape(-1)
    assert ((e.xs.double() - s).abs() <= (n / 16 + 128) * 2.0 ** -24 * want.abs().view(rows, -1, 32).sum(-1).reshape(-1)).all()
    if dtype == F32 and rows == 1:                    # and feeds the matvec's norm: the same as norm_q8's on h alone
        zero = torch.zeros_like(y)
        x, e, _ = mmvq.norm_block(zero[0], h[0], w2, 1e-6, eingang=True)
        xn, e2, _ = mmvq.norm_q8(h[0], w2, 1e-6)
        assert (x - xn).abs().max() <= (n / 16 + 64) * 2.0 ** -24 * xn.abs().max()


def test_strides_vectors_and_streams(cuda):
    g = torch.Generator(device=cuda).manual_seed(3)
    big = torch.randn(7, 3 * 160 + 1, generator=g, device=cuda)
    y, h, gate = big[:, 1:161], big[:, 161:321], big[:, 320:480]
    w = torch.rand(160, generator=g, device=cuda) + 0.5
    # rows that start off 16 bytes are summed in another order than whole pieces, so their bits may differ: both keep the
    # bound of `close`, which holds for any order of at most n / 32 + 16 additions a chain
    ref = plain(y, h, w, 1e-5, w, gate, 1.0)
    want = mmvq.norm_block(y.contiguous(), h.contiguous(), w, 1e-5, gate=gate.contiguous(), w_post=w)
    got = mmvq.norm_block(y, h, w, 1e-5, gate=gate, w_post=w)
    for x, _, new in (want, got):
        close(x, new, ref, h, 1.0, F32, 160)
    t = torch.randn(160, 7, generator=g, device=cuda).T                     # values far apart: copied first
    a = mmvq.norm_block(t, h, w, 1e-5)
    b = mmvq.norm_block(t.contiguous(), h, w, 1e-5)
    assert torch.equal(a[0], b[0])
    one = mmvq.norm_block(y[2].clone(), h[2].clone(), w, 1e-5, gate=gate[2].clone(), w_post=w)
    assert one[0].shape == (160,) and torch.equal(one[0], want[0][2]) and torch.equal(one[2], want[2][2])
    each = mmvq.norm_block(y[:1].expand(7, 160), h, w, 1e-5, w_post=w)      # one row broadcast: copied first
    assert torch.equal(each[2][3], mmvq.norm_block(y[0].contiguous(), h[3], w, 1e-5, w_post=w)[2])
    wide = big[:, 4:324].contiguous()[:, :160]                              # aligned rows with a stride
    got = mmvq.norm_block(wide, wide, w, 1e-5, w_post=w)
    assert torch.equal(got[0], mmvq.norm_block(wide.contiguous(), wide.contiguous(), w, 1e-5, w_post=w)[0])
    want = mmvq.norm_block(y, h, w, 1e-5, gate=gate, w_post=w)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mmvq.norm_block(y, h, w, 1e-5, gate=gate, w_post=w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0])
    empty = mmvq.norm_block(y[:0], h[:0], w, 1e-5)
    assert empty[0].shape == (0, 160)


def test_infinities_stay_in_their_row(cuda):
    y = torch.randn(3, 96, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    h, w = torch.zeros_like(y), torch.ones(96, device=cuda)
    want = mmvq.norm_block(y, h, w, 1e-6, w_post=w)
    y2 = y.clone()
    y2[1, 5], y2[1, 6] = float("inf"), float("nan")
    got = mmvq.norm_block(y2, h, w, 1e-6, w_post=w)
    for i in (0, 2):
        assert torch.equal(got[0][i], want[0][i]) and torch.equal(got[2][i], want[2][i])
    assert torch.isnan(got[0][1]).all()
    z = mmvq.norm_block(torch.zeros_like(y), h, w, 1e-6, w_post=w)
    assert not z[0].any() and not z[2].any()


def test_refusals(cuda):
    y, w = torch.zeros(2, 64, device=cuda), torch.ones(64, device=cuda)
    for call in (lambda: mmvq.norm_block(y, y[:1], w, 1e-6), lambda: mmvq.norm_block(y, y.half(), w, 1e-6),
                 lambda: mmvq.norm_block(y, y, w[:32], 1e-6), lambda: mmvq.norm_block(y, y, w.half(), 1e-6),
                 lambda: mmvq.norm_block(y, y, w, 1e-6, gate=y[:1]), lambda: mmvq.norm_block(y, y, None, 1e-6, eingang=True),
                 lambda: mmvq.norm_block(y[:, :33], y[:, :33], w[:33], 1e-6, eingang=True),
                 lambda: mmvq.norm_block(y.double(), y.double(), w, 1e-6), lambda: mmvq.norm_block(y, y.cpu(), w, 1e-6),
                 lambda: mmvq.norm_block(torch.zeros(1, 32800, device=cuda), torch.zeros(1, 32800, device=cuda), None, 1e-6)):
        with pytest.raises(RuntimeError):
            call()
