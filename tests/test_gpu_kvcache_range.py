"""Attention over the quantised cache where ranges end, against the plain 64-bit forms of kv_helpers."""
import pytest
import torch

from nemicli_terminal_b200 import kvcache

from tests import kv_helpers as KH
from tests.test_gpu_kvcache import BF16, F16, F32, MANY, gen, slots_of, tables_of

pytestmark = pytest.mark.gpu


def attend(c, tables, q, lens, new, most, scale=None, window=0):
    """attend for the last new[b] tokens of each sequence; MANY rows (3.0, covered by nothing) where that is the bound given."""
    starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=c.device)
    n = q.shape[0]
    if most == MANY:
        q = torch.cat([q, q.new_full((MANY - n, *q.shape[1:]), 3.0)])
    tiles = KH.tiled(c, q.shape[1], len(new), most, q.dtype, tables.shape[1], window)
    got = c.attend(q, tables, torch.tensor(lens, dtype=torch.int32, device=c.device), starts, max_new=most, scale=scale, window=window)
    return got[:n], tiles


def compare(got, tiles, q, held, lens, new, scale, window=0, tol_of=None):
    """Every row against the 64-bit form, within KH.bound or tol_of(sizes, o, keys).  A negative scale is given to the plain
    form as negative queries: the same product, and sizes that are positive."""
    at = 0
    for b, n in enumerate(new):
        rows = slice(at, at + n)
        at += n
        qb = q[rows].double() * (-1 if scale < 0 else 1)
        o, sizes = KH.attention(qb, *held[b], torch.arange(lens[b] - n, lens[b], device=q.device), abs(scale), window)
        tol = tol_of(sizes, o, lens[b]) if tol_of else KH.bound(sizes, o, q.dtype, max(lens[b], 1), tiles)
        assert torch.isfinite(got[rows]).all(), b
        err = (got[rows].double() - o).abs()
        assert (err <= tol).all(), (b, (err / tol).max().item())


# ---- values at fp16's end -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("kf, vf", [("Q8_0", "Q8_0"), ("Q4_0", "Q8_0"), ("Q8_0", "Q4_0")])
@pytest.mark.parametrize("most", [MANY])
def test_clamped_values(cuda, dtype, dim, kf, vf, most):
    """Infinities and values past fp16 are held as the largest code times fp16(65504 / 127), which is 65532: finite for every
    query that sees them, and nothing to those before.  The queries' share of K's clamped channel is small, so that its score
    is an ordinary one."""
    g = gen(1, cuda)
    tables, pages = tables_of([90], 16, 1, cuda)
    c = kvcache.KVCache(pages, 2, dim, 16, kf, vf, cuda)
    k, v = (torch.randn(90, 2, dim, generator=g, device=cuda) for _ in range(2))
    for key, x in ((40, float("inf")), (41, -float("inf")), (55, 1e30), (70, -65504.0), (71, 65501.0)):
        k[key, :, 1], v[key, :, 3], v[key, 1, dim - 2] = x, x, -x
    s = slots_of(tables[0], 90, 16)
    c.write(k, v, s)
    held = [[x.double() for x in c.read(s, F32)]]
    assert held[0][1].abs().max() > (65504 if vf == "Q8_0" else 65503)
    q = torch.randn(90, 8, dim, generator=g, device=cuda)
    q[..., :32] = 0
    q[..., 1] = 2.0 ** -13 * torch.randn(90, 8, generator=g, device=cuda).clamp(-2, 2)
    q = q.to(dtype)
    got, tiles = attend(c, tables, q, [90], [90], most)
    assert tiles == (most == MANY and dtype == BF16)
    compare(got, tiles, q, held, [90], [90], dim ** -0.5)


@pytest.mark.parametrize("fmt", ["Q4_0", "Q8_0"])
def test_clamped_values_in_float16(cuda, fmt):
    """65532 rounds to an infinity of float16: read and the attention's float16 outputs stay at 65504, half a step away."""
    k = torch.zeros(1, 1, 64, device=cuda)
    v = torch.ones(1, 1, 64, device=cuda)
    v[..., 0], v[..., 40] = float("inf"), -1e30
    k[..., 3] = float("inf")
    c = kvcache.KVCache(200, 1, 64, 16, fmt, fmt, cuda)
    c.write(k.expand(2, 1, 64).contiguous(), v.expand(2, 1, 64).contiguous(), torch.arange(2, device=cuda))
    want = torch.zeros(64, device=cuda)
    want[0], want[40] = 65504, -65504
    for x in c.read(torch.arange(2, device=cuda), F16):
        assert torch.isfinite(x).all()
    assert torch.equal(c.read(torch.arange(2, device=cuda), F16)[1][0, 0], want.half())
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
    wide = torch.zeros(1, 200, dtype=torch.int32, device=cuda)             # a table this long: keys cut over the GPU
    for t, new, most in ((table, 1, 1), (table, 2, 2), (table, 2, MANY), (wide, 1, 1), (wide, 2, 400)):
        q = torch.zeros(new, 4, 64, dtype=F16, device=cuda)
        got, _ = attend(c, t, q, [2], [new], most)
        assert torch.equal(got, want.half().expand(new, 4, 64))
