"""Attention over the quantised cache where ranges end, against the plain 64-bit forms of kv_helpers."""
import pytest
import torch

from nemicli_terminal_b200 import _lib, kvcache

from tests import kv_helpers as KH
from tests.test_gpu_kvcache import BF16, F16, F32, MANY, filled, gen, slots_of, tables_of

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
@pytest.mark.parametrize("most", [90, MANY])
def test_clamped_values(cuda, dtype, dim, kf, vf, most):
    """Infinities and values past fp16 are held as the largest code times fp16(65504 / 127), which is 65532: finite for every
    query that sees them, and nothing to those before.  The queries' share of K's clamped channel is small, so that its score
    is an ordinary one.
    One bound more than KH.bound's where the codes' bits are the operand (16-bit queries, no tiles): the tensor cores align a
    step's 16 products at the largest exponent and cut each off there, 2^-23 of it, and a code c 2^-24 (8 bits; 4 bits:
    c 2^-18), a denormal, counts as 2^-14: each loses up to 2^-37 p d, or 2^-13 p d (2^-19) once 2^24 (2^18) is taken off; 16
    of a step 2^-9 p d (2^-15), codes and offset together 2^-8 (2^-14).  A block's largest value is 127 d (7 d): 2^-15 of
    it (2^-16)."""
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
    bits = dtype == BF16 and not tiles
    compare(got, tiles, q, held, [90], [90], dim ** -0.5,
            tol_of=lambda sizes, o, keys: KH.bound(sizes, o, dtype, keys, tiles) + 2.0 ** (-15 if vf == "Q8_0" else -16) * sizes[1] * bits)


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


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kf", ["Q4_0", "Q8_0"])
@pytest.mark.parametrize("vf", ["Q4_0", "Q8_0"])
@pytest.mark.parametrize("dim, n_kv, group", [(64, 8, 1), (128, 3, 8), (256, 2, 7), (96, 2, 4)])
def test_values_under_a_larger_key(cuda, dtype, kf, vf, dim, n_kv, group):
    """Sums near 0 beside a key whose values are far larger: few keys, so that a step's largest product stands alone."""
    lens, new = [21, 22, 37, 53, 14, 33, 112, 24], [3, 9, 4, 1, 3, 3, 10, 1]
    for seed in range(6):
        c, tables, held = filled(cuda, lens, n_kv, dim, 32, kf, vf, seed=seed)
        q = torch.randn(sum(new), n_kv * group, dim, generator=gen(seed, cuda), device=cuda).to(dtype)
        got, tiles = attend(c, tables, q, lens, new, max(new))
        assert not tiles
        compare(got, tiles, q, held, lens, new, dim ** -0.5)


# ---- weights far apart, values of any size ---------------------------------------------------------------

def sink(cuda, lens, gap, small, kf, vf, same=False, dim=64, n_kv=2, heads=4, page=16):
    """Caches whose first key stands `gap` above all others in the score of a head's queries (half of it for odd heads) and
    whose first value is 0; the others' values are `small` times 1 to 1.25 (same: one row for all of them).  -> cache, tables, held, the queries' row, scale.
    Queries are one power of two on channel 0, and K there an integer times a power of two, so every score is exact."""
    g = gen(2, cuda)
    tables, pages = tables_of(lens, page, 1, cuda)
    c = kvcache.KVCache(pages, n_kv, dim, page, kf, vf, cuda)
    held = []
    for b, n in enumerate(lens):
        k = torch.zeros(n, n_kv, dim, device=cuda)
        top, d, most = (100, 0.125, 127) if kf == "Q8_0" else (7, 0.5, -8)
        k[..., 31] = most * d                                  # the block's scale is d
        k[0, :, 0] = top * d
        v = small * (1 + 0.25 * torch.rand(n, n_kv, dim, generator=g, device=cuda))
        if same:
            v[:] = v[1]
        v[0] = 0
        s = slots_of(tables[b], n, page)
        c.write(k, v, s)
        held.append([x.double() for x in c.read(s, F32)])
        assert torch.equal(held[-1][0], k.double())
    q = torch.zeros(heads, dim, device=cuda)
    q[:, 0] = 1.0
    q[1::2, 0] = 0.5
    scale = torch.tensor(gap / (top * d)).float().item()
    return c, tables, held, q, scale


def sink_bound(dtype, tiles, small=1.0):
    """The scores are exact, so a weight 2^x is off by x's rounding: x = s cs + reference, |x| <= 32: 2^-19 for the sum, three
    roundings of 2^-24 in cs times at most 25, ln 2 times both is 5e-6; ex2's 2^-22; twice, for the sum that it is divided by:
    2^-16.  Weights in fp16 2^-11 (float32: two parts, 2^-21), V in fp16 2^-11 on the tiles; sums and the output as in KH.bound.
    A product of a weight (and V's scale) in fp16, or its second part, is off by 2^-25 at least, where the largest weight has 2^9
    or more (2^10 with V's scale, as float32 queries have it): 2^-34 a key (2^-35), times V, at most 1.25 `small`."""
    rel = 2.0 ** -16 + (2.0 ** -21 if dtype == F32 else 2.0 ** -11) + (2.0 ** -11 if tiles else 0.0)

    def tol(sizes, o, keys):
        mag, top, _, _ = sizes
        return mag * rel + keys * 2.0 ** (-35 if dtype == F32 else -34) * 1.25 * small + 2 * top * (keys / 16 + 16) * 2.0 ** -22 + o.abs() * KH.HALF_STEP[dtype] + 2.0 ** -24 * (dtype == F16) + 1e-30
    return tol


CALLS = [([1500, 900], 1, 1), ([1500, 900], 6, 6), ([1500, 900], 60, MANY), ([5000], 200, 200)]     # the last: keys cut over the GPU


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("small", [1.0, 1e-2, 1e-3, 3e-5])
@pytest.mark.parametrize("kf, vf", [("Q8_0", "Q8_0"), ("Q4_0", "Q4_0")])
@pytest.mark.parametrize("lens, new, most", CALLS)
def test_small_values_keep_small_weights(cuda, dtype, small, kf, vf, lens, new, most):
    """The output does not depend on V's size."""
    c, tables, held, q, scale = sink(cuda, lens, 10.0, small, kf, vf)
    q = q.expand(new * len(lens), 4, 64).to(dtype)
    got, tiles = attend(c, tables, q, lens, [new] * len(lens), most, scale)
    assert tiles == (new >= 60 and dtype != F32)
    compare(got, tiles, q, held, lens, [new] * len(lens), scale, tol_of=sink_bound(dtype, tiles, small))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gap", [12.0, 14.0, 15.0, 17.0])
@pytest.mark.parametrize("same", [False, True])
@pytest.mark.parametrize("lens, new, most", CALLS)
def test_many_weights_under_one_key(cuda, dtype, gap, same, lens, new, most):
    """Weights down to 2^-23 of the row's largest hold their bits, those below to 2^-34 of it: a first key without a value (an attention sink) far above
    many equal ones."""
    c, tables, held, q, scale = sink(cuda, lens, gap, 1.0, "Q8_0", "Q8_0", same)
    q = q.expand(new * len(lens), 4, 64).to(dtype)
    got, tiles = attend(c, tables, q, lens, [new] * len(lens), most, scale)
    compare(got, tiles, q, held, lens, [new] * len(lens), scale, tol_of=sink_bound(dtype, tiles))


# ---- queries --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kf", ["Q4_0", "Q8_0"])
@pytest.mark.parametrize("new, most", [(1, 1), (6, 6), (70, MANY)])
def test_queries_of_far_sizes_in_a_row(cuda, dtype, kf, new, most):
    """One value of a row 2^30 (2^27 with Q4_0's upper nibbles, float16: 2^23) above the others, where K holds zeros: the others
    count in full."""
    lens, g = [200, 150], gen(3, cuda)
    tables, pages = tables_of(lens, 16, 1, cuda)
    c = kvcache.KVCache(pages, 1, 96, 16, kf, "Q8_0", cuda)
    held = []
    for b, n in enumerate(lens):
        k, v = (torch.randn(n, 1, 96, generator=g, device=cuda) for _ in range(2))
        k[..., :32] = 0
        s = slots_of(tables[b], n, 16)
        c.write(k, v, s)
        held.append([x.double() for x in c.read(s, F32)])
    far = 23 if dtype == F16 else 30 if kf == "Q8_0" else 27
    q = torch.randn(2 * new, 4, 96, generator=g, device=cuda)
    q = torch.sign(q) * q.abs().clamp(0.5, 1.9) * 2.0 ** (13 - far)
    q[..., 5] = 1.9 * 2.0 ** 13
    q = q.to(dtype)
    scale = 2.0 ** (far - 13) / 8
    got, tiles = attend(c, tables, q, lens, [new, new], most, scale)
    compare(got, tiles, q, held, lens, [new, new], scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [2.0 ** 125, 2.0 ** -120])
@pytest.mark.parametrize("new, most", [(1, 1), (6, 6), (70, MANY)])
def test_queries_of_any_size(cuda, dtype, size, new, most):
    """Queries near both ends of bf16's range, with a scale that makes their scores ordinary."""
    lens = [200, 150]
    c, tables, held = filled(cuda, lens, 1, 128, 16, "Q8_0", "Q8_0")
    q = (torch.randn(2 * new, 4, 128, generator=gen(4, cuda), device=cuda).clamp(-3.9, 3.9) * size).to(dtype)
    scale = 2.0 ** -3 / size
    got, tiles = attend(c, tables, q, lens, [new, new], most, scale)
    compare(got, tiles, q, held, lens, [new, new], scale)


def test_scale_must_be_finite(cuda):
    c, tables, _ = filled(cuda, [3], 1, 64, 16, "Q4_0", "Q4_0")
    q, lens = torch.zeros(1, 2, 64, device=cuda), torch.tensor([3], dtype=torch.int32, device=cuda)
    for scale in (float("nan"), float("inf"), -1e39, 1e300):
        with pytest.raises(RuntimeError):
            c.attend(q, tables, lens, scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("new, most", [(1, 1), (6, 6), (70, MANY)])
def test_scale_zero_and_negative(cuda, dtype, scale, window, new, most):
    """Masked keys stay masked whatever the scale's sign, the causal and the window's border inside a unit of keys."""
    lens = [200, 77]
    c, tables, held = filled(cuda, lens, 2, 128, 16, "Q8_0", "Q4_0")
    q = torch.randn(2 * new, 8, 128, generator=gen(5, cuda), device=cuda).to(dtype)
    got, tiles = attend(c, tables, q, lens, [new, new], most, scale, window)
    compare(got, tiles, q, held, lens, [new, new], scale, window)


def test_no_rows(cuda):
    c = kvcache.KVCache(2, 1, 64, 16, "Q8_0", "Q8_0", cuda)
    x, s = torch.randn(0, 1, 64, device=cuda), torch.arange(0, device=cuda)
    assert c.write(x, x, s) is None
    assert c.write(x, x, s, q=torch.randn(0, 3, 64, device=cuda)).shape == (0, 3, 64)
    k, v = c.read(s, F32)
    assert k.shape == (0, 1, 64) and v.shape == (0, 1, 64)
    assert _lib.device_status(device=cuda) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens, new, most", CALLS)
def test_out_over_the_queries(cuda, dtype, lens, new, most):
    """out may be q itself: a row's queries are read before it is written, by every part of a cut sequence too."""
    c, tables, held = filled(cuda, lens, 2, 64, 16, "Q8_0", "Q4_0")
    n = [new] * len(lens)
    q = torch.randn(most if most == MANY else new * len(lens), 8, 64, generator=gen(6, cuda), device=cuda).to(dtype)
    starts = torch.arange(len(lens) + 1, dtype=torch.int32, device=cuda) * new
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    want = c.attend(q, tables, lt, starts, max_new=most)[:sum(n)]
    out = q.clone()
    assert torch.equal(c.attend(out, tables, lt, starts, max_new=most, out=out)[:sum(n)], want)
    assert torch.equal(out[sum(n):], q[sum(n):])
