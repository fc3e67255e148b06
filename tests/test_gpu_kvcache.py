"""The quantised key / value cache and attention over it on the GPU against plain 64-bit forms (kv_helpers)."""
import numpy as np
import pytest
import torch

from nemicli_terminal_b200 import _lib, kvcache, mmvq, synth

from tests import kv_helpers as KH

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def tables_of(lens, page, extra, device, seed=0, width=None):
    """Pages in a random order; -1 behind a sequence's last page."""
    per = [(n + page - 1) // page for n in lens]
    order = torch.randperm(sum(per) + extra, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    t = torch.full((len(lens), max(1, width or max(per))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        t[b, :n] = order[at:at + n]
        at += n
    return t.to(device), sum(per) + extra


def slots_of(table, n, page):
    i = torch.arange(n, device=table.device)
    return table[i // page].long() * page + i % page


# ---- write and read ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim, kf, vf", [(64, "Q4_0", "Q8_0"), (96, "Q8_0", "Q4_0"), (128, "Q4_0", "Q4_0"), (256, "Q8_0", "Q8_0")])
@pytest.mark.parametrize("rope", ["none", "half", "pairs", "part"])
def test_write_is_exact(cuda, dtype, dim, kf, vf, rope):
    """Codes and scales equal the plain quantiser's bit for bit, other slots stay, padding rows write nothing, and the rows of
    a fused q/k/v output are read in place."""
    rows, n_kv, heads, page = 37, 3, 6, 16
    g = gen(1, cuda)
    c = kvcache.KVCache(6, n_kv, dim, page, kf, vf, cuda)
    for t in (c.k_codes, c.v_codes):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=cuda, dtype=torch.uint8))
    c.scales.uniform_(0.1, 1.0, generator=g)
    old = [t.clone() for t in (c.k_codes, c.v_codes, c.scales)]
    fused = (torch.randn(rows, (heads + 2 * n_kv) * dim, generator=g, device=cuda) * 3).to(dtype)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in fused.split([heads * dim, n_kv * dim, n_kv * dim], 1))
    slots = torch.randperm(6 * page, generator=g, device=cuda)[:rows].contiguous()
    pad = torch.zeros(rows, dtype=torch.bool, device=cuda)
    pad[5::9] = True
    given = torch.where(pad, -1, slots)
    rot = {"none": 0, "half": dim, "pairs": dim, "part": 40}[rope]
    tab = torch.arange(999, dtype=torch.float64)[:, None] * torch.pow(1e4, -torch.arange(rot // 2, dtype=torch.float64) / max(1, rot // 2))
    pos = torch.randint(0, 999, (rows,), generator=g, device=cuda)
    cos, sin = tab.cos().float().to(cuda), tab.sin().float().to(cuda)
    out = c.write(k, v, given, q=q, rope=None if rope == "none" else (cos, sin, pos), paired=rope == "pairs")
    kn, vn, qn = (x.float().cpu().numpy() for x in (k, v, q))
    if rope != "none":
        kn, qn = (KH.rotate(x, cos.cpu().numpy(), sin.cpu().numpy(), pos.cpu().numpy(), rope == "pairs") for x in (kn, qn))
    assert torch.equal(out.cpu(), torch.from_numpy(qn).to(dtype))
    live = (~pad).cpu().numpy()
    gk, gv, gs = KH.codes_of(c, slots.cpu().numpy())
    for x, fmt, got, sc in ((kn, kf, gk, gs[:, :, 0]), (vn, vf, gv, gs[:, :, 1])):
        code, d = KH.quantise(x, fmt)
        assert np.array_equal(got[live], code[live])
        assert np.array_equal(sc[live].view(np.uint16), d[live].view(np.uint16))
    rest = torch.ones(6 * page, dtype=torch.bool, device=cuda)
    rest[slots[~pad]] = False
    keep = rest.nonzero()[:, 0].cpu().numpy()
    before = kvcache.KVCache(6, n_kv, dim, page, kf, vf, buffers=old)
    for a, b in zip(KH.codes_of(c, keep), KH.codes_of(before, keep)):
        assert np.array_equal(a, b)
    rk, rv = c.read(given, dtype)
    for r, code, sc, fmt in ((rk, gk, gs[:, :, 0], kf), (rv, gv, gs[:, :, 1], vf)):
        want = torch.from_numpy(KH.values(code, sc, fmt)).float().to(dtype)        # d * code fits fp32: one rounding
        want[pad.cpu()] = 0
        assert torch.equal(r.cpu(), want)
    assert _lib.device_status(device=cuda) == 0


def test_write_special_values(cuda):
    """NaN counts as 0, infinities and values past fp16 are clamped, equal magnitudes go by the first, blocks of zeros and of
    values below fp16's smallest step hold zeros."""
    x = torch.zeros(1, 2, 128)
    x[0, 0, :32] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e30] + [1.0] * 28)
    x[0, 0, 32:64] = torch.tensor([2.0, -2.0] * 16)
    x[0, 0, 64:96] = torch.tensor([-2.0, 2.0] * 16)
    x[0, 1, :32] = 1e-9
    x[0, 1, 32:64] = torch.linspace(-3e-7, 2.9e-7, 32)              # scales among fp16's denormals
    x[0, 1, 64:96] = torch.linspace(-65504, 65504, 32)
    x[0, 1, 96:] = float("nan")
    for kf in kvcache.FORMATE:
        c = kvcache.KVCache(1, 2, 128, 16, kf, kf, cuda)
        c.write(x.to(cuda), x.to(cuda), torch.tensor([7], device=cuda))
        gk, gv, gs = KH.codes_of(c, np.array([7]))
        code, d = KH.quantise(x.numpy(), kf)
        for got, i in ((gk, 0), (gv, 1)):
            assert np.array_equal(got, code) and np.array_equal(gs[:, :, i].view(np.uint16) & 0x7FFF, d.view(np.uint16) & 0x7FFF)
        k, _ = c.read(torch.tensor([7], device=cuda), F32)
        assert torch.isfinite(k).all()


def test_write_out_of_range(cuda):
    """A slot past the cache and a position outside the tables: the row is not written, its queries are 0, the status is set."""
    c = kvcache.KVCache(2, 1, 64, 16, device=cuda)
    x = torch.randn(3, 1, 64, generator=gen(3, cuda), device=cuda)
    cos = torch.ones(4, 32, device=cuda)
    _lib.device_status(device=cuda)
    q = c.write(x, x, torch.tensor([0, 32, 2], device=cuda), q=x, rope=(cos, cos * 0, torch.tensor([1, 2, 4], device=cuda)))
    assert _lib.device_status(device=cuda) == 1
    assert torch.equal(q[:2], x[:2]) and not q[2].any()
    k, v = c.read(torch.tensor([0, 1, 2, -1, 31], device=cuda), F32)
    assert k[0].any() and not k[1:].any() and not v[2].any()
    c.read(torch.tensor([32], device=cuda))
    assert _lib.device_status(device=cuda) == 1


@pytest.mark.parametrize("rows", [0, 1, 2, 1023])
def test_write_and_read_row_counts(cuda, rows):
    c = kvcache.KVCache(64, 1, 64, 16, "Q8_0", "Q8_0", cuda)
    x = torch.randn(rows, 1, 64, generator=gen(4, cuda), device=cuda)
    s = torch.arange(rows, device=cuda)
    assert c.write(x, x, s) is None
    k, v = c.read(s, F32)
    assert k.shape == (rows, 1, 64) and (k - x).abs().max().item() < 0.05 if rows else True
    assert torch.equal(k, v)


# ---- attention --------------------------------------------------------------------------------------

def filled(cuda, lens, n_kv, dim, page, kf, vf, seed=0, extra=2, poison=True):
    """A cache with `lens` tokens of random keys and values a sequence; what no token holds is poisoned (NaN scales, all
    codes set).  -> cache, tables, [(k, v) fp64 (len, n_kv, dim)]."""
    g = gen(seed, cuda)
    tables, pages = tables_of(lens, page, extra, cuda, seed)
    c = kvcache.KVCache(pages, n_kv, dim, page, kf, vf, cuda)
    if poison:
        c.k_codes.fill_(255), c.v_codes.fill_(255), c.scales.fill_(float("nan"))
    held = []
    for b, n in enumerate(lens):
        k = torch.randn(n, n_kv, dim, generator=g, device=cuda) * torch.exp(0.5 * torch.randn(dim, generator=g, device=cuda))
        v = torch.randn(n, n_kv, dim, generator=g, device=cuda) * torch.exp(torch.randn(n, 1, 1, generator=g, device=cuda))
        s = slots_of(tables[b], n, page)
        c.write(k, v, s)
        held.append([x.double() for x in c.read(s, F32)])
    return c, tables, held


MANY = 20000                    # query rows, and bound on a sequence's, that make any batch one for the tiles


def check(c, tables, held, lens, new, heads, dtype, window=0, seed=5, scale=None, most=None, q=None, out=None, one=False):
    """attend for new[b] tokens of each sequence against the 64-bit form; -> the output.  most: the bound given, and MANY
    rows of q, which nothing covers."""
    dev = c.device
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    if q is None:
        q = torch.randn(starts[-1], heads, c.dim, generator=gen(seed, dev), device=dev).to(dtype)
    if most == MANY and q.shape[0] < MANY:
        q = torch.cat([q, q.new_full((MANY - q.shape[0], heads, c.dim), 3.0)])
    most = most or max(new)
    tiles = KH.tiled(c, heads, len(new), most, dtype, tables.shape[1])
    assert tiles or most < MANY or dtype == F32
    got = c.attend(q, tables, torch.tensor(lens, dtype=torch.int32, device=dev),
                   starts=None if one else torch.tensor(starts, dtype=torch.int32, device=dev), max_new=most, window=window,
                   scale=scale, out=out)
    for b, n in enumerate(new):
        if n == 0:
            continue
        rows = slice(starts[b], starts[b + 1])
        pos = torch.arange(lens[b] - n, lens[b], device=dev)
        o, sizes = KH.attention(q[rows].double(), *held[b], pos, scale or c.dim ** -0.5, window)
        tol = KH.bound(sizes, o, dtype, max(lens[b], 1), tiles)
        err = (got[rows].double() - o).abs()
        assert torch.isfinite(got[rows]).all(), b
        assert (err <= tol).all(), (b, (err / tol).max().item())
    return got


LENS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 300, 0, 1000]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim, n_kv, group", [(64, 2, 7), (96, 1, 8), (128, 2, 4), (256, 2, 1), (128, 1, 16), (64, 3, 3), (256, 1, 12)])
@pytest.mark.parametrize("kf, vf", [("Q4_0", "Q4_0"), ("Q8_0", "Q8_0"), ("Q4_0", "Q8_0"), ("Q8_0", "Q4_0")])
def test_one_token(cuda, dtype, dim, n_kv, group, kf, vf):
    """Decode: one row a sequence, lengths around the tile and page borders, an empty sequence (zeros)."""
    c, tables, held = filled(cuda, LENS, n_kv, dim, 16, kf, vf)
    got = check(c, tables, held, LENS, [1] * len(LENS), n_kv * group, dtype, one=True)
    assert not got[LENS.index(0)].any()
    assert _lib.device_status(device=cuda) == 0


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("window", [0, 1, 16, 100, 5000])
def test_one_token_windows_and_pages(cuda, page, window):
    lens = [1, 100, 16, 4097, 900]
    c, tables, held = filled(cuda, lens, 2, 128, page, "Q4_0", "Q8_0")
    check(c, tables, held, lens, [1] * 5, 8, BF16, window=window, one=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_kv, group, dim", [(1, 1, 128), (8, 4, 128), (2, 8, 64)])
def test_one_long_sequence(cuda, dtype, n_kv, group, dim):
    """A long cache of one sequence, split over the whole GPU."""
    c, tables, held = filled(cuda, [20011], n_kv, dim, 64, "Q4_0", "Q4_0")
    check(c, tables, held, [20011], [1], n_kv * group, dtype, one=True)


def test_one_token_many_short_sequences(cuda):
    lens = [(7 * b) % 90 for b in range(300)]
    c, tables, held = filled(cuda, lens, 1, 64, 16, "Q4_0", "Q4_0")
    check(c, tables, held, lens, [1] * 300, 4, F32, one=True)


@pytest.mark.parametrize("n_seq", [127, 128, 129, 300])
def test_many_sequences_cut_over_the_gpu(cuda, n_seq):
    """More sequences than a CTA has threads, lengths long enough to be cut between CTAs, some empty or without new tokens."""
    lens = [(397 * b) % 1500 * (b % 7 > 0) for b in range(n_seq)]
    c, tables, held = filled(cuda, lens, 1, 64, 16, "Q4_0", "Q4_0")
    check(c, tables, held, lens, [1] * n_seq, 4, BF16, one=True)
    new = [b % 3 if n > 2 else 0 for b, n in enumerate(lens)]
    check(c, tables, held, lens, new, 4, BF16)


@pytest.mark.parametrize("most", [3, MANY])
def test_rows_between_sequences(cuda, most):
    """Rows before the first sequence's stay as they were, and a sequence without new tokens writes none."""
    lens = [40, 200, 33]
    c, tables, held = filled(cuda, lens, 2, 128, 16, "Q8_0", "Q4_0")
    q = torch.randn(max(most, 12), 8, 128, generator=gen(3, cuda), device=cuda).bfloat16()
    out = torch.full_like(q, 7.0)
    starts = torch.tensor([4, 7, 7, 9], dtype=torch.int32, device=cuda)
    c.attend(q, tables, torch.tensor(lens, dtype=torch.int32, device=cuda), starts, max_new=most, out=out)
    assert (out[:4] == 7).all() and (out[9:] == 7).all()
    for b, rows in ((0, slice(4, 7)), (2, slice(7, 9))):
        n = rows.stop - rows.start
        o, sizes = KH.attention(q[rows].double(), *held[b], torch.arange(lens[b] - n, lens[b], device=cuda), 128 ** -0.5, 0)
        assert ((out[rows].double() - o).abs() <= KH.bound(sizes, o, BF16, lens[b], most == MANY)).all()
    assert _lib.device_status(device=cuda) == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("new", [[2, 3, 1, 5], [16, 16, 16, 16], [4, 0, 9, 1]])
@pytest.mark.parametrize("window", [0, 7])
def test_few_tokens(cuda, dtype, new, window):
    """Drafted tokens: unequal runs, one without new tokens; causal within the run."""
    lens = [20, 333, 64, 130]
    c, tables, held = filled(cuda, lens, 2, 128, 32, "Q8_0", "Q4_0")
    check(c, tables, held, lens, new, 8, dtype, window=window)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim, n_kv, group", [(64, 2, 7), (96, 1, 3), (128, 2, 4), (256, 1, 2), (128, 3, 1), (64, 1, 32)])
@pytest.mark.parametrize("kf, vf", [("Q4_0", "Q4_0"), ("Q8_0", "Q4_0"), ("Q4_0", "Q8_0"), ("Q8_0", "Q8_0")])
@pytest.mark.parametrize("most", [None, MANY])
def test_prompts(cuda, dtype, dim, n_kv, group, kf, vf, most):
    """Prompts of unequal length behind what the cache holds already, a fresh one (all of its tokens new), a single token."""
    lens, new = [300, 65, 257, 129, 1], [100, 65, 33, 1, 1]
    c, tables, held = filled(cuda, lens, n_kv, dim, 16, kf, vf)
    check(c, tables, held, lens, new, n_kv * group, dtype, most=most)
    assert _lib.device_status(device=cuda) == 0


@pytest.mark.parametrize("window", [1, 64, 130, 4000])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("most", [None, MANY])
def test_prompt_windows(cuda, window, dim, most):
    lens, new = [700, 200], [600, 200]
    c, tables, held = filled(cuda, lens, 1, dim, 64, "Q4_0", "Q4_0")
    check(c, tables, held, lens, new, 4, BF16, window=window, most=most)


@pytest.mark.parametrize("n", [17, 128, 255, 511])
@pytest.mark.parametrize("most", [None, MANY])
def test_prompt_lengths(cuda, n, most):
    c, tables, held = filled(cuda, [n], 2, 128, 16, "Q4_0", "Q4_0")
    check(c, tables, held, [n], [n], 2, BF16, most=most)


@pytest.mark.parametrize("most", [None, MANY])
def test_long_prompt(cuda, most):
    c, tables, held = filled(cuda, [2500], 2, 128, 64, "Q4_0", "Q4_0")
    check(c, tables, held, [2500], [2100], 4, BF16, most=most)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim, n_kv, group", [(64, 2, 8), (96, 3, 3), (128, 2, 4), (256, 1, 5)])
@pytest.mark.parametrize("window", [0, 700, 1500])
def test_tiles_with_keys_cut(cuda, dtype, dim, n_kv, group, window):
    """Few tiles with many keys: each tile's keys are cut over several CTAs; lengths that leave some of them no key."""
    lens, new = [5000, 1, 2049, 130, 0, 700], [120, 1, 97, 130, 0, 3]
    c, tables, held = filled(cuda, lens, n_kv, dim, 16, "Q4_0", "Q8_0")
    assert KH.tiled(c, n_kv * group, 6, 130, dtype, tables.shape[1])
    cut = _lib.load().qmv_kv_attend_workspace_bytes(c._ref, n_kv * group, 6, 130, 1, tables.shape[1], window) > 1
    assert cut == (window != 700)             # too few keys to cut
    check(c, tables, held, lens, new, n_kv * group, dtype, window=window)
    assert _lib.device_status(device=cuda) == 0


def test_tiles_with_keys_cut_from_graphs(cuda):
    """Two captured calls with cut keys replayed at the same time: each has its own parts."""
    lens, new = [5000, 3000], [60, 64]
    c, tables, _ = filled(cuda, lens, 2, 128, 64, "Q4_0", "Q4_0")
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 60, 124], dtype=torch.int32, device=cuda)
    assert KH.tiled(c, 8, 2, 64, BF16, tables.shape[1])
    qs = [torch.randn(124, 8, 128, generator=gen(30 + i, cuda), device=cuda).bfloat16() for i in range(2)]
    want = [c.attend(q, tables, lt, starts, max_new=64) for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.attend(q, tables, lt, starts, max_new=64))
        graphs.append(g)
    side = torch.cuda.Stream(cuda)
    torch.cuda.synchronize()
    for _ in range(5):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("new, most", [(1, None), (6, None), (90, None), (90, MANY), (1, MANY)])
def test_extreme_scores(cuda, new, most):
    """Scores far apart (one key takes all the weight), all equal (zero queries: the mean of the values), and values and
    queries of very different sizes among the heads."""
    lens = [200, 150]
    c, tables, held = filled(cuda, lens, 2, 128, 16, "Q8_0", "Q8_0")
    g = gen(9, cuda)
    q = torch.randn(2 * new, 8, 128, generator=g, device=cuda).bfloat16()
    q[:, 0] *= 300
    q[:, 1] = 0
    q[:, 2] *= 1e-6
    q[:, 5] *= 1e-3
    check(c, tables, held, lens, [new, new], 8, BF16, q=q, most=most)


@pytest.mark.parametrize("new, most", [(1, 1), (5, 5), (70, 70), (70, MANY)])
def test_rows_nobody_covers_and_positions_before_the_start(cuda, new, most):
    """Rows behind the last sequence stay as they were; more new tokens than the cache holds: those before its start see no
    key and give zeros."""
    lens = [3, 80]
    c, tables, held = filled(cuda, lens, 1, 64, 16, "Q4_0", "Q4_0")
    q = torch.randn(max(2 * new + 4, most), 2, 64, generator=gen(2, cuda), device=cuda).bfloat16()
    assert KH.tiled(c, 2, 2, most, BF16, tables.shape[1]) == (most == MANY)
    out = torch.full_like(q, 7.0)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, new, 2 * new], dtype=torch.int32, device=cuda)
    assert c.attend(q, tables, lens_t, starts, max_new=most, out=out) is out
    assert (out[2 * new:] == 7).all()
    if new > 3:
        assert not out[:new - 3].any()
        assert out[new - 3:new].any()
    o, sizes = KH.attention(q[:new].double(), *held[0], torch.arange(3 - new, 3, device=cuda), 0.125, 0)
    assert ((out[:new].double() - o).abs() <= KH.bound(sizes, o, BF16, 3, most == MANY)).all()
    assert _lib.device_status(device=cuda) == 0


@pytest.mark.parametrize("new, seqs", [(1, 2), (40, 2), (40, 100)])
def test_out_of_range_on_the_device(cuda, new, seqs):
    """Pages outside the cache count as masked, lengths beyond the table are cut, runs longer than max_new are not computed
    beyond it: each sets the status, and nothing else is touched."""
    lens = [96] * seqs                        # (100: the tiles)
    tiles = seqs > 2
    c, tables, held = filled(cuda, lens, 1, 64, 16, "Q4_0", "Q4_0", poison=False)
    _lib.device_status(device=cuda)
    q = torch.randn(seqs * new, 2, 64, generator=gen(2, cuda), device=cuda).bfloat16()
    starts = torch.arange(seqs + 1, dtype=torch.int32, device=cuda) * new
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    assert KH.tiled(c, 2, seqs, new, BF16, tables.shape[1]) == KH.tiled(c, 2, seqs, max(1, new - 3), BF16, tables.shape[1]) == tiles
    want = c.attend(q, tables, lt, starts, max_new=new)
    assert _lib.device_status(device=cuda) == 0
    for wrong in (-5, c.n_pages, 2 ** 31 - 1):
        bad = tables.clone()
        bad[0, 1] = wrong
        got = c.attend(q, bad, lt, starts, max_new=new)
        assert _lib.device_status(device=cuda) == 1
        assert torch.equal(got[new:], want[new:]) and torch.isfinite(got).all()
        k, v = ([x[i] for i in range(96) if not 16 <= i < 32] for x in held[0])
        pos = torch.arange(80 - new, 80, device=cuda)
        o, sizes = KH.attention(q[:new].double(), torch.stack(k), torch.stack(v), pos, 0.125, 0)
        assert ((got[:new].double() - o).abs() <= KH.bound(sizes, o, BF16, 96, tiles)).all()
    got = c.attend(q, tables, torch.tensor([96, 1000] + lens[2:], dtype=torch.int32, device=cuda), starts, max_new=new)
    assert _lib.device_status(device=cuda) == 1
    assert torch.equal(got, want)
    if new > 1:
        out = torch.full_like(q, 7.0)
        c.attend(q, tables, lt, starts, max_new=new - 3, out=out)
        assert _lib.device_status(device=cuda) == 1
        assert (out[new - 3:new] == 7).all() and not (out[:new - 3] == 7).all()


@pytest.mark.parametrize("new", [5, 70])
def test_window_of_any_size(cuda, new):
    """A window as long as an int holds is none, for queries before the sequence's start too."""
    c, tables, _ = filled(cuda, [3, 80], 1, 64, 16, "Q4_0", "Q4_0")
    lens = torch.tensor([3, 80], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, new, 2 * new], dtype=torch.int32, device=cuda)
    for rows in (2 * new, MANY):
        q = torch.randn(rows, 2, 64, generator=gen(4, cuda), device=cuda).bfloat16()
        want = c.attend(q, tables, lens, starts, max_new=rows)[:2 * new]
        for window in (10 ** 6, 2 ** 31 - 1, 2 ** 40):
            assert torch.equal(c.attend(q, tables, lens, starts, max_new=rows, window=window)[:2 * new], want)


def test_strided_queries_scale_and_out(cuda):
    lens = [50, 77]
    c, tables, held = filled(cuda, lens, 2, 64, 16, "Q8_0", "Q4_0")
    fused = torch.randn(2, 12 * 64, generator=gen(8, cuda), device=cuda)
    q = fused[:, :8 * 64].unflatten(1, (8, 64))
    out = torch.empty(2, 8, 64, device=cuda)
    assert check(c, tables, held, lens, [1, 1], 8, F32, scale=0.3, q=q, out=out, one=True).data_ptr() == out.data_ptr()
    odd = torch.randn(2 * 8 * 64 + 1, generator=gen(8, cuda), device=cuda)[1:].view(2, 8, 64)     # starts off four values
    check(c, tables, held, lens, [1, 1], 8, F32, q=odd, one=True)


@pytest.mark.parametrize("off", [4, 8])
@pytest.mark.parametrize("dim", [96, 128, 256])
def test_strided_queries_of_the_tiles(cuda, off, dim):
    """Rows apart that start on 8 bytes (not 16) or on 16."""
    lens, new = [150, 90], [70, 90]
    c, tables, held = filled(cuda, lens, 2, dim, 16, "Q4_0", "Q8_0")
    fused = torch.randn(MANY, 4 * dim + off + 8, generator=gen(8, cuda), device=cuda).to(F16)
    q = fused[:, off:off + 4 * dim].unflatten(1, (4, dim))
    check(c, tables, held, lens, new, 4, F16, q=q, most=MANY)


@pytest.mark.parametrize("new, most", [(1, 1), (3, 3), (60, 60), (60, MANY)])
def test_same_bits_every_time_and_on_another_stream(cuda, new, most):
    lens = [5000, 777, 64]
    c, tables, _ = filled(cuda, lens, 2, 128, 64, "Q4_0", "Q4_0")
    assert KH.tiled(c, 8, 3, most, BF16, tables.shape[1]) == (new == 60)      # (60, 60): keys cut over the GPU
    q = torch.randn(max(3 * new, most), 8, 128, generator=gen(6, cuda), device=cuda).bfloat16()
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    starts = torch.arange(4, dtype=torch.int32, device=cuda) * new
    attend = lambda: c.attend(q, tables, lt, starts, max_new=most)[:3 * new]      # noqa: E731
    want = attend()
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [attend() for _ in range(3)]
    here = attend()           # at the same time as the side stream's
    torch.cuda.current_stream().wait_stream(side)
    for o in outs + [here]:
        assert torch.equal(o, want)


@pytest.mark.parametrize("new, most", [(1, 1), (30, 30), (30, MANY)])
def test_graph_with_growing_sequences(cuda, new, most):
    """A captured write + attend, replayed as the cache grows (lengths, slots and tables change in place), two graphs in
    turn and overlapping on two streams."""
    lens = [40, 400, 63]
    c, tables, _ = filled(cuda, [n + 200 for n in lens], 2, 128, 16, "Q4_0", "Q4_0")
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    starts = torch.arange(4, dtype=torch.int32, device=cuda) * new
    assert KH.tiled(c, 8, 3, most, BF16, tables.shape[1]) == (most == MANY)
    st = []
    for i in range(2):
        g = gen(20 + i, cuda)
        st.append([torch.randn(n, h, 128, generator=g, device=cuda).bfloat16() for n, h in ((max(3 * new, most), 8), (3 * new, 2), (3 * new, 2))])
    slots = torch.arange(3 * new, device=cuda)

    def step(q, k, v):
        c.write(k, v, slots)
        return c.attend(q, tables, lt, starts, max_new=most)[:3 * new]

    step(*st[0])
    graphs, outs = [], []
    for s in st:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*s))
        graphs.append(g)
    for t in range(4):
        lt += new
        for b in range(3):
            i = torch.arange(new, device=cuda) + lt[b].long() - new
            slots[b * new:(b + 1) * new] = tables[b][i // 16].long() * 16 + i % 16
        graphs[t % 2].replay()
        got = outs[t % 2].clone()
        assert torch.equal(got, step(*st[t % 2]))
    # the same slots and inputs on two streams: each graph has its own workspace
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a):
        oa = c.attend(st[0][0], tables, lt, starts, max_new=most)[:3 * new]
    with torch.cuda.graph(b):
        ob = c.attend(st[1][0], tables, lt, starts, max_new=most)[:3 * new]
    want = [c.attend(s[0], tables, lt, starts, max_new=most)[:3 * new] for s in st]
    side = torch.cuda.Stream(cuda)
    torch.cuda.synchronize()
    for _ in range(5):
        a.replay()
        with torch.cuda.stream(side):
            b.replay()
    torch.cuda.synchronize()
    assert torch.equal(oa, want[0]) and torch.equal(ob, want[1])


def test_offsets_past_32_bits(cuda):
    """Pages whose code bytes lie beyond 2^32."""
    n_pages = (1 << 32) // (1024 * 1024) + 3          # a page of K: 1024 tokens x 8 heads x 128 bytes
    c = kvcache.KVCache(n_pages, 8, 128, 1024, "Q8_0", "Q8_0", cuda)
    assert c.k_codes.numel() > 1 << 32
    n = 1500
    tables = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device=cuda)
    g = gen(1, cuda)
    k, v = (torch.randn(n, 8, 128, generator=g, device=cuda) for _ in range(2))
    s = slots_of(tables[0], n, 1024)
    c.write(k, v, s)
    held = [[x.double() for x in c.read(s, F32)]]
    assert (held[0][0] - k).abs().max() < 0.05
    for new, most in ((1, None), (4, None), (80, MANY)):
        check(c, tables, held, [n], [new], 8, BF16, most=most)


def test_decoder_layer_step(cuda):
    """A layer's attention half as a decoder runs it, three steps of two sequences: norm_block, q/k/v products, write with RoPE,
    attend, the output product and the norm behind it; every stage against its 64-bit form on the stage's own inputs,
    and once more from a captured graph, bit for bit."""
    dim, heads, n_kv, hid, page = 64, 4, 2, 256, 16
    mk = lambda n_out, n_in, s: (synth.blocks("Q8_0", n_out, n_in, seed=s).to(cuda), n_out)      # noqa: E731
    mq, mkk, mv_, mo = mk(heads * dim, hid, 1), mk(n_kv * dim, hid, 2), mk(n_kv * dim, hid, 3), mk(hid, heads * dim, 4)
    g = gen(7, cuda)
    w_pre, w_post, w_next = (torch.rand(hid, generator=g, device=cuda) + 0.5 for _ in range(3))
    tab = torch.arange(64, dtype=torch.float64)[:, None] * torch.pow(1e4, -torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
    cos, sin = tab.cos().float().to(cuda), tab.sin().float().to(cuda)
    c = kvcache.KVCache(8, n_kv, dim, page, "Q8_0", "Q4_0", cuda)
    tables = torch.tensor([[5, 1], [0, 7]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([14, 0], dtype=torch.int32, device=cuda)
    past = torch.randn(14, n_kv, dim, generator=g, device=cuda)
    c.write(past, past, slots_of(tables[0], 14, page))
    ffn, h = (torch.randn(2, hid, generator=g, device=cuda) for _ in range(2))

    def layer(ffn, h):
        pos = lens.long()
        slots = tables.gather(1, (pos // page)[:, None])[:, 0].long() * page + pos % page
        x, e, h1 = mmvq.norm_block(ffn, h, w_pre, 1e-6, w_post=w_post, rs=0.5, eingang=True)
        q, k, v = mmvq.mv_geteilt("Q8_0", [mq, mkk, mv_], e, hid)
        qr = c.write(k.view(2, n_kv, dim), v.view(2, n_kv, dim), slots, q=q.view(2, heads, dim), rope=(cos, sin, pos))
        o = c.attend(qr, tables, lens + 1)
        y = mmvq.mv("Q8_0", mo[0], o.view(2, -1), hid, heads * dim)
        x2, _, h2 = mmvq.norm_block(y, h1, w_next, 1e-6, w_post=w_post, rs=0.5)
        return x, q, k, qr, o, y, x2, h2

    for step in range(3):
        x, q, k, qr, o, y, x2, h2 = layer(ffn, h)
        pos = lens.long().cpu().numpy()
        want_q = KH.rotate(q.view(2, heads, dim).cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy(), pos, False)
        assert np.array_equal(qr.cpu().numpy(), want_q)
        wq = mmvq.entpacken("Q8_0", mq[0], mq[1], hid, F32).double()
        assert ((q.double() - x.double() @ wq.T).abs().max() / q.abs().max()) < 1e-3          # the matvec's own bound
        for b in range(2):
            n = int(lens[b]) + 1
            held = [t.double() for t in c.read(slots_of(tables[b], n, page), F32)]
            ref, sizes = KH.attention(qr[b:b + 1].double(), *held, torch.tensor([n - 1], device=cuda), dim ** -0.5, 0)
            assert ((o[b:b + 1].double() - ref).abs() <= KH.bound(sizes, ref, F32, n, False)).all()
        z = y.double() / (y.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w_post.double()
        z0 = ffn.double() / (ffn.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w_post.double()
        ref = h.double() + 0.5 * z0 + 0.5 * z
        # two norms of 256 values: (256 / 32 + 32) 2^-24 of rs |z| each, sums and roundings below 2^-22: under 2^-18
        assert ((h2.double() - ref).abs() <= 2.0 ** -18 * (h.abs() + z.abs() + z0.abs()).double()).all()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = layer(ffn, h)
        graph.replay()
        for a, b in zip(outs, (x, q, k, qr, o, y, x2, h2)):
            assert torch.equal(a, b)
        ffn, h = y.clone(), h2.clone()
        lens += 1


def test_refusals(cuda):
    c = kvcache.KVCache(4, 2, 64, 16, device=cuda)
    x = torch.zeros(3, 2, 64, device=cuda)
    s = torch.arange(3, device=cuda)
    t, n = torch.zeros(3, 1, dtype=torch.int32, device=cuda), torch.ones(3, dtype=torch.int32, device=cuda)
    tab = torch.zeros(8, 32, device=cuda)
    for call in (lambda: c.write(x[:, :1], x, s), lambda: c.write(x, x[:2], s), lambda: c.write(x, x.half(), s),
                 lambda: c.write(x, x, s.int()), lambda: c.write(x, x, s[:2]), lambda: c.write(x.double(), x.double(), s),
                 lambda: c.write(x.cpu(), x, s), lambda: c.write(x, x, s, rope=(tab, tab[:4], s)),
                 lambda: c.write(x, x, s, rope=(tab[:, :30].contiguous(), tab[:, :30].contiguous(), s)),
                 lambda: c.write(x, x, s, rope=(tab[:0], tab[:0], s)), lambda: c.write(x, x, s, q=x[..., :32]),
                 lambda: c.read(s, torch.float64), lambda: c.read(s.cpu()), lambda: c.attend(x[:, :1], t, n),
                 lambda: c.attend(x, t.long(), n), lambda: c.attend(x, t, n[:2]), lambda: c.attend(x[:2], t, n),
                 lambda: c.attend(x, t, n, window=-1), lambda: c.attend(x, t, n, starts=n), lambda: c.attend(x, t, n, out=x.half()),
                 lambda: c.attend(x, t[:, :0].contiguous(), n), lambda: c.attend(x, t, n, out=torch.zeros(3, 4, 64, device=cuda)[:, ::2]),
                 lambda: kvcache.KVCache(4, 2, 64, 16, buffers=(c.k_codes, c.v_codes, c.scales.float())),
                 lambda: kvcache.KVCache(5, 2, 64, 16, buffers=(c.k_codes, c.v_codes, c.scales))):
        with pytest.raises(RuntimeError):
            call()
    assert c.attend(x[:0], t[:0], n[:0]).shape == (0, 2, 64)
