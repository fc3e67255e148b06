"""Page tables, beam selection, chosen pages and positions of several axes without a GPU: refusals of the C ABI and of the Python
entry points before any launch, and the plain forms that the GPU tests compare with."""
import ctypes

import pytest
import torch

from nemicli_terminal_b200 import _lib, beams, kvcache, pages

from tests import paging_helpers as PH
from tests.test_kvcache import A, ODD, cache

B = ctypes.c_void_p(8192)
HALF = ctypes.c_void_p(4096 + 128)


def plan(lens=A, add=A, tables=A, n=1, width=4, page=16, free=A, n_pages=8, counts=A, rows=1, slots=A, pos=A, starts=A, lens_out=B, counts_out=B):
    return _lib.load().qmv_page_plan(lens, add, tables, n, width, page, free, n_pages, counts, rows, slots, pos, starts, lens_out, counts_out, None)


@pytest.mark.parametrize("bad, status", [
    (dict(lens=None), 6), (dict(add=None), 6), (dict(counts_out=None), 6), (dict(slots=None), 6), (dict(page=24), 2), (dict(page=8), 2),
    (dict(page=2048), 2), (dict(width=0), 2), (dict(width=1 << 27), 2), (dict(n_pages=0), 2), (dict(n=0), 4), (dict(n=65536), 4),
    (dict(rows=-1), 4), (dict(rows=(1 << 30) + 1), 4), (dict(lens_out=A), 2), (dict(counts_out=A), 2), (dict(tables=ODD), 3),
    (dict(slots=ctypes.c_void_p(4100)), 3), (dict(lens_out=ODD), 3)])
def test_plan_refusals(bad, status):
    assert plan(**bad) == status


def release(done=A, lens=A, tables=A, n=1, width=4, page=16, free=A, n_pages=8, counts=A, lens_out=B, counts_out=B):
    return _lib.load().qmv_page_release(done, lens, tables, n, width, page, free, n_pages, counts, lens_out, counts_out, None)


@pytest.mark.parametrize("bad, status", [(dict(done=None), 6), (dict(free=None), 6), (dict(page=20), 2), (dict(n=0), 4), (dict(lens_out=A), 2),
                                         (dict(counts_out=A), 2), (dict(free=ODD), 3), (dict(n_pages=-1), 2)])
def test_release_refusals(bad, status):
    assert release(**bad) == status


def reorder(parents=A, lens=A, tables=A, own=A, n_req=2, k=4, width=4, page=16, free=A, n_pages=8, counts=A, t_out=B, l_out=B, src=A, dst=A,
            used=A, c_out=B, ws=A, nbytes=1 << 30):
    return _lib.load().qmv_page_reorder(parents, lens, tables, own, n_req, k, width, page, free, n_pages, counts, t_out, l_out, src, dst, used,
                                        c_out, ws, nbytes, None)


@pytest.mark.parametrize("bad, status", [
    (dict(parents=None), 6), (dict(ws=None), 6), (dict(used=None), 6), (dict(k=65), 2), (dict(k=0), 2), (dict(n_req=0), 4), (dict(n_req=20000), 4),
    (dict(t_out=A), 2), (dict(l_out=A), 2), (dict(c_out=A), 2), (dict(nbytes=100), 2), (dict(page=17), 2), (dict(own=ODD), 3), (dict(ws=HALF), 3),
    (dict(dst=ODD), 3)])
def test_reorder_refusals(bad, status):
    assert reorder(**bad) == status


def test_reorder_workspace():
    f = _lib.load().qmv_page_reorder_workspace_bytes
    assert f(2, 4, 4) > 0 and f(0, 4, 4) == f(2, 65, 4) == f(2, 4, 0) == f(20000, 4, 4) == 0


def select(x=A, dtype=0, stride=100, n_req=1, k=2, vocab=100, scores=A, n=2, out=A, parents=A, tokens=A, ws=A, nbytes=1 << 30):
    return _lib.load().qmv_beam_select(x, dtype, stride, n_req, k, vocab, scores, n, out, parents, tokens, ws, nbytes, None)


@pytest.mark.parametrize("bad, status", [
    (dict(x=None), 6), (dict(scores=None), 6), (dict(ws=None), 6), (dict(dtype=3), 2), (dict(n=0), 2), (dict(n=65), 2), (dict(k=65), 2), (dict(k=0), 2),
    (dict(n_req=0), 2), (dict(n_req=40000), 2), (dict(vocab=0), 2), (dict(vocab=(1 << 30) + 1, stride=1 << 31), 2), (dict(stride=99), 2),
    (dict(nbytes=10), 2), (dict(vocab=3, n=7), 2), (dict(x=ctypes.c_void_p(4098)), 3), (dict(x=ODD, dtype=1), 3), (dict(tokens=ODD), 3), (dict(ws=HALF), 3)])
def test_select_refusals(bad, status):
    assert select(**bad) == status


def test_select_workspace():
    f = _lib.load().qmv_beam_workspace_bytes
    assert f(1, 4, 1000, 8) > 0 and f(1, 4, 1, 5) == f(0, 4, 9, 1) == f(1, 65, 9, 1) == f(1, 4, 9, 65) == 0


def copy(c=None, src=A, dst=A, used=A, n=1):
    return _lib.load().qmv_kv_copy(c or cache(), src, dst, used, n, None)


@pytest.mark.parametrize("bad, status", [(dict(src=None), 6), (dict(dst=None), 6), (dict(n=-1), 4), (dict(n=1 << 30), 4), (dict(src=ODD), 3),
                                         (dict(used=ODD), 3)])
def test_copy_refusals(bad, status):
    assert copy(**bad) == status
    assert copy(n=0) == 0 and copy(cache(page=8)) == 2


def bounds(c=None, tables=A, width=1, lens=A, starts=A, n=1, new=1, b=A):
    return _lib.load().qmv_kv_bounds(c or cache(), tables, width, lens, starts, n, new, b, None)


@pytest.mark.parametrize("bad, status", [(dict(tables=None), 6), (dict(b=None), 6), (dict(width=0), 2), (dict(width=1 << 28), 2), (dict(n=0), 4),
                                         (dict(n=65536), 4), (dict(new=0), 4), (dict(b=ctypes.c_void_p(4104)), 3), (dict(starts=ODD), 3),
                                         (dict(c=cache(dim=80)), 2)])
def test_bounds_refusals(bad, status):
    assert bounds(**bad) == status


def choose(c=None, q=A, dtype=0, qs=256, heads=4, b=A, tables=A, width=9, lens=A, starts=A, n=1, rows=1, keep=4, first=1, last=1, chosen=A, held=A,
           ws=A, nbytes=1 << 30):
    return _lib.load().qmv_kv_choose(c or cache(), q, dtype, qs, heads, b, tables, width, lens, starts, n, rows, keep, first, last, chosen, held, ws,
                                     nbytes, None)


@pytest.mark.parametrize("bad, status", [
    (dict(q=None), 6), (dict(b=None), 6), (dict(held=None), 6), (dict(ws=None), 6), (dict(dtype=4), 2), (dict(heads=3), 2), (dict(heads=130, qs=1 << 14), 2),
    (dict(width=0), 2), (dict(n=0), 4), (dict(rows=65536), 4), (dict(rows=-1), 4), (dict(starts=None, rows=2, n=3), 4), (dict(first=-1), 2),
    (dict(last=0), 2), (dict(keep=1), 2), (dict(keep=1 << 30), 2), (dict(qs=252), 2), (dict(q=ODD), 3), (dict(qs=258), 3), (dict(nbytes=8), 2),
    (dict(ws=HALF), 3), (dict(b=ctypes.c_void_p(4104)), 3)])
def test_choose_refusals(bad, status):
    assert choose(**bad) == status
    assert choose(rows=0) == 0


def attend(c=None, q=A, dtype=0, qs=256, heads=4, chosen=A, keep=4, held=A, rows=1, scale=1.0, out=A, ws=A, nbytes=1 << 30):
    return _lib.load().qmv_kv_attend_chosen(c or cache(), q, dtype, qs, heads, chosen, keep, held, rows, scale, out, ws, nbytes, None)


@pytest.mark.parametrize("bad, status", [
    (dict(q=None), 6), (dict(chosen=None), 6), (dict(out=None), 6), (dict(dtype=3), 2), (dict(heads=5), 2), (dict(keep=0), 2), (dict(keep=1 << 27), 2),
    (dict(rows=65536), 4), (dict(rows=-1), 4), (dict(scale=float("nan")), 2), (dict(scale=float("inf")), 2), (dict(qs=252), 2), (dict(out=ODD), 3),
    (dict(ws=HALF), 3), (dict(nbytes=0), 2), (dict(held=ODD), 3)])
def test_attend_chosen_refusals(bad, status):
    assert attend(**bad) == status
    assert attend(rows=0) == 0


def axes(names=bytes([0, 1, 2, 2] * 8), n_axes=3, cos=A, rot=64):
    return _lib.load().qmv_kv_write_axes(cache(), A, A, 0, 128, 128, A, 0, cos, A, A, 8, rot, 0, names, n_axes, A, 256, 4, A, None)


def test_write_axes_refusals():
    assert axes() == 0                                            # (no rows: no launch)
    assert axes(cos=None) == 6 and axes(names=None) == 6
    assert axes(n_axes=0) == axes(n_axes=5) == axes(n_axes=2) == axes(rot=60) == 2
    with pytest.raises(RuntimeError):
        kvcache.rope_axes(())
    with pytest.raises(RuntimeError):
        kvcache.rope_axes((3, -1))


def test_rope_axes():
    assert kvcache.rope_axes((1, 2, 3)) == (0, 1, 1, 2, 2, 2)
    assert kvcache.rope_axes((3, 1, 2), mixed=True) == (0, 1, 2, 0, 2, 0)


def test_python_refuses_cpu_tensors_and_odd_shapes():
    t, v = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    free, counts = torch.zeros(4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        pages.plan(v, v, t, free, counts, 16, 2)
    with pytest.raises(RuntimeError):
        pages.release(v.bool(), v, t, free, counts, 16)
    with pytest.raises(RuntimeError):
        pages.reorder(v.view(1, 2), v, t, free, counts, 16)
    with pytest.raises(RuntimeError):
        beams.select(torch.zeros(1, 2, 3), torch.zeros(1, 2))


def test_plain_forms_by_hand():
    got = PH.plan([15, 0], [2, 1], [[7, -1], [-1, -1]], [3, 4, 0, 0, 0, 0, 0, 0], [2, 0], 16, 4)
    assert got[0] == [7 * 16 + 15, 4 * 16, 3 * 16, -1] and got[1] == [15, 16, 0, 0] and got[2] == [0, 2, 3] and got[4] == [0, 0]
    got = PH.reorder([[1, 1]], [20, 20], [[0, 1], [0, 2]], [5, 0, 0, 0, 0, 0], [1, 0], 16)
    assert got[0] == [[0, 2], [0, 1]] and got[3:6] == ([-1, 2], [-1, 1], [0, 4]) and got[2] == [1, 0]
