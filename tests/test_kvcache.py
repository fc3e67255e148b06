"""The quantised cache and norm_block without a GPU: refusals of the C ABI and of the Python entry points, before any
launch, and the plain forms the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

from nemicli_terminal_b200 import _lib, kvcache, mmvq
from nemicli_terminal_b200.formats import TYPE_ID

from tests import kv_helpers as KH

A = ctypes.c_void_p(4096)                    # never dereferenced: every call below is refused first
ODD = ctypes.c_void_p(4097)


def cache(**kw):
    arg = dict(k=4096, v=4096, scales=4096, n_pages=4, n_kv=2, dim=64, page=16, k_type=TYPE_ID["Q4_0"], v_type=TYPE_ID["Q8_0"])
    arg.update(kw)
    return ctypes.byref(kvcache._Cache(*[arg[n] for n, _ in kvcache._Cache._fields_]))


def write(c=None, k=A, v=A, dtype=0, ks=128, vs=128, slots=A, rows=1, cos=A, sin=A, pos=A, n_pos=8, rot=64, q=A, qs=256, nq=4,
          qo=A):
    return _lib.load().qmv_kv_write(c or cache(), k, v, dtype, ks, vs, slots, rows, cos, sin, pos, n_pos, rot, 0, q, qs, nq, qo, None)


@pytest.mark.parametrize("bad, status", [
    (dict(k=0), 6), (dict(scales=0), 6), (dict(k=4100), 3), (dict(n_pages=0), 2), (dict(n_kv=0), 2), (dict(dim=80), 2),
    (dict(dim=0), 2), (dict(page=8), 2), (dict(page=48), 2), (dict(page=2048), 2), (dict(n_pages=1 << 40), 2),
    (dict(k_type=TYPE_ID["Q4_K"]), 1), (dict(v_type=0), 1)])
def test_cache_descriptions_refused(bad, status):
    L, c = _lib.load(), cache(**bad)
    assert write(c) == status
    assert L.qmv_kv_read(c, A, 1, A, A, 0, None) == status
    assert L.qmv_kv_attend(c, A, 0, 256, 4, A, 1, A, None, 1, 1, 1, 1.0, 0, A, A, 1 << 30, None) == status
    assert L.qmv_kv_attend_workspace_bytes(c, 4, 1, 1, 0, 1, 0) == 0


@pytest.mark.parametrize("bad, status", [
    (dict(k=None), 6), (dict(slots=None), 6), (dict(sin=None), 6), (dict(pos=None), 6), (dict(qo=None), 6),
    (dict(dtype=3), 2), (dict(rows=-1), 4), (dict(rows=1 << 31), 4), (dict(nq=0), 4), (dict(ks=120), 2), (dict(vs=124), 2),
    (dict(qs=255), 2), (dict(rot=60), 2), (dict(rot=72), 2), (dict(rot=0), 2), (dict(n_pos=0), 2), (dict(ks=130), 3), (dict(k=ODD), 3),
    (dict(cos=ODD), 3), (dict(q=ctypes.c_void_p(4104)), 3), (dict(qs=258), 3)])
def test_write_refusals(bad, status):
    assert write(**bad) == status


def test_write_of_no_rows_is_no_launch():
    assert write(rows=0) == 0


def attend(q=A, dtype=0, qs=256, heads=4, tables=A, width=1, lens=A, starts=A, n_seq=1, rows=1, new=1, window=0, out=A, ws=A,
           nbytes=1 << 34):
    return _lib.load().qmv_kv_attend(cache(), q, dtype, qs, heads, tables, width, lens, starts, n_seq, rows, new, 1.0, window, out, ws,
                                     nbytes, None)


@pytest.mark.parametrize("bad, status", [
    (dict(q=None), 6), (dict(tables=None), 6), (dict(lens=None), 6), (dict(out=None), 6), (dict(ws=None), 6), (dict(dtype=3), 2),
    (dict(heads=3), 2), (dict(heads=0), 2), (dict(width=0), 2), (dict(width=1 << 28), 2), (dict(window=-1), 2), (dict(n_seq=0), 4),
    (dict(n_seq=70000), 4), (dict(rows=-1), 4), (dict(new=0), 4), (dict(starts=None, rows=2, n_seq=3), 4), (dict(qs=252), 2),
    (dict(q=ODD), 3), (dict(out=ODD), 3), (dict(ws=ctypes.c_void_p(4096 + 128)), 3), (dict(nbytes=0), 2), (dict(qs=258), 3)])
def test_attend_refusals(bad, status):
    assert attend(**bad) == status


def test_attend_refuses_a_short_workspace_for_cut_tiles():
    need = _lib.load().qmv_kv_attend_workspace_bytes(cache(), 4, 1, 2000, 1, 1000, 0)
    assert need % 2 == 1 and need > 1
    assert attend(dtype=1, new=2000, rows=2000, width=1000, nbytes=need - 2) == 2


def test_attend_of_no_rows_is_no_launch():
    assert attend(rows=0) == 0


@pytest.mark.parametrize("bad, status", [
    (dict(y=None), 6), (dict(h_out=None), 6), (dict(xn=None), 6), (dict(xq2=None), 6), (dict(w_pre=None), 6), (dict(dtype=5), 2), (dict(n=0), 2),
    (dict(n=32769), 2), (dict(n=33), 2), (dict(ys=63), 2), (dict(gs=3), 2), (dict(rows=-1), 4), (dict(h=ODD), 3),
    (dict(xq=ctypes.c_void_p(4104)), 3)])
def test_norm_block_refusals(bad, status):
    a = dict(y=A, ys=64, h=A, hs=64, gate=A, gs=0, w_post=A, w_pre=A, dtype=0, rows=1, n=64, h_out=A, xn=A, xq=A, xq2=A)
    a.update(bad)
    st = _lib.load().qmv_norm_block(a["y"], max(a["ys"], a["n"] if "n" in bad else 0), a["h"], max(a["hs"], a["n"]), a["gate"], a["gs"],
                                    a["w_post"], a["w_pre"], a["dtype"], 1e-6, 1.0, a["rows"], a["n"], a["h_out"], a["xn"], a["xq"],
                                    a["xq2"], A, A, None)
    assert st == status


def test_python_refuses_cpu_tensors_and_odd_shapes():
    with pytest.raises(RuntimeError):
        kvcache.KVCache(4, 2, 64, device="cpu")
    for kw in (dict(k_fmt="Q4_K"), dict(v_fmt="F16"), dict(dim=80), dict(page=24), dict(n_pages=0), dict(n_kv=0)):
        with pytest.raises(RuntimeError):
            kvcache.KVCache(**{**dict(n_pages=4, n_kv=2, dim=64, device="cuda"), **kw})
    with pytest.raises(RuntimeError):
        mmvq.norm_block(torch.zeros(64), torch.zeros(64), torch.ones(64), 1e-6)


def test_plain_attention_against_softmax_by_hand():
    q, k, v = (torch.randn(*s, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
               for i, s in enumerate(((2, 2, 64), (3, 1, 64), (3, 1, 64))))
    o, _ = KH.attention(q, k, v, torch.tensor([1, 2]), 0.5, 0)
    w = torch.exp(0.5 * (k[:2, 0] @ q[0, 1]))
    assert torch.allclose(o[0, 1], (w / w.sum()) @ v[:2, 0], atol=1e-12)
    o, _ = KH.attention(q, k, v, torch.tensor([-1, 2]), 0.5, 1)
    assert torch.equal(o[0], torch.zeros_like(o[0])) and torch.allclose(o[1, 0], v[2, 0], atol=1e-12)


@pytest.mark.parametrize("fmt", ["Q4_0", "Q8_0"])
def test_plain_quantiser_stays_within_half_a_step(fmt):
    """Half a step of d, plus what rounding d to fp16 moves the end of the range by (Q4_0's upper end is 7 of 8 steps)."""
    x = np.random.default_rng(1).standard_normal((5, 2, 64)).astype(np.float32)
    c, d = KH.quantise(x, fmt)
    err = np.abs(KH.values(c, d, fmt) - x).reshape(5, 2, 2, 32)
    step = np.abs(d.astype(np.float64))[..., None]
    far = 1.0 if fmt == "Q4_0" else 0.5
    assert (err <= step * (far + 128 * 2.0 ** -11)).all()
