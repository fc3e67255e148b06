"""KVCache.write with positions on several axes on the GPU: codes, scales and queries equal the plain forms' bit for bit."""
import numpy as np
import pytest
import torch

from nemicli_terminal_b200 import _lib, kvcache

from tests import kv_helpers as KH
from tests.test_gpu_kvcache import gen

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def tables(rot, n, cuda):
    a = torch.arange(n, dtype=torch.float64)[:, None] * torch.pow(1e6, -torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
    return a.cos().float().to(cuda), a.sin().float().to(cuda)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim, rot, sections, mixed, paired", [
    (128, 128, (16, 24, 24), False, False), (128, 128, (24, 20, 20), True, False), (64, 64, (8, 12, 12), False, True),
    (96, 96, (20, 14, 14), True, True), (256, 64, (11, 11, 10), True, False), (96, 40, (1, 18, 1), False, False),
    (256, 256, (40, 30, 30, 28), True, False), (64, 64, (32,), False, False), (128, 128, (0, 64), False, True)])
def test_write_is_exact(cuda, dtype, dim, rot, sections, mixed, paired):
    rows, n_kv, heads, page = 45, 3, 6, 16
    g = gen(dim + rot, cuda)
    axes = kvcache.rope_axes(sections, mixed)
    c = kvcache.KVCache(4, n_kv, dim, page, "Q8_0", "Q4_0", cuda)
    q, k, v = (torch.randn(rows, h, dim, generator=g, device=cuda).mul(3).to(dtype) for h in (heads, n_kv, n_kv))
    slots = torch.randperm(4 * page, generator=g, device=cuda)[:rows].contiguous()
    cos, sin = tables(rot, 700, cuda)
    pos = torch.randint(0, 700, (len(sections), rows), generator=g, device=cuda)
    out = c.write(k, v, slots, q=q, rope=(cos, sin, pos), paired=paired, axes=axes)
    # the plain rotation takes one table row a token: put together from the axes' rows
    at = pos.cpu().numpy()[list(axes)].T
    cn, sn = (np.take_along_axis(x.cpu().numpy(), at, 0) for x in (cos, sin))
    one = np.arange(rows)
    kn, qn = (KH.rotate(x.float().cpu().numpy(), cn, sn, one, paired) for x in (k, q))
    assert torch.equal(out.cpu(), torch.from_numpy(qn).to(dtype))
    gk, gv, gs = KH.codes_of(c, slots.cpu().numpy())
    for x, fmt, got, sc in ((kn, "Q8_0", gk, gs[:, :, 0]), (v.float().cpu().numpy(), "Q4_0", gv, gs[:, :, 1])):
        code, d = KH.quantise(x, fmt)
        assert np.array_equal(got, code) and np.array_equal(sc.view(np.uint16), d.view(np.uint16))
    assert _lib.device_status(device=cuda) == 0


def test_axes_alike_are_one_axis(cuda):
    """Text tokens have the same position on every axis: the same bytes as a write without axes."""
    g = gen(2, cuda)
    k = torch.randn(200, 4, 128, generator=g, device=cuda).bfloat16()
    cos, sin = tables(128, 500, cuda)
    pos = torch.randint(0, 500, (200,), generator=g, device=cuda)
    a, b = (kvcache.KVCache(13, 4, 128, 16, device=cuda) for _ in range(2))
    slots = torch.arange(200, device=cuda)
    qa = a.write(k, k, slots, q=k, rope=(cos, sin, pos))
    qb = b.write(k, k, slots, q=k, rope=(cos, sin, pos.expand(3, -1).contiguous()), axes=kvcache.rope_axes((16, 24, 24)))
    assert torch.equal(qa, qb) and torch.equal(a.k_codes, b.k_codes) and torch.equal(a.v_codes, b.v_codes) and torch.equal(a.scales, b.scales)


def test_positions_outside_the_tables(cuda):
    """On any axis, also one that no frequency follows: the row is not written, its queries are 0, the status is set; padding rows."""
    c = kvcache.KVCache(2, 1, 64, 16, device=cuda)
    x = torch.randn(5, 1, 64, generator=gen(3, cuda), device=cuda)
    cos, sin = tables(64, 4, cuda)
    pos = torch.tensor([[0, 1, 4, 3, 0], [0, -1, 2, 3, 0], [0, 1, 2, 9, 1]], device=cuda)
    _lib.device_status(device=cuda)
    q = c.write(x, x, torch.tensor([0, 1, 2, 3, -1], device=cuda), q=x, rope=(cos, sin, pos), axes=kvcache.rope_axes((16, 16, 0)))
    assert _lib.device_status(device=cuda) == 1
    assert q[0].any() and not q[1:4].any() and q[4].any()
    k, v = c.read(torch.arange(5, device=cuda), F32)
    assert k[0].any() and not k[1:].any() and not v[1:].any()
