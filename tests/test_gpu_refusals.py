"""Refusals of the small calls whose arguments have to be on the GPU to be looked at."""
import pytest
import torch

from nemicli_terminal_b200 import beams, kvcache, pages

pytestmark = pytest.mark.gpu
I32 = torch.int32


def chosen_call(cuda, **kw):
    c = kvcache.KVCache(4, 1, 64, 16, "Q4_0", "Q4_0", cuda)
    q = torch.zeros(2, 2, 64, device=cuda)
    return c.attend_chosen(q, torch.zeros(2, 1, 1, dtype=I32, device=cuda), torch.zeros(2, dtype=I32, device=cuda), **kw)


@pytest.mark.parametrize("scale", ["0.125", "x", (1.0,), object(), float("nan"), float("inf"), -1e300, 10 ** 400],
                         ids=["digits", "text", "tuple", "object", "nan", "inf", "below", "above"])
def test_scale_of_attend_chosen(cuda, scale):
    """Numbers that are finite in float32 are taken, whatever their type; anything else is refused as everything is."""
    with pytest.raises(RuntimeError, match="KVCache.attend_chosen: scale"):
        chosen_call(cuda, scale=scale)


def test_scales_that_are_taken(cuda):
    for scale in (None, 1, 0.5, -1.0, torch.tensor(0.25), 3e38):
        assert not chosen_call(cuda, scale=scale).any()


def test_numbers(cuda):
    x, s = torch.zeros(1, 2, 8, device=cuda), torch.zeros(1, 2, device=cuda)
    for n in (2.0, "2", None, 65, -1, 1 << 70):
        with pytest.raises(RuntimeError, match="beams.select"):
            beams.select(x, s, n)
    t, v, free, counts = torch.zeros(2, 3, dtype=I32, device=cuda), torch.zeros(2, dtype=I32, device=cuda), *pages.pool(4, cuda)
    wide = torch.zeros(64, (1 << 20) + 1, dtype=I32, device=cuda)
    with pytest.raises(RuntimeError, match="pages.reorder: tables"):
        pages.reorder(torch.zeros(1, 64, dtype=I32, device=cuda), torch.zeros(64, dtype=I32, device=cuda), wide, free, counts, 16)
    for page, rows in ((16.0, 2), (None, 2), (24, 2), (16, 2.5), (16, -1), (16, 1 << 31)):
        with pytest.raises(RuntimeError, match="pages.plan"):
            pages.plan(v, v, t, free, counts, page, rows)
