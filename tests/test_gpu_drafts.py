"""Drafted rows over chosen pages in float16, and in batches whose sequences have none, one or many of them."""
import numpy as np
import pytest
import torch

from nemicli_terminal_b200 import _lib

from tests.test_gpu_chosen import BF16, F16, F32, check, filled
from tests.test_gpu_kvcache import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim, heads, n_kv, page, kf, vf", [(128, 8, 2, 16, "Q4_0", "Q8_0"), (96, 5, 1, 32, "Q8_0", "Q4_0"), (256, 6, 3, 16, "Q4_0", "Q4_0")])
def test_rows_of_unequal_sequences(cuda, dtype, dim, heads, n_kv, page, kf, vf):
    lens, news = [300, 17, 1, 640, 33, 90], [7, 0, 1, 16, 2, 12]
    c, t, n = filled(cuda, lens, n_kv, dim, page, kf, vf, dim)
    b = c.bounds()
    c.summarise(b, t, n, torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=cuda))
    starts = torch.tensor(np.cumsum([0] + news), dtype=torch.int32, device=cuda)
    q = (torch.randn(sum(news) + 2, heads, dim, generator=gen(6, cuda), device=cuda) * 0.6).to(dtype)
    for keep, first, last in ((2, 0, 1), (5, 1, 2), (64, 1, 1)):
        check(c, q, b, t, n, keep, first, last, starts, news)
    assert _lib.device_status(device=cuda) == 0
