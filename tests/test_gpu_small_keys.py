"""The choice of pages whose keys are so small that their boxes are fp16's denormals."""
import pytest
import torch

from tests.test_gpu_chosen import BF16, F16, F32, choice, long_cache
from tests.test_gpu_kvcache import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("power", [-14, -16, -18, -20])
def test_boxes_of_denormals(cuda, dtype, power):
    """Boxes from 2^power of their usual size down to a few steps of 2^-24: the pages that fp64 chooses."""
    c, t, n, b = long_cache(cuda, 1500)
    small = (b.float() * 2.0 ** power).half()
    for seed in range(3):
        q = torch.randn(1, 4, 64, generator=gen(30 + seed, cuda), device=cuda).to(dtype)
        for keep in (20, 333):
            chosen, _ = c.choose(q, small, t, n, keep, first=0, last=1)
            want = choice(q[0], small, t[0], 1500 * 16 - 1, 16, keep, 0, 1, 1)[0]
            assert chosen[0, 0].tolist() == t[0, torch.tensor(want, device=cuda)].tolist()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sign", [1, -1])
def test_sums_of_denormals_beside_a_large_query(cuda, dtype, sign):
    """Products of tensor cores with a denormal operand are cut off as if that were 2^-14.  Of the pages here half reach 5 to 9 units (2^-38
    of the largest query value) further than the others by 59 products, of each of which a quarter of a unit is cut off on average; the
    others' score is one product without a rest."""
    c, t, n, b = long_cache(cuda, 1500)
    step = 2.0 ** -24
    large = [0, 4, 32, 36]                                        # one in each step of the products
    q = 2.0 ** -11 * (1 + torch.rand(1, 1, 64, generator=gen(5, cuda), device=cuda)).to(dtype)
    q[..., large] = 1
    few = torch.ones(64, dtype=torch.bool, device=cuda)
    few[large + [1]] = False
    q[..., 1] = torch.floor((q[0, 0, few].double().sum() * 2.0 ** 14 - 5) / 4) * 4 * 2.0 ** -14
    assert (q[0, 0, 1].double() * 2.0 ** 12) % 1 == 0             # (held by every type)
    many = torch.arange(1500, device=cuda) % 2 == 1
    box = torch.zeros_like(b)
    side = 1 if sign > 0 else 0
    for at, on in ((t[0, many].long(), few), (t[0, ~many].long(), ~few)):
        x = torch.zeros(64, device=cuda)
        x[on] = step
        x[large] = step
        box[at, 0, side] = (x * sign).half()
    q *= sign
    for keep in (300, 751, 1100):
        chosen, _ = c.choose(q, box, t, n, keep, first=0, last=1)
        want = choice(q[0], box, t[0], 1500 * 16 - 1, 16, keep, 0, 1, 1)[0]
        assert chosen[0, 0].tolist() == t[0, torch.tensor(want, device=cuda)].tolist(), keep


def test_a_written_cache_of_small_keys(cuda):
    """The same through write and summarise: keys of 2^-19."""
    c, t, n, b = long_cache(cuda, 800)
    g = gen(3, cuda)
    k = torch.randn(800, 1, 1, 64, generator=g, device=cuda) + torch.randn(800, 16, 1, 64, generator=g, device=cuda)
    slots = (t[0, :, None].long() * 16 + torch.arange(16, device=cuda)).flatten()
    c.write((k * 2.0 ** -19).flatten(0, 1), k.flatten(0, 1), slots)
    c.summarise(b, t, n, torch.tensor([0, 12800], dtype=torch.int32, device=cuda))
    q = torch.randn(1, 4, 64, generator=g, device=cuda)
    for keep in (16, 200):
        chosen, _ = c.choose(q, b, t, n, keep)
        want = choice(q[0], b, t[0], 800 * 16 - 1, 16, keep, 1, 1, 1)[0]
        assert chosen[0, 0].tolist() == t[0, torch.tensor(want, device=cuda)].tolist()
