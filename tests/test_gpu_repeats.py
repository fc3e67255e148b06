"""The same calls on the same inputs give the same bits, with other calls between them that nothing waits for."""
import pytest
import torch

from nemicli_terminal_b200 import mmvq

from tests.test_gpu_chosen import BF16, F32, filled
from tests.test_gpu_kvcache import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pdl", [False, True])
@pytest.mark.parametrize("dtype, seqs, most, keep", [(BF16, 64, 4000, 12), (F32, 1, 9000, 64), (BF16, 8, 700, 64)])
def test_chosen_pages(cuda, dtype, seqs, most, keep, pdl):
    states = []
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        lens = [most] + torch.randint(1, most, (seqs - 1,), generator=g).tolist()
        c, t, n = filled(cuda, lens, 4, 128, 64, "Q4_0", "Q4_0", seed)
        b = c.bounds()
        c.summarise(b, t, n, torch.tensor([0] + lens, device=cuda).cumsum(0).int())
        q = torch.randn(seqs, 16, 128, generator=gen(seed, cuda), device=cuda).to(dtype)
        states.append((c, q, b, t, n))

    def run(c, q, b, t, n):
        chosen, held = c.choose(q, b, t, n, keep, first=1, last=2)
        return chosen, held, c.attend_chosen(q, chosen, held)

    mmvq.pdl(pdl)
    try:
        want = [run(*s) for s in states]
        for i in range(60):
            got = run(*states[i % 2])
            assert all(torch.equal(x, y) for x, y in zip(got, want[i % 2])), i
    finally:
        mmvq.pdl(False)
