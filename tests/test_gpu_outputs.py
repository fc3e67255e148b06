"""The outputs of one call share an allocation, each with its own 16-byte aligned bytes."""
import pytest
import torch

from nemicli_terminal_b200 import beams, kvcache, pages

pytestmark = pytest.mark.gpu
I32 = torch.int32


@pytest.mark.parametrize("n", [1, 3, 7, 64])
def test_parts_of_one_allocation(cuda, n):
    free, counts = pages.pool(4 * n, cuda)
    tables, lens, new = torch.full((n, 3), -1, dtype=I32, device=cuda), torch.zeros(n, dtype=I32, device=cuda), torch.ones(n, dtype=I32, device=cuda)
    c = kvcache.KVCache(4 * n, 1, 64, 16, "Q4_0", "Q4_0", cuda)
    calls = [pages.plan(lens, new, tables, free, counts, 16, n), pages.release(new.bool(), lens, tables, free, counts, 16),
             pages.reorder(lens.view(1, n), lens, tables, free, counts, 16), beams.select(torch.zeros(n, 1, 5, device=cuda), torch.zeros(n, 1, device=cuda), 3),
             c.choose(torch.zeros(n, 2, 64, device=cuda), c.bounds(), tables, new, 5)]
    for outputs in calls:
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in outputs)
        assert all(a % 16 == 0 for a, _ in spans) and all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
        assert len({t.untyped_storage().data_ptr() for t in outputs}) == 1
        kept = [t.clone() for t in outputs]
        for t in outputs:                                         # writing to one changes no other
            t.zero_()
            kept[[x is t for x in outputs].index(True)].zero_()
            assert all(torch.equal(x, y) for x, y in zip(outputs, kept))
        assert len({t.untyped_storage().data_ptr() for t in kept}) == len(kept)
