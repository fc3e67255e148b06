"""Calls of the quantised cache's attention that the C ABI refuses before any launch (no GPU)."""
import pytest

from nemicli_terminal_b200 import _lib

from tests.test_kvcache import A, attend, cache


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("heads, new", [(64, (1 << 30) + 1), (64, (1 << 31) - 1), (64, (1 << 25) + 1), (2, (1 << 30) + 1)])
def test_more_rows_than_positions_are_refused(dtype, heads, new):
    """max_new times the heads a key head: at most 2^30 (2^32 rows in tiles of 8 came out as four tiles, for 32 rows)."""
    need = _lib.load().qmv_kv_attend_workspace_bytes
    assert need(cache(), heads, 1, new, dtype, 1, 0) == 0
    assert attend(dtype=dtype, heads=heads, qs=64 * heads, new=new) == 4
    at_most = (1 << 30) // (heads // 2)
    assert need(cache(), heads, 1, at_most, dtype, 1, 0) > 0


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_scales_without_a_size_are_refused(scale):
    L = _lib.load()
    call = lambda s: L.qmv_kv_attend(cache(), A, 0, 256, 4, A, 1, A, A, 1, 0, 1, s, 0, A, A, 1 << 34, None)      # noqa: E731
    assert call(scale) == 2
    assert call(0.0) == call(-1e38) == 0             # (no rows: no launch)
