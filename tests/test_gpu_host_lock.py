"""The small calls leave the interpreter's lock to other threads while they allocate and launch."""
import threading
import time

import pytest
import torch

from nemicli_terminal_b200 import beams, kvcache, mmvq, pages

pytestmark = pytest.mark.gpu
I32 = torch.int32


def calls(cuda):
    c = kvcache.KVCache(8, 1, 64, 16, "Q4_0", "Q4_0", cuda)
    slots = torch.arange(4, device=cuda)
    k = torch.zeros(4, 1, 64, device=cuda)
    free, counts = pages.pool(8, cuda)
    tables, lens, none = torch.arange(4, dtype=I32, device=cuda).view(2, 2), torch.zeros(2, dtype=I32, device=cuda), torch.zeros(2, dtype=torch.bool, device=cuda)
    at = torch.full((2,), -1, dtype=I32, device=cuda)
    box, q = c.bounds(), torch.zeros(2, 2, 64, device=cuda)
    held = torch.ones(2, dtype=I32, device=cuda)
    chosen = torch.zeros(2, 1, 1, dtype=I32, device=cuda)
    logits, scores = torch.zeros(1, 2, 64, device=cuda), torch.zeros(1, 2, device=cuda)
    return {"write": lambda: c.write(k, k, slots), "read": lambda: c.read(slots), "copy": lambda: c.copy(at, at),
            "summarise": lambda: c.summarise(box, tables, held), "choose": lambda: c.choose(q, box, tables, held, 3),
            "attend_chosen": lambda: c.attend_chosen(q, chosen, held), "plan": lambda: pages.plan(lens, lens, tables, free, counts, 16, 2),
            "release": lambda: pages.release(none, lens, tables, free, counts, 16),
            "reorder": lambda: pages.reorder(at.view(1, 2), lens, tables, free, counts, 16), "select": lambda: beams.select(logits, scores)}


@pytest.mark.parametrize("name", ["write", "read", "copy", "summarise", "choose", "attend_chosen", "plan", "release", "reorder", "select"])
def test_other_threads_run_while_a_launch_waits(cuda, name):
    """Behind a kernel of some tenths of a second the stream's queue fills up and a launch waits for room in it."""
    call = calls(cuda)[name]
    call()
    torch.cuda.synchronize()
    gaps, stop = [0.0], threading.Event()

    def tick():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gaps[0] = max(gaps[0], now - last)
            last = now

    other = threading.Thread(target=tick)
    other.start()
    try:
        torch.cuda._sleep(1_000_000_000)                          # about half a second
        longest = 0.0
        for _ in range(2500):
            begin = time.perf_counter()
            call()
            longest = max(longest, time.perf_counter() - begin)
    finally:
        stop.set()
        other.join()
        torch.cuda.synchronize()
    if longest < 0.1:
        pytest.skip("no launch had to wait")
    assert gaps[0] < longest / 2


@pytest.mark.parametrize("pdl", [False, True])
def test_two_threads_on_one_stream(cuda, pdl):
    """Calls of two launches each from two threads, whose launches fall between one another's."""
    g = torch.Generator(device=cuda).manual_seed(4)
    x = [torch.randn(4, 6, 20003, generator=g, device=cuda) for _ in range(2)]
    s = torch.zeros(4, 6, device=cuda)
    want = [beams.select(a, s, 12) for a in x]
    got, start = [[], []], threading.Barrier(2)

    def work(i):
        start.wait()
        got[i] += [beams.select(x[i], s, 12) for _ in range(60)]

    mmvq.pdl(pdl)
    try:
        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
    finally:
        mmvq.pdl(False)
    assert [len(o) for o in got] == [60, 60]
    assert all(torch.equal(p, q) for i in range(2) for o in got[i] for p, q in zip(o, want[i]))
