"""What a fault met in device memory reaches: every call that waits and hands out results tells it, once, to the host thread
whose call it was."""
import ctypes
import threading
import time
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

V = 5000


@pytest.fixture(scope="module")
def gv():
    import geode_amd

    geode_amd.init(0)
    return geode_amd


class BadRules:
    """queues a gv_process_logits call one of whose rows names a mask that is not there"""

    def __init__(self, gv):
        self.gv = gv
        self.bufs = [gv.DeviceBuffer.from_array(a) for a in (
            np.zeros((2, V), np.float32), np.full((1, (V + 31) // 32), 0xFFFFFFFF, np.uint32), np.array([0, 1], np.int32))]
        self.out = gv.DeviceBuffer(2 * V * 4)
        x, masks, of = self.bufs
        self.rules = gv.GvLogitsRules(masks=masks.ptr, n_masks=1, ld_mask=(V + 31) // 32, mask_of=of.ptr)
        gv.check(gv.lib.gv_synchronize(), "gv_synchronize")

    def queue(self):
        self.gv.check(self.gv.lib.gv_process_logits(ctypes.byref(self.rules), self.bufs[0].ptr, self.gv.F32, V, 2, V,
                                                    self.out.ptr, V), "gv_process_logits")


def _waiting_calls(gv):
    """(name, a call that waits for results of device memory that is in order)"""
    r = np.random.default_rng(80)
    rows = gv.DeviceBuffer.from_array((r.standard_normal((9, V)) * 3).astype(np.float32))
    batch, out, kept = np.array([7, 8, 9, 10], np.int32), np.zeros(64, np.int32), ctypes.c_int(0)
    u, uf, seen, stop = np.full(9, 0.5), np.full(9, 0.5, np.float32), np.array([3, 4], np.int32), np.arange(40, dtype=np.int32)
    host = np.zeros(4, np.float32)
    p = lambda a: a.ctypes.data   # noqa: E731
    keep = (rows, batch, out, kept, u, uf, seen, stop, host)

    def match(T, top_k, penalty=0.0, n_stop=0):
        return lambda: gv.lib.gv_accept_match_ex(rows.ptr, V, V, p(batch), 4, T, 0.9, top_k, 0, p(u), p(seen), 2, penalty,
                                                 p(stop), n_stop, p(out), ctypes.byref(kept))

    def textbook(T, top_p, greedy):
        return lambda: gv.lib.gv_accept_textbook(rows.ptr, rows.ptr + 5 * V * 4, V, V, 4, T, top_p, greedy, p(uf), p(uf), 0.5,
                                                 p(out))

    calls = {
        "memcpy_d2h": lambda: gv.lib.gv_memcpy_d2h(p(host), rows.ptr, 16),
        "sample greedy": lambda: gv.lib.gv_sample_rows(rows.ptr, V, 4, V, 0.0, 1.0, 0, 0, p(u), p(out)),
        "sample": lambda: gv.lib.gv_sample_rows(rows.ptr, V, 4, V, 0.8, 0.9, 0, 0, p(u), p(out)),
        "match greedy": match(0.0, 0), "match candidates": match(0.8, 50), "match walks": match(0.8, 0),
        "match penalty": match(0.8, 50, 0.5), "match many stops": match(0.0, 0, 0.0, 40),
        "textbook greedy": textbook(0.8, 0.9, 1), "textbook candidates": textbook(0.8, 0.9, 0), "textbook walks": textbook(0.8, 1.0, 0),
    }
    return calls, keep


CALLS = ["memcpy_d2h", "sample greedy", "sample", "match greedy", "match candidates", "match walks", "match penalty",
         "match many stops", "textbook greedy", "textbook candidates", "textbook walks"]


@pytest.mark.parametrize("name", CALLS)
def test_calls_that_hand_out_results_tell_a_fault(gv, name):
    """a row made of rules that are not there is not turned into tokens or copied out with success; the call after it is
    as without the fault"""
    bad = BadRules(gv)
    calls, keep = _waiting_calls(gv)
    assert calls[name]() >= 0
    bad.queue()
    assert calls[name]() == -1
    assert "range, bias range or mask" in gv.lib.gv_last_error().decode()
    assert calls[name]() >= 0
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")   # (told once)
    bad.queue()
    assert gv.lib.gv_synchronize() == -1
    assert calls[name]() >= 0
    del keep


def test_a_fault_is_told_to_the_thread_whose_call_it_was(gv):
    """two host threads on the one stream: the thread whose calls are in order waits and gets its results, before and after
    the other learns of its own fault"""
    a, b = BadRules(gv), BadRules(gv)
    b.bufs[2].upload(np.array([0, -1], np.int32))   # (in order)
    sync = gv.lib.gv_synchronize
    with ThreadPoolExecutor(1) as one, ThreadPoolExecutor(1) as two:
        do = lambda t, f: t.submit(f).result()   # noqa: E731
        for _ in range(3):
            do(one, a.queue)
            do(two, b.queue)
            assert do(two, sync) == 0
            assert np.array_equal(do(two, lambda: b.out.download(np.float32, (2, V))), np.zeros((2, V), np.float32))
            assert do(one, sync) == -1
            assert do(one, sync) == 0 and do(two, sync) == 0 and sync() == 0


def test_the_fault_of_a_thread_that_has_ended(gv):
    """a thread that queued a call and ended without a wait: the next thread that waits is told, once; and many threads one
    after the other each learn of their own faults alone"""
    bad = BadRules(gv)
    t = threading.Thread(target=bad.queue)
    t.start()
    t.join()
    told = []
    for _ in range(200):   # (the thread's own end comes a little after its join)
        told.append(gv.lib.gv_synchronize())
        if told[-1] != 0:
            break
        time.sleep(0.01)
    assert told[-1] == -1 and gv.lib.gv_synchronize() == 0
    good = BadRules(gv)
    good.bufs[2].upload(np.array([0, -1], np.int32))
    said = []

    def work(i):
        (bad if i % 3 == 0 else good).queue()
        said.append((gv.lib.gv_synchronize(), gv.lib.gv_synchronize()))

    for i in range(150):
        t = threading.Thread(target=work, args=(i,))
        t.start()
        t.join()
    assert said == [(-1 if i % 3 == 0 else 0, 0) for i in range(150)]
    assert gv.lib.gv_synchronize() == 0


@pytest.mark.parametrize("start", [
    [2, 1, 4], [0, 3, 2, 4],
    # (300 sequences, the row starts of two without rows exchanged: no row of the batch lies in either)
    list(range(100)) + [100] * 150 + [101, 100] + [101 + i for i in range(49)]])
def test_row_starts_that_descend_are_told_whichever_rows_they_give(gv, start):
    """also where every row of the batch lies in a sequence that fits"""
    n, hd, page = len(start) - 1, 16, 16
    rows = max(start)
    cache = gv.PagedCache(gv.F16, n, page, 1, hd)
    good = np.minimum(np.arange(n + 1), rows)
    batch = gv.PagedBatch(np.diff(good), np.full(n, 16), np.arange(n)[:, None], n_rows=rows, max_rows=16)
    z = np.zeros((rows, 1, hd))
    gv.paged_append(cache, batch, z, z, z)
    gv.paged_attention(cache, batch, z)
    batch.bufs[0].upload(np.array(start, np.int32))
    with pytest.raises(gv.GeodeError, match="row starts"):
        gv.paged_append(cache, batch, z, z, z)
    with pytest.raises(gv.GeodeError, match="row starts"):
        gv.paged_attention(cache, batch, z)
    gv.check(gv.lib.gv_synchronize(), "gv_synchronize")
