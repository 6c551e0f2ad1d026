"""clip_grads_(error_if_nonfinite=True) waits for the GPU: what other threads do meanwhile."""
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_other_threads_run_while_a_clip_waits(genre, dev):
    """behind half a second of products and more, a thread that wakes every millisecond does so; were it held up, it would wake once or twice"""
    ts = [torch.randn(1000, device=dev), torch.randn(33, device=dev)]
    want = [t.clone() for t in ts]
    genre.clip_grads_(want, 1.0)
    a, b = (torch.randn(8192, 8192, device=dev) for _ in range(2))
    out = a @ b
    torch.cuda.synchronize()
    woken, stop = [0], threading.Event()

    def wake():
        while not stop.is_set():
            woken[0] += 1
            time.sleep(1e-3)

    thread = threading.Thread(target=wake)
    thread.start()
    for _ in range(80):
        torch.mm(a, b, out=out)
    listed = list(ts)
    before, start = woken[0], time.perf_counter()
    norm = genre.clip_grads_(listed, 1.0, error_if_nonfinite=True)
    took, more = time.perf_counter() - start, woken[0] - before
    stop.set()
    thread.join()
    assert took > 0.1 and more >= 20, (took, more)
    assert norm.item() > 1 and all(torch.equal(t, w) for t, w in zip(ts, want))
