"""The 8-bit checkpoint operators called from several threads at once."""
import threading
import time

import pytest
import torch

from sandmuon_b200 import _lib, activations
from test_gpu_activations import activation, cotangent

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_threads_with_streams_of_their_own():
    """Each thread's results are what one thread alone gets."""
    sizes = [(3000, 264, 520), (1000, 136, 260), (257, 1000, 96), (4100, 96, 64)]

    def passes(k, n):
        rows, d_in, d_out = sizes[k]
        x, d = activation(rows, d_in, torch.bfloat16, seed=k), cotangent(rows, d_out, torch.bfloat16, seed=k)
        w = torch.ones(d_out, d_in, device=DEV).mul_(.01).requires_grad_()
        e = cotangent(rows, d_in, torch.bfloat16, seed=k + 9)
        for _ in range(n):
            leaf = x.clone().requires_grad_()
            y, py = activations.gelu(leaf, pack_output=True, stats=True)
            dx, dw = torch.autograd.grad([y, activations.linear(leaf, w)], [leaf, w], [e, d])
            last = [dx, dw, py.sums, activations.unpack(py), activations.weight_gradient(d, py)]
        torch.cuda.current_stream().synchronize()
        return last

    want = [passes(k, 1) for k in range(len(sizes))]
    got, errors = [None] * len(sizes), []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[k] = passes(k, 30)
        except BaseException as e:  # noqa: BLE001 -- reported by the test's own thread
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for g, w in zip(a, b):
            assert torch.equal(g, w)
    assert _lib.device_status(DEV) == 0


def test_a_call_that_waits_for_the_launch_queue_holds_no_python_lock():
    """Behind half a second of GPU time the launch queue fills up and a call
    waits in its launch; other threads run meanwhile."""
    x = activation(64, 128, torch.float32)
    activations.pack(x)
    torch.cuda.synchronize()
    stop, gaps = threading.Event(), []

    def tick():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gaps.append(now - last)
            last = now

    thread = threading.Thread(target=tick)
    thread.start()
    longest = 0.0
    try:
        torch.cuda._sleep(1_000_000_000)
        for _ in range(20000):
            t = time.perf_counter()
            activations.pack(x)
            longest = max(longest, time.perf_counter() - t)
            if longest > 0.1:
                break
    finally:
        stop.set()
        thread.join()
        torch.cuda.synchronize()
    assert longest > 0.1, "the launch queue never filled up"
    assert max(gaps) < 0.8 * longest
