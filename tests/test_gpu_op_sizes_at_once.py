"""Calls of one kernel with different amounts of shared memory, from two threads at once (through the C ABI, whose calls do not hold Python's lock) and one after the other in one capture: a call's
launch does not depend on the sizes of another call."""
import ctypes as C
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


class Heads(C.Structure):
    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64), ("heads", C.c_int32), ("reserved", C.c_int32)]


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


def _distill(dev, vocab):
    """(call on a stream, what it writes) for rows of `vocab` whole 16-byte pieces: the same kernel whatever the vocabulary."""
    from goneuron_b200 import _lib
    L, gen = _lib.load(), torch.Generator("cuda").manual_seed(vocab)
    logits = torch.randn(75, vocab, device="cuda", generator=gen).half()
    ids, top = torch.randint(0, vocab, (75, 8), device="cuda", generator=gen), torch.randn(75, 8, device="cuda", generator=gen)
    loss, grad = torch.zeros(75, device="cuda"), torch.zeros_like(logits)
    keep = (logits, ids, top)
    return lambda stream: L.gn_op_distill(dev.handle, 1, 75, vocab, 8, 1.5, keep[0].data_ptr(), vocab, keep[1].data_ptr(), 1, keep[2].data_ptr(), None, loss.data_ptr(), grad.data_ptr(), vocab, stream), (loss, grad)


def _qk(dev, size):
    """The gradient for heads of an odd size, element by element: shared memory for a row of every warp."""
    from goneuron_b200 import _lib
    L, gen = _lib.load(), torch.Generator("cuda").manual_seed(size)
    x, dy = (torch.randn(64, 3, size, device="cuda", generator=gen) for _ in range(2))
    dx = torch.zeros_like(x)
    hx, hdy, hdx = (Heads(t.data_ptr(), 3 * size, size, 3, 0) for t in (x, dy, dx))
    keep = (x, dy)
    return lambda stream: keep and L.gn_op_qk_norm_rope_backward(dev.handle, 0, 64, size, 0, 0, 1e-5, C.addressof(hx), None, None, None, None, 0, None, C.addressof(hdy), None, C.addressof(hdx), None, None, None, None, 0,
                                                                 stream), (dx,)


@pytest.mark.parametrize("make,sizes", [(_distill, (100000, 32768)), (_qk, (1023, 701))])
def test_two_threads(dev, make, sizes):
    calls = [make(dev, n) for n in sizes]
    torch.cuda.synchronize()
    want = []
    for call, out in calls:
        assert call(torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        want.append([t.clone() for t in out])
    refused, start = [0, 0], threading.Barrier(2)

    def work(i):
        s = torch.cuda.Stream()
        start.wait()
        for _ in range(20000):
            refused[i] += calls[i][0](s.cuda_stream) != 0
        s.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert refused == [0, 0]
    for (_, out), w in zip(calls, want):
        assert all(torch.equal(a, b) for a, b in zip(out, w))


@pytest.mark.parametrize("make,sizes", [(_distill, (100000, 32768)), (_qk, (1023, 701))])
def test_a_large_call_captured_before_a_small_one(dev, make, sizes):
    calls = [make(dev, n) for n in sizes]
    torch.cuda.synchronize()
    want = []
    for call, out in calls:
        assert call(torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        want.append([t.clone() for t in out])
    for _, out in calls:
        for t in out:
            t.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert [call(torch.cuda.current_stream().cuda_stream) for call, _ in calls] == [0, 0]
    graph.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(calls, want):
        assert all(torch.equal(a, b) for a, b in zip(out, w))
