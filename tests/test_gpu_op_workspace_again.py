"""One workspace for call after call, without waiting in between: what a launch reads there is what the launch before it wrote, not what an earlier call left."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


@pytest.mark.parametrize("tokens,vocab", [(9000, 70000), (9000, 300), (40000, 70000), (300000, 70000), (3000, 70000)])
def test_embedding_gradients_one_after_the_other(dev, tokens, vocab):
    """Passes over digits of 8 bits with few tiles and with many, and places counted directly; whole numbers, so that every sum is exact."""
    from goneuron_b200 import _lib
    L, gen = _lib.load(), torch.Generator("cuda").manual_seed(tokens)
    n = C.c_int64()
    _lib.check(L.gn_op_embedding_workspace(dev.handle, tokens, vocab, 4, C.byref(n)))
    ws, stream = torch.empty(n.value, dtype=torch.uint8, device="cuda"), torch.cuda.current_stream().cuda_stream
    ids = [torch.randint(-1, vocab, (tokens,), device="cuda", generator=gen) for _ in range(4)] + [torch.randint(0, 3, (tokens,), device="cuda", generator=gen)]
    dout = [torch.randint(-8, 9, (tokens, 4), device="cuda", generator=gen).float() for _ in ids]
    got = [torch.empty(vocab, 4, device="cuda") for _ in range(20)]
    for k, d in enumerate(got):
        i = k % len(ids)
        _lib.check(L.gn_op_embedding_backward(dev.handle, 0, tokens, vocab, 4, 1.0, dout[i].data_ptr(), 4, ids[i].data_ptr(), 1, d.data_ptr(), ws.data_ptr(), n.value, stream))
    for k, d in enumerate(got):
        i = k % len(ids)
        there = ids[i] >= 0
        assert torch.equal(d, torch.zeros(vocab, 4, device="cuda", dtype=torch.float64).index_add_(0, ids[i][there], dout[i][there].double()).float()), k


def test_gain_gradients_one_after_the_other(dev):
    """Partial sums of the blocks; rows of ones and powers of two, so that every sum is exact."""
    from goneuron_b200 import _lib
    from tests.test_gpu_op_sizes_at_once import Heads
    L, heads, size, tokens = _lib.load(), 4, 64, 3000
    n = C.c_int64()
    _lib.check(L.gn_op_qk_norm_rope_workspace(dev.handle, tokens, heads, 0, size, C.byref(n)))
    ws, stream = torch.empty(n.value, dtype=torch.uint8, device="cuda"), torch.cuda.current_stream().cuda_stream
    x, dx = torch.ones(tokens, heads, size, device="cuda"), torch.empty(tokens, heads, size, device="cuda")
    scales = [2.0 ** (k % 5) for k in range(30)]
    dy, gains = [torch.full_like(x, 2.0 ** k) for k in range(5)], torch.empty(30, size, device="cuda")
    h = lambda t: Heads(t.data_ptr(), heads * size, size, heads, 0)
    hx, hdx, hdy = h(x), h(dx), [h(t) for t in dy]
    for k in range(30):
        _lib.check(L.gn_op_qk_norm_rope_backward(dev.handle, 0, tokens, size, 0, 0, 0.0, C.addressof(hx), None, None, None, None, 0, None, C.addressof(hdy[k % 5]), None, C.addressof(hdx), None, gains[k].data_ptr(), None,
                                                 ws.data_ptr(), n.value, stream))
    want = torch.tensor(scales, device="cuda")[:, None] * (tokens * heads)
    # 1 / sqrt(1) by rsqrtf, 2 steps of float32 off at most; the sums of equal numbers below 2^24 of them are exact but for that factor's rounding, 2^-24 for each of fewer than 64 additions one after the other
    assert ((gains - want).abs() <= want * (2 * 2.0 ** -23 + 64 * 2.0 ** -24)).all()
