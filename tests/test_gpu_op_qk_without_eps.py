"""Norm of queries and keys with eps = 0: numbers of tokens and heads that leave lanes without a row, every way in which rows are read, against float64."""
import pytest
import torch

from tests.operator_checks import TYPES, assert_near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,size", [(1, 1, 64), (3, 5, 64), (301, 3, 128), (7, 1, 80), (50, 3, 4), (5, 1, 512), (2, 3, 66), (1500, 7, 32)])
def test_gradients(dev, type, tokens, heads, size):
    from goneuron_b200 import operators as ops
    gen = torch.Generator("cuda").manual_seed(tokens + size)
    x, dy = (torch.randn(tokens, heads, size, device="cuda", generator=gen).to(TYPES[type]) for _ in range(2))
    gain = 1 + 0.2 * torch.randn(size, device="cuda", generator=gen)
    dx, _, dgain, _ = ops.qk_norm_rope_backward(dev, dy, None, x, None, gain, eps=0.0)
    X, G = x.double().requires_grad_(), gain.double().requires_grad_()
    r = X / torch.sqrt(X.square().mean(-1, keepdim=True))
    want_x, want_g = torch.autograd.grad(r * G, (X, G), dy.double())
    # float32: sums of `size` products (4 to 1024 additions, most of them side by side), the root 2^-22, a few products; relative to the sums of sizes
    slack = 2.0 ** -24 * (size + 32)
    rs = 1 / torch.sqrt(X.detach().square().mean(-1, keepdim=True))
    gdy = dy.double().abs() * gain.double().abs()
    xn = X.detach().abs() * rs
    assert_near(dx, want_x, slack * rs * (gdy + xn * (gdy * xn).mean(-1, keepdim=True)), "dx")
    # a column of the gain: the products above, then a sum of tokens * heads of them
    assert_near(dgain, want_g, 2.0 ** -24 * (size + 32 + tokens * heads) * (dy.double().abs() * xn).sum((0, 1)), "dgain")
