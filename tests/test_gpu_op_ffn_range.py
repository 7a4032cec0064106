"""What float16 cannot hold between the products of the gated feed-forward block (h, dg, du): the row that it belongs to is not finite afterwards, as a loss scale's check wants it, and no other row is touched; in
bfloat16 the same numbers are finite and right."""
import pytest
import torch

from tests.operator_checks import TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


def _weights(type):
    """relu(x0) x0 in h[:, 7], all other h about 1; y, dx and the gradients of the weights are small sums of them."""
    gen = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).mul(0.125).to(TYPES[type])
    x, wg, wu, wd, dy = r(300, 64), r(136, 64), r(136, 64), r(64, 136), r(300, 64)
    wg[:, 0], wu[:, 0] = 0, 0
    wg[7], wu[7] = 0, 0
    wg[7, 0], wu[7, 0] = 1, 1
    return x, wg, wu, wd.abs() + 2.0 ** -6, dy


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("tokens", [5, 16, 300])
def test_forward(dev, type, tokens):
    from goneuron_b200 import operators as ops
    x, wg, wu, wd, _ = _weights(type)
    x = x[:tokens].clone()
    x[2, 0] = 300                                      # h: 90000, above 65504
    for y in (ops.gated_ffn(dev, x, wg, wu, wd, "relu"), ops.gated_ffn(dev, x, wg, wu, wd, "relu", save=True)[0]):
        rows = torch.isfinite(y).all(1)
        if type == "f16":
            assert not torch.isfinite(y[2]).any() and rows.sum() == tokens - 1
        else:                                          # 90000 wd and numbers about 1 beside it; h and y are rounded once each, the sum of the others is below 2^7
            want = 90000.0 * wd[:, 7].double()
            assert rows.all() and ((y[2].double() - want).abs() <= 2 ** -7 * want + 2 ** 7).all()


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_backward(dev, type):
    from goneuron_b200 import operators as ops
    x, wg, wu, wd, dy = _weights(type)
    x[:, 0] = 1
    x[2, 0] = 300
    wd[:, 7] = 1
    dy[2] = 8                                          # dh: 512, dg and du: 512 * 300 = 153600
    _, saved = ops.gated_ffn(dev, x, wg, wu, wd, "relu", save=True)
    dx, dwg, dwu, _ = ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved, "relu")
    rows = torch.isfinite(dx).all(1)
    if type == "f16":
        assert not rows[2] and rows.sum() == 299 and not torch.isfinite(dwg[7]).any() and not torch.isfinite(dwu[7]).any()
    else:
        assert rows.all() and torch.isfinite(dwg).all() and torch.isfinite(dwu).all()
        assert abs(float(dx[2, 0]) - 2 * 153600) <= 2 * 153600 * 2 ** -7 + 2 ** 10      # (the other columns of wg and wu are zero there)
    others = [i for i in range(136) if i != 7]
    assert torch.isfinite(dwg[others]).all() and torch.isfinite(dwu[others]).all()
