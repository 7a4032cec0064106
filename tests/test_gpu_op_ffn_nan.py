"""A gate that is not a number, with a projection beside it that is: no activation hides it."""
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


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("tokens", [1, 8, 16, 300])
def test_nan_gates(dev, type, act, tokens):
    from goneuron_b200 import operators as ops
    gen = torch.Generator("cuda").manual_seed(tokens)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).mul(0.2).to(TYPES[type])
    x, wg, wu, wd, dy = r(tokens, 64), r(136, 64), r(136, 64), r(64, 136), r(tokens, 64)
    wg[3, 5] = float("nan")
    y, saved = ops.gated_ffn(dev, x, wg, wu, wd, act, save=True)
    dx, dwg, dwu, dwd = ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved, act)
    ops.check(dev)
    # h[:, 3] is not a number, nor is what it or its gradient is a factor of; nothing else is touched
    for t in (y, ops.gated_ffn(dev, x, wg, wu, wd, act), dx, dwd[:, 3], dwu[3]):
        assert torch.isnan(t).all()
    others = [i for i in range(136) if i != 3]
    assert torch.isfinite(dwd[:, others]).all() and torch.isfinite(dwu[others]).all() and torch.isfinite(dwg[others]).all()
