"""Tensors given as `out` and autograd: one that a backward pass has kept, one that requires a gradient, a parameter without gradients, views, inference mode."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


def _distill(dev, out_of):
    """Writes over out_of [5, 40] as the gradient of a loss."""
    from goneuron_b200 import operators as ops
    ids, top = torch.arange(15, device="cuda").view(5, 3), torch.randn(5, 3, device="cuda")
    return ops.distill_loss_grad(dev, out_of, ids, top, out=out_of)[1]


def _qk(dev, out_of):
    from goneuron_b200 import operators as ops
    x = out_of.view(5, 5, 8)
    return ops.qk_norm_rope(dev, x, None, out=(x, None))[0]


def _k(dev, out_of):
    from goneuron_b200 import operators as ops
    x = out_of.view(5, 5, 8)
    return ops.qk_norm_rope(dev, torch.randn_like(x), x, out=(torch.empty_like(x), x))[1]


@pytest.mark.parametrize("write", [_distill, _qk, _k])
def test_what_a_backward_pass_has_kept(dev, write):
    """exp keeps its result for its gradient."""
    w = torch.randn(5, 40, device="cuda", requires_grad=True)
    y = torch.exp(w)
    kept = y.detach()                                  # the same memory and version
    before = y._version
    write(dev, kept)
    assert y._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("write", [_distill, _qk, _k])
def test_what_requires_a_gradient(dev, write):
    w = torch.randn(5, 40, device="cuda", requires_grad=True)
    for t in (w, w * 2):
        before, version = t.detach().clone(), t._version
        with pytest.raises(ValueError, match="requires a gradient"):
            write(dev, t)
        assert torch.equal(t, before) and t._version == version
    with torch.no_grad():
        version = w._version
        write(dev, w)
        assert w._version > version


def test_inference_mode(dev):
    with torch.inference_mode():
        x = torch.randn(5, 40, device="cuda")
        _distill(dev, x)
        _qk(dev, x)
    with pytest.raises(ValueError, match="inference"):
        _qk(dev, x)


def test_other_outputs_are_the_calls_own(dev):
    """Inputs that require gradients are read, their versions stay, outputs have no history."""
    from goneuron_b200 import operators as ops
    q = torch.randn(5, 5, 8, device="cuda", requires_grad=True)
    y = ops.qk_norm_rope(dev, q, None)[0]
    assert not y.requires_grad and q._version == 0
