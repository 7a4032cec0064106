"""A tensor given as `out` that requires a gradient is refused before anything is launched; without gradients it is not refused for that."""
import pytest
import torch


class _NoDevice:
    """Stands in for a Device where a call must not get as far as the library."""
    device, handle = 0, None


def test_out_that_requires_a_gradient():
    from goneuron_b200 import operators as ops
    dev, ids, top = _NoDevice(), torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    logits = torch.zeros(4, 10, requires_grad=True)
    for out in (logits, logits * 2):
        call = lambda: ops.distill_loss_grad(dev, logits, ids, top, out=out)      # noqa: B023
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="runs on cuda:0"):
            call()
