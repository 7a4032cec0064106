"""Outputs of queries and keys given the other way round, both the same, and distillation's gradient a little beside the logits are refused; views of one projection in place are written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


def test_queries_and_keys(dev):
    from goneuron_b200 import _lib, operators as ops
    gen = torch.Generator("cuda").manual_seed(1)
    q, k = (torch.randn(5000, 4, 64, device="cuda", generator=gen) for _ in range(2))
    want = ops.qk_norm_rope(dev, q, k)
    new = torch.empty_like(q)
    before = q.clone(), k.clone()
    for out in ((k, q), (k, new), (new, q), (new, new)):
        with pytest.raises(_lib.GoNeuronCudaError):
            ops.qk_norm_rope(dev, q, k, out=out)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    both = torch.stack((q, k), 2)                      # heads of queries and keys in turn
    ops.qk_norm_rope(dev, both[:, :, 0], both[:, :, 1], out=(both[:, :, 0], both[:, :, 1]))
    assert torch.equal(both[:, :, 0], want[0]) and torch.equal(both[:, :, 1], want[1])
    side = torch.cat((q, k), 1)
    ops.qk_norm_rope(dev, side[:, :4], side[:, 4:], out=(side[:, :4], side[:, 4:]))
    assert torch.equal(side, torch.cat(want, 1))
    ops.check(dev)


def test_distillation(dev):
    from goneuron_b200 import _lib, operators as ops
    wide = torch.randn(30, 2100, device="cuda")
    ids, top = torch.arange(90, device="cuda").view(30, 3), torch.randn(30, 3, device="cuda")
    logits = wide[:, :1000]
    want = ops.distill_loss_grad(dev, logits, ids, top)
    for out in (wide[:, 2:1002], wide[:, 900:1900]):
        with pytest.raises(_lib.GoNeuronCudaError):
            ops.distill_loss_grad(dev, logits, ids, top, out=out)
    with pytest.raises(_lib.GoNeuronCudaError):
        ops.distill_loss_grad(dev, logits[1:], ids[1:], top[1:], out=logits[:-1])
    got = ops.distill_loss_grad(dev, logits, ids, top, out=wide[:, 1000:2000])
    assert all(torch.equal(x, y) for x, y in zip(got, want))
