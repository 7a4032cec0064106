"""gn_op_distill against float64: vocabularies around every change of plan, entries that are missing, repeated or without probability, rows without weight, values that are not
finite, odd strides, in place, captured; the gradient also against differences of the loss."""
import math

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


def _want(logits, ids, top, tau, weight):
    z = logits.double() / tau
    there = (ids >= 0) & (ids < logits.shape[1])
    t = torch.where(there, top.double() / tau, -math.inf)
    some = (t > -math.inf).any(1) | torch.isnan(t).any(1)
    on = some & (weight != 0)
    p = torch.softmax(torch.where(some[:, None], t, 0.0), 1) * some[:, None]
    log_q = torch.log_softmax(z, 1)
    at = ids.clamp(0, logits.shape[1] - 1).long()
    term = torch.where(p > 0, p * (torch.log(p) - log_q.gather(1, at)), torch.where(torch.isnan(p), p, 0.0))
    loss = torch.where(on, weight.double() * tau * tau * term.sum(1), 0.0)
    d = torch.exp(log_q).scatter_add(1, at, -torch.where(there, p, 0.0)) * (tau * weight.double())[:, None]
    return loss, torch.where(on[:, None], d, 0.0)


def _check(dev, logits, ids, top, tau=1.0, weight=None, out=None):
    from goneuron_b200 import operators as ops
    w = torch.ones(logits.shape[0], device="cuda") if weight is None else weight
    loss_want, d_want = _want(logits, ids, top, tau, w)
    alone = ops.distill_loss(dev, logits, ids, top, tau, weight)
    loss, d = ops.distill_loss_grad(dev, logits, ids, top, tau, weight, out=out)
    # float32 with exponents rounded to 2^-24 of their size: |s - lse| and |t - lse| below 100 here, so 1e-5 of a probability, 2e-5 tau^2 in the loss
    size = (w.abs() * tau * tau).double()
    for x in (loss, alone):
        assert_near(x, loss_want, 2e-5 * size + 1e-6 * loss_want.abs().nan_to_num(0, 0, 0), "loss")
    p_size = (torch.softmax(logits.double() / tau, 1).nan_to_num(0) + 0.0)
    hit = torch.zeros_like(p_size).scatter_add(1, ids.clamp(0, logits.shape[1] - 1).long(), (ids >= 0).double())
    assert_near(d, d_want, 1e-5 * (w.abs() * tau).double()[:, None] * (p_size + hit) + 1e-37, "dlogits")
    return loss, d


def _case(rows, vocab, top, type, seed, spread=2.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    logits = torch.randn(rows, vocab, device="cuda", generator=gen).mul(spread).to(TYPES[type])
    ids = torch.randint(0, vocab, (rows, top), device="cuda", generator=gen)
    return logits, ids, torch.randn(rows, top, device="cuda", generator=gen) * 3, gen


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (1, 32000, 64), (700, 500, 16), (9, 2032, 8), (9, 2033, 8), (300, 8176, 8), (300, 8177, 8), (150, 16369, 33), (200, 32751, 64),
                                            (160, 32753, 64), (20, 65505, 100), (150, 70001, 20), (40, 131072, 1024), (3, 262016, 5), (2, 262500, 300), (30, 8192, 0), (2, 300007, 17), (500, 53241, 9), (500, 53257, 9), (200, 90113, 9), (2, 720881, 3), (2, 720897, 3), (2, 730000, 1024)])
def test_against_float64(dev, type, rows, vocab, top):
    logits, ids, t, gen = _case(rows, vocab, top, type, rows + vocab)
    weight = torch.rand(rows, device="cuda", generator=gen) + 0.1
    _check(dev, logits, ids, t, 1.0, weight)
    if rows < 40:
        _check(dev, logits, ids.int(), t, 2.5)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [106485, 106496, 106501, 128000, 180225, 212981, 212993, 250000, 360449])
def test_rows_over_four_and_eight_blocks(dev, type, vocab):
    """More rows than fill the multiprocessors at once, lengths on either side of those at which a row is cut into more parts."""
    logits, ids, t, gen = _case(60, vocab, 70, type, vocab)
    ids[:, 5] = ids[:, 4]                                # the same index twice
    weight = torch.rand(60, device="cuda", generator=gen) + 0.1
    weight[3] = 0
    _check(dev, logits, ids, t, 2.0, weight)
    _check(dev, logits.clone(), ids, t, 2.0, weight, out=torch.empty(60, vocab + 3, device="cuda", dtype=logits.dtype)[:, 1:vocab + 1])


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [777, 40000, 270000])
def test_entries_and_rows_that_say_nothing(dev, type, vocab):
    from goneuron_b200 import operators as ops
    logits, ids, t, gen = _case(12, vocab, 40, type, vocab)
    ids[0, 5:] = -1                                    # few entries
    ids[1] = -1                                        # none
    t[2] = -math.inf                                   # none with probability
    t[3, 1:] = -math.inf                               # a single one
    ids[4] = 17                                        # one index forty times
    ids[5, 10:20] = ids[5, :10]                        # some twice
    weight = torch.rand(12, device="cuda", generator=gen) + 0.1
    weight[6] = 0
    logits[6] = float("nan")                           # a row of padding may hold anything
    logits[7, 100:] = -math.inf                        # a masked vocabulary
    ids[7] %= 100
    logits[8, ids[8, 0]] = -math.inf                   # the teacher wants what the student masks: an infinite loss
    logits[9] = torch.finfo(logits.dtype).min          # the lowest value of the type everywhere
    logits[9, :2] = 0
    t[9] = -math.inf
    t[9, 0], ids[9, 0] = 0.0, 1
    t[10] = torch.finfo(torch.float32).min             # the teacher's lowest value everywhere: equal entries
    loss, d = _check(dev, logits, ids, t, 1.5, weight)
    ops.check(dev)
    assert loss[1] == 0 and loss[2] == 0 and loss[6] == 0 and float(d[[1, 2, 6]].abs().sum()) == 0
    assert math.isinf(float(loss[8]))
    logits[3, 7] = float("nan")
    logits[4, 9] = float("inf")
    t[5, 3] = float("nan")
    loss, d = ops.distill_loss_grad(dev, logits, ids, t, 1.5, weight)
    assert torch.isnan(loss[[3, 4, 5]]).all() and torch.isnan(d[3]).all() and torch.isnan(d[4]).all()
    assert torch.isfinite(loss[[0, 1, 2, 6, 7, 9, 10, 11]]).all() and torch.isfinite(d[[0, 1, 2, 6, 7, 9, 10, 11]]).all()


def test_index_out_of_range_is_reported(dev):
    from goneuron_b200 import _lib, operators as ops
    logits, ids, t, _ = _case(5, 1000, 6, "f32", 1)
    ids[2, 3] = 1000
    ids[3, 0] = -7
    loss, d = ops.distill_loss_grad(dev, logits, ids, t)
    with pytest.raises(_lib.GoNeuronCudaError):
        ops.check(dev)
    ops.check(dev)                                     # reported once
    ids[2, 3] = ids[3, 0] = -1
    assert all(torch.equal(x, y) for x, y in zip((loss, d), ops.distill_loss_grad(dev, logits, ids, t)))


@pytest.mark.parametrize("type", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [501, 33001])
def test_strides_and_in_place(dev, type, vocab):
    """Rows that begin anywhere within 16 bytes, outputs that begin elsewhere; nothing around them is written; in place."""
    from goneuron_b200 import operators as ops
    _, ids, t, gen = _case(21, vocab, 30, type, 8)
    wide = torch.randn(21, vocab + 13, device="cuda", generator=gen).to(TYPES[type])
    logits = wide[:, 3:3 + vocab]
    out = torch.full((21, vocab + 6), 5.0, device="cuda").to(TYPES[type])
    loss, d = _check(dev, logits, ids, t, 2.0, None, out[:, 5:5 + vocab])
    assert (out[:, :5] == 5).all() and (out[:, 5 + vocab:] == 5).all()
    before = wide.clone()
    d = d.clone()
    loss2, d2 = ops.distill_loss_grad(dev, logits, ids, t, 2.0, out=logits)
    assert torch.equal(loss, loss2) and torch.equal(d, d2)
    assert torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, 3 + vocab:], before[:, 3 + vocab:])
    one = torch.randn(1, vocab, device="cuda", generator=gen).to(TYPES[type]).expand(21, vocab)      # the same row for all
    _check(dev, one, ids, t)


def test_gradient_against_differences(dev):
    from goneuron_b200 import operators as ops
    logits, ids, t, gen = _case(4, 50, 6, "f32", 3, 1.0)
    ids[1, 3:] = ids[1, 0]
    _, d = ops.distill_loss_grad(dev, logits, ids, t, 1.7)
    h = 2e-2                                           # error h^2 / 6 of the third derivative (below 1), and 2e-5 / 2h of the losses' own
    for e in range(50):
        step = torch.zeros_like(logits)
        step[:, e] = h
        diff = (ops.distill_loss(dev, logits + step, ids, t, 1.7).double() - ops.distill_loss(dev, logits - step, ids, t, 1.7).double()) / (2 * h)
        assert float((diff - d[:, e].double()).abs().max()) < 2e-3


def test_streams_and_graphs(dev):
    from goneuron_b200 import operators as ops
    logits, ids, t, gen = _case(333, 40000, 24, "bf16", 6)
    want = ops.distill_loss_grad(dev, logits, ids, t, 2.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.distill_loss_grad(dev, logits, ids, t, 2.0)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = ops.distill_loss_grad(dev, logits, ids, t, 2.0)
    logits.copy_(logits.flip(0))
    g.replay()
    again = ops.distill_loss_grad(dev, logits, ids, t, 2.0)
    assert all(torch.equal(x, y) for x, y in zip(held, again)) and not torch.equal(held[0], want[0])


def test_no_rows(dev):
    from goneuron_b200 import operators as ops
    loss, d = ops.distill_loss_grad(dev, torch.empty(0, 100, device="cuda"), torch.empty(0, 3, device="cuda", dtype=torch.int64), torch.empty(0, 3, device="cuda"))
    assert loss.shape == (0,) and d.shape == (0, 100)
