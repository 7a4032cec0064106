"""gn_op_qk_norm_rope and its gradient against float64, over head sizes, layouts, types, views and positions; in place, on another stream, captured."""
import pytest
import torch

from tests.operator_checks import TYPES, assert_near

pytestmark = pytest.mark.gpu

EPS = 1e-5


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


def _turned(x, positions, frequencies, interleaved, back=False):
    """Rotation of the first pairs of [tokens, heads, size] in float64."""
    if frequencies is None:
        return x
    r = 2 * frequencies.numel()
    a = positions.reshape(-1).double()[:, None] * frequencies * (-1 if back else 1)
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    y = x.clone()
    i, j = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    return y


def _one(x, gain, positions, frequencies, interleaved, dy=None):
    """Output, and with dy the gradients, in float64; also the sizes that the float32 arithmetic's errors are relative to."""
    x = x.double()
    g = torch.ones(x.shape[-1], device=x.device, dtype=torch.float64) if gain is None else gain.double()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    y = _turned(x * r * g, positions, frequencies, interleaved)
    out = {"y": y, "y_size": y.abs().amax(-1, keepdim=True)}
    if dy is not None:
        u = _turned(dy.double(), positions, frequencies, interleaved, back=True)
        gu = g * u
        out["dx"] = r * (gu - x * r * r * (gu * x).mean(-1, keepdim=True))
        out["dx_size"] = r * (gu.abs().amax(-1, keepdim=True) + x.abs().amax(-1, keepdim=True) * r * r * (gu * x).abs().mean(-1, keepdim=True))
        out["dgain"] = (u * x * r).sum((0, 1))
        out["dgain_size"] = (u * x * r).abs().sum((0, 1))
    return out


def _check(dev, q, k, gq, gk, pos, freq, interleaved):
    from goneuron_b200 import operators as ops
    gen = torch.Generator("cuda").manual_seed(3)
    dqo = torch.randn(q.shape, device="cuda", generator=gen).to(q.dtype)
    dko = None if k is None else torch.randn(k.shape, device="cuda", generator=gen).to(q.dtype)
    q0, k0 = q.clone(), None if k is None else k.clone()
    qo, ko = ops.qk_norm_rope(dev, q, k, gq, gk, pos, freq, eps=EPS, interleaved=interleaved)
    dq, dk, dgq, dgk = ops.qk_norm_rope_backward(dev, dqo, dko, q, k, gq, gk, pos, freq, eps=EPS, interleaved=interleaved)
    ops.check(dev)
    for x, x0, g, o, d, dx, dg, n in ((q, q0, gq, qo, dqo, dq, dgq, "q"), (k, k0, gk, ko, dko, dk, dgk, "k")):
        if x is None:
            assert o is None and dx is None and dg is None
            continue
        assert torch.equal(x, x0)
        if x.numel() == 0:
            assert o.shape == x.shape and dx.shape == x.shape and float(dg.abs().sum()) == 0
            continue
        flat = lambda t: t.reshape(-1, t.shape[-2], t.shape[-1])
        want = _one(flat(x), g, pos, freq, interleaved, flat(d))
        # mean of squares: at most 32 + 5 additions in a row for the sizes here, half of it behind the root; two products, sine and cosine with 2 ulp and an angle rounded to
        # 2^-25 turns (1.9e-7): below 3e-6 of the row's largest element.  The gradient has two such sums.
        assert_near(flat(o), want["y"], 3e-6 * want["y_size"], n)
        assert_near(flat(dx), want["dx"], 8e-6 * want["dx_size"], "d" + n)
        if g is not None:
            assert_near(dg, want["dgain"], 1e-5 * want["dgain_size"] + 1e-30, "dgain_" + n)      # some 100 additions in a row, 2^-24 each
        else:
            assert dg is None


def _freq(rotated, base=10000.0):
    return base ** (-torch.arange(0, rotated, 2, device="cuda", dtype=torch.float64) / rotated) if rotated else None


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv,size,rotated,interleaved", [
    (1, 1, 1, 64, 64, False), (1, 16, 4, 64, 64, False), (5, 3, 3, 128, 128, False), (333, 6, 2, 80, 40, True), (257, 5, 1, 96, 96, False), (64, 2, 2, 256, 256, False),
    (2500, 4, 1, 64, 64, False), (1500, 4, 1, 64, 32, True), (40, 2, 1, 512, 512, False), (33, 2, 2, 1024, 512, False), (17, 3, 2, 65, 64, True), (17, 3, 2, 33, 6, False),
    (9, 1, 1, 2, 2, False), (9, 2, 1, 1, 0, False), (30, 2, 1, 64, 0, False), (12, 1, 1, 16, 16, True), (12, 2, 2, 8, 8, False), (31, 2, 1, 80, 16, False), (7, 1, 2, 128, 2, True)])
def test_against_float64(dev, type, tokens, heads, kv, size, rotated, interleaved):
    gen = torch.Generator("cuda").manual_seed(tokens + size)
    t = TYPES[type]
    q, k = (torch.randn(tokens, h, size, device="cuda", generator=gen).mul(2).to(t) for h in (heads, kv))
    gq, gk = (1 + 0.3 * torch.randn(size, device="cuda", generator=gen) for _ in range(2))
    pos = torch.randint(0, 4096, (tokens,), device="cuda", generator=gen)
    _check(dev, q, k, gq, gk, pos if rotated else None, _freq(rotated), interleaved)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv,size,rotated,interleaved,room", [
    (333, 6, 2, 80, 40, False, 0), (1, 6, 2, 80, 40, False, 0), (2100, 2, 1, 80, 40, False, 0), (100, 4, 3, 72, 24, False, 0), (50, 3, 2, 12, 8, False, 0), (50, 3, 2, 4, 4, True, 0), (40, 2, 1, 252, 248, False, 0),
    (40, 2, 1, 252, 250, True, 0), (60, 5, 2, 64, 64, False, 4), (60, 5, 2, 64, 64, True, 4), (60, 5, 2, 64, 64, False, 2), (60, 5, 2, 64, 48, False, 1), (1500, 3, 2, 66, 66, False, 0), (20, 1, 1, 1024, 1024, False, 1),
    (3, 40, 1, 260, 256, False, 4)])
def test_pieces_of_every_width(dev, type, tokens, heads, kv, size, rotated, interleaved, room):
    """Rows that fit pieces of 16 bytes, of 8 or none, by their size, by where the rotated part's halves end, or by the room between heads."""
    gen = torch.Generator("cuda").manual_seed(tokens + size + room)
    t = TYPES[type]
    q, k = (torch.randn(tokens, h, size + room, device="cuda", generator=gen).mul(2).to(t)[:, :, :size] for h in (heads, kv))
    gq, gk = (1 + 0.3 * torch.randn(size, device="cuda", generator=gen) for _ in range(2))
    pos = torch.randint(0, 4096, (tokens,), device="cuda", generator=gen)
    _check(dev, q, k, gq, gk, pos, _freq(rotated), interleaved)


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_views_batches_and_missing_parts(dev, type):
    """Views of a fused projection (aligned for 16-byte accesses and not), a batch, 32-bit positions, no gains, no keys, broadcast gradients."""
    gen = torch.Generator("cuda").manual_seed(9)
    t = TYPES[type]
    qkv = torch.randn(70, 3, 4, 64, device="cuda", generator=gen).to(t)
    pos = torch.randint(0, 1000, (70,), device="cuda", generator=gen, dtype=torch.int32)
    _check(dev, qkv[:, 0], qkv[:, 1], None, None, pos, _freq(64), False)
    odd = torch.randn(70, 8 * 65 + 1, device="cuda", generator=gen).to(t)[:, 1:].view(70, 8, 65)[..., :64]
    _check(dev, odd[:, :5], odd[:, 5:], None, torch.rand(64, device="cuda", generator=gen), pos, _freq(64), True)
    _check(dev, qkv[:, 0], None, torch.rand(64, device="cuda", generator=gen), None, pos, _freq(32), False)
    batch = qkv.view(7, 10, 3, 4, 64)[:, :, 0]
    _check(dev, batch, batch, None, None, pos.view(7, 10), _freq(64), False)
    _check(dev, torch.randn(1, 4, 64, device="cuda", generator=gen).to(t).expand(70, 4, 64), qkv[:, 1], None, None, pos, _freq(64), False)
    _check(dev, qkv[:, 0, :0], qkv[:, 1], torch.ones(64, device="cuda"), torch.ones(64, device="cuda"), pos, _freq(64), False)


def test_far_positions_and_extreme_rows(dev):
    """Angles of positions near 2^40 come out as in float64; rows of zeros, infinities and NaN stay in their rows."""
    from goneuron_b200 import operators as ops
    gen = torch.Generator("cuda").manual_seed(2)
    q = torch.randn(40, 2, 64, device="cuda", generator=gen)
    # 2^40 positions leave 2^-53 2^40 / (2 pi) turns of the float64 product unresolved, both here and there: 3e-4 of a turn would be lost in float32
    pos = torch.randint(1 << 39, 1 << 40, (40,), device="cuda", generator=gen)
    freq = 2.0 ** -torch.arange(32, device="cuda", dtype=torch.float64)      # products with positions are exact
    qo, _ = ops.qk_norm_rope(dev, q, None, None, None, pos, freq, eps=EPS)
    turns = (pos.double()[:, None] * freq / (2 * torch.pi)).frac()
    want = _one(q, None, torch.ones(1, device="cuda"), None, False)["y"]
    c, s = torch.cos(2 * torch.pi * turns)[:, None], torch.sin(2 * torch.pi * turns)[:, None]
    want = torch.cat((want[..., :32] * c - want[..., 32:] * s, want[..., :32] * s + want[..., 32:] * c), -1)
    # 2^40 / 2 pi turns, of which 2^-53 is lost by the product and as much by the rounding of 1 / (2 pi), here and there: below 8e-5 turns or 5e-4 radians between the
    # two, of a pair whose size is at most sqrt(2) of the largest element
    assert float((qo.double() - want).abs().max()) <= 7e-4 * float(want.abs().max())
    q[3] = 0
    q[5, 1, 7] = float("inf")
    q[6, 0, 9] = float("nan")
    p = torch.arange(40, device="cuda")
    qo, _ = ops.qk_norm_rope(dev, q, None, None, None, p, _freq(64), eps=EPS)
    assert torch.equal(qo[3], torch.zeros_like(qo[3]))
    bad = ~torch.isfinite(qo).all(-1)
    assert bad[5].tolist() == [False, True] and bad[6].tolist() == [True, False] and int(bad.sum()) == 2


@pytest.mark.parametrize("size", [64, 65])
def test_in_place_is_the_same(dev, size):
    from goneuron_b200 import operators as ops
    gen = torch.Generator("cuda").manual_seed(4)
    q, k = (torch.randn(300, h, size, device="cuda", generator=gen).bfloat16() for h in (4, 2))
    pos, freq = torch.arange(300, device="cuda"), _freq(64)
    a = ops.qk_norm_rope(dev, q, k, None, None, pos, freq)
    ops.qk_norm_rope(dev, q, k, None, None, pos, freq, out=(q, k))
    assert torch.equal(a[0], q) and torch.equal(a[1], k)


def test_streams_and_graphs(dev):
    """On a stream of its own, and captured forward and backward, replayed on new values; the same call twice gives the same bits."""
    from goneuron_b200 import operators as ops
    gen = torch.Generator("cuda").manual_seed(5)
    q, k, dqo, dko = (torch.randn(900, h, 64, device="cuda", generator=gen).half() for h in (8, 2, 8, 2))
    gq, gk = torch.rand(64, device="cuda", generator=gen), torch.rand(64, device="cuda", generator=gen)
    pos, freq = torch.arange(900, device="cuda"), _freq(64)
    both = lambda: (*ops.qk_norm_rope(dev, q, k, gq, gk, pos, freq), *ops.qk_norm_rope_backward(dev, dqo, dko, q, k, gq, gk, pos, freq))
    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = both()
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = both()
    q.copy_(q.flip(0)), dqo.copy_(dqo.flip(0))
    g.replay()
    again = both()
    assert all(torch.equal(x, y) for x, y in zip(held, again))
    assert not torch.equal(held[0], want[0])


def test_no_tokens(dev):
    from goneuron_b200 import operators as ops
    q, g = torch.empty(0, 4, 64, device="cuda"), torch.ones(64, device="cuda")
    pos = torch.empty(0, device="cuda", dtype=torch.int64)
    qo, ko = ops.qk_norm_rope(dev, q, q, g, g, pos, _freq(64))
    assert qo.shape == q.shape and ko.shape == q.shape
    dq, dk, dgq, dgk = ops.qk_norm_rope_backward(dev, q, q, q, q, g, g, pos, _freq(64))
    assert float(dgq.abs().sum()) == 0 and float(dgk.abs().sum()) == 0


def test_gains_anywhere_and_one_missing(dev):
    """Gains that begin 4 bytes after an 8-byte boundary; a gain for the keys alone."""
    gen = torch.Generator("cuda").manual_seed(6)
    q, k = (torch.randn(50, h, 64, device="cuda", generator=gen).bfloat16() for h in (3, 2))
    gains = torch.rand(130, device="cuda", generator=gen)
    pos = torch.arange(50, device="cuda")
    _check(dev, q, k, gains[1:65], gains[65:129], pos, _freq(64), False)
    _check(dev, q, k, None, gains[65:129], pos, _freq(64), True)


def test_in_place_with_other_strides_is_refused(dev):
    from goneuron_b200 import _lib, operators as ops
    wide = torch.randn(20, 8, 64, device="cuda")
    with pytest.raises(_lib.GoNeuronCudaError):
        ops.qk_norm_rope(dev, wide[:, :2], None, out=(wide.view(40, 4, 64)[:20, :2], None))
