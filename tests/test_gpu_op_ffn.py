"""gn_op_gated_ffn and its gradient against float64: token counts from one to several tiles, widths that end inside tiles, every cut of the contraction, views, special values, a wait that
gives up, another stream, captured."""
import pytest
import torch

from tests.operator_checks import TYPES, rounding

pytestmark = pytest.mark.gpu

ACT = {"silu": torch.nn.functional.silu, "relu": torch.relu, "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


def _case(m, d, f, type, seed, scale=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    t = TYPES[type]
    r = lambda *s, k=1.0: torch.randn(*s, device="cuda", generator=gen).mul(k).to(t)
    return r(m, d, k=scale), r(f, d, k=d ** -0.5), r(f, d, k=d ** -0.5), r(d, f, k=f ** -0.5), r(m, d)


def _accumulated(indices):
    """Error of float32 accumulation of that many products relative to the sum of their sizes: the tensor core adds 16 at a time and truncates (2^-23 each), slices' sums and what is done with the
    result in float32 are below 64 more."""
    return 2.0 ** -23 * (indices / 16 + 64)


def _near(got, want, error, what):
    """got against want (float64), element by element, within `error` and one rounding to got's type."""
    rel, small = rounding(got.dtype)
    bound = error + rel * (want.abs() + error) + small
    over = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all() and float(over.max()) <= 0, f"{what}: {float((got.double() - want).abs().max()):.3g} off, {float(over.max()):.3g} over the bound"


def _check(dev, x, wg, wu, wd, dy, act):
    from goneuron_b200 import operators as ops
    m, d = x.reshape(-1, x.shape[-1]).shape
    f = wg.shape[0]
    y0 = ops.gated_ffn(dev, x, wg, wu, wd, act)
    y, saved = ops.gated_ffn(dev, x, wg, wu, wd, act, save=True)
    grads = ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved, act)
    ops.check(dev)
    X, G, U, D, DY = (v.double().reshape(-1, v.shape[-1]) for v in (x, wg, wu, wd, dy))
    g, u = (X @ G.T).requires_grad_(), (X @ U.T).requires_grad_()
    h = ACT[act](g) * u
    dh = DY @ D
    dg, du = torch.autograd.grad(h, (g, u), dh)
    g, u, h = g.detach(), u.detach(), h.detach()
    # What the second products read is rounded once to 16 bits (half a step, or that of the subnormal numbers), behind float32: g, u and dh are sums over d with errors relative to the sums of
    # their sizes, which reach h, dg and du by the derivatives (act'' is at most 1.2); activation, derivative and products have 2^-19 (exponential and quotient of a few 2^-22).
    # The gradient reads g and u with 24 bits: cut off below 2^-15 of them.
    rel, small = rounding(x.dtype)
    a, da = ACT[act](g).abs(), torch.autograd.functional.jvp(ACT[act], (g,), (torch.ones_like(g),))[1].abs()
    cd, eg, eu, edh = _accumulated(d), X.abs() @ G.abs().T, X.abs() @ U.abs().T, DY.abs() @ D.abs()
    Eh = rel * h.abs() + small + cd * (da * u.abs() * eg + a * eu) + 2.0 ** -19 * h.abs()
    eg, eu = eg + 2.0 ** -15 * g.abs() / cd, eu + 2.0 ** -15 * u.abs() / cd
    Edg = rel * dg.abs() + small + cd * (u.abs() * da * edh + dh.abs() * da * eu + 1.2 * dh.abs() * u.abs() * eg) + 2.0 ** -19 * dh.abs() * u.abs() * (da + 0.1)
    Edu = rel * du.abs() + small + cd * (a * edh + dh.abs() * da * eg) + 2.0 ** -19 * du.abs()
    down = Eh @ D.abs().T + _accumulated(f) * (h.abs() @ D.abs().T)
    _near(y.reshape(m, d), h @ D.T, down, "y")
    _near(y0.reshape(m, d), h @ D.T, down, "y alone")
    dx, dwg, dwu, dwd = grads
    _near(dx.reshape(m, d), dg @ G + du @ U, Edg @ G.abs() + Edu @ U.abs() + _accumulated(2 * f) * (dg.abs() @ G.abs() + du.abs() @ U.abs()), "dx")
    _near(dwg, dg.T @ X, Edg.T @ X.abs() + _accumulated(m) * (dg.abs().T @ X.abs()), "dw_gate")
    _near(dwu, du.T @ X, Edu.T @ X.abs() + _accumulated(m) * (du.abs().T @ X.abs()), "dw_up")
    _near(dwd, DY.T @ h, DY.abs().T @ Eh + _accumulated(m) * (DY.abs().T @ h.abs()), "dw_down")
    return y, grads


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("m,d,f,act", [(1, 8, 8, "silu"), (1, 1024, 4096, "silu"), (7, 264, 520, "gelu"), (8, 64, 128, "relu"), (9, 1032, 72, "silu"), (16, 512, 2048, "gelu"), (17, 64, 64, "silu"), (33, 200, 136, "relu"),
                                       (128, 64, 256, "silu"), (129, 72, 264, "gelu"), (333, 520, 1400, "gelu"), (1000, 256, 1024, "silu"), (2500, 136, 408, "relu"), (4000, 64, 64, "silu"), (2048, 1024, 2048, "silu"),
                                       (70, 2048, 4096, "silu"), (5000, 768, 640, "gelu")])
def test_against_float64(dev, type, m, d, f, act):
    _check(dev, *_case(m, d, f, type, m + d), act)


@pytest.mark.parametrize("bad", [0.0, 3.0])
def test_special_values(dev, bad):
    """Zero rows, gates far on either side, a row that is not finite stays in its row of y and dx."""
    from goneuron_b200 import operators as ops
    for act in ACT:
        x, wg, wu, wd, dy = _case(40, 128, 256, "bf16", 5, 20.0 + bad)
        x[3] = 0
        _check(dev, x, wg, wu, wd, dy, act)
        x[7, 5] = float("nan")
        x[9, 0] = float("inf")
        y, saved = ops.gated_ffn(dev, x, wg, wu, wd, act, save=True)
        dx = ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved, act)[0]
        for v in (y, ops.gated_ffn(dev, x, wg, wu, wd, act), dx):
            rows = torch.isfinite(v).all(1)
            assert not rows[7] and rows.sum() >= 38 and all(rows[i] for i in range(40) if i not in (7, 9))


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("m,d,f,act", [(1, 8, 8, "silu"), (1, 1024, 4096, "silu"), (3, 264, 520, "gelu"), (8, 64, 128, "relu"), (7, 1032, 72, "silu"), (8, 512, 2048, "gelu")])
def test_few_tokens_are_rounded_once(dev, type, m, d, f, act):
    """Up to 8 tokens without a gradient: h enters the second product as two 16-bit numbers, half a step of half a step off; y has its own rounding and no other."""
    from goneuron_b200 import operators as ops
    x, wg, wu, wd, _ = _case(m, d, f, type, m + f)
    X, G, U, D = (v.double() for v in (x, wg, wu, wd))
    g, u = X @ G.T, X @ U.T
    h = ACT[act](g) * u
    rel, small = rounding(x.dtype)
    a, da = ACT[act](g).abs(), torch.autograd.functional.jvp(ACT[act], (g,), (torch.ones_like(g),))[1].abs()
    eh = rel * rel * h.abs() + small + _accumulated(d) * (da * u.abs() * (X.abs() @ G.abs().T) + a * (X.abs() @ U.abs().T)) + 2.0 ** -19 * h.abs()
    _near(ops.gated_ffn(dev, x, wg, wu, wd, act), h @ D.T, eh @ D.abs().T + _accumulated(2 * f) * (h.abs() @ D.abs().T), "y")


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_few_tokens_whose_h_is_not_finite(dev, type):
    """A product beyond the type's range, or not finite itself, makes its row's outputs not finite and no other row's, with an h of one infinity the same infinity."""
    from goneuron_b200 import operators as ops
    x, wg, wu, wd, _ = _case(5, 64, 64, type, 9)
    x[:, 0], wg[:], wu[:] = 1, 0, 0
    x[2, 0] = 3e4 if type == "f16" else 3e38
    wg[7, 0], wu[7, 0] = 3, 2                            # h[:, 7] = 6 x^2, the others 0
    y = ops.gated_ffn(dev, x, wg, wu, wd, "relu")
    rows = torch.isfinite(y).all(1)
    assert not rows[2] and rows.sum() == 4 and torch.equal(y[2][wd[:, 7] != 0], (wd[:, 7][wd[:, 7] != 0].float() * torch.inf).to(y.dtype))
    assert torch.equal(y[0], (6 * wd[:, 7].double()).to(y.dtype))


def test_gates_whose_square_is_not_finite(dev):
    """Gates of some 2^80, finite in bfloat16 though their square is not in float32: every activation is relu there, and relu's results are those of gates of about 1 times powers of two, bit for bit."""
    from goneuron_b200 import operators as ops
    x, wg, wu, wd, dy = _case(40, 128, 256, "bf16", 8)
    up, down = 2.0 ** 40, 2.0 ** -40

    def run(x, wg, wu, wd, act):
        y, saved = ops.gated_ffn(dev, x, wg, wu, wd, act, save=True)
        return [y, ops.gated_ffn(dev, x[:5], wg, wu, wd, act), *ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved, act)]
    _check(dev, x, wg, wu, wd, dy, "relu")
    want = [v * k for v, k in zip(run(x, wg, wu, wd, "relu"), (up, up, 1.0, 1.0, up * up, up * up))]
    for act in ACT:
        got = run(x * up, wg * up, wu * down, wd * down, act)
        for v, r in zip(got, want):
            assert torch.isfinite(v).all()
            if act == "relu":
                assert torch.equal(v, r)
            else:                                        # h, dg, du and the result may be rounded to the neighbouring number, 2^-7 off: the quotient in the sigmoid has some 2^-22
                assert (v.double() - r.double()).norm() <= 2 * 2.0 ** -7 * r.double().norm()


def test_views_and_batches(dev):
    x, wg, wu, wd, dy = _case(60, 96, 200, "f16", 6)
    wide = torch.randn(60, 400, device="cuda").half()
    for v in (x.view(5, 12, 96), wide[:, 8:104], wide.view(5, 12, 400)[:, :, 96:192]):
        _check(dev, v, wg, wu, wd, dy.view(v.shape), "silu")
    _check(dev, x, wg, wu, wd, wide[:, 16:112], "gelu")
    x1 = wide[:1, 8:104]
    _check(dev, x1, wg, wu, wd, dy[:1], "silu")


def test_refusals(dev):
    from goneuron_b200 import _lib, operators as ops
    x, wg, wu, wd, dy = _case(20, 64, 128, "f16", 7)
    _, saved = ops.gated_ffn(dev, x, wg, wu, wd, save=True)
    for call in (lambda: ops.gated_ffn(dev, x, wg, wu, wd, "tanh"), lambda: ops.gated_ffn(dev, x.float(), wg.float(), wu.float(), wd.float()), lambda: ops.gated_ffn(dev, x.bfloat16(), wg, wu, wd),
                 lambda: ops.gated_ffn(dev, x, wg, wu[:64], wd), lambda: ops.gated_ffn(dev, x, wg, wu, wd.t()), lambda: ops.gated_ffn(dev, x[:, :56], wg, wu, wd), lambda: ops.gated_ffn(dev, x.cpu(), wg, wu, wd),
                 lambda: ops.gated_ffn_backward(dev, dy[:19], x, wg, wu, wd, saved), lambda: ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved[:-1])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.gated_ffn(dev, x[:, :60], wg[:, :60].contiguous(), wu[:, :60].contiguous(), wd[:60]),                 # no multiple of 8
                 lambda: ops.gated_ffn(dev, torch.zeros(20, 65, device="cuda").half()[:, :64], wg, wu, wd),                        # rows 130 bytes apart
                 lambda: ops.gated_ffn(dev, torch.zeros(20, 72, device="cuda").half()[:, 1:65], wg, wu, wd),                       # begins at 2 bytes
                 lambda: ops.gated_ffn(dev, x[:1].expand(20, 64), wg, wu, wd)):                                                    # one row for all
        with pytest.raises(_lib.GoNeuronCudaError):
            call()
    ops.check(dev)


def test_a_wait_that_gives_up_is_reported_and_the_device_stays_usable(dev):
    from goneuron_b200 import _lib, operators as ops
    a = _case(300, 256, 512, "bf16", 8)
    want = ops.gated_ffn(dev, *a[:4])
    _lib.check(_lib.load().gn_ctx_set_spin_limit(dev.handle, 1))
    try:
        ops.gated_ffn(dev, *a[:4])
        with pytest.raises(_lib.GoNeuronCudaError) as e:
            ops.check(dev)
        assert e.value.code == -6
    finally:
        _lib.check(_lib.load().gn_ctx_set_spin_limit(dev.handle, 0))
    assert torch.equal(ops.gated_ffn(dev, *a[:4]), want)
    ops.check(dev)


def test_streams_and_graphs(dev):
    from goneuron_b200 import operators as ops
    for m in (4, 300):
        x, wg, wu, wd, dy = _case(m, 256, 512, "f16", 9)

        def both():
            y, saved = ops.gated_ffn(dev, x, wg, wu, wd, save=True)
            return (ops.gated_ffn(dev, x, wg, wu, wd), y, *ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved))
        want = both()
        streams = [torch.cuda.Stream() for _ in range(2)]
        other = []
        for s in streams:                              # two at once
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                other.append(both())
        for s in streams:
            s.synchronize()
        assert all(torch.equal(a, b) for o in other for a, b in zip(want, o))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = both()
        x.copy_(x.flip(1))
        g.replay()
        again = both()
        assert all(torch.equal(a, b) for a, b in zip(held, again)) and not torch.equal(held[0], want[0])


def test_gradient_against_differences(dev):
    """The directional derivative of sum(y dy) along dx."""
    from goneuron_b200 import operators as ops
    x, wg, wu, wd, dy = _case(64, 64, 128, "f16", 10)
    _, saved = ops.gated_ffn(dev, x, wg, wu, wd, save=True)
    dx = ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved)[0].double()
    step = torch.zeros_like(x)
    for row in range(0, 64, 9):
        step.zero_()
        step[row] = (2.0 ** -4 * torch.sign(dx[row])).half()
        hi, lo = (x + step).half(), (x - step).half()
        f = lambda v: (ops.gated_ffn(dev, v, wg, wu, wd).double() * dy.double()).sum(1)[row]
        # y's rounding 2^-11 of about 1 in each of 64 elements; third derivatives of silu times the step's cube
        assert abs(float(f(hi) - f(lo)) - float(((hi - lo)[row].double() * dx[row]).sum())) <= 0.05 * float(((hi - lo)[row].double() * dx[row]).sum()) + 0.05


def test_no_tokens(dev):
    from goneuron_b200 import operators as ops
    x, wg, wu, wd, dy = _case(0, 64, 128, "f16", 11)
    y, saved = ops.gated_ffn(dev, x, wg, wu, wd, save=True)
    assert y.shape == (0, 64)
    dx, *dw = ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved)
    assert dx.shape == (0, 64) and all(float(w.abs().sum()) == 0 for w in dw)
