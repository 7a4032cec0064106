"""The operators on device memory as they would be used together: a training step of a one-layer student (embedding, norm and rotation of queries and keys, attention by torch, gated feed-forward block,
distillation from a teacher's top logits) against float64 autograd; the same model answering token by token; from two threads at once; with gradients left out."""
import ctypes as C
import os
import subprocess
import sys
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

V, D, H, KV, E, F, K = 640, 128, 4, 2, 32, 320, 12


@pytest.fixture(scope="module")
def dev():
    from goneuron_b200.sequential import Device
    d = Device(0)
    yield d
    d.close()


def _weights(seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s, k: torch.randn(*s, device="cuda", generator=gen).mul(k).half()
    w = {"table": r(V, D, k=D ** -0.5), "wq": r(H * E, D, k=D ** -0.5), "wk": r(KV * E, D, k=D ** -0.5), "wv": r(KV * E, D, k=D ** -0.5), "wo": r(D, H * E, k=D ** -0.5),
         "wg": r(F, D, k=D ** -0.5), "wu": r(F, D, k=D ** -0.5), "wd": r(D, F, k=F ** -0.5), "head": r(V, D, k=D ** -0.5),
         "gq": 1 + 0.2 * torch.randn(E, device="cuda", generator=gen), "gk": 1 + 0.2 * torch.randn(E, device="cuda", generator=gen)}
    return w, gen


FREQ = lambda: 10000.0 ** (-torch.arange(0, E, 2, device="cuda", dtype=torch.float64) / E)


def _attend(q, k, v):
    """Causal attention of [T, H, E] over [T, KV, E] in q's type, and the probabilities."""
    k, v = (x.repeat_interleave(H // KV, 1) for x in (k, v))
    s = torch.einsum("thd,shd->hts", q, k) * E ** -0.5
    p = torch.softmax(s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -torch.inf), -1)
    return torch.einsum("hts,shd->thd", p, v), p


def _step(dev, w, ids, pos, top_ids, top, weight):
    """Loss and gradients; what is not one of the operators runs in float32."""
    from goneuron_b200 import operators as ops
    f, T = (lambda x: x.float()), ids.numel()
    x0 = ops.embedding(dev, w["table"], ids, scale=D ** 0.5)
    q, k, v = ((f(x0) @ f(w[n]).T).half().view(T, -1, E) for n in ("wq", "wk", "wv"))
    qr, kr = ops.qk_norm_rope(dev, q, k, w["gq"], w["gk"], pos, FREQ())
    a, p = _attend(f(qr), f(kr), f(v))
    x1 = (f(x0) + a.reshape(T, -1) @ f(w["wo"]).T).half()
    y, saved = ops.gated_ffn(dev, x1, w["wg"], w["wu"], w["wd"], save=True)
    x2 = f(x1) + f(y)
    logits = (x2 @ f(w["head"]).T).half()
    loss, dl = ops.distill_loss_grad(dev, logits, top_ids, top, 2.0, weight)
    g = {"head": f(dl).T @ x2}
    dx2 = f(dl) @ f(w["head"])
    dx1, g["wg"], g["wu"], g["wd"] = ops.gated_ffn_backward(dev, dx2.half(), x1, w["wg"], w["wu"], w["wd"], saved)
    dx1 = f(dx1) + dx2
    g["wo"], da = dx1.T @ a.reshape(T, -1), (dx1 @ f(w["wo"])).view(T, H, E)
    kk, vv = (f(t).repeat_interleave(H // KV, 1) for t in (kr, v))
    dp = torch.einsum("thd,shd->hts", da, vv)
    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * E ** -0.5
    dqr = torch.einsum("hts,shd->thd", ds, kk).half()
    dkr, dv = (torch.einsum("hts,thd->shd", m, t).view(T, KV, H // KV, E).sum(2).half() for m, t in ((ds, f(qr)), (p, da)))
    dq, dk, g["gq"], g["gk"] = ops.qk_norm_rope_backward(dev, dqr, dkr, q, k, w["gq"], w["gk"], pos, FREQ())
    dx0 = dx1
    for n, d in (("wq", dq), ("wk", dk), ("wv", dv)):
        g[n], dx0 = f(d).reshape(T, -1).T @ f(x0), dx0 + f(d).reshape(T, -1) @ f(w[n])
    g["table"] = ops.embedding_backward(dev, dx0.half(), ids, V, scale=D ** 0.5)
    return loss, g


def _model(w, ids, pos, top_ids, top, weight):
    """The same in float64, by its definition; gradients by autograd."""
    w = {n: t.double().requires_grad_() for n, t in w.items()}
    T, there = ids.numel(), (ids >= 0)[:, None]
    x0 = torch.where(there, w["table"][ids.clamp(min=0)], 0.0) * D ** 0.5
    turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), pos.double()[:, None] * FREQ())[:, None]

    def heads(n, gain):
        t = (x0 @ w[n].T).view(T, -1, E)
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-5) * w[gain]
        z = torch.complex(t[..., :E // 2], t[..., E // 2:]) * turn
        return torch.cat((z.real, z.imag), -1)
    a, _ = _attend(heads("wq", "gq"), heads("wk", "gk"), (x0 @ w["wv"].T).view(T, -1, E))
    x1 = x0 + a.reshape(T, -1) @ w["wo"].T
    x2 = x1 + (torch.nn.functional.silu(x1 @ w["wg"].T) * (x1 @ w["wu"].T)) @ w["wd"].T
    log_q = torch.log_softmax(x2 @ w["head"].T / 2.0, 1)
    t = torch.where(top_ids >= 0, top.double() / 2.0, -torch.inf)
    p = torch.softmax(t, 1)
    loss = weight.double() * 4.0 * (torch.special.xlogy(p, p) - p * log_q.gather(1, top_ids.clamp(min=0))).sum(1)
    names = list(w)
    return loss.detach(), dict(zip(names, torch.autograd.grad(loss.sum(), [w[n] for n in names])))


def _batch(gen, T=150):
    ids = torch.randint(0, V, (T,), device="cuda", generator=gen)
    ids[-7:] = -1                                        # padding at the end: zero rows that nobody before them sees, without a loss
    weight = torch.ones(T, device="cuda")
    weight[-7:] = 0
    top, top_ids = torch.topk(torch.randn(T, V, device="cuda", generator=gen) * 3, K, 1)
    return ids, torch.arange(T, device="cuda") + 1000, top_ids, top, weight * 16


def test_training_step(dev):
    from goneuron_b200 import operators as ops
    w, gen = _weights(1)
    batch = _batch(gen)
    loss, g = _step(dev, w, *batch)
    ops.check(dev)
    want_loss, want = _model(w, *batch)
    # Some 12 roundings to float16 (2^-11 of a value at most) lie on the way to the logits, 10 more on the way back to the table; each moves what follows by about as much in the 2-norm.
    off = lambda x, y: float((x.double() - y).norm() / y.norm())
    assert off(loss, want_loss) < 12 * 2 ** -11 and float(loss[-7:].abs().sum()) == 0
    for n, x in g.items():
        assert off(x, want[n]) < 22 * 2 ** -11, (n, off(x, want[n]))


def test_captured_training_step_is_the_same(dev):
    w, gen = _weights(2)
    batch = _batch(gen)
    want = _step(dev, w, *batch)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _step(dev, w, *batch)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, g = _step(dev, w, *batch)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    same = lambda x, y: float((x.double() - y.double()).norm()) <= 1e-3 * float(y.double().norm())      # (torch's own products may be cut differently)
    assert same(loss, want[0]) and all(same(g[n], want[1][n]) for n in g)


def test_token_by_token(dev):
    """Queries, keys and feed-forward rows of one token at a time are those of the whole sequence, up to the rounding of other orders of sums."""
    from goneuron_b200 import operators as ops
    w, gen = _weights(3)
    ids, pos, *_ = _batch(gen, 40)
    x = ops.embedding(dev, w["table"], ids, scale=D ** 0.5)
    q = (x.float() @ w["wq"].float().T).half().view(40, H, E)
    whole_q = ops.qk_norm_rope(dev, q, None, w["gq"], None, pos, FREQ())[0]
    whole_y = ops.gated_ffn(dev, x, w["wg"], w["wu"], w["wd"])
    size = (x.double().abs() @ w["wg"].double().abs().T) * (x.double().abs() @ w["wu"].double().abs().T) @ w["wd"].double().abs().T
    for n in (1, 5, 16):
        for i in range(0, 40 - n, 7):
            one = slice(i, i + n)
            assert torch.equal(ops.embedding(dev, w["table"], ids[one], scale=D ** 0.5), x[one])
            assert torch.equal(ops.qk_norm_rope(dev, q[one], None, w["gq"], None, pos[one], FREQ())[0], whole_q[one])
            # h and y are each rounded to float16 on both sides
            assert ((ops.gated_ffn(dev, x[one], w["wg"], w["wu"], w["wd"]).double() - whole_y[one].double()).abs() <= 2 ** -11 * (2 * whole_y[one].double().abs() + 2 * size[one])).all()


def test_two_threads(dev):
    """The same step on two streams of two threads: calls share nothing."""
    w, gen = _weights(4)
    batches = [_batch(gen), _batch(gen, 77)]
    want = [_step(dev, w, *b) for b in batches]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i] = _step(dev, w, *batches[i])
            s.synchronize()
        except Exception as e:      # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    same = lambda x, y: float((x.double() - y.double()).norm()) <= 1e-3 * float(y.double().norm())
    for i in range(2):
        assert same(got[i][0], want[i][0]) and all(same(got[i][1][n], want[i][1][n]) for n in want[i][1])


def test_gradients_that_are_not_wanted(dev):
    """The C ABI leaves out what it gets no pointer for, and writes the rest as with all of them; a workspace that is too small is refused."""
    from goneuron_b200 import _lib, operators as ops
    L = _lib.load()
    gen = torch.Generator("cuda").manual_seed(5)
    m, d, f = 300, 128, 256
    x, dy = (torch.randn(m, d, device="cuda", generator=gen).half() for _ in range(2))
    wg, wu = (torch.randn(f, d, device="cuda", generator=gen).mul(0.1).half() for _ in range(2))
    wd = torch.randn(d, f, device="cuda", generator=gen).mul(0.1).half()
    _, saved = ops.gated_ffn(dev, x, wg, wu, wd, save=True)
    want = ops.gated_ffn_backward(dev, dy, x, wg, wu, wd, saved)
    n = C.c_int64()
    _lib.check(L.gn_op_gated_ffn_workspace(dev.handle, m, d, f, 1, C.byref(n)))
    ws, stream = torch.empty(n.value, dtype=torch.uint8, device="cuda"), torch.cuda.current_stream().cuda_stream
    p = lambda t: None if t is None else t.data_ptr()

    def call(out, size=n.value):
        return L.gn_op_gated_ffn_backward(dev.handle, 1, 7, m, d, f, p(dy), d, p(x), d, p(wg), p(wu), p(wd), p(saved), p(out[0]), d, p(out[1]), p(out[2]), p(out[3]), p(ws), size, stream)
    for wanted in ((0,), (1,), (2, 3), (0, 3), (3,), ()):
        out = [torch.full_like(t, 7.0) if i in wanted else None for i, t in enumerate(want)]
        _lib.check(call(out))
        for i in wanted:
            assert (out[i].double() - want[i].double()).norm() <= 2 ** -11 * want[i].double().norm()      # (fewer weights: other cuts of the contraction)
    assert call([None] * 4, n.value - 1) == -1 and b"workspace" in L.gn_last_error()
    # a gain's gradient alone, of the keys
    q, k = (torch.randn(70, h, 64, device="cuda", generator=gen) for h in (3, 2))
    g = torch.ones(64, device="cuda")
    *_, dgk = ops.qk_norm_rope_backward(dev, q, k, q, k, None, g)
    assert ops.qk_norm_rope_backward(dev, q, k, q, k, None, g)[2] is None and torch.equal(dgk, ops.qk_norm_rope_backward(dev, q, k, q, k, g, g)[3])


def test_captured_branches(dev):
    """Two branches of a captured graph, each with kernels of these operators, joined by one that reads both: kernels placed under their predecessors wait for both branches."""
    from goneuron_b200 import operators as ops
    w, gen = _weights(6)
    ids, pos, *_ = _batch(gen)
    q = torch.randn(150, H, E, device="cuda", generator=gen).half()

    def step(side):
        main = torch.cuda.current_stream()
        x = ops.embedding(dev, w["table"], ids, scale=D ** 0.5)
        if side:
            side.wait_stream(main)
        with torch.cuda.stream(side or main):
            a = ops.qk_norm_rope(dev, q, None, w["gq"], None, pos, FREQ())[0]
            a = ops.gated_ffn(dev, a.reshape(150, D), w["wg"], w["wu"], w["wd"])
        y = ops.gated_ffn(dev, x, w["wg"], w["wu"], w["wd"])
        if side:
            main.wait_stream(side)
        return ops.qk_norm_rope(dev, a.view(150, H, E), y.view(150, H, E), None, None, pos, FREQ())
    want = step(None)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(side)
    for i in range(5):
        for t in got:
            t.fill_(7.0)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i
    ops.check(dev)


FIRST = """
import torch
from goneuron_b200 import operators as ops
from goneuron_b200.sequential import Device
dev = Device(0)
r = lambda *s: torch.randn(*s, device="cuda").half()
x, wg, wu, wd, q, table, logits = r(40, 64), r(128, 64), r(128, 64), r(64, 128), r(40, 4, 64), r(90, 64), r(40, 500)
ids, top = torch.randint(0, 90, (40,), device="cuda"), torch.randn(40, 5, device="cuda")
def step():
    y, saved = ops.gated_ffn(dev, x, wg, wu, wd, save=True)
    return [y, ops.gated_ffn(dev, x[:1], wg, wu, wd), *ops.gated_ffn_backward(dev, x, x, wg, wu, wd, saved), ops.qk_norm_rope(dev, q, None)[0], ops.embedding(dev, table, ids),
            ops.embedding_backward(dev, x, ids, 90), *ops.distill_loss_grad(dev, logits, ids[:, None].expand(40, 5).contiguous(), top)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
want = step()
ops.check(dev)
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("the same")
"""


def test_first_calls_of_a_process_are_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "the same" in r.stdout, r.stderr[-2000:]


def test_status_is_not_read_while_capturing(dev):
    from goneuron_b200 import _lib, operators as ops
    x = torch.zeros(4, 8, device="cuda")
    ids = torch.zeros(2, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.embedding(dev, x, ids)
        with pytest.raises(_lib.GoNeuronCudaError):
            ops.check(dev)
    graph.replay()
    ops.check(dev)


def test_closed_device_is_refused():
    from goneuron_b200 import _lib, operators as ops
    from goneuron_b200.sequential import Device
    d = Device(0)
    x, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    ops.embedding(d, x, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.embedding(d, x, ids)
    d.close()
    with pytest.raises(_lib.GoNeuronCudaError):
        ops.embedding(d, x, ids)
    x.fill_(3)
    graph.replay()                                       # what was captured does not need the device any more
    assert float(out.sum()) == 48
