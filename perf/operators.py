"""Operators of language models on device tensors: norms of queries and keys with the position rotation, the gated
feed-forward block, distillation from a teacher's top logits, embedding lookup with scaling; each with its gradient where a
case trains.  Where `own` is false they are computed from elementary torch operations in 32 bits, where it is true by this
framework's kernels (goneuron_b200.operators).  Sizes are those of the framework's Transformer configurations (widths 256 and
1024, vocabularies 8192 and 32000, 128 and 512 tokens) and odd ones around them."""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def listed():
    return [
        # one token of one sequence through the large Transformer's feed-forward block: the weights are what it reads
        dict(name="ffn one token", op="ffn", tokens=1, dim=1024, ff=4096, act="silu", type="bf16", train=False),
        # training on a ragged batch: sizes that end inside every tile
        dict(name="ffn train ragged", op="ffn", tokens=333, dim=520, ff=1400, act="gelu", type="f16", train=True),
        # a training step of the small Transformer, 64 sequences of 128 tokens
        dict(name="ffn train 256 wide", op="ffn", tokens=8192, dim=256, ff=1024, act="silu", type="bf16", train=True),
        # a training step of the large Transformer, 32 sequences of 512 tokens
        dict(name="ffn train 1024 wide", op="ffn", tokens=16384, dim=1024, ff=4096, act="silu", type="bf16", train=True),
        # one decoding step of five sequences at far positions
        dict(name="qk decode", op="qk", tokens=5, heads=16, kv_heads=4, head=64, rotated=64, interleaved=False, fused=True, far=True, type="bf16", train=False),
        # odd head size, part of it rotated as neighbouring pairs, views of one projection's output
        dict(name="qk train ragged", op="qk", tokens=2049, heads=6, kv_heads=2, head=80, rotated=40, interleaved=True, fused=True, far=False, type="f16", train=True),
        # a training step of 128 sequences of 512 tokens with shared key heads
        dict(name="qk train", op="qk", tokens=65536, heads=16, kv_heads=4, head=64, rotated=64, interleaved=False, fused=False, far=False, type="bf16", train=True),
        # evaluation: the loss alone
        dict(name="distill loss", op="distill", rows=24, vocab=8192, top=8, temperature=1.0, type="f32", train=False),
        # a training step over the large Transformer's vocabulary
        dict(name="distill train", op="distill", rows=4096, vocab=32000, top=64, temperature=2.0, type="bf16", train=True),
        # a vocabulary of odd size that does not fit one multiprocessor
        dict(name="distill train odd", op="distill", rows=515, vocab=100003, top=100, temperature=1.5, type="f16", train=True),
        # a ragged batch in 32 bits
        dict(name="embedding train ragged", op="embedding", tokens=3001, vocab=8192, dim=300, type="f32", train=True),
        # a training step of 256 sequences of 512 tokens
        dict(name="embedding train", op="embedding", tokens=131072, vocab=32000, dim=1024, type="bf16", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ffn", "qk", "distill", "embedding"])
    half = rng.choice(["bf16", "f16"])
    any_type = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.6
    if op == "ffn":
        c = dict(op=op, tokens=_log(rng, 1, 16384), dim=8 * _log(rng, 8, 128), act=rng.choice(["silu", "gelu", "relu"]), type=half, train=train)
        c["ff"] = min(4096, 8 * max(1, round(c["dim"] * rng.uniform(1.0, 4.0) / 8)))
        return c
    if op == "qk":
        head = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        c = dict(op=op, tokens=_log(rng, 1, 32768), heads=rng.randint(1, 32), head=head, rotated=rng.choice([head, head, head // 2]),
                 interleaved=rng.random() < 0.3, fused=rng.random() < 0.5, far=rng.random() < 0.5, type=any_type, train=train)
        c["kv_heads"] = rng.randint(1, c["heads"])
        while c["tokens"] > 1 and c["tokens"] * (c["heads"] + c["kv_heads"]) * head > 60e6:
            c["tokens"] = c["tokens"] * 2 // 3
        return c
    if op == "distill":
        c = dict(op=op, vocab=_log(rng, 500, 130000), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), type=any_type, train=train)
        c.update(rows=_log(rng, 1, min(8192, 131e6 / c["vocab"])), top=_log(rng, 1, 256))
        return c
    c = dict(op=op, tokens=_log(rng, 1, 131072), vocab=_log(rng, 500, 50000), dim=rng.choice([8 * _log(rng, 4, 128), _log(rng, 30, 1024)]), type=any_type, train=train)
    while c["tokens"] > 1 and c["tokens"] * c["dim"] > 130e6:
        c["tokens"] = c["tokens"] * 2 // 3
    return c


# ------------------------------------------------------------------ inputs
class _Random:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, scale=1.0, type=torch.float32):
        return torch.randn(*shape, device="cuda", generator=self.g).mul_(scale).to(type)

    def uniform(self, *shape):
        return torch.rand(*shape, device="cuda", generator=self.g)

    def below(self, n, *shape):
        return torch.randint(0, n, shape, device="cuda", generator=self.g)


def prepare(case, seed):
    r, t, s = _Random(seed), TYPES[case["type"]], {"case": case}
    if case["op"] == "ffn":
        m, d, f = case["tokens"], case["dim"], case["ff"]
        s.update(x=r.normal(m, d, type=t), w_gate=r.normal(f, d, scale=d ** -0.5, type=t), w_up=r.normal(f, d, scale=d ** -0.5, type=t),
                 w_down=r.normal(d, f, scale=f ** -0.5, type=t), dy=r.normal(m, d, type=t) if case["train"] else None)
    elif case["op"] == "qk":
        n, h, k, e = case["tokens"], case["heads"], case["kv_heads"], case["head"]
        if case["fused"]:                               # query, key and value side by side, as one projection leaves them
            qkv = r.normal(n, h + 2 * k, e, scale=2.0, type=t)
            s.update(q=qkv[:, :h], k=qkv[:, h:h + k])
        else:
            s.update(q=r.normal(n, h, e, scale=2.0, type=t), k=r.normal(n, k, e, scale=2.0, type=t))
        s.update(gain_q=1 + 0.2 * r.normal(e), gain_k=1 + 0.2 * r.normal(e),
                 positions=r.below(1 << 20, n) if case["far"] else torch.arange(n, device="cuda") % 512,
                 frequencies=10000.0 ** (-torch.arange(0, case["rotated"], 2, device="cuda", dtype=torch.float64) / case["rotated"]))
        if case["train"]:
            s.update(dq_out=r.normal(n, h, e, type=t), dk_out=r.normal(n, k, e, type=t))
    elif case["op"] == "distill":
        n, v, k = case["rows"], case["vocab"], min(case["top"], case["vocab"])
        teacher = r.normal(n, v, scale=3.0)
        s.update(logits=(0.5 * teacher).add_(r.normal(n, v, scale=1.5)).to(t))
        s["top_logits"], s["top_ids"] = torch.topk(teacher, k, dim=1)
        del teacher
        cut = r.below(k + 1, n).clamp_(min=(k + 1) // 2)                            # some rows keep fewer entries of the teacher's
        s["top_ids"] = s["top_ids"].masked_fill(torch.arange(k, device="cuda")[None, :] >= cut[:, None], -1)
        used = (r.uniform(n) > 0.1).float()                                         # rows of padding have no loss
        used[0] = 1.0
        s["row_weight"] = used * ((65536.0 if case["type"] == "f16" else 1.0) / used.sum())      # 16-bit gradients carry a loss scale
    else:
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        order = torch.randperm(v, device="cuda", generator=r.g)
        ids = order[(r.uniform(n).double() ** 3 * v).long().clamp_(max=v - 1)]      # few tokens are frequent, most are rare
        s.update(table=r.normal(v, d, scale=d ** -0.5, type=t), ids=ids.masked_fill(r.uniform(n) < 0.02, -1), scale=math.sqrt(d))
        if case["train"]:
            s["dout"] = r.normal(n, d, type=t)
    return s


# ------------------------------------------------------------------ this framework's operators
_device = None


def _own(s):
    global _device
    from goneuron_b200 import operators as ops
    if _device is None:
        from goneuron_b200.sequential import Device
        _device = Device(torch.cuda.current_device())
    c, dev = s["case"], _device
    if c["op"] == "ffn":
        w = (s["w_gate"], s["w_up"], s["w_down"])
        if not c["train"]:
            return {"y": ops.gated_ffn(dev, s["x"], *w, activation=c["act"])}
        y, saved = ops.gated_ffn(dev, s["x"], *w, activation=c["act"], save=True)
        dx, d_gate, d_up, d_down = ops.gated_ffn_backward(dev, s["dy"], s["x"], *w, saved, activation=c["act"])
        return {"y": y, "dx": dx, "dw_gate": d_gate, "dw_up": d_up, "dw_down": d_down}
    if c["op"] == "qk":
        a = (s["q"], s["k"], s["gain_q"], s["gain_k"], s["positions"], s["frequencies"])
        q, k = ops.qk_norm_rope(dev, *a, eps=EPS, interleaved=c["interleaved"])
        if not c["train"]:
            return {"q": q, "k": k}
        dq, dk, dgq, dgk = ops.qk_norm_rope_backward(dev, s["dq_out"], s["dk_out"], *a, eps=EPS, interleaved=c["interleaved"])
        return {"q": q, "k": k, "dq": dq, "dk": dk, "dgain_q": dgq, "dgain_k": dgk}
    if c["op"] == "distill":
        a = (s["logits"], s["top_ids"], s["top_logits"], c["temperature"])
        if not c["train"]:
            return {"loss": ops.distill_loss(dev, *a)}
        loss, dlogits = ops.distill_loss_grad(dev, *a, s["row_weight"])
        return {"loss": loss, "dlogits": dlogits}
    out = ops.embedding(dev, s["table"], s["ids"], scale=s["scale"])
    if not c["train"]:
        return {"out": out}
    return {"out": out, "dtable": ops.embedding_backward(dev, s["dout"], s["ids"], c["vocab"], scale=s["scale"])}


# ------------------------------------------------------------------ plain forms
_GELU = math.sqrt(2.0 / math.pi)


def _activation(act, g):
    """act(g) and its derivative."""
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return g * p, p * (1.0 + g * (1.0 - p))
    if act == "gelu":
        t = torch.tanh(_GELU * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * _GELU * (1.0 + 3 * 0.044715 * g * g)
    return torch.clamp(g, min=0.0), (g > 0).float()


def _plain_ffn(s):
    c, t = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.T, x @ wu.T
    a, da = _activation(c["act"], g)
    h = a * u
    y = (h @ wd.T).to(t)
    if not c["train"]:
        return {"y": y}
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    return {"y": y, "dx": (dg @ wg + du @ wu).to(t), "dw_gate": (dg.T @ x).to(t), "dw_up": (du.T @ x).to(t), "dw_down": (dy.T @ h).to(t)}


def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] elements of each head as pairs, turned by the angles; the others as they are."""
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_qk(s):
    c, t, out = s["case"], s["q"].dtype, {}
    angle = s["positions"].double()[:, None, None] * s["frequencies"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    for n in ("q", "k"):
        x, gain = s[n].float(), s["gain_" + n]
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xn = x * r
        out[n] = _rotate(xn * gain, cos, sin, c["interleaved"]).to(t)
        if c["train"]:
            dy = _rotate(s["d%s_out" % n].float(), cos, -sin, c["interleaved"])
            dxn = dy * gain
            out["d" + n] = (r * (dxn - xn * (dxn * xn).mean(-1, keepdim=True))).to(t)
            out["dgain_" + n] = (dy * xn).sum((0, 1))
    return out


def _plain_distill(s):
    c, t = s["case"], s["logits"].dtype
    z, tau, ids = s["logits"].float() / c["temperature"], c["temperature"], s["top_ids"]
    there = ids >= 0
    top = (s["top_logits"] / tau).masked_fill(~there, -math.inf)
    p = torch.exp(top - top.max(1, keepdim=True).values)
    p = p / p.sum(1, keepdim=True)
    e = z - z.max(1, keepdim=True).values
    log_q = e - torch.log(torch.exp(e).sum(1, keepdim=True))
    at = ids.clamp(min=0)
    loss = tau * tau * torch.where(there, p * (torch.log(torch.where(there, p, 1.0)) - torch.gather(log_q, 1, at)), 0.0).sum(1)
    if not c["train"]:
        return {"loss": loss}
    w = s["row_weight"][:, None]
    d = torch.exp(log_q).scatter_add(1, at, -p) * (tau * w)
    return {"loss": loss * s["row_weight"], "dlogits": d.to(t)}


def _plain_embedding(s):
    c, t, ids = s["case"], s["table"].dtype, s["ids"]
    there = (ids >= 0)[:, None]
    at = ids.clamp(min=0)
    out = torch.where(there, s["table"][at].float() * s["scale"], 0.0).to(t)
    if not c["train"]:
        return {"out": out}
    rows = torch.where(there, s["dout"].float() * s["scale"], 0.0)
    return {"out": out, "dtable": torch.zeros(c["vocab"], c["dim"], device=rows.device).index_add_(0, at, rows)}


_PLAIN = {"ffn": _plain_ffn, "qk": _plain_qk, "distill": _plain_distill, "embedding": _plain_embedding}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ definitions in 64 bits
def _grads(y, leaves, dy):
    return torch.autograd.grad(y, leaves, dy)


def _exact_ffn(s):
    c = s["case"]
    x, wg, wu, wd = leaves = [s[n].double().requires_grad_(c["train"]) for n in ("x", "w_gate", "w_up", "w_down")]
    g = torch.einsum("md,fd->mf", x, wg)
    act = {"silu": torch.nn.functional.silu, "relu": torch.relu, "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[c["act"]]
    y = torch.einsum("mf,df->md", act(g) * torch.einsum("md,fd->mf", x, wu), wd)
    if not c["train"]:
        return {"y": y}
    dx, dg, du, dd = _grads(y, leaves, s["dy"].double())
    return {"y": y, "dx": dx, "dw_gate": dg, "dw_up": du, "dw_down": dd}


def _exact_qk(s):
    c, out = s["case"], {}
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * s["frequencies"][None, :])[:, None, :]
    r = c["rotated"]
    for n in ("q", "k"):
        x, gain = s[n].double().requires_grad_(c["train"]), s["gain_" + n].double().requires_grad_(c["train"])
        v = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["head"] + EPS) * gain
        pairs = v[..., :r].unflatten(-1, (r // 2, 2)) if c["interleaved"] else v[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        w = torch.cat(((w if c["interleaved"] else w.transpose(-1, -2)).flatten(-2), v[..., r:]), -1)
        out[n] = w.detach()
        if c["train"]:
            out["d" + n], out["dgain_" + n] = _grads(w, [x, gain], s["d%s_out" % n].double())
    return out


def _exact_distill(s):
    c, tau = s["case"], s["case"]["temperature"]
    z = s["logits"].double().requires_grad_(c["train"])
    log_q = torch.log_softmax(z / tau, 1)
    top = torch.where(s["top_ids"] >= 0, s["top_logits"].double() / tau, -math.inf)
    p = torch.softmax(top, 1)
    cross = -(p * log_q.gather(1, s["top_ids"].clamp(min=0))).sum(1)
    loss = tau ** 2 * (torch.special.xlogy(p, p).sum(1) + cross)
    if not c["train"]:
        return {"loss": loss}
    loss = loss * s["row_weight"].double()
    return {"loss": loss.detach(), "dlogits": _grads(loss, [z], torch.ones_like(loss))[0]}


def _exact_embedding(s):
    c, ids = s["case"], s["ids"]
    there = ids >= 0
    out = torch.zeros(c["tokens"], c["dim"], dtype=torch.float64, device="cuda")
    out[there] = s["table"].double()[ids[there]] * s["scale"]
    if not c["train"]:
        return {"out": out}
    d = torch.zeros(c["vocab"], c["dim"], dtype=torch.float64, device="cuda")
    d.index_put_((ids[there],), s["dout"][there].double(), accumulate=True)
    return {"out": out, "dtable": d * s["scale"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"ffn": _exact_ffn, "qk": _exact_qk, "distill": _exact_distill, "embedding": _exact_embedding}[case["op"]](s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b, train = BYTES[case["type"]], case["train"]
    if case["op"] == "ffn":
        m, d, f = case["tokens"], case["dim"], case["ff"]
        return {"bytes": float(b * (m * d + 3 * d * f) * 2 + b * m * d * 2 if train else b * (2 * m * d + 3 * d * f)), "flops": (18.0 if train else 6.0) * m * d * f}
    if case["op"] == "qk":
        n, rows = case["tokens"], case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": float(rows * case["head"] * b * (4 if train else 2) + 8 * n), "flops": (20.0 if train else 8.0) * rows * case["head"]}
    if case["op"] == "distill":
        n, v, k = case["rows"], case["vocab"], min(case["top"], case["vocab"])
        return {"bytes": float(n * v * b * (2 if train else 1) + n * k * 12 + 8 * n), "flops": (8.0 if train else 5.0) * n * v}
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    edge = (np.arange(v + 1) / v) ** (1.0 / 3.0)
    rows = float((1.0 - (1.0 - np.diff(edge)) ** (0.98 * n)).sum())                 # table rows that such a batch touches
    return {"bytes": rows * d * b + float(n * d * b + 8 * n) + (float(n * d * b + v * d * 4) if train else 0.0), "flops": (2.0 if train else 1.0) * n * d}
