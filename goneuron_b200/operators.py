"""Operators of language models on torch CUDA tensors, over the C ABI of libgoneuron_cuda.so (the last part of
include/goneuron_cuda.h, which states each operator's formula and limits).

They have no counterpart in the reference, whose layers are float32 on host slices.  Every function takes a `Device`
(goneuron_b200.sequential) and tensors on that GPU; it enqueues its kernels on torch's current stream there, waits for nothing
and can be captured into a CUDA graph.  Outputs and workspaces are torch allocations of the call.  Wrong arguments raise
ValueError, failures of the library GoNeuronCudaError; what only the kernels can find (an index out of range) is kept until
`check` reads it."""
import ctypes as C

from . import _lib


class _Heads(C.Structure):
    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64), ("heads", C.c_int32), ("reserved", C.c_int32)]


def _torch():
    import torch
    return torch


def _dtype(t):
    torch = _torch()
    return {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}.get(t.dtype)


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _tensor(dev, name, t, dims=None, dtype=None, dense=False):
    """Checks one argument; its values are not looked at."""
    torch = _torch()
    _need(isinstance(t, torch.Tensor), f"{name} is not a torch tensor")
    _need(t.is_cuda and t.device.index == dev.device, f"{name} is on {t.device}, the operator runs on cuda:{dev.device}")
    _need(dims is None or t.dim() in ((dims,) if isinstance(dims, int) else dims), f"{name} has {t.dim()} dimensions, {dims} are needed")
    _need(dtype is None or t.dtype == dtype, f"{name} is {t.dtype}, {dtype} is needed")
    _need(not dense or t.is_contiguous(), f"{name} is not contiguous")
    return t


def _floating(dev, name, t, dims, dtype=None):
    _tensor(dev, name, t, dims, dtype)
    _need(_dtype(t) is not None, f"{name} is {t.dtype}: float32, float16 or bfloat16 is needed")
    _need(t.numel() == 0 or t.shape[-1] <= 1 or t.stride(-1) == 1, f"the last dimension of {name} is not contiguous")
    return t


def _index(dev, name, t):
    torch = _torch()
    _tensor(dev, name, t, dense=True)
    _need(t.dtype in (torch.int32, torch.int64), f"{name} is {t.dtype}: int32 or int64 is needed")
    return t, int(t.dtype == torch.int64)


def _p(t):
    return None if t is None or t.numel() == 0 else C.c_void_p(t.data_ptr())


def _stream(dev):
    return C.c_void_p(_torch().cuda.current_stream(dev.device).cuda_stream)


def _workspace(dev, function, *args):
    """A workspace of the bytes that the C function gives, and those."""
    n = C.c_int64()
    _lib.check(function(dev.handle, *args, C.byref(n)))
    torch = _torch()
    return torch.empty(n.value, dtype=torch.uint8, device=f"cuda:{dev.device}"), n.value


def check(dev):
    """Waits for the current stream and raises GoNeuronCudaError for what operators found wrong on the GPU since the last call
    that did: an id or index out of range, a bounded wait that gave up."""
    _lib.check(_lib.load().gn_op_status(dev.handle, _stream(dev)))


# ------------------------------------------------------------------ norm of queries and keys with the rotation
def _as_heads(dev, name, t, like=None):
    """[tokens, heads, size] of a tensor [..., heads, size] without copying."""
    _floating(dev, name, t, (3, 4), None if like is None else like.dtype)
    _need(like is None or t.shape == like.shape, f"{name} has shape {tuple(t.shape)}" + ("" if like is None else f", {tuple(like.shape)} is needed"))
    if t.dim() == 4:
        try:
            t = t.view(t.shape[0] * t.shape[1], t.shape[2], t.shape[3])
        except RuntimeError:
            raise ValueError(f"{name}: the strides of its first two dimensions do not make one of tokens") from None
    return t


def _heads(t):
    return None if t is None else C.byref(_Heads(t.data_ptr() if t.numel() else None, t.stride(0), t.stride(1), t.shape[1], 0))


def _qk(dev, q, k, gain_q, gain_k, positions, frequencies):
    torch = _torch()
    q3 = _as_heads(dev, "q", q)
    n, _, size = q3.shape
    k3 = None if k is None else _as_heads(dev, "k", k)
    _need(k3 is None or (k3.dtype == q3.dtype and k3.shape[0] == n and k3.shape[2] == size), "q and k differ in type, tokens or head size")
    for name, g in (("gain_q", gain_q), ("gain_k", gain_k)):
        _need(g is None or _tensor(dev, name, g, 1, torch.float32, True).shape[0] == size, f"{name} has another length than a head")
    wide, rotated = 0, 0
    if frequencies is not None:
        rotated = 2 * _tensor(dev, "frequencies", frequencies, 1, torch.float64, True).shape[0]
        _need(positions is not None, "positions are needed for a rotation")
        positions, wide = _index(dev, "positions", positions)
        _need(positions.numel() == n, "positions: one for each token is needed")
    return q3, k3, rotated, wide


def _qk_args(q3, k3, gain_q, gain_k, positions, frequencies, eps, interleaved, rotated, wide):
    return (_dtype(q3), q3.shape[0], q3.shape[2], rotated, int(bool(interleaved)), eps, _heads(q3), _heads(k3), _p(gain_q), _p(gain_k),
            _p(positions) if rotated else None, wide, _p(frequencies))


def qk_norm_rope(dev, q, k, gain_q=None, gain_k=None, positions=None, frequencies=None, eps=1e-5, interleaved=False, out=None):
    """RMS norm of every head of q and k ([tokens, heads, size] or [batch, tokens, heads, size]; any strides of the first dimensions,
    k may be None) with gains [size] (float32), then the rotation of the pairs by positions * frequencies.  Without frequencies
    ([rotated / 2], float64) nothing is rotated.  out: a pair of tensors for the results, q and k themselves among them."""
    q3, k3, rotated, wide = _qk(dev, q, k, gain_q, gain_k, positions, frequencies)
    torch = _torch()
    qo, ko = out if out is not None else (torch.empty(q.shape, dtype=q.dtype, device=q.device), None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device))
    qo3, ko3 = _as_heads(dev, "out[0]", qo, q), None if k is None else _as_heads(dev, "out[1]", ko, k)
    _lib.check(_lib.load().gn_op_qk_norm_rope(dev.handle, *_qk_args(q3, k3, gain_q, gain_k, positions, frequencies, eps, interleaved, rotated, wide),
                                              _heads(qo3), _heads(ko3), _stream(dev)))
    return qo, ko


def qk_norm_rope_backward(dev, dq_out, dk_out, q, k, gain_q=None, gain_k=None, positions=None, frequencies=None, eps=1e-5, interleaved=False):
    """Gradients (dq, dk, dgain_q, dgain_k) from those of the outputs and the forward call's inputs; those of the gains are float32."""
    q3, k3, rotated, wide = _qk(dev, q, k, gain_q, gain_k, positions, frequencies)
    torch = _torch()
    dqo = _as_heads(dev, "dq_out", dq_out, q)
    dko = None if k is None else _as_heads(dev, "dk_out", dk_out, k)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    size = q3.shape[2]
    gains = [None if g is None or t is None else torch.empty(size, dtype=torch.float32, device=q.device) for g, t in ((gain_q, q), (gain_k, k))]
    L = _lib.load()
    ws, n = _workspace(dev, L.gn_op_qk_norm_rope_workspace, q3.shape[0], q3.shape[1], 0 if k3 is None else k3.shape[1], size)
    _lib.check(L.gn_op_qk_norm_rope_backward(dev.handle, *_qk_args(q3, k3, gain_q, gain_k, positions, frequencies, eps, interleaved, rotated, wide),
                                             _heads(dqo), _heads(dko), _heads(_as_heads(dev, "dq", dq)), _heads(None if dk is None else _as_heads(dev, "dk", dk)),
                                             _p(gains[0]), _p(gains[1]), _p(ws), n, _stream(dev)))
    return dq, dk, gains[0], gains[1]


# ------------------------------------------------------------------ distillation
def _distill(dev, logits, top_ids, top_logits, temperature, row_weight, dlogits):
    torch = _torch()
    _floating(dev, "logits", logits, 2)
    rows, vocab = logits.shape
    top_ids, wide = _index(dev, "top_ids", top_ids)
    _tensor(dev, "top_logits", top_logits, 2, torch.float32, True)
    _need(top_ids.shape == top_logits.shape and top_ids.shape[0] == rows, "top_ids and top_logits: [rows, top] each are needed")
    if row_weight is not None:
        _need(_tensor(dev, "row_weight", row_weight, 1, torch.float32, True).shape[0] == rows, "row_weight: one for each row is needed")
    loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _lib.check(_lib.load().gn_op_distill(dev.handle, _dtype(logits), rows, vocab, top_ids.shape[1], temperature, _p(logits), logits.stride(0), _p(top_ids), wide,
                                         _p(top_logits), _p(row_weight), _p(loss), _p(dlogits), 0 if dlogits is None else dlogits.stride(0), _stream(dev)))
    return loss


def distill_loss(dev, logits, top_ids, top_logits, temperature=1.0, row_weight=None):
    """Loss of each row of logits [rows, vocab] against the teacher's top logits (top_ids with -1 for unused entries, top_logits float32,
    [rows, top] each), times row_weight."""
    return _distill(dev, logits, top_ids, top_logits, temperature, row_weight, None)


def distill_loss_grad(dev, logits, top_ids, top_logits, temperature=1.0, row_weight=None, out=None):
    """(loss, dlogits): the same with the derivative of each row's loss by its logits, which are read once.  out: a tensor for dlogits, logits among them."""
    torch = _torch()
    _floating(dev, "logits", logits, 2)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if out is None else _floating(dev, "out", out, 2, logits.dtype)
    _need(d.shape == logits.shape, "out has another shape than logits")
    return _distill(dev, logits, top_ids, top_logits, temperature, row_weight, d), d


# ------------------------------------------------------------------ embedding
def embedding(dev, table, ids, scale=1.0):
    """scale * table[ids]: [..., dim] for ids of any shape; rows of zeros where an id is -1."""
    torch = _torch()
    _floating(dev, "table", table, 2)
    ids, wide = _index(dev, "ids", ids)
    out = torch.empty(*ids.shape, table.shape[1], dtype=table.dtype, device=table.device)
    _lib.check(_lib.load().gn_op_embedding(dev.handle, _dtype(table), ids.numel(), table.shape[0], table.shape[1], scale, _p(table), table.stride(0), _p(ids), wide,
                                           _p(out), table.shape[1], _stream(dev)))
    return out


def embedding_backward(dev, dout, ids, vocab, scale=1.0):
    """Gradient of the table, float32 [vocab, dim], from that of the lookup's output [..., dim]."""
    torch = _torch()
    ids, wide = _index(dev, "ids", ids)
    _tensor(dev, "dout", dout)
    _need(dout.dim() == ids.dim() + 1 and dout.shape[:-1] == ids.shape, "dout: a row for each id is needed")
    dim = dout.shape[-1]
    try:
        rows = dout.view(ids.numel(), dim)
    except RuntimeError:
        raise ValueError("dout: the strides of its first dimensions do not make one of tokens") from None
    _floating(dev, "dout", rows, 2)
    dtable = torch.empty(vocab, dim, dtype=torch.float32, device=dout.device)
    L = _lib.load()
    ws, n = _workspace(dev, L.gn_op_embedding_workspace, ids.numel(), vocab, dim)
    _lib.check(L.gn_op_embedding_backward(dev.handle, _dtype(rows), ids.numel(), vocab, dim, scale, _p(rows), rows.stride(0), _p(ids), wide, _p(dtable), _p(ws), n, _stream(dev)))
    return dtable
