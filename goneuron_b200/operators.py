"""Operators of language models on torch CUDA tensors, over the C ABI of libgoneuron_cuda.so (the last part of
include/goneuron_cuda.h, which states each operator's formula and limits).

They have no counterpart in the reference, whose layers are float32 on host slices.  Every function takes a `Device`
(goneuron_b200.sequential) and tensors on that GPU; it enqueues its kernels on torch's current stream there, waits for nothing
and can be captured into a CUDA graph.  Outputs and workspaces are torch allocations of the call.  Wrong arguments raise
ValueError, failures of the library GoNeuronCudaError; what only the kernels can find (an index out of range) is kept until
`check` reads it.

A decoding step's kernel takes less time than an ordinary Python function around it: messages are formatted only when they are
raised, and structures go to the library as packed bytes (norm of queries and keys for five tokens: 52 us a call with messages
formatted ahead and ctypes structures)."""
import ctypes as C
from struct import Struct

import torch

from . import _lib
from .descriptors import GELU, RELU, SILU

_F32, _F64, _I32, _I64 = torch.float32, torch.float64, torch.int32, torch.int64
_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ACTIVATION = {"silu": SILU, "gelu": GELU, "relu": RELU}
_heads_struct = Struct("@qqqii").pack      # gn_heads: data, token_stride, head_stride, heads, reserved
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else lambda i: torch.cuda.current_stream(i).cuda_stream


def _here(dev, name, t):
    """Refuses what is not a tensor on the device's GPU."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} is not a torch tensor")
    if not t.is_cuda or t.get_device() != dev.device:
        raise ValueError(f"{name} is on {t.device}, the operator runs on cuda:{dev.device}")


def _floating(dev, name, t, dtype=None):
    """... or not of a floating type (of `dtype`), or without a contiguous last dimension; returns its shape."""
    _here(dev, name, t)
    if t.dtype is not dtype and (dtype is not None or t.dtype not in _DTYPE):
        raise ValueError(f"{name} is {t.dtype}: {dtype or 'float32, float16 or bfloat16'} is needed")
    shape = t.shape
    if len(shape) == 0 or (t.stride(-1) != 1 and shape[-1] > 1 and t.numel()):
        raise ValueError(f"the last dimension of {name} is not contiguous")
    return shape


def _dense(dev, name, t, dtype, *shape):
    """... or not a contiguous tensor of this type and shape (-1: any)."""
    _here(dev, name, t)
    if t.dtype is not dtype or not t.is_contiguous():
        raise ValueError(f"{name} is {t.dtype}{'' if t.is_contiguous() else ' and not contiguous'}: contiguous {dtype} is needed")
    if t.dim() != len(shape) or any(n != m for n, m in zip(t.shape, shape) if m >= 0):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, {shape} is needed")


def _index(dev, name, t):
    """... or not contiguous int32 or int64; returns its gn_index_type."""
    _here(dev, name, t)
    if t.dtype is _I64:
        wide = 1
    elif t.dtype is _I32:
        wide = 0
    else:
        raise ValueError(f"{name} is {t.dtype}: int32 or int64 is needed")
    if not t.is_contiguous():
        raise ValueError(f"{name} is not contiguous")
    return wide


def _p(t):
    return None if t is None else t.data_ptr() or None


def _workspace(dev, like, function, *args):
    """A workspace of the bytes that the C function gives, and those."""
    n = C.c_int64()
    _lib.check(function(dev.handle, *args, C.byref(n)))
    return like.new_empty(n.value, dtype=torch.uint8), n.value


def check(dev):
    """Waits for the current stream and raises GoNeuronCudaError for what operators found wrong on the GPU since the last call
    that did: an id or index out of range, a bounded wait that gave up."""
    _lib.check(_lib.load().gn_op_status(dev.handle, _raw_stream(dev.device)))


# ------------------------------------------------------------------ norm of queries and keys with the rotation
def _heads(dev, name, t, like=None):
    """gn_heads of a tensor [..., heads, size] without copying, and its tokens, heads and head size."""
    shape = _floating(dev, name, t, None if like is None else like.dtype)
    if like is not None and shape != like.shape:
        raise ValueError(f"{name} has shape {tuple(shape)}, {tuple(like.shape)} is needed")
    if len(shape) == 4:
        try:
            t = t.view(shape[0] * shape[1], shape[2], shape[3])
        except RuntimeError:
            raise ValueError(f"{name}: the strides of its first two dimensions do not make one of tokens") from None
        shape = t.shape
    elif len(shape) != 3:
        raise ValueError(f"{name} has {len(shape)} dimensions: [tokens, heads, size] or [batch, tokens, heads, size] is needed")
    stride = t.stride()
    return _heads_struct(t.data_ptr(), stride[0], stride[1], shape[1], 0), shape


def _qk(dev, q, k, gain_q, gain_k, positions, frequencies, eps, interleaved):
    """The arguments that both directions begin with; tokens, heads of q and k, head size."""
    hq, (n, heads, size) = _heads(dev, "q", q)
    hk, kv = None, 0
    if k is not None:
        hk, (n_k, kv, size_k) = _heads(dev, "k", k)
        if k.dtype is not q.dtype or n_k != n or size_k != size:
            raise ValueError("q and k differ in type, tokens or head size")
    if gain_q is not None:
        _dense(dev, "gain_q", gain_q, _F32, size)
    if gain_k is not None:
        _dense(dev, "gain_k", gain_k, _F32, size)
    wide, rotated, at = 0, 0, None
    if frequencies is not None:
        _dense(dev, "frequencies", frequencies, _F64, -1)
        rotated = 2 * frequencies.shape[0]
        if positions is None:
            raise ValueError("positions are needed for a rotation")
        wide, at = _index(dev, "positions", positions), positions.data_ptr() or None
        if positions.numel() != n:
            raise ValueError("positions: one for each token is needed")
    return (_DTYPE[q.dtype], n, size, rotated, 1 if interleaved else 0, eps, hq, hk, _p(gain_q), _p(gain_k), at, wide, _p(frequencies)), n, heads, kv, size


def qk_norm_rope(dev, q, k, gain_q=None, gain_k=None, positions=None, frequencies=None, eps=1e-5, interleaved=False, out=None):
    """RMS norm of every head of q and k ([tokens, heads, size] or [batch, tokens, heads, size]; any strides of the first dimensions,
    k may be None) with gains [size] (float32), then the rotation of the pairs by positions * frequencies.  Without frequencies
    ([rotated / 2], float64) nothing is rotated.  out: a pair of tensors for the results, q and k themselves among them."""
    args = _qk(dev, q, k, gain_q, gain_k, positions, frequencies, eps, interleaved)[0]
    qo, ko = out if out is not None else (q.new_empty(q.shape), None if k is None else k.new_empty(k.shape))
    _lib.check(_lib.load().gn_op_qk_norm_rope(dev.handle, *args, _heads(dev, "out[0]", qo, q)[0], None if k is None else _heads(dev, "out[1]", ko, k)[0], _raw_stream(dev.device)))
    return qo, ko


def qk_norm_rope_backward(dev, dq_out, dk_out, q, k, gain_q=None, gain_k=None, positions=None, frequencies=None, eps=1e-5, interleaved=False):
    """Gradients (dq, dk, dgain_q, dgain_k) from those of the outputs and the forward call's inputs; those of the gains are float32."""
    args, n, heads, kv, size = _qk(dev, q, k, gain_q, gain_k, positions, frequencies, eps, interleaved)
    hdq, hdk = _heads(dev, "dq_out", dq_out, q)[0], None if k is None else _heads(dev, "dk_out", dk_out, k)[0]
    dq, dk = q.new_empty(q.shape), None if k is None else k.new_empty(k.shape)
    dgq = None if gain_q is None else gain_q.new_empty(size)
    dgk = None if gain_k is None or k is None else gain_k.new_empty(size)
    L = _lib.load()
    ws, bytes_ = _workspace(dev, q, L.gn_op_qk_norm_rope_workspace, n, heads, kv, size) if dgq is not None or dgk is not None else (None, 0)
    _lib.check(L.gn_op_qk_norm_rope_backward(dev.handle, *args, hdq, hdk, _heads(dev, "dq", dq)[0], None if k is None else _heads(dev, "dk", dk)[0],
                                             _p(dgq), _p(dgk), _p(ws), bytes_, _raw_stream(dev.device)))
    return dq, dk, dgq, dgk


# ------------------------------------------------------------------ distillation
def _distill(dev, logits, shape, top_ids, top_logits, temperature, row_weight, dlogits):
    if len(shape) != 2:
        raise ValueError(f"logits has shape {tuple(shape)}: [rows, vocabulary] is needed")
    rows, vocab = shape
    wide = _index(dev, "top_ids", top_ids)
    _dense(dev, "top_logits", top_logits, _F32, rows, -1)
    if top_ids.shape != top_logits.shape:
        raise ValueError(f"top_ids has shape {tuple(top_ids.shape)}, top_logits {tuple(top_logits.shape)}")
    if row_weight is not None:
        _dense(dev, "row_weight", row_weight, _F32, rows)
    loss, L = top_logits.new_empty(rows), _lib.load()
    ws, bytes_ = _workspace(dev, logits, L.gn_op_distill_workspace, rows, top_ids.shape[1], dlogits is not None)
    _lib.check(L.gn_op_distill(dev.handle, _DTYPE[logits.dtype], rows, vocab, top_ids.shape[1], temperature, _p(logits), logits.stride(0), _p(top_ids), wide, _p(top_logits),
                               _p(row_weight), _p(loss), _p(dlogits), 0 if dlogits is None else dlogits.stride(0), _p(ws), bytes_, _raw_stream(dev.device)))
    return loss


def distill_loss(dev, logits, top_ids, top_logits, temperature=1.0, row_weight=None):
    """Loss of each row of logits [rows, vocab] against the teacher's top logits (top_ids with -1 for unused entries, top_logits float32,
    [rows, top] each), times row_weight."""
    return _distill(dev, logits, _floating(dev, "logits", logits), top_ids, top_logits, temperature, row_weight, None)


def distill_loss_grad(dev, logits, top_ids, top_logits, temperature=1.0, row_weight=None, out=None):
    """(loss, dlogits): the same with the derivative of each row's loss by its logits, which are read once.  out: a tensor for dlogits, logits among them."""
    shape = _floating(dev, "logits", logits)
    if out is None:
        out = logits.new_empty(shape)
    elif _floating(dev, "out", out, logits.dtype) != shape:
        raise ValueError("out has another shape than logits")
    return _distill(dev, logits, shape, top_ids, top_logits, temperature, row_weight, out), out


# ------------------------------------------------------------------ embedding
def embedding(dev, table, ids, scale=1.0):
    """scale * table[ids]: [..., dim] for ids of any shape; rows of zeros where an id is -1."""
    shape = _floating(dev, "table", table)
    if len(shape) != 2:
        raise ValueError(f"table has shape {tuple(shape)}: [vocab, dim] is needed")
    wide = _index(dev, "ids", ids)
    vocab, dim = shape
    out = table.new_empty((*ids.shape, dim))
    _lib.check(_lib.load().gn_op_embedding(dev.handle, _DTYPE[table.dtype], ids.numel(), vocab, dim, scale, _p(table), table.stride(0), _p(ids), wide, _p(out), dim, _raw_stream(dev.device)))
    return out


def embedding_backward(dev, dout, ids, vocab, scale=1.0):
    """Gradient of the table, float32 [vocab, dim], from that of the lookup's output [..., dim]."""
    wide = _index(dev, "ids", ids)
    rows, dim = _rows(dev, "dout", dout)
    if dout.shape[:-1] != ids.shape:
        raise ValueError("dout: a row for each id is needed")
    dtable = dout.new_empty((vocab, dim), dtype=_F32)
    L, n = _lib.load(), ids.numel()
    ws, bytes_ = _workspace(dev, dout, L.gn_op_embedding_workspace, n, vocab, dim)
    _lib.check(L.gn_op_embedding_backward(dev.handle, _DTYPE[dout.dtype], n, vocab, dim, scale, _p(rows), rows.stride(0), _p(ids), wide, _p(dtable), _p(ws), bytes_, _raw_stream(dev.device)))
    return dtable


def _rows(dev, name, t, like=None):
    """[tokens, dim] of a tensor [..., dim] without copying, and dim."""
    shape = _floating(dev, name, t, None if like is None else like.dtype)
    if like is not None and shape != like.shape:
        raise ValueError(f"{name} has shape {tuple(shape)}, {tuple(like.shape)} is needed")
    dim = shape[-1]
    if len(shape) == 2:
        return t, dim
    try:
        return t.view(t.numel() // dim if dim else 0, dim), dim
    except RuntimeError:
        raise ValueError(f"{name}: the strides of its first dimensions do not make one of tokens") from None


# ------------------------------------------------------------------ gated feed-forward block
def _ffn(dev, x, w_gate, w_up, w_down, activation):
    """x as rows, dim and ff."""
    if activation not in _ACTIVATION:
        raise ValueError(f"activation {activation!r} is none of {sorted(_ACTIVATION)}")
    rows, dim = _rows(dev, "x", x)
    t = x.dtype
    if t is _F32:
        raise ValueError("x is float32: float16 or bfloat16 is needed (TransformerBlock has the 32-bit form)")
    _dense(dev, "w_gate", w_gate, t, -1, dim)
    ff = w_gate.shape[0]
    _dense(dev, "w_up", w_up, t, ff, dim)
    _dense(dev, "w_down", w_down, t, dim, ff)
    return rows, dim, ff


def gated_ffn(dev, x, w_gate, w_up, w_down, activation="silu", save=False):
    """(act(x w_gate^T) * (x w_up^T)) w_down^T for x [..., dim], w_gate and w_up [ff, dim], w_down [dim, ff]; activation "silu", "gelu" (tanh form)
    or "relu".  save: also returns what gated_ffn_backward reads, (y, saved)."""
    rows, dim, ff = _ffn(dev, x, w_gate, w_up, w_down, activation)
    L, n = _lib.load(), rows.shape[0]
    y = x.new_empty(x.shape)
    saved = _workspace(dev, x, L.gn_op_gated_ffn_saved, n, dim, ff)[0] if save else None
    ws, bytes_ = _workspace(dev, x, L.gn_op_gated_ffn_workspace, n, dim, ff, 0)
    _lib.check(L.gn_op_gated_ffn(dev.handle, _DTYPE[x.dtype], _ACTIVATION[activation], n, dim, ff, _p(rows), rows.stride(0), _p(w_gate), _p(w_up), _p(w_down),
                                 _p(y), dim, _p(saved), _p(ws), bytes_, _raw_stream(dev.device)))
    return (y, saved) if save else y


def gated_ffn_backward(dev, dy, x, w_gate, w_up, w_down, saved, activation="silu"):
    """Gradients (dx, dw_gate, dw_up, dw_down) from that of y, the forward call's inputs and what it saved."""
    rows, dim, ff = _ffn(dev, x, w_gate, w_up, w_down, activation)
    d = _rows(dev, "dy", dy, x)[0]
    L, n, size = _lib.load(), rows.shape[0], C.c_int64()
    _lib.check(L.gn_op_gated_ffn_saved(dev.handle, n, dim, ff, C.byref(size)))
    _dense(dev, "saved", saved, torch.uint8, size.value)
    dx, dwg, dwu, dwd = x.new_empty(x.shape), w_gate.new_empty((ff, dim)), w_gate.new_empty((ff, dim)), w_gate.new_empty((dim, ff))
    ws, bytes_ = _workspace(dev, x, L.gn_op_gated_ffn_workspace, n, dim, ff, 1)
    _lib.check(L.gn_op_gated_ffn_backward(dev.handle, _DTYPE[x.dtype], _ACTIVATION[activation], n, dim, ff, _p(d), d.stride(0), _p(rows), rows.stride(0), _p(w_gate), _p(w_up), _p(w_down),
                                          _p(saved), _p(dx), dim, _p(dwg), _p(dwu), _p(dwd), _p(ws), bytes_, _raw_stream(dev.device)))
    return dx, dwg, dwu, dwd
