"""Operators of language models on torch CUDA tensors, over the C ABI of libgoneuron_cuda.so (the last part of
include/goneuron_cuda.h, which states each operator's formula and limits).

They have no counterpart in the reference, whose layers are float32 on host slices.  Every function takes a `Device`
(goneuron_b200.sequential) and tensors on that GPU; it enqueues its kernels on torch's current stream there, waits for nothing
and can be captured into a CUDA graph.  Outputs and workspaces are torch allocations of the call.  Inputs' autograd history is not
followed: outputs do not require a gradient, and each operator's gradient is a call of its own.  A tensor given as `out` is
written like any that torch changes in place: one that requires a gradient is refused outside torch.no_grad(), and a backward
pass that has kept it raises torch's error.  Wrong arguments raise ValueError (TypeError where a tensor is none), failures of
the library GoNeuronCudaError; what only the kernels can find (an index out of range, a bounded wait that gave up) is kept
until `check` reads it.

The functions' bodies are compiled (csrc/torch_operators.cpp)."""
import torch  # noqa: F401  (its libraries have to be there before the module below)

from . import _lib
from .descriptors import GELU, RELU, SILU

_lib.load()
try:
    from . import _torch_operators as _ops
except ImportError as e:
    raise ImportError("goneuron_b200/_torch_operators.so is missing or does not fit this torch: build it with `python -m goneuron_b200.build`") from e
_ops.set_error(_lib.GoNeuronCudaError)

_ACTIVATION = {"silu": SILU, "gelu": GELU, "relu": RELU}


def _handle(dev):
    return dev.handle.value if dev.handle else 0      # (a closed device: the library refuses the call)


def check(dev):
    """Waits for the current stream and raises GoNeuronCudaError for what operators found wrong on the GPU since the last call
    that did, on whatever stream, thread or Device of it: an id or index out of range, a bounded wait that gave up."""
    _ops.status(_handle(dev), dev.device)


def qk_norm_rope(dev, q, k, gain_q=None, gain_k=None, positions=None, frequencies=None, eps=1e-5, interleaved=False, out=None):
    """RMS norm of every head of q and k ([tokens, heads, size] or [batch, tokens, heads, size]; any strides of the first dimensions,
    k may be None) with gains [size] (float32), then the rotation of the pairs by positions * frequencies.  Without frequencies
    ([rotated / 2], float64) nothing is rotated.  out: a pair of tensors for the results, (q, k) themselves for in place; the queries' must not lie on the
    keys', nor the other way round."""
    qo, ko = (None, None) if out is None else out
    return _ops.qk_norm_rope(_handle(dev), dev.device, q, k, gain_q, gain_k, positions, frequencies, eps, interleaved, qo, ko)


def qk_norm_rope_backward(dev, dq_out, dk_out, q, k, gain_q=None, gain_k=None, positions=None, frequencies=None, eps=1e-5, interleaved=False):
    """Gradients (dq, dk, dgain_q, dgain_k) from those of the outputs and the forward call's inputs; those of the gains are float32."""
    return _ops.qk_norm_rope_backward(_handle(dev), dev.device, dq_out, dk_out, q, k, gain_q, gain_k, positions, frequencies, eps, interleaved)


def distill_loss(dev, logits, top_ids, top_logits, temperature=1.0, row_weight=None):
    """Loss of each row of logits [rows, vocab] against the teacher's top logits (top_ids with -1 for unused entries, top_logits float32,
    [rows, top] each), times row_weight."""
    return _ops.distill(_handle(dev), dev.device, logits, top_ids, top_logits, temperature, row_weight, False, None)[0]


def distill_loss_grad(dev, logits, top_ids, top_logits, temperature=1.0, row_weight=None, out=None):
    """(loss, dlogits): the same with the derivative of each row's loss by its logits, which are read once.  out: a tensor for dlogits, logits itself for in place, else
    not on any part of it."""
    return _ops.distill(_handle(dev), dev.device, logits, top_ids, top_logits, temperature, row_weight, True, out)


def embedding(dev, table, ids, scale=1.0):
    """scale * table[ids]: [..., dim] for ids of any shape; rows of zeros where an id is -1."""
    return _ops.embedding(_handle(dev), dev.device, table, ids, scale)


def embedding_backward(dev, dout, ids, vocab, scale=1.0):
    """Gradient of the table, float32 [vocab, dim], from that of the lookup's output [..., dim]."""
    return _ops.embedding_backward(_handle(dev), dev.device, dout, ids, vocab, scale)


def _activation(name):
    try:
        return _ACTIVATION[name]
    except KeyError:
        raise ValueError(f"activation {name!r} is none of {sorted(_ACTIVATION)}") from None


def gated_ffn(dev, x, w_gate, w_up, w_down, activation="silu", save=False):
    """(act(x w_gate^T) * (x w_up^T)) w_down^T for x [..., dim], w_gate and w_up [ff, dim], w_down [dim, ff]; activation "silu", "gelu" (tanh form)
    or "relu".  save: also returns what gated_ffn_backward reads, (y, saved).  act(..) * (..) is rounded to x's type between the
    products: in float16 above 65504 it is infinite, and so is its row of y, where bfloat16 would hold it."""
    r = _ops.gated_ffn(_handle(dev), dev.device, x, w_gate, w_up, w_down, _activation(activation), save)
    return r if save else r[0]


def gated_ffn_backward(dev, dy, x, w_gate, w_up, w_down, saved, activation="silu"):
    """Gradients (dx, dw_gate, dw_up, dw_down) from that of y, the forward call's inputs and what it saved.  The gradients of
    both projections are rounded to x's type on the way: in float16 a loss scale has to leave room for them (65504), and what is below 2^-25 is lost."""
    return _ops.gated_ffn_backward(_handle(dev), dev.device, dy, x, w_gate, w_up, w_down, saved, _activation(activation))
