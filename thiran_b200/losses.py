"""Losses over a large vocabulary, with their gradients (thb_linear_loss_*, thb_distill_*).

Three operators over rows (tokens) of torch CUDA tensors:

* `linear_cross_entropy`: softmax cross entropy of z = scale * hidden @ weight.T
  against labels. z is never stored.
* `linear_distillation`: the divergence of softmax(hidden @ weight.T / temperature)
  from a teacher's top logits, q = softmax(teacher_logits / temperature). z is never stored.
* `distillation`: the same divergence for student logits in memory.

loss = sum_k q_k (log q_k - z_{id_k}) + log sum_v exp(z_v) per row; for a label q = 1. The
divergence is that of the softened distributions (no factor temperature ** 2). A row whose label
is `ignore_index`, or whose teacher list has no entry (ids < 0 and logits of -inf are not there),
has loss, log-sum-exp and gradients 0 and costs no products. A label or id outside the vocabulary
makes the row's loss NaN, leaves it out of the gradients, and raises TH-SPEC-BOUNDS from
`check_device_status`.

Outputs are passed in, as for `gemm`, and every call is ordered on `stream` (a raw handle, the
default stream if 0): tensors that another stream allocated or uses must be kept alive and ordered
by the caller. hidden, weight and their gradients are bf16 [rows][dim] and [vocab][dim] with any
row stride; labels and teacher_ids are int64; loss, lse and grad_loss are f32 and contiguous.
A workspace holds nothing between calls, but calls that may run at the same time (other streams,
graphs replayed side by side) need one each.
"""
from __future__ import annotations

import ctypes as C
import threading


class LinearLossDesc(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("vocab", C.c_uint64), ("dim", C.c_uint64), ("hidden", C.c_void_p),
                ("ld_hidden", C.c_uint64), ("weight", C.c_void_p), ("ld_weight", C.c_uint64), ("labels", C.c_void_p),
                ("ignore_index", C.c_int64), ("teacher_ids", C.c_void_p), ("teacher_logits", C.c_void_p),
                ("teacher_dtype", C.c_uint32), ("entries", C.c_uint64), ("scale", C.c_float), ("loss", C.c_void_p),
                ("lse", C.c_void_p), ("grad_loss", C.c_void_p), ("grad_hidden", C.c_void_p),
                ("ld_grad_hidden", C.c_uint64), ("grad_weight", C.c_void_p), ("ld_grad_weight", C.c_uint64),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


class DistillDesc(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("vocab", C.c_uint64), ("logits", C.c_void_p), ("ld_logits", C.c_uint64),
                ("dtype", C.c_uint32), ("teacher_ids", C.c_void_p), ("teacher_logits", C.c_void_p),
                ("teacher_dtype", C.c_uint32), ("entries", C.c_uint64), ("scale", C.c_float), ("loss", C.c_void_p),
                ("lse", C.c_void_p), ("grad_loss", C.c_void_p), ("grad_logits", C.c_void_p),
                ("ld_grad_logits", C.c_uint64)]


SIGNATURES = {
    "thb_linear_loss_workspace": (C.c_int, [C.c_int, C.c_uint64, C.c_uint64, C.c_uint64, C.c_uint64, C.c_int, C.c_int,
                                            C.POINTER(C.c_uint64), C.c_char_p, C.c_uint64]),
    "thb_linear_loss_forward": (C.c_int, [C.c_int, C.POINTER(LinearLossDesc), C.c_void_p, C.c_char_p, C.c_uint64]),
    "thb_linear_loss_backward": (C.c_int, [C.c_int, C.POINTER(LinearLossDesc), C.c_void_p, C.c_char_p, C.c_uint64]),
    "thb_distill_forward": (C.c_int, [C.c_int, C.POINTER(DistillDesc), C.c_void_p, C.c_char_p, C.c_uint64]),
    "thb_distill_backward": (C.c_int, [C.c_int, C.POINTER(DistillDesc), C.c_void_p, C.c_char_p, C.c_uint64]),
}

_F32, _BF16 = 2, 3  # THB_DTYPE_*
_DTYPES = {}        # torch dtype -> THB_DTYPE_*, filled with the rest on the first call
_f32 = _bf16 = _i64 = _lib = _raise = None
_local = threading.local()  # a failure buffer for each thread


def _bad(text):
    from . import STATUS_ABI, GpuError
    raise GpuError(STATUS_ABI, "GPU-LOSS-ARGUMENT: " + text)


def _load():
    """torch's types and the library, looked up once (the package itself needs no torch)."""
    global _f32, _bf16, _i64, _lib, _raise
    import torch

    import thiran_b200 as package
    _f32, _bf16, _i64 = torch.float32, torch.bfloat16, torch.int64
    _DTYPES.update({_f32: _F32, _bf16: _BF16})
    _raise, _lib = package._raise, package.lib()


def _failure():
    try:
        return _local.buffer
    except AttributeError:
        _local.buffer = C.create_string_buffer(1024)
        return _local.buffer


def _call(function, device, desc, stream):
    fail = _failure()
    status = function(device, C.byref(desc), stream, fail, 1024)
    if status:
        _raise(status, fail)


def _wrong(name, t, dtype, ordinal):
    if t.dtype is not dtype:
        _bad(f"{name} is {t.dtype}, expected {dtype}")
    _bad(f"{name} is on {t.device}, expected CUDA device {ordinal}")


def _matrix(name, t, rows, cols, dtype, ordinal):
    """(pointer, row stride) of a [rows][cols] tensor with contiguous rows on CUDA device `ordinal`."""
    if t.shape != (rows, cols):
        _bad(f"{name} has shape {list(t.shape)}, expected {[rows, cols]}")
    if t.dtype is not dtype or t.get_device() != ordinal:
        _wrong(name, t, dtype, ordinal)
    step, inner = t.stride()
    if inner != 1 and cols > 1:
        _bad(f"{name} has rows that are not contiguous")
    if step < cols:
        if rows > 1:
            _bad(f"{name} has overlapping rows")
        step = cols
    return t.data_ptr(), step


def _vector(name, t, rows, dtype, ordinal):
    if t.shape != (rows,):
        _bad(f"{name} has shape {list(t.shape)}, expected {[rows]}")
    if t.dtype is not dtype or t.get_device() != ordinal:
        _wrong(name, t, dtype, ordinal)
    if rows > 1 and t.stride(0) != 1:
        _bad(f"{name} is not contiguous")
    return t.data_ptr()


def _place(t, name):
    """The CUDA ordinal of the tensor that decides it; loads what the calls need."""
    if _lib is None:
        _load()
    ordinal = t.get_device()
    if ordinal < 0:
        _bad(f"{name} is on {t.device}, expected a CUDA device")
    if t.dim() != 2:
        _bad(f"{name} has shape {list(t.shape)}, expected two dimensions")
    return ordinal


def _teacher(desc, ids, logits, rows, ordinal):
    if ids.dim() != 2:
        _bad(f"teacher_ids has shape {list(ids.shape)}, expected two dimensions")
    entries = ids.shape[1]
    dtype = logits.dtype
    kind = _DTYPES.get(dtype)
    if kind is None:
        _bad(f"teacher_logits is {dtype}, expected torch.float32 or torch.bfloat16")
    desc.teacher_ids, ld = _matrix("teacher_ids", ids, rows, entries, _i64, ordinal)
    desc.teacher_logits, ld2 = _matrix("teacher_logits", logits, rows, entries, dtype, ordinal)
    if rows > 1 and (ld != entries or ld2 != entries):
        _bad("teacher_ids and teacher_logits must be contiguous")
    desc.teacher_dtype, desc.entries = kind, entries


def _temperature(value):
    if not value > 0.0:
        _bad("temperature must be positive")
    return 1.0 / value


def linear_loss_workspace(rows, vocab, dim, entries=1, backward=True, aligned=None, device=0):
    """Bytes of workspace that a linear loss over these sizes needs. With `backward` it serves the
    forward and the backward call over these rows; fewer rows may need more, so each size is to be
    asked for. `entries` is the length of the teacher's lists (labels: 1);
    `aligned` says whether every weight row starts at a multiple of 16 bytes (by default: whether
    contiguous rows do)."""
    if _lib is None:
        _load()
    fail = _failure()
    out = C.c_uint64()
    aligned = dim % 8 == 0 if aligned is None else aligned
    status = _lib.thb_linear_loss_workspace(device, rows, vocab, dim, entries, int(backward), int(aligned), C.byref(out),
                                            fail, 1024)
    if status:
        _raise(status, fail)
    return out.value


def _linear(hidden, weight, workspace, scale):
    ordinal = _place(hidden, "hidden")
    if weight.dim() != 2:
        _bad(f"weight has shape {list(weight.shape)}, expected two dimensions")
    rows, dim = hidden.shape
    vocab = weight.shape[0]
    pointer, ld = _matrix("hidden", hidden, rows, dim, _bf16, ordinal)
    weights, ldw = _matrix("weight", weight, vocab, dim, _bf16, ordinal)
    if workspace.get_device() != ordinal:
        _bad(f"workspace is on {workspace.device}, expected CUDA device {ordinal}")
    if not workspace.is_contiguous():
        _bad("workspace is not contiguous")
    desc = LinearLossDesc(rows, vocab, dim, pointer, ld, weights, ldw)
    desc.scale, desc.workspace, desc.workspace_bytes = scale, workspace.data_ptr(), workspace.nbytes
    return desc, rows, vocab, dim, ordinal


def _forward(desc, rows, ordinal, loss, lse, stream):
    desc.loss = _vector("loss", loss, rows, _f32, ordinal)
    desc.lse = _vector("lse", lse, rows, _f32, ordinal)
    _call(_lib.thb_linear_loss_forward, ordinal, desc, stream)


def _backward(desc, rows, vocab, dim, ordinal, lse, grad_loss, grad_hidden, grad_weight, stream):
    desc.lse = _vector("lse", lse, rows, _f32, ordinal)
    desc.grad_loss = _vector("grad_loss", grad_loss, rows, _f32, ordinal)
    desc.grad_hidden, desc.ld_grad_hidden = _matrix("grad_hidden", grad_hidden, rows, dim, _bf16, ordinal)
    desc.grad_weight, desc.ld_grad_weight = _matrix("grad_weight", grad_weight, vocab, dim, _bf16, ordinal)
    _call(_lib.thb_linear_loss_backward, ordinal, desc, stream)


def linear_cross_entropy(hidden, weight, labels, loss, lse, workspace, scale=1.0, ignore_index=-100, stream=0):
    """loss[t] = lse[t] - z[t, labels[t]], lse[t] = log sum_v exp(z[t, v]) for
    z = scale * hidden @ weight.T (bf16 operands, f32 sums)."""
    desc, rows, _, _, ordinal = _linear(hidden, weight, workspace, scale)
    desc.labels, desc.ignore_index = _vector("labels", labels, rows, _i64, ordinal), ignore_index
    _forward(desc, rows, ordinal, loss, lse, stream)


def linear_cross_entropy_backward(hidden, weight, labels, lse, grad_loss, grad_hidden, grad_weight, workspace,
                                  scale=1.0, ignore_index=-100, stream=0):
    """Gradients of sum_t grad_loss[t] * loss[t] with respect to hidden and weight, from the `lse` of
    a forward call with the same rows; z is computed again, summed as it was there, a piece of the
    vocabulary at a time."""
    desc, rows, vocab, dim, ordinal = _linear(hidden, weight, workspace, scale)
    desc.labels, desc.ignore_index = _vector("labels", labels, rows, _i64, ordinal), ignore_index
    _backward(desc, rows, vocab, dim, ordinal, lse, grad_loss, grad_hidden, grad_weight, stream)


def linear_distillation(hidden, weight, teacher_ids, teacher_logits, loss, lse, workspace, temperature=1.0, stream=0):
    """loss[t] = sum_k q_k (log q_k - z[t, id_k]) + lse[t] for z = hidden @ weight.T / temperature
    and q = softmax(teacher_logits[t] / temperature) over row t's entries; lse is that of z."""
    desc, rows, _, _, ordinal = _linear(hidden, weight, workspace, _temperature(temperature))
    _teacher(desc, teacher_ids, teacher_logits, rows, ordinal)
    _forward(desc, rows, ordinal, loss, lse, stream)


def linear_distillation_backward(hidden, weight, teacher_ids, teacher_logits, lse, grad_loss, grad_hidden, grad_weight,
                                 workspace, temperature=1.0, stream=0):
    """Gradients of sum_t grad_loss[t] * loss[t] with respect to hidden and weight."""
    desc, rows, vocab, dim, ordinal = _linear(hidden, weight, workspace, _temperature(temperature))
    _teacher(desc, teacher_ids, teacher_logits, rows, ordinal)
    _backward(desc, rows, vocab, dim, ordinal, lse, grad_loss, grad_hidden, grad_weight, stream)


def _distill(logits, teacher_ids, teacher_logits, temperature):
    ordinal = _place(logits, "logits")
    dtype = logits.dtype
    if dtype not in _DTYPES:
        _bad(f"logits is {dtype}, expected torch.float32 or torch.bfloat16")
    rows, vocab = logits.shape
    pointer, ld = _matrix("logits", logits, rows, vocab, dtype, ordinal)
    desc = DistillDesc(rows, vocab, pointer, ld, _DTYPES[dtype])
    desc.scale = _temperature(temperature)
    _teacher(desc, teacher_ids, teacher_logits, rows, ordinal)
    return desc, rows, vocab, dtype, ordinal


def distillation(logits, teacher_ids, teacher_logits, loss, lse, temperature=1.0, grad_loss=None, grad_logits=None,
                 stream=0):
    """The divergence for logits in memory (f32 or bf16): loss and lse per row. With `grad_logits`
    (and `grad_loss`, the upstream gradient of each row's loss) the gradient is written in the same
    pass; `grad_logits` may be `logits`."""
    desc, rows, vocab, dtype, ordinal = _distill(logits, teacher_ids, teacher_logits, temperature)
    desc.loss = _vector("loss", loss, rows, _f32, ordinal)
    desc.lse = _vector("lse", lse, rows, _f32, ordinal)
    if (grad_loss is None) != (grad_logits is None):
        _bad("grad_loss and grad_logits go together")
    if grad_logits is not None:
        desc.grad_loss = _vector("grad_loss", grad_loss, rows, _f32, ordinal)
        desc.grad_logits, desc.ld_grad_logits = _matrix("grad_logits", grad_logits, rows, vocab, dtype, ordinal)
    _call(_lib.thb_distill_forward, ordinal, desc, stream)


def distillation_backward(logits, teacher_ids, teacher_logits, lse, grad_loss, grad_logits, temperature=1.0, stream=0):
    """grad_logits from the forward call's `lse`; `grad_logits` may be `logits`."""
    desc, rows, vocab, dtype, ordinal = _distill(logits, teacher_ids, teacher_logits, temperature)
    desc.lse = _vector("lse", lse, rows, _f32, ordinal)
    desc.grad_loss = _vector("grad_loss", grad_loss, rows, _f32, ordinal)
    desc.grad_logits, desc.ld_grad_logits = _matrix("grad_logits", grad_logits, rows, vocab, dtype, ordinal)
    _call(_lib.thb_distill_backward, ordinal, desc, stream)
