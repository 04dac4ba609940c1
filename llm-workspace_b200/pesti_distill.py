"""Distillation from a teacher's top logits over the library's logit rows
(include/pesti_sampler.h): the loss, its gradient, or both in one pass.

The teacher's lists are what the library's teacher side makes: kept lists
(probabilities: pass their logarithm), or pesti_beam.top_logprobs, whose tokens
are padded with -1.  Every call runs the CUDA kernels of libpesti_sampler.so on
the logits' device and the current stream; there is no CPU path.
"""
from __future__ import annotations

import functools

import torch

from pesti_beam import _DTYPES, _launch, _need, _on_device, _ptr, _row_stride, _rows_dtype
from pesti_sampler import _check, load_library

MAX_TOP = 256  # PESTI_DISTILL_MAX_TOP


def _stats(k: int) -> int:
    """PESTI_DISTILL_STATS(k)."""
    return 8 + k


@functools.lru_cache(maxsize=256)
def _workspace(dtype: int, N: int, V: int, k: int) -> int:
    need = load_library().pesti_distill_topk_workspace(dtype, N, V, k)
    _check(min(0, need))
    return need


def _lists(logits, idx, val, temperature, teacher_lse, weight):
    """Checks the arguments and returns them in the C call's order."""
    dtype, vtype = _rows_dtype(logits), _DTYPES.get(val.dtype)
    (N, V), dev, shape = logits.shape, logits.device, idx.shape
    (ld, _), to_idx, to_val = logits.stride(), idx.stride(), val.stride()
    if V < 1:
        raise ValueError("V must be at least 1")
    if idx.device != dev or val.device != dev:
        raise ValueError("idx and val must be on the logits' device")
    if shape != val.shape:
        raise ValueError("idx and val must have the same shape")
    if len(shape) != 2 or shape[0] != N or (shape[1] > 1 and (to_idx[1] != 1 or to_val[1] != 1)):
        raise ValueError("idx and val must be [N, k] with contiguous rows")
    k = shape[1]
    if not 1 <= k <= MAX_TOP:
        raise ValueError(f"k must be 1 to {MAX_TOP}")
    if idx.dtype != torch.int32:
        raise ValueError("idx must be int32")
    if vtype is None:
        raise ValueError("val must be float32, bfloat16 or float16")
    for t, name in ((teacher_lse, "teacher_lse"), (weight, "weight")):
        if t is not None and not (t.device == dev and t.dtype == torch.float32 and t.shape == (N,)
                                  and t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous [N] float32 tensor on the logits' device")
    return (logits.data_ptr(), dtype, N, V, ld if N > 1 else max(ld, V), idx.data_ptr(), to_idx[0], val.data_ptr(),
            vtype, to_val[0], k, _ptr(teacher_lse), _ptr(weight), float(temperature))


class _DistillTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, idx, val, temperature, teacher_lse, weight):
        args = _lists(logits, idx, val, temperature, teacher_lse, weight)
        N, dev, keep = logits.shape[0], logits.device, ctx.needs_input_grad[0]

        def call(st):
            loss = logits.new_empty(N, dtype=torch.float32)
            stats = logits.new_empty((N, _stats(args[10])), dtype=torch.float64) if keep else None
            need = _workspace(args[1], N, args[3], args[10])
            ws = logits.new_empty(need, dtype=torch.uint8)
            rc = load_library().pesti_distill_topk(*args, loss.data_ptr(), _ptr(stats), None, 0, ws.data_ptr(), need,
                                                   st)
            if rc:
                _check(rc)
            return loss, stats

        loss, stats = _launch(dev, None, call)
        if keep:
            ctx.temperature = temperature
            ctx.save_for_backward(logits, idx, val, teacher_lse, weight, stats)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        # refuses tensors that were written to since; hooks (activation checkpointing, offloading to the host) may
        # hand back others of the same values, at other addresses and with other strides
        logits, idx, val, teacher_lse, weight, stats = ctx.saved_tensors
        args = _lists(logits, idx, val, ctx.temperature, teacher_lse, weight)
        stats = stats.contiguous()
        if up.dtype != torch.float32:
            up = up.to(torch.float32)

        def call(st):
            grad = logits.new_empty(logits.shape)
            rc = load_library().pesti_distill_topk_backward(*args, stats.data_ptr(), up.data_ptr(), up.stride(0),
                                                            grad.data_ptr(), logits.shape[1], st)
            if rc:
                _check(rc)
            return grad

        return _launch(logits.device, None, call), None, None, None, None, None


def distill_topk(logits, idx, val, temperature: float = 1.0, teacher_lse=None, weight=None):
    """Each row's distillation loss ([N] float32), differentiable for `logits`.

    logits: [N, V] float32, bfloat16 or float16 student logits (rows may be
    strided).  idx [N, k] int32 and val [N, k] (float32, bfloat16 or float16):
    the teacher's tokens and logits or log-probabilities; tokens outside [0, V)
    are padding.  teacher_lse: None (the list is renormalised), or [N] float32,
    the log sum exp of the teacher's logits / temperature over its whole
    vocabulary (0 for log-probabilities at temperature 1): the mass outside the
    list is then one more outcome.  weight: optional [N] float32; rows of weight
    0 are not read.  loss = weight * T^2 * KL(teacher || student).
    The teacher and the weights are constants: no gradient reaches idx, val,
    teacher_lse or weight."""
    # what is not differentiable must not make the loss require a gradient
    if val.requires_grad:
        val = val.detach()
    if teacher_lse is not None and teacher_lse.requires_grad:
        teacher_lse = teacher_lse.detach()
    if weight is not None and weight.requires_grad:
        weight = weight.detach()
    return _DistillTopk.apply(logits, idx, val, temperature, teacher_lse, weight)


def distill_topk_grad(logits, idx, val, temperature: float = 1.0, teacher_lse=None, weight=None, grad=None,
                      stream=None):
    """(loss [N], gradient of loss.sum() for the logits) in one pass over them:
    for a training step that folds what follows the loss into `weight` (a mean's
    1/N, a mask) and continues with logits.backward(gradient).  grad: the tensor
    to fill, `logits` itself to overwrite them."""
    logits = logits.detach()
    args = _lists(logits, idx, val, temperature, teacher_lse, weight)
    N, V = logits.shape
    dev = logits.device
    if grad is not None:
        _on_device(grad, dev, "grad")
        _need(grad.shape == logits.shape and grad.dtype == logits.dtype and (V <= 1 or grad.stride(1) == 1),
              "grad must match the logits and have contiguous rows")

    def call(st):
        loss = logits.new_empty(N, dtype=torch.float32)
        to = logits.new_empty((N, V)) if grad is None else grad
        need = _workspace(args[1], N, V, args[10])
        ws = logits.new_empty(need, dtype=torch.uint8)
        rc = load_library().pesti_distill_topk(*args, loss.data_ptr(), None, to.data_ptr(), _row_stride(to),
                                               ws.data_ptr(), need, st)
        if rc:
            _check(rc)
        if grad is not None and not grad.is_inference():
            torch.autograd.graph.increment_version(grad)  # a backward pass that needs its old values is refused
        return loss, to

    return _launch(dev, stream, call)
