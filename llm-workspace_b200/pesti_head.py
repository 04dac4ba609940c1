"""The vocabulary projection around the library's logit rows (include/pesti_sampler.h):

    linear_cross_entropy, linear_cross_entropy_grad
        the loss of training and scoring straight from the hidden states and the
        projection's weight, with its gradients; the logits are not kept

    quantize_head, QuantizedHead
        that weight in 4 bits with group scales, and back
    head_logits
        logits from it, for pesti_sampler and pesti_beam

    loss = linear_cross_entropy(hidden, head, target)       # [N], differentiable
    loss.sum().backward()
    held = quantize_head(head)
    logits = head_logits(hidden, held)                      # [B, V]
    tokens = sampler.sample_batch(logits, config, u)        # or sampler.sample_hidden(hidden, held, config, u)

Every call runs the CUDA kernels of libpesti_sampler.so on the tensors' device
and the current stream (or `stream`, a cudaStream_t); there is no CPU path, and
no call synchronises.
"""
from __future__ import annotations

import functools

import torch

from pesti_beam import _DTYPES, _launch, _need, _ptr, _row_stride, _written
from pesti_sampler import PESTI_BF16, PESTI_F16, _check, load_library

_HALVES = {torch.bfloat16: PESTI_BF16, torch.float16: PESTI_F16}
_TARGETS = {torch.int64: 8, torch.int32: 4}
_FORWARD, _GRADS = 1, 2  # PESTI_LINEAR_CE_*


@functools.lru_cache(maxsize=256)
def _ce_workspace(dtype: int, N: int, V: int, D: int, passes: int) -> int:
    need = load_library().pesti_linear_ce_workspace(dtype, N, V, D, passes)
    _check(min(0, need))
    return need


def _ce_args(hidden, head, target, weight, label_smoothing, z_loss):
    """Checks the arguments and returns them in the C call's order."""
    kind, dev, shape, to_hidden, to_head = hidden.dtype, hidden.device, hidden.shape, hidden.stride(), head.stride()
    dtype = _HALVES.get(kind)
    if dtype is None or head.dtype != kind:
        raise ValueError("hidden and head must both be bfloat16 or both float16")
    if len(to_hidden) != 2 or len(to_head) != 2 or shape[1] != head.shape[1]:
        raise ValueError("hidden must be [N, D] and head [V, D]")
    (N, D), V = shape, head.shape[0]
    if D < 1 or V < 1:
        raise ValueError("D and V must be at least 1")
    if head.device != dev or target.device != dev:
        raise ValueError("head and target must be on the hidden states' device")
    if D > 1 and (to_hidden[1] != 1 or to_head[1] != 1):
        raise ValueError("rows of hidden and head must be contiguous")
    size = _TARGETS.get(target.dtype)
    if size is None or target.shape != (N,) or not target.is_contiguous():
        raise ValueError("target must be a contiguous [N] int64 or int32 tensor")
    if weight is not None and not (weight.device == dev and weight.dtype == torch.float32 and weight.shape == (N,)
                                   and weight.is_contiguous()):
        raise ValueError("weight must be a contiguous [N] float32 tensor on the hidden states' device")
    return (hidden.data_ptr(), dtype, N, D, to_hidden[0] if N > 1 else D, head.data_ptr(), V,
            to_head[0] if V > 1 else -(-D // 8) * 8, target.data_ptr(), size, _ptr(weight), float(label_smoothing),
            float(z_loss))


def _rows_like(t, rows: int, D: int):
    """[rows, D] with rows that begin at multiples of 16 bytes."""
    return t.new_empty((rows, D)) if D % 8 == 0 else t.new_empty((rows, -(-D // 8) * 8))[:, :D]


def _ce_forward(args, like, keep: bool, grads: bool, st):
    dtype, N, D, V = args[1], args[2], args[3], args[6]
    loss = like.new_empty(N, dtype=torch.float32)
    lse, nll = (like.new_empty(N, dtype=torch.float32) for _ in range(2)) if keep else (None, None)
    gh = like.new_empty((N, D)) if grads else None
    gw = _rows_like(like, V, D) if grads else None
    need = _ce_workspace(dtype, N, V, D, _FORWARD | _GRADS if grads else _FORWARD)
    ws = like.new_empty(need, dtype=torch.uint8)
    rc = load_library().pesti_linear_ce_nll(*args, loss.data_ptr(), _ptr(lse), _ptr(nll), _ptr(gh), D, _ptr(gw),
                                            -(-D // 8) * 8, ws.data_ptr(), need, st)
    if rc:
        _check(rc)
    return loss, lse, nll, gh, gw


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, head, target, weight, label_smoothing, z_loss):
        args = _ce_args(hidden, head, target, weight, label_smoothing, z_loss)
        keep = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        loss, lse, nll, _, _ = _launch(hidden.device, None, lambda st: _ce_forward(args, hidden, keep, False, st))
        if keep:
            ctx.more = label_smoothing, z_loss
            ctx.save_for_backward(hidden, head, target, weight, lse, nll)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        hidden, head, target, weight, lse, nll = ctx.saved_tensors
        # hooks (activation checkpointing, offloading) may hand back tensors at other addresses and of other strides: without
        # the room behind the rows of a head whose D is no multiple of 8, for one
        if hidden.stride(1) != 1:
            hidden = hidden.contiguous()
        if head.stride(1) != 1 or head.stride(0) % 8 or head.data_ptr() % 16:
            head = _rows_like(head, *head.shape).copy_(head)
        target, lse, nll = target.contiguous(), lse.contiguous(), nll.contiguous()
        if weight is not None:
            weight = weight.contiguous()
        args = _ce_args(hidden, head, target, weight, *ctx.more)
        if up.dtype != torch.float32:
            up = up.to(torch.float32)
        dtype, N, D, V = args[1], args[2], args[3], args[6]

        def call(st):
            gh = hidden.new_empty((N, D)) if ctx.needs_input_grad[0] else None
            gw = _rows_like(head, V, D) if ctx.needs_input_grad[1] else None
            need = _ce_workspace(dtype, N, V, D, _GRADS)
            ws = hidden.new_empty(need, dtype=torch.uint8)
            rc = load_library().pesti_linear_ce_nll_backward(
                *args, lse.data_ptr(), nll.data_ptr(), up.data_ptr(), up.stride(0), _ptr(gh), D, _ptr(gw), -(-D // 8) * 8,
                ws.data_ptr(), need, st)
            if rc:
                _check(rc)
            return gh, gw

        return *_launch(hidden.device, None, call), None, None, None, None


def linear_cross_entropy(hidden, head, target, weight=None, label_smoothing: float = 0.0, z_loss: float = 0.0):
    """Each row's cross entropy under softmax(hidden @ head.T) ([N] float32),
    differentiable for `hidden` and `head`.

    hidden [N, D] and head [V, D]: bfloat16 or float16, both the same (rows may
    be strided; head's begin at multiples of 16 bytes).  target [N] int64 or
    int32: rows whose target is outside [0, V) are padding.  weight: optional
    [N] float32.  Padded rows and rows of weight 0 are not read and cost nothing:
    their loss and gradients are 0.
    loss = weight * (lse - (1 - label_smoothing) * z[target] - label_smoothing * mean(z) + z_loss * lse^2)
    The weights are constants: no gradient reaches them."""
    if weight is not None and weight.requires_grad:
        weight = weight.detach()
    return _LinearCrossEntropy.apply(hidden, head, target, weight, label_smoothing, z_loss)


def linear_cross_entropy_grad(hidden, head, target, weight=None, label_smoothing: float = 0.0, z_loss: float = 0.0,
                              stream=None):
    """(loss [N], gradients of loss.sum() for hidden and head) in one call: for a
    training step that folds what follows the loss into `weight` (a mean's 1/N, a
    mask)."""
    hidden, head = hidden.detach(), head.detach()
    args = _ce_args(hidden, head, target, weight, label_smoothing, z_loss)
    loss, _, _, gh, gw = _launch(hidden.device, stream, lambda st: _ce_forward(args, hidden, False, True, st))
    return loss, gh, gw


_BLOCK, _ROWS = 128, 64  # of a tile of the held layout


class QuantizedHead:
    """A [V, D] weight in 4 bits with a scale for every `group` columns of a row
    (quantize_head), about (4.5, 4.25 or 4.125) / 16 of its bfloat16 size.

    packed [ceil(V / 64), ceil(D / 128), 64, 64] uint8 and tile_scale
    [ceil(V / 64), ceil(D / 128), 64, 128 / group] bfloat16 are the library's
    layout (pesti_q4_quantize); scale is tile_scale by rows, [V, ceil(D / group)]."""

    def __init__(self, packed, tile_scale, V: int, D: int, group: int):
        _need(V >= 1 and D >= 1 and group in (32, 64, 128), "V and D must be at least 1, group 32, 64 or 128")
        tiles = -(-V // _ROWS), -(-D // _BLOCK), _ROWS
        _need(packed.dtype == torch.uint8 and packed.shape == (*tiles, _BLOCK // 2) and packed.is_contiguous(),
              "packed must be a contiguous [ceil(V / 64), ceil(D / 128), 64, 64] uint8 tensor")
        _need(tile_scale.dtype == torch.bfloat16 and tile_scale.shape == (*tiles, _BLOCK // group)
              and tile_scale.is_contiguous() and tile_scale.device == packed.device,
              "tile_scale must be a contiguous [ceil(V / 64), ceil(D / 128), 64, 128 / group] bfloat16 tensor on "
              "packed's device")
        self.packed, self.tile_scale, self.V, self.D, self.group = packed, tile_scale, int(V), int(D), int(group)

    @property
    def device(self):
        return self.packed.device

    @property
    def scale(self):
        tiles, blocks, rows, per = self.tile_scale.shape
        by_rows = self.tile_scale.new_empty((tiles * rows, blocks * per))
        whole = {1: torch.int16, 2: torch.int32, 4: torch.int64}[per]  # a row's scales of a tile, moved as one number
        by_rows.view(whole).view(tiles, rows, blocks).copy_(self.tile_scale.view(whole).squeeze(3).transpose(1, 2))
        return by_rows[:self.V, :-(-self.D // self.group)]

    def dequantize(self, dtype=torch.bfloat16, out=None, stream=None):
        """The [V, D] weight that is held (or `out` filled with it): float32 holds it exactly."""
        dev = self.device
        if out is not None:
            _need(out.device == dev and out.shape == (self.V, self.D) and out.dtype in _DTYPES
                  and (self.D == 1 or out.stride(1) == 1),
                  "out must be a [V, D] float32, bfloat16 or float16 tensor with contiguous rows on the held weight's "
                  "device")
        else:
            _need(dtype in _DTYPES, "dtype must be float32, bfloat16 or float16")

        def call(st):
            to = out if out is not None else torch.empty((self.V, self.D), dtype=dtype, device=dev)
            _check(load_library().pesti_q4_dequantize(
                self.packed.data_ptr(), self.tile_scale.data_ptr(), self.V, self.D, self.group, to.data_ptr(),
                _DTYPES[to.dtype], _row_stride(to), st))
            if out is not None:
                _written((out,))
            return to

        return _launch(dev, stream, call)


def quantize_head(head, group: int = 64, stream=None) -> QuantizedHead:
    """pesti_q4_quantize: `head` [V, D] (float32, bfloat16 or float16, rows may be
    strided) in 4 bits with a bfloat16 scale for every `group` (32, 64 or 128)
    columns.  A group's scale is minus an eighth of its largest value by
    magnitude; its values are the nearest of the scale's multiples -8 to 7.  A
    group with an infinity or a NaN is held as NaN."""
    _need(head.dim() == 2 and head.dtype in _DTYPES, "head must be a [V, D] float32, bfloat16 or float16 tensor")
    V, D = head.shape
    _need(D == 1 or head.stride(1) == 1, "head rows must be contiguous")
    _need(group in (32, 64, 128), "group must be 32, 64 or 128")
    head = head.detach()

    def call(st):
        tiles = -(-V // _ROWS), -(-D // _BLOCK), _ROWS
        packed = torch.empty((*tiles, _BLOCK // 2), dtype=torch.uint8, device=head.device)
        scale = torch.empty((*tiles, _BLOCK // group), dtype=torch.bfloat16, device=head.device)
        _check(load_library().pesti_q4_quantize(head.data_ptr(), _DTYPES[head.dtype], V, D, _row_stride(head), group,
                                                packed.data_ptr(), scale.data_ptr(), st))
        return QuantizedHead(packed, scale, V, D, group)

    return _launch(head.device, stream, call)


@functools.lru_cache(maxsize=256)
def _logits_workspace(dtype: int, B: int, D: int) -> int:
    need = load_library().pesti_q4_logits_workspace(dtype, B, D)
    _check(min(0, need))
    return need


def head_logits(x, held: QuantizedHead, dtype=None, out=None, stream=None):
    """pesti_q4_logits: x [B, D] times the held weight, [B, V] logits.

    x: float32, bfloat16 or float16 (rows may be strided); products are
    summed in float32, times the scales in float32 (pesti_sampler.h says how x
    enters them).  dtype: the logits' type
    (None: x's), or out: the [B, V] tensor to fill (rows may be strided).  Made
    for the few rows of a decode step: the weight is read once for every 64 rows
    of x, and no gradient reaches it."""
    code, shape, to_x, dev = _DTYPES.get(x.dtype), x.shape, x.stride(), x.device
    if code is None or len(shape) != 2:
        raise ValueError("x must be a [B, D] float32, bfloat16 or float16 tensor")
    (B, D), V, packed = shape, held.V, held.packed
    if D != held.D:
        raise ValueError("x and the held weight have different D")
    if packed.device != dev:
        raise ValueError("x and the held weight must be on the same device")
    if D > 1 and to_x[1] != 1:
        raise ValueError("x rows must be contiguous")
    if out is not None:
        _need(out.device == dev and out.shape == (B, V) and out.dtype in _DTYPES and (V == 1 or out.stride(1) == 1),
              "out must be a [B, V] float32, bfloat16 or float16 tensor with contiguous rows on x's device")
        kind = out.dtype
    else:
        kind = dtype or x.dtype
        if kind not in _DTYPES:
            raise ValueError("dtype must be float32, bfloat16 or float16")

    def call(st):
        to = out if out is not None else x.new_empty((B, V), dtype=kind)
        if B:
            need = _logits_workspace(code, B, D)
            ws = x.new_empty(need, dtype=torch.uint8) if need else None
            rc = load_library().pesti_q4_logits(
                x.data_ptr(), code, B, D, to_x[0] if B > 1 else D, packed.data_ptr(), held.tile_scale.data_ptr(), V,
                held.group, to.data_ptr(), _DTYPES[kind], _row_stride(to) if out is not None else V, _ptr(ws), need, st)
            if rc:
                _check(rc)
            if out is not None:
                _written((out,))
        return to

    return _launch(dev, stream, call)
