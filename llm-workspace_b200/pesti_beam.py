"""Beam search over the library's logit rows (include/pesti_sampler.h):
selection over beams and vocabulary, the loop control of the beams on the
device, and the reordering of per-beam states.

    state = BeamState(groups, beams, max_tokens, max_seq_len, stop_tokens=[2])
    while ...:
        score, token, parent = beam_select(logits, beams, 2 * beams, cum=state.cum, done=state.done)
        state.advance(score, token, parent)
        beam_reorder(caches, state.parent)
        logits = model(state.last)      # [groups*beams, V]
    state.hypotheses()

With S stop tokens, (1 + S) * beams candidates always leave enough live beams.
Every call runs the CUDA kernels of libpesti_sampler.so on the tensors' device
and the current stream (or `stream`, a cudaStream_t); there is no CPU path.
No call synchronises, except hypotheses() and active(), which read back on the
current stream.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Sequence

import torch

from pesti_sampler import PESTI_BF16, PESTI_F16, PESTI_F32, _check, load_library

MAX_BEAMS = 64        # PESTI_BEAM_MAX_WIDTH
MAX_CANDIDATES = 128  # PESTI_BEAM_MAX_CAND

_DTYPES = {torch.float32: PESTI_F32, torch.bfloat16: PESTI_BF16, torch.float16: PESTI_F16}


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _rows_dtype(logits) -> int:
    dtype, strides = _DTYPES.get(logits.dtype), logits.stride()
    if len(strides) != 2:
        raise ValueError("logits must be [rows, V]")
    if dtype is None:
        raise ValueError("logits must be float32, bfloat16 or float16")
    if strides[1] != 1 and logits.shape[1] > 1:
        raise ValueError("logits rows must be contiguous")
    return dtype


def _row_stride(t) -> int:
    """Elements between rows (a single row's stride is never used: its length then)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _on_device(t, dev, what: str) -> None:
    if t.device != dev:
        raise ValueError(f"{what} must be on the logits' device")


# For a list of tensors that a call wrote: a backward pass that needs their old values is refused.
_written = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)

_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(device, stream, call):
    """call(cudaStream_t) with the tensors' device current, and with what it
    allocates belonging to the stream that uses it."""
    if device.type != "cuda":
        raise ValueError("tensors must be on a CUDA device (there is no CPU path)")
    index = device.index
    if index == _current_device():
        current = _current_stream(index)
        if stream is None or stream == current:
            return call(current)
    with torch.cuda.device(device):
        if stream is None:
            return call(_current_stream(index))
        # (an ExternalStream of handle 0 would be a stream of its own)
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device) if stream
                               else torch.cuda.default_stream(device)):
            return call(stream)


@functools.lru_cache(maxsize=256)
def _select_workspace(dtype: int, G: int, W: int, V: int, K: int) -> int:
    need = load_library().pesti_beam_select_workspace(dtype, G, W, V, K)
    _check(min(0, need))
    return need


def _ptr(t):
    return t.data_ptr() if t is not None else None


def beam_select(logits, beams: int, k: int, cum=None, done=None, lse=None, out=None, stream=None):
    """pesti_beam_select: the k best continuations of each group of beams.

    logits: [groups*beams, V] float32, bfloat16 or float16 CUDA tensor (rows may
    be strided).  cum: [groups, beams] float32 scores so far (None: 0).  done:
    optional [groups] uint8 or bool, groups to leave out.  lse: optional
    [groups*beams] float32 tensor that receives each row's log sum exp.
    Returns (score float32, token int32, parent int32), [groups, k] each, best
    first; slots without a candidate hold (-inf, -1, -1).  out: the three
    tensors to fill instead."""
    dtype = _rows_dtype(logits)
    rows, V = logits.shape
    _need(1 <= beams <= MAX_BEAMS, f"beams must be 1 to {MAX_BEAMS}")
    _need(1 <= k <= MAX_CANDIDATES, f"k must be 1 to {MAX_CANDIDATES}")
    _need(rows % beams == 0, "rows must be a multiple of beams")
    _need(V >= 1, "V must be at least 1")
    G, dev = rows // beams, logits.device
    if cum is not None:
        _on_device(cum, dev, "cum")
        _need(cum.dtype == torch.float32 and cum.numel() == rows and cum.is_contiguous(),
              "cum must be a contiguous [groups, beams] float32 tensor")
    if done is not None:
        _on_device(done, dev, "done")
        _need(done.dtype in (torch.uint8, torch.bool) and done.numel() == G and done.is_contiguous(),
              "done must be a contiguous [groups] uint8 or bool tensor")
    if lse is not None:
        _on_device(lse, dev, "lse")
        _need(lse.dtype == torch.float32 and lse.numel() == rows and lse.is_contiguous(),
              "lse must be a contiguous [groups*beams] float32 tensor")
    if out is not None:
        for t, want in zip(out, (torch.float32, torch.int32, torch.int32)):
            _on_device(t, dev, "out")
            _need(t.dtype == want and t.shape == (G, k) and t.is_contiguous(),
                  "out must be contiguous [groups, k] float32, int32 and int32 tensors")

    def call(st):
        if out is None:
            score = logits.new_empty((G, k), dtype=torch.float32)
            token = logits.new_empty((G, k), dtype=torch.int32)
            parent = logits.new_empty((G, k), dtype=torch.int32)
        else:
            score, token, parent = out
        if G:
            need = _select_workspace(dtype, G, beams, V, k)
            ws = logits.new_empty(need, dtype=torch.uint8)
            rc = load_library().pesti_beam_select(
                logits.data_ptr(), dtype, G, beams, V, _row_stride(logits), _ptr(cum), _ptr(done), k,
                score.data_ptr(), token.data_ptr(), parent.data_ptr(), _ptr(lse), ws.data_ptr(), need, st)
            if rc:
                _check(rc)
            if out is not None:
                _written(out)
            if lse is not None:
                _written((lse,))
        return score, token, parent

    return _launch(dev, stream, call)


def top_logprobs(logits, k: int, stream=None):
    """The k largest log-probabilities of each row of `logits` ([B, V]), as a
    distillation teacher records them: (logprob [B, k] float32, token [B, k]
    int32, lse [B] float32), best first, (-inf, -1) where a row has fewer."""
    lse = _launch(logits.device, stream,
                  lambda st: torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device))
    logprob, token, _ = beam_select(logits, 1, k, lse=lse, stream=stream)
    return logprob, token, lse


class _StateC(ctypes.Structure):
    """pesti_beam_state."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("cum", "last", "parent", "tokens", "count", "done", "fin_tokens",
                                               "fin_len", "fin_score", "fin_count")] + [("cap", ctypes.c_int64)]


class _LimitsC(ctypes.Structure):
    """pesti_beam_limits."""
    _fields_ = [("max_tokens", ctypes.c_int64), ("max_seq_len", ctypes.c_int64), ("length_penalty", ctypes.c_double),
                ("early_stop", ctypes.c_int32)]


class BeamState:
    """The loop control of a beam search on the device (pesti_beam_advance),
    DecodeState's counterpart for `groups` prompts of `beams` beams.

    cum [G, W] scores for the next beam_select; last [G, W] the next step's
    input tokens; parent [G, W] for beam_reorder; tokens [G, W, cap] and count
    [G] the live beams; done [G] (0 running, 1 finished, 2 max_tokens, 3
    max_seq_len); fin_tokens, fin_len, fin_score, fin_count the pool of finished
    hypotheses, scored s / length^length_penalty."""

    def __init__(self, groups: int, beams: int, max_tokens: int, max_seq_len: int, stop_tokens: Sequence[int] = (),
                 length_penalty: float = 1.0, early_stop: bool = False, device=0, stream=None):
        _need(groups >= 0, "groups must not be negative")
        _need(1 <= beams <= MAX_BEAMS, f"beams must be 1 to {MAX_BEAMS}")
        _need(max_tokens >= 0 and max_seq_len >= 0, "max_tokens and max_seq_len must not be negative")
        self._lib = load_library()
        self.groups, self.beams = int(groups), int(beams)
        self.max_tokens, self.max_seq_len = int(max_tokens), int(max_seq_len)
        self.cap = max(1, min(self.max_tokens, self.max_seq_len))
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if dev.type == "cuda":
            current = torch.cuda.current_device()  # sets CUDA up
            dev = torch.device("cuda", current if dev.index is None else dev.index)
        G, W, i32 = self.groups, self.beams, torch.int32

        def make(*shape, dtype=i32):
            return torch.empty(*shape, dtype=dtype, device=dev)

        def allocate(st):
            self.cum, self.fin_score = make(G, W, dtype=torch.float32), make(G, W, dtype=torch.float32)
            self.last, self.parent, self.fin_len = make(G, W), make(G, W), make(G, W)
            self.tokens, self.fin_tokens = make(G, W, self.cap), make(G, W, self.cap)
            self.count, self.fin_count, self.done = make(G), make(G), make(G, dtype=torch.uint8)
            self.stop = torch.tensor(list(stop_tokens) or [0], dtype=torch.int64).to(i32).to(dev)

        _launch(dev, stream, allocate)
        dev = self.device = self.cum.device
        self.n_stop = len(stop_tokens)
        self._c = _StateC(*[getattr(self, n).data_ptr() for n, _ in _StateC._fields_[:-1]], self.cap)
        self._limits = _LimitsC(self.max_tokens, self.max_seq_len, float(length_penalty), int(bool(early_stop)))
        self._arrays = [getattr(self, n) for n, _ in _StateC._fields_[:-1]]
        self._at = (ctypes.addressof(self._c), self.stop.data_ptr(), ctypes.addressof(self._limits),
                    self._lib.pesti_beam_advance)
        self.reset(stream)

    def reset(self, stream=None) -> None:
        """Begins a new search: one live beam per group with score 0."""
        _launch(self.device, stream,
                lambda st: _check(self._lib.pesti_beam_reset(self._at[0], self.groups, self.beams, st)))
        _written(self._arrays)

    def advance(self, score, token, parent, stream=None) -> None:
        """Takes one step's candidates ([groups, k], as beam_select returns them)."""
        shape, dev, i32 = score.shape, self.device, torch.int32
        if not (len(shape) == 2 and shape[0] == self.groups and shape == token.shape == parent.shape
                and score.dtype == torch.float32 and token.dtype == i32 and parent.dtype == i32
                and score.is_contiguous() and token.is_contiguous() and parent.is_contiguous()):
            raise ValueError("candidates must be contiguous [groups, k] float32, int32 and int32 tensors")
        index = dev.index
        if not (score.get_device() == index and token.get_device() == index and parent.get_device() == index):
            raise ValueError("candidates must be on the state's device")
        state, stop, limits, advance = self._at

        def call(st):
            rc = advance(state, score.data_ptr(), token.data_ptr(), parent.data_ptr(), shape[0], self.beams, shape[1],
                         stop, self.n_stop, limits, st)
            if rc:
                _check(rc)

        _launch(dev, stream, call)
        _written(self._arrays)

    def active(self) -> int:
        """Groups still running (a host read: call it now and then)."""
        return int((self.done == 0).sum().item())

    def hypotheses(self):
        """Every group's finished hypotheses, best first: lists of (score,
        [tokens]); live beams of groups still running are not among them."""
        toks, lens = self.fin_tokens.cpu(), self.fin_len.cpu()
        scores, counts = self.fin_score.cpu(), self.fin_count.cpu()
        out = []
        for g in range(self.groups):
            have = [(float(scores[g, i]), toks[g, i, :int(lens[g, i])].tolist()) for i in range(int(counts[g]))]
            out.append(sorted(have, key=lambda h: -h[0]))
        return out


class _RowsC(ctypes.Structure):
    """pesti_beam_rows."""
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p)] + [
        (n, ctypes.c_int64) for n in ("src_row_stride", "dst_row_stride", "src_block_stride", "dst_block_stride",
                                      "blocks", "block_bytes")]


@functools.lru_cache(maxsize=1024)
def _layout(shape, strides):
    """A row (all but the first dimension) as (blocks, block elements, elements
    between blocks)."""
    run, i = 1, len(shape) - 1
    while i >= 1 and (shape[i] == 1 or strides[i] == run):
        run *= shape[i]
        i -= 1
    blocks, step, at = 1, 0, 0
    for j in range(i, 0, -1):
        if shape[j] == 1:
            continue
        if blocks == 1:
            step = at = strides[j]
        elif strides[j] != at:
            raise ValueError("a state's rows must be contiguous or equally spaced contiguous blocks")
        blocks *= shape[j]
        at = strides[j] * shape[j]
    return blocks, run, step


@functools.lru_cache(maxsize=1024)
def _reorder_strides(shape, src, dst, esize: int):
    """The six numbers of a pesti_beam_rows behind its pointers, in bytes."""
    blocks, run, step = _layout(shape, src)
    to = _layout(shape, dst)
    if to[:2] != (blocks, run):
        raise ValueError("out must be laid out in the same blocks as its state")
    return src[0] * esize, dst[0] * esize, step * esize, to[2] * esize, blocks, run * esize


def beam_reorder(states, parent, out=None, stream=None):
    """pesti_beam_reorder: row g*beams + w of every state becomes row g*beams +
    parent[g, w] (a parent outside the group's beams: the beam itself).

    states: a tensor or a list of tensors of any type whose first dimension is
    groups*beams (for caches [rows, heads, room, dim], pass cache[:, :, :used]).
    In place, or into `out` (tensors of the same shapes).  States must not share
    memory, and what is written none with `parent`.  Returns the reordered
    states."""
    single = isinstance(states, torch.Tensor)
    src = [states] if single else list(states)
    dst = src if out is None else ([out] if single else list(out))
    _need(len(src) == len(dst), "out must have one tensor per state")
    _need(parent.dim() == 2 and parent.dtype == torch.int32 and parent.is_contiguous(),
          "parent must be a contiguous [groups, beams] int32 tensor")
    G, W = parent.shape
    dev, first, fields = parent.device, G * W, []
    for a, b in zip(src, dst):
        shape = a.shape
        if not shape or shape[0] != first:
            raise ValueError("a state's first dimension must be groups*beams")
        if a.device != dev:
            raise ValueError("states must be on the parents' device")
        strides = to = a.stride()
        if b is not a:
            if b.shape != shape or b.dtype != a.dtype or b.device != dev:
                raise ValueError("out must match the states' shapes, types and device")
            to = b.stride()
        fields += a.data_ptr(), b.data_ptr()
        fields += _reorder_strides(shape, strides, to, a.element_size())
    rows = (ctypes.c_int64 * max(1, len(fields)))(*fields)

    def call(st):
        rc = load_library().pesti_beam_reorder(ctypes.addressof(rows), len(src), parent.data_ptr(), G, W, st)
        if rc:
            _check(rc)

    _launch(dev, stream, call)
    _written(dst)
    return dst[0] if single else dst
