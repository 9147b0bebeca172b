"""Operators around a training step over torch tensors: GradClip and
LogProbs, which a server uses as well.

Thin classes over the C ABI's apk_clip_* and apk_logprobs_* (include/apk.h), in the manner of
layers.py: torch is used for memory and streams only.  No counterpart in the
reference, which multiplies bare matrices (src/tcyield.cu:91-356).
"""
from __future__ import annotations

import array
import ctypes
import math
import operator

import torch

from . import _lib as L
from .layers import _ANY, _CODE, _Handle, _like, _new, _overlap, _raw_stream, _rows, _tensor

_TYPES = set(_ANY)
_dtype, _shape = operator.attrgetter("dtype"), operator.attrgetter("shape")
_data_ptr, _numel, _get_device, _is_contiguous = (
    torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous)


def _device_index(device) -> int:
    """The index of a CUDA device given as torch takes it; None: the current one."""
    if device is None:
        return torch.cuda.current_device()
    d = torch.device(device)
    if d.type != "cuda":
        raise ValueError(f"device is {d}, not a CUDA device")
    return torch.cuda.current_device() if d.index is None else d.index


def _dense(t) -> bool:
    """Whether t's elements fill one stretch of memory, each once, in any order of axes."""
    if t.is_contiguous():
        return True
    step = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride != step:
            return False
        step *= size
    return True


class GradClip(_Handle):
    """The global norm of many gradients, and clipping them by it.

    Gradients may be fp32 or bf16, of any shape, dense in memory.  Nones (of
    parameters without one) are passed over."""
    _create, _destroy, _error = "apk_clip_create", "apk_clip_destroy", "apk_clip_last_error"

    def __init__(self, max_norm: float, device=None):
        self.max_norm = float(max_norm)
        if not self.max_norm >= 0.0:
            raise ValueError(f"max_norm is {max_norm}: 0 or above")
        self._index = _device_index(device)
        self.device = torch.device("cuda", self._index)
        self._open(L.ClipConfig(self._index))
        self._io = L.ClipIO()
        self._io_ref = ctypes.byref(self._io)

    def _check_list(self, tensors, what):
        """Their types, and whether all are contiguous."""
        # the usual case in few steps: there may be hundreds of them
        try:
            kinds = list(map(_dtype, tensors))
            if (set(map(_get_device, tensors)) <= {self._index} and set(kinds) <= _TYPES
                    and all(map(_is_contiguous, tensors))):
                return kinds, True
        except (AttributeError, RuntimeError, TypeError):
            pass
        for i, t in enumerate(tensors):
            _tensor(t, f"{what}[{i}]", self.device, _ANY)
            if not _dense(t):
                raise ValueError(f"{what}[{i}], of strides {t.stride()}, is not dense in memory")
        return list(map(_dtype, tensors)), False

    def _run(self, grads, out, function):
        grads = list(grads)
        if out is not None:
            out = list(out)
            if len(out) != len(grads):
                raise ValueError(f"{len(out)} tensors in out for {len(grads)} gradients")
            out = [o for o, t in zip(out, grads) if t is not None]
        grads = [t for t in grads if t is not None]
        kinds, plain = self._check_list(grads, "grads")
        if out is not None:
            to, both = self._check_list(out, "out")
            if to != kinds or not (plain and both) or list(map(_shape, out)) != list(map(_shape, grads)):
                for i, (t, o) in enumerate(zip(grads, out)):
                    if t.shape != o.shape or t.dtype != o.dtype:
                        raise ValueError(f"out[{i}] is {o.dtype} {tuple(o.shape)}, its gradient {t.dtype} {tuple(t.shape)}")
                    if t.stride() != o.stride() and not (t.is_contiguous() and o.is_contiguous()):
                        raise ValueError(f"out[{i}] has strides {o.stride()}, its gradient {t.stride()}")
        norm = torch.empty_strided((), (), dtype=torch.float32, device=self.device)
        at = array.array("q", list(map(_data_ptr, grads)))
        to = at if out is None else array.array("q", list(map(_data_ptr, out)))
        n = array.array("q", list(map(_numel, grads)))
        kinds = array.array("i", [_CODE[d] for d in kinds])
        with self._lock:
            io = self._io
            io.count, io.max_norm = len(grads), self.max_norm
            io.in_, io.out, io.n, io.dtype = (a.buffer_info()[0] for a in (at, to, n, kinds))
            io.norm, io.stream = norm.data_ptr(), _raw_stream(self._index)
            st = function(self._h, self._io_ref)
            if st:
                self._check(st)
        return norm

    def norm(self, grads):
        """The 2-norm of all gradients together: an fp32 tensor without axes, on the device."""
        return self._run(grads, None, self._lib.apk_clip_norm)

    def clip(self, grads, out=None):
        """Multiplies the gradients by min(1, max_norm / (norm + 1e-6)), in
        place or into the tensors of `out`; returns the norm before that.  No
        two of them may share memory.  An infinite norm makes the factor 0 (NaN
        where max_norm is infinite too), a NaN makes it NaN: look at the norm
        before the weights are updated."""
        if not self.max_norm >= 0.0 or math.isnan(self.max_norm):
            raise ValueError(f"max_norm is {self.max_norm}: 0 or above")
        return self._run(grads, out, self._lib.apk_clip_scale)

    __call__ = clip


class LogProbs(_Handle):
    """Log probabilities of given tokens, entropies and the `top` largest
    alternatives of rows of logits (fp32 or bf16), and their gradient."""
    _create, _destroy, _error = "apk_logprobs_create", "apk_logprobs_destroy", "apk_logprobs_last_error"

    def __init__(self, top: int = 0, device=None):
        if top not in range(33):
            raise ValueError(f"top is {top!r}: 0 to 32")
        self.top = int(top)
        self._index = _device_index(device)
        self.device = torch.device("cuda", self._index)
        self._open(L.LogprobsConfig(self._index, self.top))
        self._io, self._grads = L.LogprobsIO(), L.LogprobsGrads()
        self._io_ref, self._grads_ref = ctypes.byref(self._io), ctypes.byref(self._grads)

    def _logits(self, logits, a):
        if not isinstance(logits, torch.Tensor) or logits.dim() < 1 or logits.shape[-1] < max(1, self.top):
            raise ValueError(f"logits: a tensor [..., vocabulary] of at least {max(1, self.top)} is wanted")
        V = logits.shape[-1]
        a.logits, a.rows, a.ld = _rows(logits, "logits", self.device, V, _ANY)
        a.vocabulary = V
        a.dtype = _CODE[logits.dtype]

    def _per_row(self, t, what, shape, dtypes):
        try:  # the usual case first
            if t.shape == shape and t.dtype in dtypes and t.device == self.device and t.is_contiguous():
                return t.data_ptr()
        except AttributeError:
            pass
        _tensor(t, what, self.device, dtypes)
        if t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{what} is {tuple(t.shape)} with strides {t.stride()}: contiguous {tuple(shape)} is wanted")
        return t.data_ptr()

    def _tokens(self, tokens, shape, a):
        a.tokens = self._per_row(tokens, "tokens", shape, (torch.int64, torch.int32))
        a.tokens_64 = tokens.dtype is torch.int64

    def forward(self, logits, tokens=None, save_stats: bool = False):
        """(logprob, entropy, top_ids, top_logprobs) for logits [..., V] and
        tokens [...]; None without tokens, or where top is 0; with save_stats
        a fifth: what backward() takes.  A negative token is padding, with log
        probability 0.  ids are int32, the others fp32."""
        with self._lock:
            io = self._io
            self._logits(logits, io)
            shape = logits.shape[:-1]
            logprob = ids = tops = stats = None
            entropy = _new(logits, shape, torch.float32)
            if tokens is None:
                io.tokens = io.logprob = None
            else:
                self._tokens(tokens, shape, io)
                logprob = torch.empty_like(entropy)
                io.logprob = logprob.data_ptr()
            io.entropy = entropy.data_ptr()
            if self.top:
                tops = _new(logits, (*shape, self.top), torch.float32)
                ids = torch.empty_like(tops, dtype=torch.int32)
                io.top_ids, io.top_logprobs = ids.data_ptr(), tops.data_ptr()
            if save_stats:
                stats = _new(logits, (*shape, 2), torch.float32)
                io.stats = stats.data_ptr()
            else:
                io.stats = None
            io.stream = _raw_stream(self._index)
            st = self._lib.apk_logprobs_forward(self._h, self._io_ref)
            if st:
                self._check(st)
            return (logprob, entropy, ids, tops, stats) if save_stats else (logprob, entropy, ids, tops)

    __call__ = forward

    def backward(self, dlogprob, logits, tokens, stats, dentropy=None, entropy=None, out=None):
        """The logits' gradient, of their type, for the outputs' gradients
        dlogprob and dentropy (fp32 [...]; None: not used).  stats and, with
        dentropy, entropy: what forward(save_stats=True) returned.  out: the
        gradient's tensor; it may be the logits, but share no memory with them
        otherwise."""
        with self._lock:
            g = self._grads
            self._logits(logits, g)
            shape, f32 = logits.shape[:-1], (torch.float32,)
            if dlogprob is None and dentropy is None:
                raise ValueError("dlogprob or dentropy is wanted")
            g.tokens = g.dlogprob = g.dentropy = g.entropy = None
            if dlogprob is not None:
                self._tokens(tokens, shape, g)
                g.dlogprob = self._per_row(dlogprob, "dlogprob", shape, f32)
            if dentropy is not None:
                g.dentropy = self._per_row(dentropy, "dentropy", shape, f32)
                g.entropy = self._per_row(entropy, "entropy", shape, f32)
            g.stats = self._per_row(stats, "stats", (*shape, 2), f32)
            if out is None:
                out = _like(logits, logits.shape)
                g.dlogits, g.ld_d = out.data_ptr(), g.vocabulary
            else:
                if not isinstance(out, torch.Tensor) or out.shape != logits.shape:
                    raise ValueError(f"out: a tensor {tuple(logits.shape)} is wanted")
                g.dlogits, _, g.ld_d = _rows(out, "out", self.device, g.vocabulary, (logits.dtype,))
                es = out.element_size()
                to, of = (g.dlogits, g.ld_d * es, g.vocabulary * es), (g.logits, g.ld * es, g.vocabulary * es)
                if to != of and _overlap(to, of, g.rows):
                    raise ValueError("out shares memory with logits, but is not it")
            g.stream = _raw_stream(self._index)
            st = self._lib.apk_logprobs_backward(self._h, self._grads_ref)
            if st:
                self._check(st)
            return out
