"""Operators around a training step over torch tensors: GradClip.

Thin classes over the C ABI's apk_clip_* (include/apk.h), in the manner of
layers.py: torch is used for memory and streams only.  No counterpart in the
reference, which multiplies bare matrices (src/tcyield.cu:91-356).
"""
from __future__ import annotations

import array
import ctypes
import math

import torch

from . import _lib as L
from .layers import _ANY, _CODE, _Handle, _raw_stream, _tensor

_TYPES = set(_ANY)


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
        # the usual case in few steps: there may be hundreds of them
        try:
            if ({t.get_device() for t in tensors} <= {self._index} and {t.dtype for t in tensors} <= _TYPES
                    and all([t.is_contiguous() for t in tensors])):
                return
        except (AttributeError, RuntimeError):
            pass
        for i, t in enumerate(tensors):
            _tensor(t, f"{what}[{i}]", self.device, _ANY)
            if not _dense(t):
                raise ValueError(f"{what}[{i}], of strides {t.stride()}, is not dense in memory")

    def _run(self, grads, out, function):
        grads = list(grads)
        if out is not None:
            out = list(out)
            if len(out) != len(grads):
                raise ValueError(f"{len(out)} tensors in out for {len(grads)} gradients")
            out = [o for o, t in zip(out, grads) if t is not None]
        grads = [t for t in grads if t is not None]
        self._check_list(grads, "grads")
        if out is not None:
            self._check_list(out, "out")
            for i, (t, o) in enumerate(zip(grads, out)):
                if t.shape != o.shape or t.dtype != o.dtype:
                    raise ValueError(f"out[{i}] is {o.dtype} {tuple(o.shape)}, its gradient {t.dtype} {tuple(t.shape)}")
                if t.stride() != o.stride() and not (t.is_contiguous() and o.is_contiguous()):
                    raise ValueError(f"out[{i}] has strides {o.stride()}, its gradient {t.stride()}")
        norm = torch.empty((), dtype=torch.float32, device=self.device)
        at = array.array("q", [t.data_ptr() for t in grads])
        to = at if out is None else array.array("q", [t.data_ptr() for t in out])
        n = array.array("q", [t.numel() for t in grads])
        kinds = array.array("i", [_CODE[t.dtype] for t in grads])
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
        two of them may share memory.  An infinite norm makes the factor 0, a
        NaN makes it NaN: look at the norm before the weights are updated."""
        if not self.max_norm >= 0.0 or math.isnan(self.max_norm):
            raise ValueError(f"max_norm is {self.max_norm}: 0 or above")
        return self._run(grads, out, self._lib.apk_clip_scale)

    __call__ = clip
