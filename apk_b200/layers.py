"""Layer operators over torch tensors: Linear (forward, backward) and MoE.

Thin classes over the C ABI's apk_linear_* and apk_moe_* (include/apk.h):
they check shapes, types and strides, allocate outputs with torch, and run
on torch's current stream of the weights' device.  torch is used for memory
and streams only; the arithmetic is libapk's.  No counterpart in the
reference, which multiplies bare matrices (src/tcyield.cu:91-356).
"""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib as L
from .runtime import ApkError

_ACT = {"none": L.APK_ACT_NONE, "relu": L.APK_ACT_RELU, "gelu": L.APK_ACT_GELU,
        "gelu_tanh": L.APK_ACT_GELU_TANH, "silu": L.APK_ACT_SILU}
_LAYOUT = {"kn": L.APK_W_KN, "nk": L.APK_W_NK}
_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_CODE = {torch.float32: L.APK_F32, torch.bfloat16: L.APK_BF16}
_ANY = tuple(_CODE)
# the current stream's handle; building a torch.cuda.Stream for it costs 2 us a call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)
_DEFAULT_WAIT_NS = 2_000_000_000
# the native handles have the tensors' addresses
_MOVED = "weights are in other memory than when the layer was made: make a new layer"


def _pick(table, value, what):
    try:
        return table[value]
    except (KeyError, TypeError):
        raise ValueError(f"{what} is {value!r}: one of {', '.join(table)}") from None


def _tensor(t, what, device=None, dtypes=(torch.bfloat16,), dim=None):
    """t itself, or a ValueError that says what is wrong with it."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what} is not a torch tensor")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{what} is on {t.device}, not on {device or 'a CUDA device'}")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} is {t.dtype}: one of {', '.join(str(d) for d in dtypes)}")
    if dim is not None and t.dim() != dim:
        raise ValueError(f"{what} has {t.dim()} axes, not {dim}")
    return t


def _rows(t, what, device, width, dtypes=(torch.bfloat16,)):
    """(address, rows, row stride) of a [..., width] tensor whose last axis is
    contiguous.  Called for every operand of every call: the usual case first."""
    try:
        shape = t.shape
        if len(shape) == 2 and shape[1] == width and t.dtype in dtypes and t.device == device:
            s0, s1 = t.stride()
            if s1 == 1 or width == 1:
                m = shape[0]
                return t.data_ptr(), m, (s0 if m > 1 else width)
    except (AttributeError, TypeError):
        pass
    _tensor(t, what, device, dtypes)
    if t.dim() < 1 or t.shape[-1] != width:
        raise ValueError(f"{what} is {tuple(t.shape)}: its last axis has to be {width}")
    if width > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: its last axis has stride {t.stride(-1)}, not 1")
    try:
        v = t.view(-1, width) if t.numel() else t.new_empty((t.numel() // width, width))
    except RuntimeError:
        raise ValueError(f"{what}: its leading axes, of strides {t.stride()}, are not rows of one stride") from None
    return v.data_ptr(), v.shape[0], (v.stride(0) if v.shape[0] > 1 else width)


def _overlap(a, b, rows):
    """Whether two views of `rows` rows, each (address, row pitch, row length) in
    bytes, share memory: exact where the pitches agree, else whether their
    extents meet."""
    (at, pitch, length), (at2, pitch2, length2) = a, b
    if rows == 0 or at + (rows - 1) * pitch + length <= at2 or at2 + (rows - 1) * pitch2 + length2 <= at:
        return False
    off = (at2 - at) % pitch
    return pitch != pitch2 or off < length or off + length2 > pitch


def _like(t, shape):
    """A new tensor of t's type and device; of t's own shape the cheaper way."""
    return torch.empty_like(t) if t.shape == shape and t.is_contiguous() else t.new_empty(shape)


class _Handle:
    """Owner of one native handle; subclasses name its functions."""
    _create = _destroy = _error = _status = ""

    def _open(self, cfg):
        self._lib = L.load()
        # a layer's argument structures are reused from call to call, and the
        # interpreter lets other threads run during one
        self._lock = threading.Lock()
        self._h = ctypes.c_void_p()
        st = getattr(self._lib, self._create)(ctypes.byref(cfg), ctypes.byref(self._h))
        if st != L.APK_OK:
            message = self._message()
            self.close()
            raise ApkError(st, message)

    def _message(self):
        return getattr(self._lib, self._error)(self._h).decode()

    def _check(self, st):
        if st != L.APK_OK:
            raise ApkError(st, self._message())

    def status(self) -> int:
        """The first device error since the last query (0: none); waits for the current stream."""
        st = ctypes.c_int()
        self._check(getattr(self._lib, self._status)(self._h, self._stream(), ctypes.byref(st)))
        return st.value

    def _stream(self):
        return _raw_stream(self._index)

    def close(self):
        if getattr(self, "_h", None) is not None and self._h.value:
            getattr(self._lib, self._destroy)(self._h)
            self._h = ctypes.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Linear(_Handle):
    """y = act(x W + b) + r with bf16 weights, and its gradients.

    weight: [in, out] for layout "kn" (the GEMM runtime's row-major B) or
    [out, in] for "nk", bf16, rows of any stride.  bias: [out] fp32 or bf16.
    act: none, relu, gelu, gelu_tanh or silu.  The layer keeps a reference to
    the tensors, not a copy: an optimizer may update them in place.  Other
    tensors, or other memory for these, need another layer: a call refuses
    weights that have moved.  Nothing is recorded for autograd: outputs carry
    no gradient function, backward() computes the gradients."""
    _create, _destroy = "apk_linear_create", "apk_linear_destroy"
    _error, _status = "apk_linear_last_error", "apk_linear_status"

    def __init__(self, weight, bias=None, act: str = "none", layout: str = "kn", out_dtype: str = "bf16",
                 sms: int = 0, wait_limit_ns: int = _DEFAULT_WAIT_NS):
        _tensor(weight, "weight", dim=2)
        kn = _pick(_LAYOUT, layout, "layout") == L.APK_W_KN
        self.device, self._index = weight.device, weight.device.index
        self.in_features, self.out_features = weight.shape if kn else weight.shape[::-1]
        w, _, ldw = _rows(weight, "weight", self.device, weight.shape[1])
        if bias is not None:
            _tensor(bias, "bias", self.device, tuple(_CODE), 1)
            if bias.shape[0] != self.out_features or (bias.shape[0] > 1 and bias.stride(0) != 1):
                raise ValueError(f"bias is {tuple(bias.shape)} with strides {bias.stride()}: "
                                 f"{self.out_features} contiguous values are wanted")
        self.weight, self.bias, self.act, self.layout = weight, bias, act, layout
        self._w_shape, self._w_at, self._b_at = weight.shape, w, None if bias is None else bias.data_ptr()
        self.out_dtype = _pick(_TORCH, out_dtype, "out_dtype")
        self._y_code = _CODE[self.out_dtype]
        self._act = _pick(_ACT, act, "act")
        self._open(L.LinearConfig(self.device.index, self.in_features, self.out_features, _LAYOUT[layout], self._act,
                                  _CODE[bias.dtype] if bias is not None else L.APK_F32, w, ldw,
                                  bias.data_ptr() if bias is not None else None, sms, wait_limit_ns))
        self._io, self._grads = L.LinearIO(), L.LinearGrads()
        self._io_ref, self._grads_ref = ctypes.byref(self._io), ctypes.byref(self._grads)

    def forward(self, x, residual=None, save_preact: bool = False, out=None):
        """act(x W + b) + residual for x [..., in]; with save_preact also
        x W + b in bf16, as backward() takes it.  out: the output's tensor;
        it may be the residual, but share no memory with x."""
        with self._lock:
            b = self.bias
            if self.weight.data_ptr() != self._w_at or (None if b is None else b.data_ptr()) != self._b_at:
                raise ValueError(_MOVED)
            io, n = self._io, self.out_features
            io.x, io.rows, io.ldx = _rows(x, "x", self.device, self.in_features)
            shape = (io.rows, n) if len(x.shape) == 2 else (*x.shape[:-1], n)
            if out is None:
                y = x.new_empty(shape) if self._y_code == L.APK_BF16 else x.new_empty(shape, dtype=self.out_dtype)
                io.y, io.ldy = y.data_ptr(), n
            else:
                y = out
                if y.shape != shape:
                    raise ValueError(f"out is {tuple(y.shape)}, not {shape}")
                io.y, _, io.ldy = _rows(y, "out", self.device, n, (self.out_dtype,))
            if residual is None:
                io.residual = None
            else:
                if residual.shape != shape:
                    raise ValueError(f"residual is {tuple(residual.shape)}, not {shape}")
                io.residual, _, io.ld_residual = _rows(residual, "residual", self.device, n, _ANY)
                io.residual_dtype = _CODE[residual.dtype]
            if out is not None:
                es = y.element_size()
                to = (io.y, io.ldy * es, n * es)
                if _overlap(to, (io.x, io.ldx * 2, self.in_features * 2), io.rows):
                    raise ValueError("out shares memory with x")
                if residual is not None:
                    rs = residual.element_size()
                    of = (io.residual, io.ld_residual * rs, n * rs)
                    if of != to and _overlap(to, of, io.rows):
                        raise ValueError("out shares memory with residual, but is not it")
            z = None
            if save_preact:
                z = x.new_empty(shape)
                io.preact, io.ld_preact = z.data_ptr(), n
            else:
                io.preact = None
            io.y_dtype, io.stream = self._y_code, _raw_stream(self._index)
            st = self._lib.apk_linear_forward(self._h, self._io_ref)
            if st:
                self._check(st)
            return (y, z) if save_preact else y

    __call__ = forward

    def backward(self, dy, x, preact=None, need_dx: bool = True, need_dw: bool = True, need_db: bool = True,
                 dw_dtype: str = "bf16"):
        """(dx, dw, db) for the output gradient dy (the residual's is dy
        itself); None where one is not needed or the layer has no bias.
        preact: what forward(save_preact=True) returned, for a layer with an
        activation."""
        with self._lock:
            b = self.bias
            if self.weight.data_ptr() != self._w_at or (None if b is None else b.data_ptr()) != self._b_at:
                raise ValueError(_MOVED)
            g, n, k = self._grads, self.out_features, self.in_features
            g.dy, g.rows, g.ld_dy = _rows(dy, "dy", self.device, n)
            if dy.shape[:-1] != x.shape[:-1]:
                raise ValueError(f"dy is {tuple(dy.shape)} and x {tuple(x.shape)}")
            g.x, _, g.ldx = _rows(x, "x", self.device, k)
            if self._act != L.APK_ACT_NONE:
                if preact is None or preact.shape != dy.shape:
                    raise ValueError("preact: the pre-activation that forward(save_preact=True) returned is wanted")
                g.preact, _, g.ld_preact = _rows(preact, "preact", self.device, n)
            else:
                g.preact = None
            g.dx = g.dw = g.db = None
            dx = dw = db = None
            if need_dx:
                dx = _like(x, x.shape)
                g.dx, g.ld_dx = dx.data_ptr(), k
            if need_dw:
                dt = _pick(_TORCH, dw_dtype, "dw_dtype")
                shape = self._w_shape
                dw = _like(self.weight, shape) if dt is torch.bfloat16 else self.weight.new_empty(shape, dtype=dt)
                g.dw, g.ld_dw, g.dw_dtype = dw.data_ptr(), shape[1], _CODE[dt]
            if need_db and self.bias is not None:
                db = torch.empty_like(self.bias)
                g.db = db.data_ptr()
            g.stream = _raw_stream(self._index)
            if dw is not None or db is not None or (dx is not None and g.rows > 0):
                st = self._lib.apk_linear_backward(self._h, self._grads_ref)
                if st:
                    self._check(st)
            return dx, dw, db


class MoE(_Handle):
    """A mixture-of-experts layer for at most 64 tokens at a time.

    router [E, D], w_in [E, 2F, D] (gate rows, then up rows; [E, F, D] when
    not gated) and w_out [E, D, F], bf16 and contiguous.  Each token goes to
    its top_k experts, weighted by their softmax probabilities over all
    experts, divided by the chosen ones' sum if renormalize.  The hidden values
    are rounded to bf16, or with out_dtype "f32" to two bf16 terms.  Weights are
    kept by reference, as Linear keeps them; nothing is recorded for autograd."""
    _create, _destroy = "apk_moe_create", "apk_moe_destroy"
    _error, _status = "apk_moe_last_error", "apk_moe_status"

    def __init__(self, router, w_in, w_out, top_k: int, act: str = "silu", gated: bool = True,
                 renormalize: bool = True, out_dtype: str = "bf16", sms: int = 0,
                 wait_limit_ns: int = _DEFAULT_WAIT_NS):
        _tensor(router, "router", dim=2)
        self.device, self._index = router.device, router.device.index
        self.experts, self.d_model = router.shape
        _tensor(w_in, "w_in", self.device, dim=3)
        _tensor(w_out, "w_out", self.device, dim=3)
        self.d_ff = w_out.shape[2]
        want_in = (self.experts, 2 * self.d_ff if gated else self.d_ff, self.d_model)
        if tuple(w_in.shape) != want_in or tuple(w_out.shape) != (self.experts, self.d_model, self.d_ff):
            raise ValueError(f"router is {tuple(router.shape)}, w_in {tuple(w_in.shape)}, w_out {tuple(w_out.shape)}: "
                             "[E, D], [E, 2F or F, D] and [E, D, F] are wanted")
        for t, what in ((router, "router"), (w_in, "w_in"), (w_out, "w_out")):
            if not t.is_contiguous():
                raise ValueError(f"{what} is not contiguous")
        self.router, self.w_in, self.w_out, self.top_k = router, w_in, w_out, top_k
        self._at = (router.data_ptr(), w_in.data_ptr(), w_out.data_ptr())
        self.out_dtype = _pick(_TORCH, out_dtype, "out_dtype")
        self._y_code = _CODE[self.out_dtype]
        self._open(L.MoeConfig(self.device.index, self.experts, top_k, self.d_model, self.d_ff, _pick(_ACT, act, "act"),
                               int(gated), int(renormalize), router.data_ptr(), w_in.data_ptr(), w_out.data_ptr(),
                               sms, wait_limit_ns))
        self._io = L.MoeIO()
        self._io_ref = ctypes.byref(self._io)

    def forward(self, x, return_routing: bool = False):
        """The layer's output for x [..., D]; with return_routing also the
        chosen experts (int32 [..., top_k]) and their weights (fp32)."""
        with self._lock:
            if (self.router.data_ptr(), self.w_in.data_ptr(), self.w_out.data_ptr()) != self._at:
                raise ValueError(_MOVED)
            io = self._io
            io.x, io.tokens, io.ldx = _rows(x, "x", self.device, self.d_model)
            y = _like(x, x.shape) if self._y_code == L.APK_BF16 else x.new_empty(x.shape, dtype=self.out_dtype)
            io.y, io.ldy, io.y_dtype = y.data_ptr(), self.d_model, self._y_code
            ids = probs = None
            if return_routing:
                shape = (*x.shape[:-1], self.top_k)
                ids, probs = x.new_empty(shape, dtype=torch.int32), x.new_empty(shape, dtype=torch.float32)
                io.ids, io.probs = ids.data_ptr(), probs.data_ptr()
            else:
                io.ids = io.probs = None
            io.stream = _raw_stream(self._index)
            st = self._lib.apk_moe_forward(self._h, self._io_ref)
            if st:
                self._check(st)
            return (y, ids, probs) if return_routing else y

    __call__ = forward
