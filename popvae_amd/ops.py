"""Operators on the caller's own GPU tensors (include/pvae_ops.h through ctypes): a dense layer with bias, activation and
residual in one pass, its gradients, the global gradient norm, clipping by it, and the Adam update with that clipping.

They are what the engine's layers and optimizer do, for tensors that do not live in an ``Engine``: any size, float32, bfloat16
or float16, other activations.  Everything runs on torch's current stream of the tensors' device, allocates through torch's
allocator (outputs and scratch memory), never waits for the GPU and may be captured into a graph.  A call that cannot be
computed raises ValueError before anything is launched.  There is no CPU path.  Autograd records nothing here, gradients are
calls of their own: where grad mode is on, ``dense`` and ``dense_backward`` refuse tensors that require a gradient (call them
under ``torch.no_grad()``).  What is written in place counts as changed for what autograd has saved.

    y = ops.dense(x, w, b, "elu", residual=x, pre=z)               # z: float32, kept for the backward
    dx, dw, db = ops.dense_backward(dy, x, w, z, "elu", dx_add=dy)  # dx_add: the layer's residual was its own input
    grads = ops.TensorSet([...])
    norm = ops.adam_step(params, grads, m, v, step, clip_norm=1.0)
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import engine

OPS_SYMBOLS = ["pvae_ops_last_error", "pvae_dense_workspace", "pvae_dense", "pvae_dense_bwd_workspace", "pvae_dense_bwd",
               "pvae_norm_workspace", "pvae_global_norm", "pvae_clip_by_global_norm", "pvae_adam_step"]
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"linear": 0, "relu": 1, "elu": 2, "sigmoid": 3, "tanh": 4, "silu": 5, "gelu": 6}


class _Dense(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("act", C.c_int32), ("m", C.c_int64), ("k", C.c_int64), ("n", C.c_int64),
                ("x", C.c_void_p), ("ldx", C.c_int64), ("w", C.c_void_p), ("w_sk", C.c_int64), ("w_sn", C.c_int64),
                ("bias", C.c_void_p), ("residual", C.c_void_p), ("ldr", C.c_int64), ("y", C.c_void_p), ("ldy", C.c_int64),
                ("pre", C.c_void_p), ("ldp", C.c_int64)]


class _DenseBwd(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("act", C.c_int32), ("m", C.c_int64), ("k", C.c_int64), ("n", C.c_int64),
                ("dy", C.c_void_p), ("lddy", C.c_int64), ("x", C.c_void_p), ("ldx", C.c_int64), ("w", C.c_void_p),
                ("w_sk", C.c_int64), ("w_sn", C.c_int64), ("pre", C.c_void_p), ("ldp", C.c_int64), ("dx", C.c_void_p),
                ("lddx", C.c_int64), ("dx_add", C.c_void_p), ("ldadd", C.c_int64), ("dw", C.c_void_p), ("dbias", C.c_void_p),
                ("dpre", C.c_void_p)]


class _Tensor(C.Structure):
    _fields_ = [("data", C.c_void_p), ("n", C.c_int64), ("dtype", C.c_int32), ("tile", C.c_int32)]


# the same structures as bytes, which costs a call a third of what building a ctypes object does
_pack_dense = struct.Struct("@2i3qPqP2q2PqPqPq").pack
_pack_bwd = struct.Struct("@2i3qPqPqP2qPqPqPq3P").pack

_lib = None
_norm_workspace = 0  # bytes


def lib():
    """libpvae.so with the operators' signatures set."""
    global _lib, _norm_workspace
    if _lib is None:
        L = engine.lib()
        vp, i32, i64, f64, tp = C.c_void_p, C.c_int32, C.c_int64, C.c_double, C.POINTER(_Tensor)
        L.pvae_ops_last_error.restype = C.c_char_p
        for name in ("pvae_dense", "pvae_dense_bwd"):
            work = getattr(L, name + "_workspace")
            work.restype, work.argtypes = i64, [vp]
            getattr(L, name).argtypes = [vp, vp, i64, vp]
        L.pvae_norm_workspace.restype = i64
        L.pvae_global_norm.argtypes = [tp, i64, vp, vp, i64, vp]
        L.pvae_clip_by_global_norm.argtypes = [tp, tp, i64, f64, vp, vp, i64, vp]
        L.pvae_adam_step.argtypes = [tp, tp, tp, tp, i64, f64, f64, f64, f64, i64, vp, f64, vp, vp, i64, vp]
        _norm_workspace = L.pvae_norm_workspace()
        _lib = L
    return _lib


def _check(rc):
    if rc:
        text = lib().pvae_ops_last_error().decode()
        if rc <= -9:
            raise RuntimeError(f"libpvae ({rc}): {text}")
        raise ValueError(text)


def _matrix(name, t, rows, cols, dtype, device, expand=False):
    """Row stride of a [rows, cols] tensor whose rows are contiguous."""
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name}: expected {dtype} on {device}, got {t.dtype} on {t.device}")
    if t.shape != (rows, cols):
        raise ValueError(f"{name}: expected shape ({rows}, {cols}), got {tuple(t.shape)}")
    ld, sn = t.stride()
    if sn != 1 and cols > 1:
        raise ValueError(f"{name}: rows are not contiguous (strides {t.stride()})")
    if rows <= 1:
        return cols
    if ld < cols and not (expand and ld == 0):
        raise ValueError(f"{name}: rows overlap (strides {t.stride()})")
    return ld


def _vector(name, t, n, dtype, device):
    if t.dtype != dtype or t.device != device or t.shape != (n,):
        raise ValueError(f"{name}: expected {dtype} of shape ({n},) on {device}, got {t.dtype} of {tuple(t.shape)} on {t.device}")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} is not contiguous")


def _act(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"activation {name!r}: one of {', '.join(ACTIVATIONS)}") from None


def _layer(x, w):
    """Checks x [m, k] and w [k, n]; returns (type, device, m, k, n, row stride of x)."""
    dtype, device = x.dtype, x.device
    if dtype not in DTYPES:
        raise ValueError(f"x: {dtype} is not one of float32, bfloat16, float16")
    if device.type != "cuda":
        raise ValueError(f"x is on {device}: the operators run on a GPU only")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[0]:
        raise ValueError(f"x {tuple(x.shape)} and w {tuple(w.shape)}: expected [m, k] and [k, n]")
    if w.dtype != dtype or w.device != device:
        raise ValueError(f"w: expected {dtype} on {device}, got {w.dtype} on {w.device}")
    m, k = x.shape
    return dtype, device, m, k, w.shape[1], _matrix("x", x, m, k, dtype, device)


_recording = torch.is_grad_enabled


def _no_history(*tensors):
    """Where autograd would record, a result without history would pass for one that depends on nothing."""
    for t in tensors:
        if t is not None and t.requires_grad:
            raise ValueError("a tensor requires a gradient, and autograd records nothing here: call under torch.no_grad() and "
                             "take the gradients from dense_backward")


# of a list of tensors: a later backward refuses those that it has saved (directly: the public function looks at types first)
_changed = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)


def _stream(device):
    """torch's current stream of a device as a hipStream_t."""
    return torch.cuda.current_stream(device).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the same without a Stream object: a microsecond less
if _raw_stream is not None:
    def _stream(device):  # noqa: F811
        return _raw_stream(device.index)


def _call(f, packed, need, device):
    """A call whose arguments are packed; most need no workspace, and a refused one has launched nothing."""
    rc = f(packed, None, 0, _stream(device))
    if rc == -8:
        n = need(packed)
        work = torch.empty(n, dtype=torch.uint8, device=device)
        rc = f(packed, work.data_ptr(), n, _stream(device))
    if rc:
        _check(rc)


def dense(x, w, bias=None, activation="linear", residual=None, pre=None, out=None):
    """``activation(x @ w + bias) + residual``, one rounding at the end.

    x [m, k] (contiguous rows, any row stride), w [k, n] (a Keras kernel, or a transposed view), bias [n], residual [m, n]
    (an expanded row is fine), all of one type; sums are float32.  pre: float32 [m, n], receives ``x @ w + bias`` for
    ``dense_backward``.  out: [m, n] to write to (may be the residual), otherwise a new tensor.  Returns it."""
    dtype, device, m, k, n, ldx = _layer(x, w)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return dense(x, w, bias, activation, residual, pre, out)
    if _recording():
        _no_history(x, w, bias, residual, pre, out)
    bp = rp = zp = ldr = ldp = 0
    if bias is not None:
        _vector("bias", bias, n, dtype, device)
        bp = bias.data_ptr()
    changed = []
    if residual is not None:
        ldr, rp = _matrix("residual", residual, m, n, dtype, device, expand=True), residual.data_ptr()
    if pre is not None:
        ldp, zp = _matrix("pre", pre, m, n, torch.float32, device), pre.data_ptr()
        changed.append(pre)
    if out is None:
        out, ldy = torch.empty((m, n), dtype=dtype, device=device), n
    else:
        ldy = _matrix("out", out, m, n, dtype, device)
        changed.append(out)
    sk, sn = w.stride()
    L = _lib or lib()
    _call(L.pvae_dense, _pack_dense(DTYPES[dtype], _act(activation), m, k, n, x.data_ptr(), ldx, w.data_ptr(), sk, sn, bp, rp, ldr,
                                    out.data_ptr(), ldy, zp, ldp), L.pvae_dense_workspace, device)
    if changed:
        _changed(changed)
    return out


def dense_backward(dy, x, w, pre=None, activation="linear", dx_add=None, need_dx=True, need_dw=True, need_bias=True):
    """Gradients of ``dense``: ``(dx, dw, db)``, with None for what is not needed.

    dy [m, n] (an expanded row is fine); x, w and activation as in the forward, pre what it left (not needed for "linear").  dx_add [m, k] is added to
    dx before its rounding: a layer whose residual is its own input passes dy.  (The gradient of the residual is dy itself;
    summed over the rows for an expanded one.)  dx, dw and db are rounded to their type once, at their end."""
    dtype, device, m, k, n, ldx = _layer(x, w)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return dense_backward(dy, x, w, pre, activation, dx_add, need_dx, need_dw, need_bias)
    if _recording():
        _no_history(dy, x, w, pre, dx_add)
    act = _act(activation)
    lddy = _matrix("dy", dy, m, n, dtype, device, expand=True)
    zp = ldp = ap = ldadd = 0
    if pre is not None:
        ldp, zp = _matrix("pre", pre, m, n, torch.float32, device), pre.data_ptr()
    elif act:
        raise ValueError(f"the gradient of {activation!r} needs pre, which dense leaves")
    if dx_add is not None:
        ldadd, ap = _matrix("dx_add", dx_add, m, k, dtype, device, expand=True), dx_add.data_ptr()
    dx = torch.empty((m, k), dtype=dtype, device=device) if need_dx else None
    dw = torch.empty((k, n), dtype=dtype, device=device) if need_dw else None
    db = torch.empty(n, dtype=dtype, device=device) if need_bias else None
    sk, sn = w.stride()
    L = _lib or lib()
    _call(L.pvae_dense_bwd, _pack_bwd(DTYPES[dtype], act, m, k, n, dy.data_ptr(), lddy, x.data_ptr(), ldx, w.data_ptr(), sk, sn, zp, ldp,
                                      _ptr(dx), k, ap, ldadd, _ptr(dw), _ptr(db), 0), L.pvae_dense_bwd_workspace, device)
    return dx, dw, db


_data_ptr = torch.Tensor.data_ptr


def _ptr(t):
    return 0 if t is None else t.data_ptr()


class TensorSet:
    """A list of contiguous tensors on one GPU, checked and described once: what the operators over all tensors of a model take
    (a plain list works too, and is described anew by every call).  The tensors must keep their storage, which the set holds on
    to: a set one of whose tensors has moved is refused."""

    def __init__(self, tensors):
        self._describe(list(tensors))
        # while the set lives nothing else is allocated where its tensors are, whatever becomes of them
        self._storages = [t.detach() for t in self.tensors]

    def _describe(self, ts):
        self.device = ts[0].device if ts else None
        for i, t in enumerate(ts):
            if t.dtype not in DTYPES:
                raise ValueError(f"tensor {i}: {t.dtype} is not one of float32, bfloat16, float16")
            if t.device.type != "cuda" or t.device != self.device:
                raise ValueError(f"tensor {i} is on {t.device}: all tensors are on one GPU")
            if not t.is_contiguous():
                raise ValueError(f"tensor {i} is not contiguous")
        self.tensors = ts
        self._ptrs = [t.data_ptr() for t in ts]
        self._sizes = [t.numel() for t in ts]
        self._types = [t.dtype for t in ts]
        self._table = (_Tensor * len(ts))(*[(p, n, DTYPES[d], 0) for p, n, d in zip(self._ptrs, self._sizes, self._types)])

    def __len__(self):
        return len(self._sizes)

    def _same(self):
        if list(map(_data_ptr, self.tensors)) != self._ptrs:
            raise ValueError("a tensor of the set has another storage than when the set was made")
        return self._table


def _set(t):
    if isinstance(t, TensorSet):
        return t
    s = TensorSet.__new__(TensorSet)  # for one call
    s._describe(list(t))
    return s


def _device_of(s):
    if s.device is None:
        raise ValueError("no tensors")
    return s.device


def _scratch(device):
    """The norm that a call returns and its workspace."""
    lib()
    need = _norm_workspace
    return torch.empty((), dtype=torch.float32, device=device), torch.empty(need, dtype=torch.uint8, device=device), need


def global_norm(tensors):
    """``sqrt(sum of squares)`` over all tensors, summed in float64: a 0-d float32 tensor."""
    s = _set(tensors)
    device = _device_of(s)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return global_norm(s)
    table = s._same()
    norm, work, need = _scratch(device)
    _check(_lib.pvae_global_norm(table, len(s), norm.data_ptr(), work.data_ptr(), need, _stream(device)))
    return norm


def clip_by_global_norm(tensors, max_norm, out=None):
    """Scales all tensors by ``min(1, max_norm / norm)`` into ``out`` (tensors of the same sizes and types; default: in place)
    and returns the norm before clipping, a 0-d float32 tensor.  A norm that is not finite makes every output NaN."""
    s = _set(tensors)
    o = s if out is None else _set(out)
    device = _device_of(s)
    if len(o) != len(s) or o.device != device:
        raise ValueError("out: as many tensors as there are gradients, on their GPU")
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return clip_by_global_norm(s, max_norm, o)
    table = s._same()
    into = table if o is s else o._same()
    norm, work, need = _scratch(device)
    _check(_lib.pvae_clip_by_global_norm(table, into, len(s), float(max_norm), norm.data_ptr(), work.data_ptr(), need, _stream(device)))
    _changed(o.tensors)
    return norm


def adam_step(params, grads, m, v, step, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-7, clip_norm=None):
    """One update of the engine's Adam (Keras') over all tensors, in place: params, m and v float32, grads of any type.

    step: the update's number, counted from 1, or an int32 tensor of one element on the GPU holding it (a captured graph's
    replays read it anew).  clip_norm: the gradients enter scaled by ``min(1, clip_norm / norm)``; the norm before clipping is
    returned (a 0-d float32 tensor; None without clipping)."""
    p, g, m, v = _set(params), _set(grads), _set(m), _set(v)
    device = _device_of(p)
    for name, s in (("grads", g), ("m", m), ("v", v)):
        if s.device != device or s._sizes != p._sizes:
            raise ValueError(f"{name}: as many tensors of the same sizes as there are parameters, on their GPU")
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return adam_step(p, g, m, v, step, lr, beta1, beta2, eps, clip_norm)
    at = None
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int32 or step.numel() != 1 or step.device != device:
            raise ValueError("step: a number, or an int32 tensor of one element on the parameters' GPU")
        at, step = step.data_ptr(), 0
    L, norm, work, need = lib(), None, None, 0
    if clip_norm is not None:
        if not clip_norm > 0:
            raise ValueError(f"clip_norm {clip_norm}: a positive number, or None")
        norm, work, need = _scratch(device)
    _check(L.pvae_adam_step(p._same(), g._same(), m._same(), v._same(), len(p), lr, beta1, beta2, eps, int(step), at,
                            float(clip_norm or 0.0), _ptr(norm), _ptr(work), need, _stream(device)))
    for written in (p, m, v):
        _changed(written.tensors)
    return norm
