"""Python binding of the projection with low-rank adapters (include/gemmaedge_projection.h).

The layer that makes the logits which ``sampler`` reads, or any other linear layer
that many requests share, each with an adapter of its own, and the adapters'
gradients: ctypes over the same library as ``sampler``; torch supplies device memory
and streams, as in ``head`` (streams, and what is recorded on them, are described
there). There is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

from . import head as H
from . import sampler as S

EXPORTS = ("ge_projection_create", "ge_projection_destroy", "ge_project", "ge_project_backward")

_P, _I32, _I64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class ProjectArgs(ctypes.Structure):
    _fields_ = [
        ("hidden", _P), ("hidden_stride", _I64), ("weight", _P), ("weight_stride", _I64), ("rows", _I32), ("dim", _I32),
        ("out_dim", _I32), ("rank", _I32), ("adapters", _I32), ("a", _P), ("b", _P), ("scale", _P), ("adapter", _P), ("out", _P),
        ("out_stride", _I64), ("out_dtype", _I32), ("dout", _P), ("dout_stride", _I64), ("dhidden", _P), ("dhidden_stride", _I64),
        ("da", _P), ("db", _P),
    ]


_ready = False


def _library() -> ctypes.CDLL:
    global _ready
    L = S.load_library()
    if not _ready:
        for name in EXPORTS:
            getattr(L, name).restype = ctypes.c_int
        L.ge_projection_create.argtypes = [ctypes.c_int] * 8 + [ctypes.POINTER(_P)]
        L.ge_projection_destroy.restype = None
        L.ge_projection_destroy.argtypes = [_P]
        for name in ("ge_project", "ge_project_backward"):
            getattr(L, name).argtypes = [_P, _P, ctypes.POINTER(ProjectArgs)]
        _ready = True
    return L


class Projection:
    """One ge_projection handle: workspaces for up to ``max_rows`` rows of up to ``max_dim``
    channels, weights of up to ``max_out`` rows and up to ``max_adapters`` adapters of
    up to ``max_rank`` (0: none), elements of ``dtype`` (float32 or bfloat16). ``train``
    adds the backward call's workspace. A handle must not be used by two streams at once."""

    def __init__(self, max_rows: int, max_dim: int, max_out: int, max_rank: int = 0, max_adapters: int = 0, dtype=None,
                 train: bool = False, device: int = 0):
        self._h = None
        self.dtype = torch.bfloat16 if dtype is None else dtype
        if self.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"unsupported dtype {self.dtype}")
        h = ctypes.c_void_p()
        code = S.GE_DTYPE_F32 if self.dtype == torch.float32 else S.GE_DTYPE_BF16
        H._check(_library().ge_projection_create(device, max_rows, max_dim, max_out, max_rank, max_adapters, code, int(train),
                                                 ctypes.byref(h)))
        self._h = h
        self.device = torch.device("cuda", device)

    def close(self):
        if getattr(self, "_h", None):
            _library().ge_projection_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def _args(self, hidden, weight, a, b, scale, adapter):
        """The fields up to ``adapter``, checked."""
        if hidden.dim() != 2 or weight.dim() != 2:
            raise ValueError(f"hidden {tuple(hidden.shape)}, weight {tuple(weight.shape)}: [rows, dim] and [out, dim] are wanted")
        device, dtype = self.device, self.dtype
        rows, dim = shape = hidden.shape
        out = weight.shape[0]
        H._want(hidden, "hidden", dtype, shape, device)
        H._want(weight, "weight", dtype, (out, dim), device)
        head = (hidden.data_ptr(), hidden.stride(0) if rows > 1 else dim, weight.data_ptr(), weight.stride(0) if out > 1 else dim, rows, dim, out)
        if a is None and b is None and scale is None and adapter is None:
            return head + (0, 0, None, None, None, None)
        if a is None or b is None or scale is None or adapter is None:
            raise ValueError("a, b, scale and adapter are given together")
        if a.dim() != 3:
            raise ValueError(f"a has shape {tuple(a.shape)}: [adapters, rank, dim] is wanted")
        k, r, _ = a.shape
        H._want(a, "a", dtype, (k, r, dim), device)
        H._want(b, "b", dtype, (k, out, r), device)
        H._want(scale, "scale", torch.float32, (k,), device)
        H._want(adapter, "adapter", torch.int32, (rows,), device)
        if not (a.is_contiguous() and b.is_contiguous() and scale.is_contiguous() and adapter.is_contiguous()):
            raise ValueError("a, b, scale and adapter must be contiguous")
        return head + (r, k, a.data_ptr(), b.data_ptr(), scale.data_ptr(), adapter.data_ptr())

    def project(self, hidden, weight, a=None, b=None, scale=None, adapter=None, out=None, out_dtype=None, stream=None):
        """[rows, dim] hidden states times [out, dim] weights, and for each row whose
        ``adapter`` (int32 [rows]) k lies within [0, adapters) also scale[k] * b[k] @ (a[k] @ row):
        ``a`` [adapters, rank, dim], ``b`` [adapters, out, rank], ``scale`` float32 [adapters].
        Returns [rows, out] of ``out_dtype`` (None: the operands'; float32 or bfloat16), ``out`` if given."""
        x = self._args(hidden, weight, a, b, scale, adapter)
        rows, n = x[4], x[6]
        if out is not None and out_dtype is not None and out.dtype != out_dtype:
            raise ValueError(f"out has dtype {out.dtype}: {out_dtype} is wanted")
        handle, side = H._stream(stream, self.device)
        out = H._output(out, "out", (out.dtype if out is not None else out_dtype or self.dtype), (rows, n), self.device, side)
        x = ProjectArgs(*x, out.data_ptr(), H._stride(out), H._dtype(out, "out"))
        H._check(_library().ge_project(self._h, handle, ctypes.byref(x)))
        H._used(side, hidden, weight, a, b, scale, adapter, out)
        return out

    def project_backward(self, dout, hidden, weight, a=None, b=None, scale=None, adapter=None, dhidden=None, da=None, db=None,
                         need_hidden: bool = True, need_adapters: bool = True, stream=None):
        """Gradients of ``project`` for the gradient ``dout`` [rows, out] (the operands' dtype) of
        its output. Returns (dhidden, da, db), None for what is not wanted (``need_hidden``,
        ``need_adapters``) or, without adapters, not there. The weight has no gradient here."""
        x = ProjectArgs(*self._args(hidden, weight, a, b, scale, adapter))
        rows, dim, n = x.rows, x.dim, x.out_dim
        H._want(dout, "dout", self.dtype, (rows, n), self.device)
        if a is None and (da is not None or db is not None):
            raise ValueError("da or db without adapters")
        handle, side = H._stream(stream, self.device)
        if need_hidden or dhidden is not None:
            dhidden = H._output(dhidden, "dhidden", self.dtype, (rows, dim), self.device, side)
            x.dhidden, x.dhidden_stride = dhidden.data_ptr(), H._stride(dhidden)
        grads = []
        for t, what, like in ((da, "da", a), (db, "db", b)):
            if t is not None or (need_adapters and like is not None):
                t = H._output(t, what, self.dtype, like.shape, self.device, side)
                if not t.is_contiguous():
                    raise ValueError(f"{what} must be contiguous")
            grads.append(t)
        da, db = grads
        x.dout, x.dout_stride, x.da, x.db = dout.data_ptr(), H._stride(dout), S._ptr(da), S._ptr(db)
        H._check(_library().ge_project_backward(self._h, handle, ctypes.byref(x)))
        H._used(side, dout, hidden, weight, a, b, scale, adapter, dhidden, da, db)
        return dhidden, da, db
