"""Python binding of the trainable answer head (include/gemmaedge_head.h).

The norm in front of the vocabulary projection, the projection's cross entropy
with its gradients, and the AdamW step: ctypes over the same library as
``sampler``; torch supplies device memory and streams. There is no CPU path.

Calls run on the current torch stream of the tensors' device unless ``stream``
is given, and outputs that are not passed in are allocated on it. Ordering that
stream after the work that fills the inputs is the caller's. A torch.cuda.Stream
other than the current one is recorded on every tensor of the call, so tensors may
be dropped right after it; with a raw handle or an ExternalStream the caller keeps
them until the stream has passed the call.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import sampler as S

GE_ADAMW_BLOCK = 256

EXPORTS = (
    "ge_head_create",
    "ge_head_destroy",
    "ge_head_norm",
    "ge_head_norm_backward",
    "ge_head_loss",
    "ge_head_loss_backward",
    "ge_adamw_table_bytes",
    "ge_adamw_table",
    "ge_adamw_step",
)

_P, _I32, _I64, _F32, _F64, _U32 = (ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_double,
                                    ctypes.c_uint32)


class NormArgs(ctypes.Structure):
    _fields_ = [
        ("x", _P), ("x_stride", _I64), ("rows", _I32), ("dim", _I32), ("weight_dtype", _I32), ("center", _I32),
        ("eps", _F32), ("weight", _P), ("bias", _P), ("y", _P), ("y_stride", _I64), ("mean", _P), ("rstd", _P),
        ("dy", _P), ("dy_stride", _I64), ("dx", _P), ("dx_stride", _I64), ("dweight", _P), ("dbias", _P),
    ]


class LossArgs(ctypes.Structure):
    _fields_ = [
        ("hidden", _P), ("hidden_stride", _I64), ("weight", _P), ("weight_stride", _I64), ("rows", _I32), ("dim", _I32),
        ("vocab", _I32), ("softcap", _F32), ("targets", _P), ("loss", _P), ("lse", _P), ("grad", _P), ("dhidden", _P),
        ("dhidden_stride", _I64), ("dweight", _P), ("dweight_stride", _I64),
    ]


class AdamwTensor(ctypes.Structure):
    _fields_ = [
        ("param", _P), ("grad", _P), ("master", _P), ("m", _P), ("v", _P), ("m_scale", _P), ("v_scale", _P), ("n", _I64),
        ("param_dtype", _I32), ("grad_dtype", _I32),
    ]


class AdamwParams(ctypes.Structure):
    _fields_ = [
        ("lr", _F64), ("beta1", _F64), ("beta2", _F64), ("eps", _F64), ("weight_decay", _F64), ("grad_scale", _F64),
        ("step", _U32), ("seed", _U32),
    ]


class AdamwArgs(ctypes.Structure):
    _fields_ = [
        ("table", _P), ("table_bytes", _I64), ("count", _I32), ("state_bits", _I32), ("params", AdamwParams),
        ("device_params", _P),
    ]


_ready = False


def _library() -> ctypes.CDLL:
    global _ready
    L = S.load_library()
    if not _ready:
        for name in EXPORTS:
            getattr(L, name).restype = ctypes.c_int
        L.ge_head_create.argtypes = [ctypes.c_int] * 6 + [ctypes.POINTER(_P)]
        L.ge_head_destroy.restype = None
        L.ge_head_destroy.argtypes = [_P]
        for name in ("ge_head_norm", "ge_head_norm_backward"):
            getattr(L, name).argtypes = [_P, _P, ctypes.POINTER(NormArgs)]
        for name in ("ge_head_loss", "ge_head_loss_backward"):
            getattr(L, name).argtypes = [_P, _P, ctypes.POINTER(LossArgs)]
        L.ge_adamw_table_bytes.argtypes = [ctypes.POINTER(AdamwTensor), ctypes.c_int, ctypes.c_int, ctypes.POINTER(_I64)]
        L.ge_adamw_table.argtypes = [ctypes.POINTER(AdamwTensor), ctypes.c_int, ctypes.c_int, _P, _I64]
        L.ge_adamw_step.argtypes = [_P, ctypes.POINTER(AdamwArgs)]
        _ready = True
    return L


def _check(rc: int) -> None:
    if rc != S.GE_OK:
        raise S.SamplerError(rc, S.last_error())


def _dtype(t, what: str) -> int:
    if t.dtype == torch.float32:
        return S.GE_DTYPE_F32
    if t.dtype == torch.bfloat16:
        return S.GE_DTYPE_BF16
    raise ValueError(f"{what} has dtype {t.dtype}: float32 or bfloat16 is wanted")


def _want(t, what: str, dtype, shape, device) -> None:
    """A tensor of this dtype, shape and device with contiguous last axis (all axes but the first)."""
    if t.dtype == dtype and t.shape == shape and t.device == device and t.is_contiguous():
        return
    if t.dtype != dtype:
        raise ValueError(f"{what} has dtype {t.dtype}: {dtype} is wanted")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} has shape {tuple(t.shape)}: {tuple(shape)} is wanted")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, not on {device}")
    if t.dim() and t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: the last axis must be contiguous")
    if t.dim() == 2 and t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: rows overlap (row stride < {t.shape[1]})")


def _stride(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _on_gpu(t, what: str):
    if t.device.type != "cuda":
        raise ValueError(f"{what} is on {t.device}: a GPU tensor is wanted")
    return t.device


def _stream(stream, device):
    """(handle for the launch, the stream itself if it is not the current one)."""
    current = torch._C._cuda_getCurrentRawStream(device.index)
    if stream is None:
        return current, None
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device)
    return stream.cuda_stream, stream if stream.cuda_stream != current else None


def _used(side, *tensors):
    """Notes that work on ``side`` uses the tensors, so that their memory is not handed
    out again before it is done. Streams that torch does not own may be gone by the
    time a tensor is freed: there the caller keeps the tensors."""
    if side is not None and not isinstance(side, torch.cuda.ExternalStream):
        for t in tensors:
            if t is not None:
                t.record_stream(side)


def _output(t, what: str, dtype, shape, device, side):
    """The given output, checked, or a new one of the call's stream."""
    if t is not None:
        _want(t, what, dtype, shape, device)
        return t
    if side is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(side):
        return torch.empty(shape, dtype=dtype, device=device)


class Head:
    """One ge_head handle: workspaces for up to ``max_rows`` hidden states of up
    to ``max_dim`` channels and a vocabulary of up to ``max_vocab``, elements of
    ``dtype`` (float32 or bfloat16). ``train`` adds the backward calls' workspace.
    A handle must not be used by two streams at once."""

    def __init__(self, max_rows: int, max_dim: int, max_vocab: int, dtype=None, train: bool = False, device: int = 0):
        self._h = None
        self.dtype = torch.bfloat16 if dtype is None else dtype
        if self.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"unsupported dtype {self.dtype}")
        h = ctypes.c_void_p()
        code = S.GE_DTYPE_F32 if self.dtype == torch.float32 else S.GE_DTYPE_BF16
        _check(_library().ge_head_create(device, max_rows, max_dim, max_vocab, code, int(train), ctypes.byref(h)))
        self._h = h
        self.device = torch.device("cuda", device)

    def close(self):
        if getattr(self, "_h", None):
            _library().ge_head_destroy(self._h)
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

    def _rows(self, x, what):
        if x.dim() != 2:
            raise ValueError(f"{what} has shape {tuple(x.shape)}: [rows, dim] is wanted")
        _want(x, what, self.dtype, x.shape, self.device)
        return x.shape

    def norm(self, x, weight, bias=None, eps: float = 1e-6, center: bool = True, y=None, mean=None, rstd=None, stream=None):
        """y = (x - mean) * rstd * weight + bias over the last axis of [rows, dim];
        without ``center`` the mean is left at 0 (root-mean-square norm), a ``mean``
        that is passed in is filled with zeros, and None is returned for it, which is
        what ``norm_backward`` knows the norm by. Returns (y, mean, rstd)."""
        rows, dim = self._rows(x, "x")
        a = NormArgs()
        a.weight_dtype = _dtype(weight, "weight")
        _want(weight, "weight", weight.dtype, (dim,), self.device)
        if bias is not None:
            _want(bias, "bias", weight.dtype, (dim,), self.device)
        handle, side = _stream(stream, self.device)
        y = _output(y, "y", self.dtype, (rows, dim), self.device, side)
        rstd = _output(rstd, "rstd", torch.float32, (rows,), self.device, side)
        if center or mean is not None:
            mean = _output(mean, "mean", torch.float32, (rows,), self.device, side)
        a.x, a.x_stride, a.rows, a.dim = x.data_ptr(), _stride(x), rows, dim
        a.center, a.eps = int(center), eps
        a.weight, a.bias = weight.data_ptr(), S._ptr(bias)
        a.y, a.y_stride, a.mean, a.rstd = y.data_ptr(), _stride(y), S._ptr(mean), rstd.data_ptr()
        _check(_library().ge_head_norm(self._h, handle, ctypes.byref(a)))
        _used(side, x, weight, bias, y, mean, rstd)
        return y, mean if center else None, rstd

    def norm_backward(self, grad, x, weight, mean, rstd, bias: bool = False, dx=None, dweight=None, dbias=None,
                      need_input: bool = True, need_weight: bool = True, stream=None):
        """Gradients of ``norm`` for the gradient ``grad`` of its y, with the mean
        (None: not centred) and rstd it returned. Returns (dx, dweight, dbias), None
        for what is not wanted (``need_input``, ``need_weight``, ``bias``)."""
        rows, dim = self._rows(x, "x")
        a = NormArgs()
        a.weight_dtype = _dtype(weight, "weight")
        _want(weight, "weight", weight.dtype, (dim,), self.device)
        _want(grad, "grad", self.dtype, (rows, dim), self.device)
        _want(rstd, "rstd", torch.float32, (rows,), self.device)
        if mean is not None:
            _want(mean, "mean", torch.float32, (rows,), self.device)
        handle, side = _stream(stream, self.device)
        if need_input or dx is not None:
            dx = _output(dx, "dx", self.dtype, (rows, dim), self.device, side)
            a.dx_stride = _stride(dx)
        if need_weight or dweight is not None:
            dweight = _output(dweight, "dweight", weight.dtype, (dim,), self.device, side)
        if bias or dbias is not None:
            dbias = _output(dbias, "dbias", weight.dtype, (dim,), self.device, side)
        a.x, a.x_stride, a.rows, a.dim = x.data_ptr(), _stride(x), rows, dim
        a.center = int(mean is not None)
        a.weight, a.mean, a.rstd = weight.data_ptr(), S._ptr(mean), rstd.data_ptr()
        a.dy, a.dy_stride, a.dx = grad.data_ptr(), _stride(grad), S._ptr(dx)
        a.dweight, a.dbias = S._ptr(dweight), S._ptr(dbias)
        _check(_library().ge_head_norm_backward(self._h, handle, ctypes.byref(a)))
        _used(side, grad, x, weight, mean, rstd, dx, dweight, dbias)
        return dx, dweight, dbias

    def _loss_args(self, hidden, weight, targets, softcap):
        rows, dim = self._rows(hidden, "hidden")
        if weight.dim() != 2:
            raise ValueError(f"weight has shape {tuple(weight.shape)}: [vocab, dim] is wanted")
        vocab = weight.shape[0]
        _want(weight, "weight", self.dtype, (vocab, dim), self.device)
        _want(targets, "targets", torch.int32, (rows,), self.device)
        a = LossArgs()
        a.hidden, a.hidden_stride, a.weight, a.weight_stride = hidden.data_ptr(), _stride(hidden), weight.data_ptr(), _stride(weight)
        a.rows, a.dim, a.vocab, a.softcap, a.targets = rows, dim, vocab, softcap, targets.data_ptr()
        return a, rows, dim, vocab

    def loss(self, hidden, weight, targets, softcap: float = 0.0, loss=None, lse=None, stream=None):
        """Cross entropy of [rows, dim] hidden states against their ``targets``
        (int32 [rows]; outside [0, vocab): no loss) over [vocab, dim] weights.
        -loss is the target's log-probability. Returns (loss, lse), float32 [rows]."""
        a, rows, _, _ = self._loss_args(hidden, weight, targets, softcap)
        handle, side = _stream(stream, self.device)
        loss = _output(loss, "loss", torch.float32, (rows,), self.device, side)
        lse = _output(lse, "lse", torch.float32, (rows,), self.device, side)
        a.loss, a.lse = loss.data_ptr(), lse.data_ptr()
        _check(_library().ge_head_loss(self._h, handle, ctypes.byref(a)))
        _used(side, hidden, weight, targets, loss, lse)
        return loss, lse

    def loss_backward(self, grad, hidden, weight, targets, lse, softcap: float = 0.0, dhidden=None, dweight=None,
                      need_hidden: bool = True, need_weight: bool = True, stream=None):
        """Gradients of ``loss`` for ``grad`` (float32 [rows], the objective's
        derivative by each row's loss) and the lse it returned. Returns (dhidden,
        dweight), None for what is not wanted."""
        a, rows, dim, vocab = self._loss_args(hidden, weight, targets, softcap)
        _want(grad, "grad", torch.float32, (rows,), self.device)
        _want(lse, "lse", torch.float32, (rows,), self.device)
        handle, side = _stream(stream, self.device)
        if need_hidden or dhidden is not None:
            dhidden = _output(dhidden, "dhidden", self.dtype, (rows, dim), self.device, side)
            a.dhidden, a.dhidden_stride = dhidden.data_ptr(), _stride(dhidden)
        if need_weight or dweight is not None:
            dweight = _output(dweight, "dweight", self.dtype, (vocab, dim), self.device, side)
            a.dweight, a.dweight_stride = dweight.data_ptr(), _stride(dweight)
        a.grad, a.lse = grad.data_ptr(), lse.data_ptr()
        _check(_library().ge_head_loss_backward(self._h, handle, ctypes.byref(a)))
        _used(side, grad, hidden, weight, targets, lse, dhidden, dweight)
        return dhidden, dweight


def _disjoint(spans):
    """Refuses memory that a step writes and that another of its tensors shares.
    ``spans``: (first byte, end, what it is, whether it is written)."""
    written, any_ = (0, ""), (0, "")
    for start, end, what, writes in sorted(spans):
        for other, name in (written, any_ if writes else written):
            if start < other:
                raise ValueError(f"{what} shares memory with {name}")
        if writes:
            written = max(written, (end, what))
        any_ = max(any_, (end, what))


class AdamW:
    """AdamW over a list of parameters, one launch a step (ge_adamw_step).

    ``params`` and ``grads`` are contiguous float32 or bfloat16 GPU tensors that
    stay where they are (gradients are written into the same buffers before each
    step) and share no memory with one another: a tied parameter is listed once, with
    the sum of its gradients. ``masters`` gives float32 copies of some or all parameters (None: none).
    ``state_bits`` is 32 or 8. States are created as zeros unless given: ``m`` and
    ``v`` float32, or float8_e4m3fn and float8_e5m2 with ``m_scale`` and ``v_scale``
    (float32, one for each 256 elements). ``steps`` counts the steps taken.

    For a step replayed from a graph, ``device_params()`` makes the device copy of
    the parameters that ``step(device_params=...)`` reads instead of the host's."""

    def __init__(self, params: Sequence, grads: Sequence, masters: Optional[Sequence] = None, lr: float = 1e-3,
                 beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32, seed: int = 0, m=None, v=None, m_scale=None, v_scale=None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits {state_bits}: 8 or 32 is wanted")
        params, grads = list(params), list(grads)
        masters = [None] * len(params) if masters is None else list(masters)
        if not params:
            raise ValueError("no parameters")
        device = _on_gpu(params[0], "params[0]")
        mt = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        vt = torch.float32 if state_bits == 32 else torch.float8_e5m2

        def states(given, dtype, sizes):
            return [torch.zeros(n, dtype=dtype, device=device) for n in sizes] if given is None else list(given)

        sizes = [p.numel() for p in params]
        blocks = [-(-n // GE_ADAMW_BLOCK) for n in sizes]
        self.m, self.v = states(m, mt, sizes), states(v, vt, sizes)
        self.m_scale = self.v_scale = [None] * len(params)
        if state_bits == 8:
            self.m_scale, self.v_scale = states(m_scale, torch.float32, blocks), states(v_scale, torch.float32, blocks)
        lists = (grads, masters, self.m, self.v, self.m_scale, self.v_scale)
        if any(len(x) != len(params) for x in lists):
            raise ValueError("params, grads, masters and states differ in number")

        spans = []

        def flat(t, what, n, dtype=None, writes=True):
            if t.device != device or not t.is_contiguous() or t.numel() != n:
                raise ValueError(f"{what}: {n} contiguous elements on {device} are wanted")
            if dtype is not None and t.dtype != dtype:
                raise ValueError(f"{what} has dtype {t.dtype}: {dtype} is wanted")
            if n:
                spans.append((t.data_ptr(), t.data_ptr() + n * t.element_size(), what, writes))
            return t.data_ptr()

        table = (AdamwTensor * len(params))()
        for i, p in enumerate(params):
            t, n = table[i], sizes[i]
            t.param, t.param_dtype, t.n = flat(p, f"params[{i}]", n), _dtype(p, f"params[{i}]"), n
            t.grad, t.grad_dtype = flat(grads[i], f"grads[{i}]", n, writes=False), _dtype(grads[i], f"grads[{i}]")
            if masters[i] is not None:
                t.master = flat(masters[i], f"masters[{i}]", n, torch.float32)
                if t.master == t.param:  # a float32 parameter that is its own master
                    spans.pop()
            t.m, t.v = flat(self.m[i], f"m[{i}]", n, mt), flat(self.v[i], f"v[{i}]", n, vt)
            if state_bits == 8:
                t.m_scale = flat(self.m_scale[i], f"m_scale[{i}]", blocks[i], torch.float32)
                t.v_scale = flat(self.v_scale[i], f"v_scale[{i}]", blocks[i], torch.float32)
        _disjoint(spans)
        L = _library()
        size = _I64()
        _check(L.ge_adamw_table_bytes(table, len(params), state_bits, ctypes.byref(size)))
        host = torch.empty((size.value + 7) // 8, dtype=torch.int64)
        _check(L.ge_adamw_table(table, len(params), state_bits, host.data_ptr(), size.value))
        self._table = host.to(device)
        self._args = AdamwArgs(self._table.data_ptr(), size.value, len(params), state_bits)
        self.params, self.grads, self.masters, self.device = params, grads, masters, device
        self._streams = set()
        self.state_bits, self.seed, self.steps = state_bits, seed, 0
        self.lr, self.beta1, self.beta2, self.eps, self.weight_decay = lr, beta1, beta2, eps, weight_decay

    def _params(self, step, lr, grad_scale) -> AdamwParams:
        return AdamwParams(self.lr if lr is None else lr, self.beta1, self.beta2, self.eps, self.weight_decay, grad_scale,
                           step, self.seed)

    def device_params(self, lr: Optional[float] = None, grad_scale: float = 1.0, out=None):
        """The next step's parameters, checked, as a uint8 device tensor (``out`` is
        overwritten if given), and counts the step."""
        if out is not None:
            _want(out, "out", torch.uint8, (ctypes.sizeof(AdamwParams),), self.device)
        params = self._params(self.steps + 1, lr, grad_scale)
        # a step over no tensors: the checks alone
        _check(_library().ge_adamw_step(None, ctypes.byref(AdamwArgs(None, 0, 0, self.state_bits, params))))
        host = torch.frombuffer(bytearray(params), dtype=torch.uint8)
        out = host.to(self.device) if out is None else out.copy_(host)
        self.steps += 1
        return out

    def step(self, lr: Optional[float] = None, grad_scale: float = 1.0, stream=None, device_params=None):
        """One step with the gradients in ``grads``, each times ``grad_scale``. With
        ``device_params`` (see there) the launch reads those and counts nothing."""
        a = self._args
        if device_params is None:
            a.params = self._params(self.steps + 1, lr, grad_scale)
            a.device_params = None
        else:
            _want(device_params, "device_params", torch.uint8, (ctypes.sizeof(AdamwParams),), self.device)
            a.device_params = device_params.data_ptr()
        handle, side = _stream(stream, self.device)
        if torch.cuda.current_device() == self.device.index:
            rc = _library().ge_adamw_step(handle, ctypes.byref(a))
        else:
            with torch.cuda.device(self.device):
                rc = _library().ge_adamw_step(handle, ctypes.byref(a))
        _check(rc)
        if side is not None:
            _used(side, device_params)
            if handle not in self._streams:  # the list's tensors stay what they are: once a stream
                self._streams.add(handle)
                _used(side, self._table, *self.params, *self.grads, *self.masters, *self.m, *self.v, *self.m_scale, *self.v_scale)
        if device_params is None:
            self.steps += 1
