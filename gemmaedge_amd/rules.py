"""Python binding of the rules on logits (include/gemmaedge_rules.h): penalties for
repeated tokens, biases and grammar masks, between the logits and ``sampler``.

ctypes over the same library as ``sampler``; torch supplies device memory and
streams, as in ``head`` (streams, and what is recorded on them, are described there).
There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Sequence

import torch

from . import head as H
from . import sampler as S

GE_RULE_EMPTY = 1  # the row's mask allows no token

EXPORTS = ("ge_apply_rules",)

_P, _I32, _I64, _F32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class RuleParams(ctypes.Structure):
    _fields_ = [("softcap", _F32), ("repetition_penalty", _F32), ("presence_penalty", _F32), ("frequency_penalty", _F32)]


class RuleArgs(ctypes.Structure):
    _fields_ = [
        ("logits", _P), ("dtype", _I32), ("rows", _I32), ("vocab", _I32), ("row_stride", _I64), ("out", _P), ("out_dtype", _I32),
        ("out_stride", _I64), ("params", RuleParams), ("row_params", _P), ("history", _P), ("history_offsets", _P), ("ring", _P),
        ("ring_len", _P), ("ring_capacity", _I32), ("prompt_len", _P), ("bias_ids", _P), ("bias_values", _P), ("bias_offsets", _P),
        ("mask", _P), ("mask_stride", _I64), ("masks", _I32), ("mask_rows", _P), ("flags_out", _P),
    ]


@dataclass
class RuleConfig:
    """One request's rules; the defaults change nothing. The softcap belongs here or in the
    sampler's configuration, not in both: it comes before the penalties."""

    softcap: float = 0.0
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0

    def params(self) -> RuleParams:
        return RuleParams(self.softcap, self.repetition_penalty, self.presence_penalty, self.frequency_penalty)

    def check(self) -> None:
        values = (self.softcap, self.repetition_penalty, self.presence_penalty, self.frequency_penalty)
        if not all(math.isfinite(v) for v in values) or not self.repetition_penalty > 0:
            raise ValueError(f"{self}: finite values and a repetition_penalty above 0 are wanted")


_ready = False


def _library() -> ctypes.CDLL:
    global _ready
    L = S.load_library()
    if not _ready:
        L.ge_apply_rules.restype = ctypes.c_int
        L.ge_apply_rules.argtypes = [_P, ctypes.POINTER(RuleArgs)]
        _ready = True
    return L


def row_params(configs: Sequence[RuleConfig], device="cuda"):
    """A device tensor of the rows' rules, checked, for ``apply``'s ``row_params``."""
    configs = list(configs)
    for c in configs:
        c.check()
    host = (RuleParams * len(configs))(*[c.params() for c in configs])
    t = torch.frombuffer(bytearray(host), dtype=torch.uint8) if configs else torch.empty(0, dtype=torch.uint8)
    return t.to(device)


def _list(t, what, dtype, device):
    """A flat list of any length."""
    H._want(t, what, dtype, (t.numel(),), device)


def apply(logits, config: RuleConfig | None = None, out=None, out_dtype=None, history=None, history_offsets=None, ring=None,
          ring_len=None, prompt_len=None, bias_ids=None, bias_values=None, bias_offsets=None, mask=None, mask_rows=None,
          row_params=None, flags=None, stream=None):
    """The rules of ``config`` (or of ``row_params``, see there) on [rows, vocab] (or [vocab])
    float32 or bfloat16 GPU logits. Returns the output: ``out`` if given, which may be
    ``logits`` itself, else a new tensor of ``out_dtype`` (the logits' if None).

    ``history`` int32 with ``history_offsets`` int32 [rows + 1], or the sampler's ``ring`` int32
    [rows, capacity] with ``ring_len`` int32 [rows]: the tokens that are penalised;
    ``prompt_len`` int32 [rows]: how many of them, the first, are the prompt, which the
    presence and frequency penalties do not count.
    ``bias_ids`` int32 and ``bias_values`` float32 with ``bias_offsets`` int32 [rows + 1]: added
    to the tokens' logits; of several entries for a token the last counts.
    ``mask`` int32 [masks, words] with ceil(vocab / 32) words at least: bit t % 32 of word
    t // 32 is set where token t is allowed; ``mask_rows`` int32 [rows]: each row's mask,
    none if it is outside [0, masks); without it row r takes mask r.
    ``flags`` int32 [rows] is set to GE_RULE_EMPTY where the mask allows nothing, else to 0."""
    device = H._on_gpu(logits, "logits")
    shape = logits.shape
    if logits.dim() == 1:
        logits = logits.unsqueeze(0)
        if out is not None and out.dim() == 1:
            out = out.unsqueeze(0)
    if logits.dim() != 2:
        raise ValueError(f"logits have shape {tuple(shape)}: [rows, vocab] is wanted")
    rows, vocab = logits.shape
    if vocab == 0:
        raise ValueError("empty logits")
    a = RuleArgs()
    a.dtype = H._dtype(logits, "logits")
    H._want(logits, "logits", logits.dtype, logits.shape, device)
    if row_params is None:
        config = RuleConfig() if config is None else config
        config.check()
        a.params = config.params()
    else:
        H._want(row_params, "row_params", torch.uint8, (rows * ctypes.sizeof(RuleParams),), device)
    if out is not None and out_dtype is not None and out.dtype != out_dtype:
        raise ValueError(f"out has dtype {out.dtype}: {out_dtype} is wanted")
    if history is not None:
        if history_offsets is None:
            raise ValueError("history without history_offsets")
        _list(history, "history", torch.int32, device)
        H._want(history_offsets, "history_offsets", torch.int32, (rows + 1,), device)
        a.history, a.history_offsets = history.data_ptr(), history_offsets.data_ptr()
        if history.numel() == 0:  # its address may be NULL: no ids at all
            a.history = None
    if ring is not None:
        if history is not None:
            raise ValueError("history and ring are exclusive")
        if ring.dim() != 2 or not ring.is_contiguous() or ring.shape[1] < 1 or ring_len is None:
            raise ValueError("ring: contiguous [rows, capacity] with ring_len is wanted")
        H._want(ring, "ring", torch.int32, (rows, ring.shape[1]), device)
        H._want(ring_len, "ring_len", torch.int32, (rows,), device)
        a.ring, a.ring_len, a.ring_capacity = ring.data_ptr(), ring_len.data_ptr(), ring.shape[1]
    if prompt_len is not None:
        H._want(prompt_len, "prompt_len", torch.int32, (rows,), device)
    if bias_ids is not None:
        if bias_values is None or bias_offsets is None:
            raise ValueError("bias_ids without bias_values or bias_offsets")
        _list(bias_ids, "bias_ids", torch.int32, device)
        H._want(bias_values, "bias_values", torch.float32, (bias_ids.numel(),), device)
        H._want(bias_offsets, "bias_offsets", torch.int32, (rows + 1,), device)
        if bias_ids.numel():
            a.bias_ids, a.bias_values, a.bias_offsets = bias_ids.data_ptr(), bias_values.data_ptr(), bias_offsets.data_ptr()
    if mask is not None:
        if mask.dim() != 2 or mask.shape[1] < -(-vocab // 32):
            raise ValueError(f"mask has shape {tuple(mask.shape)}: [masks, {-(-vocab // 32)} words] is wanted")
        H._want(mask, "mask", torch.int32, mask.shape, device)
        if mask_rows is not None:
            H._want(mask_rows, "mask_rows", torch.int32, (rows,), device)
        elif mask.shape[0] < rows:
            raise ValueError(f"{mask.shape[0]} masks for {rows} rows without mask_rows")
        if mask.shape[0]:
            a.mask, a.mask_stride, a.masks, a.mask_rows = mask.data_ptr(), H._stride(mask), mask.shape[0], S._ptr(mask_rows)
    elif mask_rows is not None:
        raise ValueError("mask_rows without mask")
    if flags is not None:
        H._want(flags, "flags", torch.int32, (rows,), device)
    handle, side = H._stream(stream, device)
    out = H._output(out, "out", (out.dtype if out is not None else out_dtype or logits.dtype), (rows, vocab), device, side)
    a.out_dtype = H._dtype(out, "out")
    a.logits, a.rows, a.vocab, a.row_stride = logits.data_ptr(), rows, vocab, H._stride(logits)
    a.out, a.out_stride = out.data_ptr(), H._stride(out)
    a.row_params, a.prompt_len, a.flags_out = S._ptr(row_params), S._ptr(prompt_len), S._ptr(flags)
    if torch.cuda.current_device() == device.index:
        rc = _library().ge_apply_rules(handle, ctypes.byref(a))
    else:
        with torch.cuda.device(device):
            rc = _library().ge_apply_rules(handle, ctypes.byref(a))
    H._check(rc)
    H._used(side, logits, out, history, history_offsets, ring, ring_len, prompt_len, bias_ids, bias_values, bias_offsets, mask,
            mask_rows, row_params, flags)
    return out.view(shape) if len(shape) == 1 else out
