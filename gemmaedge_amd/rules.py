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


_NOTHING = RuleConfig().params()
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


def _list(t, what, dtype, n, device):
    """The address of a flat list of n elements."""
    if t.dtype != dtype or t.numel() != n or t.get_device() != device.index or not t.is_contiguous():
        H._want(t, what, dtype, (n,), device)
    return t.data_ptr()


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
    i32 = torch.int32
    dtype = H._dtype(logits, "logits")
    H._want(logits, "logits", logits.dtype, logits.shape, device)
    if row_params is None:
        params, rule_rows = (_NOTHING if config is None else config.params()), None
    else:
        params, rule_rows = _NOTHING, _list(row_params, "row_params", torch.uint8, rows * ctypes.sizeof(RuleParams), device)
    if out is not None and out_dtype is not None and out.dtype != out_dtype:
        raise ValueError(f"out has dtype {out.dtype}: {out_dtype} is wanted")
    ids = offsets = places = lens = prompt = None
    capacity = 0
    if history is not None:
        if history_offsets is None:
            raise ValueError("history without history_offsets")
        n = history.numel()
        ids, offsets = _list(history, "history", i32, n, device), _list(history_offsets, "history_offsets", i32, rows + 1, device)
        if n == 0:  # its address may be NULL: no ids at all
            ids = offsets = None
    if ring is not None:
        if history is not None:
            raise ValueError("history and ring are exclusive")
        if ring.dim() != 2 or not ring.is_contiguous() or ring.shape[1] < 1 or ring_len is None:
            raise ValueError("ring: contiguous [rows, capacity] with ring_len is wanted")
        capacity = ring.shape[1]
        H._want(ring, "ring", i32, (rows, capacity), device)
        places, lens = ring.data_ptr(), _list(ring_len, "ring_len", i32, rows, device)
    if prompt_len is not None:
        prompt = _list(prompt_len, "prompt_len", i32, rows, device)
    bias = bias_at = bias_to = None
    if bias_ids is not None:
        if bias_values is None or bias_offsets is None:
            raise ValueError("bias_ids without bias_values or bias_offsets")
        n = bias_ids.numel()
        bias, bias_to = _list(bias_ids, "bias_ids", i32, n, device), _list(bias_values, "bias_values", torch.float32, n, device)
        bias_at = _list(bias_offsets, "bias_offsets", i32, rows + 1, device)
        if n == 0:
            bias = bias_at = bias_to = None
    words = which = None
    masks = mask_stride = 0
    if mask is not None:
        if mask.dim() != 2 or mask.shape[1] < -(-vocab // 32):
            raise ValueError(f"mask has shape {tuple(mask.shape)}: [masks, {-(-vocab // 32)} words] is wanted")
        masks = mask.shape[0]
        H._want(mask, "mask", i32, mask.shape, device)
        if mask_rows is not None:
            which = _list(mask_rows, "mask_rows", i32, rows, device)
        elif masks < rows:
            raise ValueError(f"{masks} masks for {rows} rows without mask_rows")
        if masks:
            words, mask_stride = mask.data_ptr(), H._stride(mask)
        else:
            which = None
    elif mask_rows is not None:
        raise ValueError("mask_rows without mask")
    flags_out = None if flags is None else _list(flags, "flags", i32, rows, device)
    handle, side = H._stream(stream, device)
    out = H._output(out, "out", (out.dtype if out is not None else out_dtype or logits.dtype), (rows, vocab), device, side)
    a = RuleArgs(logits.data_ptr(), dtype, rows, vocab, H._stride(logits), out.data_ptr(), H._dtype(out, "out"), H._stride(out), params,
                 rule_rows, ids, offsets, places, lens, capacity, prompt, bias, bias_to, bias_at, words, mask_stride, masks, which, flags_out)
    if torch._C._cuda_getDevice() == device.index:
        rc = _library().ge_apply_rules(handle, ctypes.byref(a))
    else:
        with torch.cuda.device(device):
            rc = _library().ge_apply_rules(handle, ctypes.byref(a))
    H._check(rc)
    if side is not None:
        H._used(side, logits, out, history, history_offsets, ring, ring_len, prompt_len, bias_ids, bias_values, bias_offsets, mask,
                mask_rows, row_params, flags)
    return out.view(shape) if len(shape) == 1 else out
