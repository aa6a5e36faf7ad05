"""The rules' C ABI and binding without a GPU: the entry point is exported, the
ctypes structs match the C layout, and arguments are refused before a device is
touched."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from gemmaedge_amd import rules as R
from gemmaedge_amd import sampler as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "gemmaedge_rules.h")


def test_every_declared_function_is_exported():
    names = set(re.findall(r"^\s*(?:int|void)\s+(ge_\w+)\s*\(", open(HEADER).read(), re.M))
    assert names == set(R.EXPORTS)
    lib = S.load_library()
    for n in names:
        assert hasattr(lib, n), n


def test_struct_layouts_match_c(tmp_path):
    pairs = [("ge_rule_params", R.RuleParams), ("ge_rule_args", R.RuleArgs)]
    lines = []
    for name, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gemmaedge_rules.h"\nint main(void){' + "\n".join(lines) +
                   "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def _args(**kw):
    a = R.RuleArgs()
    a.logits, a.out, a.dtype, a.out_dtype = 1 << 20, 1 << 30, S.GE_DTYPE_BF16, S.GE_DTYPE_F32
    a.rows, a.vocab, a.row_stride, a.out_stride = 4, 1000, 1000, 1000
    a.params = R.RuleConfig().params()
    for k, v in kw.items():
        setattr(a, k, v)
    return a


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(vocab=0), dict(vocab=-5), dict(dtype=2), dict(out_dtype=-1), dict(logits=None), dict(out=None),
    dict(logits=4097), dict(out=(1 << 30) + 2), dict(row_stride=999), dict(out_stride=999), dict(row_stride=1 << 41),
    dict(out=1 << 20), dict(out=(1 << 20) + 4000), dict(out=(1 << 20) - 4, out_stride=1000),
    dict(out=1 << 20, out_dtype=S.GE_DTYPE_BF16, out_stride=1001),
    dict(params=R.RuleParams(INF, 1, 0, 0)), dict(params=R.RuleParams(0, 0, 0, 0)), dict(params=R.RuleParams(0, -1, 0, 0)),
    dict(params=R.RuleParams(0, NAN, 0, 0)), dict(params=R.RuleParams(0, 1, NAN, 0)), dict(params=R.RuleParams(0, 1, 0, INF)),
    dict(history=4096), dict(ring=4096, ring_capacity=8), dict(ring=4096, ring_len=4096), dict(history=4098, history_offsets=4096),
    dict(ring=4096, ring_len=4096, ring_capacity=8, history=4096, history_offsets=4096),
    dict(bias_ids=4096, bias_values=4096), dict(bias_ids=4096, bias_offsets=4096), dict(prompt_len=4098), dict(flags_out=4097),
    dict(mask=4096, masks=0, mask_rows=4096), dict(mask=4096, masks=4, mask_stride=31), dict(mask=4096, masks=3, mask_stride=32),
    dict(mask_rows=4096), dict(mask=4098, masks=4, mask_stride=32), dict(row_params=4098),
])
def test_refusals(bad):
    L = R._library()
    assert L.ge_apply_rules(None, ctypes.byref(_args(**bad))) == S.GE_ERR_INVALID_ARG, S.last_error()


def test_other_refusals():
    L = R._library()
    assert L.ge_apply_rules(None, None) == S.GE_ERR_INVALID_ARG
    assert L.ge_apply_rules(None, ctypes.byref(_args(vocab=(1 << 30) + 1, row_stride=1 << 31, out_stride=1 << 31))) == S.GE_ERR_CAPACITY
    assert L.ge_apply_rules(None, ctypes.byref(_args(rows=(1 << 24) + 1))) == S.GE_ERR_CAPACITY
    assert L.ge_apply_rules(None, ctypes.byref(_args(rows=(1 << 31) - 1, mask=None))) == S.GE_ERR_CAPACITY
    assert L.ge_apply_rules(None, ctypes.byref(_args(rows=0, logits=None, out=None))) == S.GE_OK


def test_binding_refusals():
    with pytest.raises(ValueError, match="GPU"):
        R.apply(torch.zeros(2, 8))
    for bad in (dict(repetition_penalty=0.0), dict(softcap=NAN), dict(presence_penalty=INF), dict(frequency_penalty=-INF)):
        with pytest.raises(ValueError, match="finite"):
            R.row_params([R.RuleConfig(), R.RuleConfig(**bad)], device="cpu")
    t = R.row_params([R.RuleConfig(30.0, 1.5, 0.25, 0.125)] * 3, device="cpu")
    assert t.dtype == torch.uint8 and t.view(torch.float32).tolist() == [30.0, 1.5, 0.25, 0.125] * 3
    assert R.row_params([], device="cpu").numel() == 0
