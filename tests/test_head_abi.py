"""The answer head's C ABI without a GPU: every declared entry point is
exported, the ctypes structs match the C layout, arguments are refused before a
device is touched, and the host's checks hold under the sanitizers."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from gemmaedge_amd import head as H
from gemmaedge_amd import sampler as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "gemmaedge_head.h")
BIN = os.path.join(ROOT, "tests", "cpp", "bin", "head_check")


def test_every_declared_function_is_exported():
    names = set(re.findall(r"^\s*(?:int|void)\s+(ge_\w+)\s*\(", open(HEADER).read(), re.M))
    assert names == set(H.EXPORTS)
    lib = S.load_library()
    for n in names:
        assert hasattr(lib, n), n


def test_struct_layouts_match_c(tmp_path):
    pairs = [("ge_norm_args", H.NormArgs), ("ge_loss_args", H.LossArgs), ("ge_adamw_tensor", H.AdamwTensor),
             ("ge_adamw_params", H.AdamwParams), ("ge_adamw_args", H.AdamwArgs)]
    lines = []
    for name, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gemmaedge_head.h"\nint main(void){' + "\n".join(lines) +
                   "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def test_host_checks_under_sanitizers():
    assert os.path.exists(BIN), "build tests/cpp first (make -C tests/cpp)"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1:verify_asan_link_order=0"))
    assert r.returncode == 0, r.stdout + r.stderr
    assert "head checks passed" in r.stdout


def test_refusals_without_a_device():
    L = H._library()
    h = ctypes.c_void_p()
    assert L.ge_head_create(0, 0, 8, 8, 0, 0, ctypes.byref(h)) == S.GE_ERR_INVALID_ARG
    assert "max_rows=0" in S.last_error()
    assert L.ge_head_create(0, 1, 8, 8, 5, 0, ctypes.byref(h)) == S.GE_ERR_INVALID_ARG
    assert L.ge_head_create(0, 1, 1 << 20, 8, 0, 0, ctypes.byref(h)) == S.GE_ERR_CAPACITY
    assert L.ge_head_create(0, 1, 8, 8, 0, 0, None) == S.GE_ERR_INVALID_ARG
    assert not h
    L.ge_head_destroy(None)
    for f in (L.ge_head_norm, L.ge_head_norm_backward, L.ge_head_loss, L.ge_head_loss_backward):
        assert f(None, None, None) == S.GE_ERR_INVALID_ARG
    assert L.ge_adamw_step(None, None) == S.GE_ERR_INVALID_ARG
    if not os.path.exists("/dev/kfd"):
        assert L.ge_head_create(0, 1, 8, 8, 0, 0, ctypes.byref(h)) == S.GE_ERR_NO_DEVICE
        with pytest.raises(S.SamplerError):
            H.Head(1, 8, 8)


def _tensor(**kw):
    t = H.AdamwTensor()
    t.param = t.grad = t.m = t.v = t.m_scale = t.v_scale = 4096
    t.n, t.param_dtype, t.grad_dtype = 5000, S.GE_DTYPE_BF16, S.GE_DTYPE_F32
    for k, v in kw.items():
        setattr(t, k, v)
    return (H.AdamwTensor * 1)(t)


@pytest.mark.parametrize("bits", (8, 32))
def test_optimiser_table(bits):
    L, size = H._library(), ctypes.c_int64()
    bad = [dict(param=None), dict(grad=None), dict(m=None), dict(v=None), dict(n=-1), dict(param_dtype=2), dict(grad_dtype=-1),
           dict(param=4097), dict(grad=4098), dict(master=4098)]
    bad += [dict(m_scale=None), dict(v_scale=None), dict(m_scale=4098)] if bits == 8 else [dict(m=4098), dict(v=4097)]
    for kw in bad:
        assert L.ge_adamw_table_bytes(_tensor(**kw), 1, bits, ctypes.byref(size)) == S.GE_ERR_INVALID_ARG, kw
        assert "tensor 0" in S.last_error()
    assert L.ge_adamw_table_bytes(None, 1, bits, ctypes.byref(size)) == S.GE_ERR_INVALID_ARG
    assert L.ge_adamw_table_bytes(_tensor(), 1, 16, ctypes.byref(size)) == S.GE_ERR_INVALID_ARG
    assert L.ge_adamw_table_bytes(_tensor(n=1 << 62), 1, bits, ctypes.byref(size)) == S.GE_ERR_CAPACITY
    assert L.ge_adamw_table_bytes(_tensor(), 1, bits, ctypes.byref(size)) == S.GE_OK
    table = (ctypes.c_int64 * (size.value // 8 + 1))()
    assert L.ge_adamw_table(_tensor(), 1, bits, table, size.value + 8) == S.GE_ERR_INVALID_ARG
    assert L.ge_adamw_table(_tensor(), 1, bits, None, size.value) == S.GE_ERR_INVALID_ARG
    assert L.ge_adamw_table(_tensor(), 1, bits, table, size.value) == S.GE_OK
    assert L.ge_adamw_table_bytes(_tensor(n=0, param=None), 1, bits, ctypes.byref(size)) == S.GE_OK


def test_step_refusals():
    L = H._library()
    a = H.AdamwArgs()
    a.table, a.count, a.state_bits = 4096, 1, 32
    size = ctypes.c_int64()
    assert L.ge_adamw_table_bytes(_tensor(), 1, 32, ctypes.byref(size)) == S.GE_OK
    ok = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, step=1)
    for field, value in (("table_bytes", 8), ("table_bytes", size.value + 1), ("table", None), ("table", 4104), ("state_bits", 4),
                         ("count", -1)):
        a.table, a.table_bytes, a.count, a.state_bits, a.params = 4096, size.value, 1, 32, H.AdamwParams(**ok)
        setattr(a, field, value)
        assert L.ge_adamw_step(None, ctypes.byref(a)) == S.GE_ERR_INVALID_ARG, field
    for field, value in (("beta1", 1.0), ("beta2", -0.5), ("eps", -1.0), ("lr", float("inf")), ("step", 0), ("grad_scale", float("nan"))):
        a.table, a.table_bytes, a.count, a.state_bits, a.params = 4096, size.value, 1, 32, H.AdamwParams(**{**ok, field: value})
        assert L.ge_adamw_step(None, ctypes.byref(a)) == S.GE_ERR_INVALID_ARG, field


def test_cpu_tensors_are_refused():
    p = [torch.zeros(4)]
    with pytest.raises(ValueError, match="GPU"):
        H.AdamW(p, [torch.zeros(4)])
    with pytest.raises(ValueError, match="no parameters"):
        H.AdamW([], [])
    with pytest.raises(ValueError, match="state_bits"):
        H.AdamW(p, p, state_bits=4)
