"""The projection's C ABI without a GPU: every declared entry point is exported, the
ctypes struct matches the C layout, arguments are refused before a device is
touched, and the host's checks hold under the sanitizers."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from gemmaedge_amd import projection as P
from gemmaedge_amd import sampler as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "gemmaedge_projection.h")
BIN = os.path.join(ROOT, "tests", "cpp", "bin", "projection_check")


def test_every_declared_function_is_exported():
    names = set(re.findall(r"^\s*(?:int|void)\s+(ge_\w+)\s*\(", open(HEADER).read(), re.M))
    assert names == set(P.EXPORTS)
    lib = S.load_library()
    for n in names:
        assert hasattr(lib, n), n


def test_struct_layout_matches_c(tmp_path):
    cls = P.ProjectArgs
    lines = ['printf("%zu\\n", sizeof(ge_project_args));']
    lines += [f'printf("%zu\\n", offsetof(ge_project_args, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gemmaedge_projection.h"\nint main(void){' + "\n".join(lines) +
                   "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]


def test_host_checks_under_sanitizers():
    assert os.path.exists(BIN), "build tests/cpp first (make -C tests/cpp)"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1:verify_asan_link_order=0"))
    assert r.returncode == 0, r.stdout + r.stderr
    assert "projection checks passed" in r.stdout


def test_refusals_without_a_device():
    L = P._library()
    h = ctypes.c_void_p()
    good = [0, 4, 8, 8, 2, 3, 0, 0]
    for at, value, code in ((1, 0, S.GE_ERR_INVALID_ARG), (2, 0, S.GE_ERR_INVALID_ARG), (3, -1, S.GE_ERR_INVALID_ARG),
                            (4, 0, S.GE_ERR_INVALID_ARG), (5, 0, S.GE_ERR_INVALID_ARG), (6, 2, S.GE_ERR_INVALID_ARG),
                            (1, 1 << 23, S.GE_ERR_CAPACITY), (2, 1 << 17, S.GE_ERR_CAPACITY), (3, 1 << 25, S.GE_ERR_CAPACITY),
                            (4, 257, S.GE_ERR_CAPACITY), (5, 65536, S.GE_ERR_CAPACITY)):
        args = list(good)
        args[at] = value
        assert L.ge_projection_create(*args, ctypes.byref(h)) == code, (at, value)
    assert L.ge_projection_create(*good, None) == S.GE_ERR_INVALID_ARG
    assert not h
    L.ge_projection_destroy(None)
    assert L.ge_project(None, None, None) == S.GE_ERR_INVALID_ARG
    assert L.ge_project_backward(None, None, None) == S.GE_ERR_INVALID_ARG
    if not os.path.exists("/dev/kfd"):
        assert L.ge_projection_create(*good, ctypes.byref(h)) == S.GE_ERR_NO_DEVICE
        with pytest.raises(S.SamplerError):
            P.Projection(1, 8, 8)
    with pytest.raises(ValueError, match="dtype"):
        P.Projection(1, 8, 8, dtype=torch.float16)
