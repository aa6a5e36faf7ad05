"""The large tiles of the matrix products write their products as instructions on the
accumulation registers, of whose latency the compiler knows nothing: in their loops it
must neither move accumulators nor spill. This reads the library's own device
code, without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

from gemmaedge_amd import sampler as S

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
LARGE = re.compile(r"gemm_kernelILi256E")


def kernels(path):
    """(name, [(address, text)]) of the large tiles' kernels."""
    out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], capture_output=True, text=True, check=True).stdout
    name, body = None, []
    for line in out.splitlines():
        m = re.match(r"^[0-9a-f]+ <(.*)>:$", line)
        if m:
            if name:
                yield name, body
            name, body = (m[1] if LARGE.search(m[1]) and not m[1].endswith(".kd") else None), []
        elif name and "//" in line:
            text, _, rest = line.partition("//")
            body.append((int(rest.split(":")[0], 16), text.strip()))
    if name:
        yield name, body


def loops(body):
    """Bodies of the backward branches, innermost first."""
    start = body[0][0]
    at = {a: i for i, (a, _) in enumerate(body)}
    found = []
    for i, (a, text) in enumerate(body):
        if not text.startswith("s_cbranch") and not text.startswith("s_branch"):
            continue
        m = re.match(r"s_c?branch\S*\s+(\d+)", text)
        if not m:
            continue
        off = int(m[1])
        to = a + 4 + 4 * (off - 65536 if off >= 32768 else off)
        if start <= to < a and to in at:
            found.append((i - at[to], at[to], i))
    return [body[lo:hi + 1] for _, lo, hi in sorted(found)]


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs ROCm's llvm-objdump")
def test_large_tiles_keep_their_accumulators(tmp_path):
    lib = shutil.copy(S.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(lib)], cwd=tmp_path, capture_output=True, check=True)
    seen = 0
    for f in sorted(os.listdir(tmp_path)):
        if "gfx950" not in f:
            continue
        for name, body in kernels(str(tmp_path / f)):
            # the innermost loop with the steps' products, 64 or 128 a half pair
            main = [b for b in loops(body) if sum("v_mfma" in t for _, t in b) >= 128]
            assert main, name
            bad = [t for _, t in main[0] if "accvgpr" in t or t.startswith("scratch_")]
            assert not bad, (name, bad[:4])
            seen += 1
    assert seen >= 10, seen
