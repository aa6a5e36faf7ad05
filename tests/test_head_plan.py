"""How the loss's calls are divided, on the host under the sanitizers
(tests/cpp/head_plan_check.cpp)."""
import os
import subprocess

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin", "head_plan_check")


def test_plans_under_sanitizers():
    assert os.path.exists(BIN), "build tests/cpp first (make -C tests/cpp)"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1:verify_asan_link_order=0"))
    assert r.returncode == 0, r.stdout + r.stderr
    assert "head plans passed" in r.stdout
