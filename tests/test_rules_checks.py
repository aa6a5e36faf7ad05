"""The rules' argument checks at the largest sizes, without a GPU: under the sanitizers."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_checks_under_sanitizers():
    path = os.path.join(ROOT, "tests", "cpp", "bin", "rules_check")
    assert os.path.exists(path), "build tests/cpp first (make -C tests/cpp)"
    r = subprocess.run([path], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1:verify_asan_link_order=0"))
    assert r.returncode == 0, r.stdout + r.stderr
    assert "rules checks passed" in r.stdout
