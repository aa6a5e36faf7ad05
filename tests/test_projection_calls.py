"""The projection's plans at the sizes where they can go wrong, without a GPU: under the sanitizers."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_calls_under_sanitizers():
    path = os.path.join(ROOT, "tests", "cpp", "bin", "projection_call_check")
    assert os.path.exists(path), "build tests/cpp first (make -C tests/cpp)"
    r = subprocess.run([path], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=1:verify_asan_link_order=0"))
    assert r.returncode == 0, r.stdout + r.stderr
    assert "projection call checks passed" in r.stdout
