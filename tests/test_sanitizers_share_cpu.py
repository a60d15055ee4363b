"""The host code of chunk attention and shared pages under AddressSanitizer and
UndefinedBehaviorSanitizer (CPU only): tests/sanitize/kvq_share_check sweeps that
part of the C ABI with stand-in pointers and never launches a kernel."""
import os
import subprocess

from test_sanitizers_cpu import REPORTS, SAN_DIR, _san_env


def test_share_host_code():
    subprocess.run(["make", "-s", "-j8", "-C", SAN_DIR, "-f", "share.mk", "share"], check=True, capture_output=True, timeout=900)
    r = subprocess.run([os.path.join(SAN_DIR, "_build", "kvq_share_check")], env=_san_env(), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert not any(x in r.stdout + r.stderr for x in REPORTS) and ", 0 failures" in r.stdout
