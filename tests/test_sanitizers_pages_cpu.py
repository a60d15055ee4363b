"""The host code around a paged cache under AddressSanitizer and
UndefinedBehaviorSanitizer (CPU only): tests/sanitize/kvq_pages_check sweeps
that part of the C ABI with stand-in pointers and never launches a kernel."""
import os
import subprocess

import pytest

from test_sanitizers_cpu import REPORTS, SAN_DIR, _san_env


@pytest.fixture(scope="module")
def pages_check():
    subprocess.run(["make", "-s", "-j8", "-C", SAN_DIR, "-f", "pages.mk", "pages"], check=True, capture_output=True, timeout=900)
    return os.path.join(SAN_DIR, "_build", "kvq_pages_check")


@pytest.mark.parametrize("switch", [{}, {"KVQ_FORCE_KERNEL": "valu"}, {"KVQ_FORCE_KERNEL": "generic"}])
def test_pages_host_code(pages_check, switch):
    r = subprocess.run([pages_check], env=_san_env(**switch), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert not any(x in r.stdout + r.stderr for x in REPORTS) and ", 0 failures" in r.stdout
