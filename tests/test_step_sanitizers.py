"""The host code of ssq_qk_norm_rope, ssq_append and ssq_decode_prefix under AddressSanitizer and
UndefinedBehaviorSanitizer (CPU only), as tests/test_host_sanitizers.py does for the other entry points."""

import os
import subprocess
import sys

import pytest

from sunshape_amd import build as B
from test_host_sanitizers import HERE, _gpu_visible


@pytest.mark.skipif(B.asan_runtime() is None, reason="no shared AddressSanitizer runtime in this toolchain")
def test_step_host_code_under_asan_and_ubsan():
    if _gpu_visible():
        pytest.skip("runs where no GPU is visible")
    lib = B.build_host_sanitized()
    env = dict(os.environ)
    env.update(LD_PRELOAD=B.asan_runtime(), ASAN_OPTIONS="detect_leaks=0:abort_on_error=1:halt_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1", HIP_VISIBLE_DEVICES="-1",
               ROCR_VISIBLE_DEVICES="-1", CUDA_VISIBLE_DEVICES="-1", PYTHONHASHSEED="0")
    r = subprocess.run([sys.executable, os.path.join(HERE, "host_step_fuzz.py"), lib, "3000"], env=env,
                       capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, (r.stdout[-2000:], r.stderr[-6000:])
    assert "no sanitizer report" in r.stdout
