"""The sampling entry points' host side after refused and failed calls, on the CPU: the library under AddressSanitizer and
UndefinedBehaviorSanitizer with no device behind it (tests/sampling_host_driver.py)."""
import os
import subprocess
import sys

import pytest

import test_host_asan as host

ROOT = host.ROOT


@pytest.mark.skipif(not os.path.exists('/opt/rocm/bin/hipcc') or host._asan_runtime() is None, reason='needs hipcc and the sanitizer runtime')
def test_host_side_under_asan_and_ubsan():
    r = subprocess.run(['make', '-C', ROOT, '-j6', 'asan-host'], capture_output=True, text=True, timeout=1500)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    env = dict(os.environ, SNK_LIBRARY=os.path.join(ROOT, 'build', 'asan', 'libsnkhip_host_asan.so'), LD_PRELOAD=host._asan_runtime(),
               ASAN_OPTIONS='detect_leaks=0:abort_on_error=0:halt_on_error=1', UBSAN_OPTIONS='print_stacktrace=1:halt_on_error=1')
    r = subprocess.run([sys.executable, os.path.join(ROOT, 'tests', 'sampling_host_driver.py')], capture_output=True, text=True, timeout=900, env=env, cwd=ROOT)
    report = r.stdout[-3000:] + '\n' + r.stderr[-6000:]
    assert r.returncode == 0 and 'SAMPLING-HOST-OK' in r.stdout, report
    assert 'ERROR: AddressSanitizer' not in r.stderr and 'runtime error:' not in r.stderr, report
