"""The attention entry points' host code under AddressSanitizer and
UndefinedBehaviorSanitizer, driven by tests/native/attention_sanitize.cpp: without
a GPU the argument checks and no-device paths, on one small calls of every kernel
choice.  The build and the environment are those of the other entry points' run."""
import os
import shutil
import subprocess

import pytest

from test_host_sanitize import CSRC

EXE = os.path.join(CSRC, "_build_san", "attention_sanitize")


def _run(gpu):
    env = dict(os.environ)
    env["ASAN_OPTIONS"] = "detect_leaks=0:abort_on_error=0" + (":protect_shadow_gap=0" if gpu else "")
    env["UBSAN_OPTIONS"] = "print_stacktrace=1:halt_on_error=1"
    r = subprocess.run([EXE], capture_output=True, text=True, env=env, timeout=300)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-4000:]
    assert f"attention_sanitize: all checks passed ({'device 0' if gpu else 'no device'})" in out, out[-4000:]


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="no hipcc")
def test_attention_host_code_sanitized_without_device():
    r = subprocess.run(["make", "-s", "-j8", "-C", CSRC, "_build_san/attention_sanitize"],
                       capture_output=True, text=True, timeout=1500)
    assert r.returncode == 0, (r.stdout + r.stderr)[-4000:]
    import torch
    if torch.cuda.device_count() > 0:
        pytest.skip("a GPU is visible: the device run is the gpu-marked test")
    _run(gpu=False)


@pytest.mark.gpu
def test_attention_host_code_sanitized_on_device():
    assert os.path.exists(EXE), "sanitized build missing: run `make -C %s sanitize` first" % CSRC
    _run(gpu=True)
