"""The stream guard and the launch of the entry points without a context
(kimi-k3-in-rust_amd/csrc/k3g_host.h), compiled for the host on a stand-in for the HIP runtime
(tests/host/hip_stub.h) whose calls fail on request."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "kimi-k3-in-rust_amd", "csrc")
HOST = os.path.join(ROOT, "tests", "host")


@pytest.fixture(scope="module")
def audit(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("host_guard")
    os.mkdir(d / "hip")
    shutil.copy(os.path.join(HOST, "hip_stub.h"), d / "hip" / "hip_runtime.h")
    shutil.copy(os.path.join(CSRC, "k3g_host.h"), d / "k3g_host.h")
    exe = d / "host_guard"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", str(d), os.path.join(HOST, "host_guard.cpp"),
                    "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, check=True)


def test_every_case_holds(audit):
    lines = audit.stdout.split("\n")[:-1]
    assert lines and all(l.startswith("ok ") for l in lines), audit.stdout


def test_every_refusal_has_its_message(audit):
    for cause in ("told:", "current:"):
        assert f"{cause}k3moe: " in audit.stderr, audit.stderr
