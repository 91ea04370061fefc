"""State that the launch code keeps between calls, with a CUDA runtime that runs nothing (``tests/host_state``): the
library's own sources are compiled and linked against it, so threads and failures can be lined up at will."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HERE = os.path.join(ROOT, "tests", "host_state")
CSRC = os.path.join(ROOT, "sbnet_b200", "csrc")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _run(cmd):
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, " ".join(cmd) + "\n" + res.stdout[-3000:] + res.stderr[-3000:]
    return res.stdout


def _program(tmp_path, name, source):
    """``tests/host_state/<name>.cc`` with the library's ``<source>.cu`` (its device code stays PTX)."""
    from sbnet_b200 import build
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    try:
        nvcc = build._nvcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    obj, exe = str(tmp_path / (source + ".o")), str(tmp_path / name)
    _run([nvcc, "-ccbin", cxx, "-gencode", "arch=compute_100a,code=compute_100a", "-O0", "-std=c++17", "-Xcompiler", "-fPIC",
          "-c", os.path.join(CSRC, source + ".cu"), "-o", obj])
    _run([cxx, "-std=c++17", "-O1", "-I", CSRC, "-I", HERE, "-isystem", os.path.join(CUDA, "include"),
          os.path.join(HERE, name + ".cc"), os.path.join(HERE, "fake_runtime.cc"), obj, "-o", exe, "-lpthread"])
    return exe


def test_layer_norm_calls_of_two_widths_from_two_threads(tmp_path):
    assert "PASS" in _run([_program(tmp_path, "norm_threads", "layer_norm")])


def test_few_row_kernels_ask_for_clusters_one_by_one(tmp_path):
    assert "PASS" in _run([_program(tmp_path, "few_clusters", "gated_ffn_few")])
