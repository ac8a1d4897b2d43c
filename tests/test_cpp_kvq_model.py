"""nn::Model over a quantised KV cache: it compiles and links on any host; on a B200 Model::forward gives what its layers give one after the
other."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "emberlm_b200")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    assert os.path.exists(os.path.join(PKG, "libctdk.so")), "build the library first: python -m emberlm_b200.build"
    exe = str(tmp_path_factory.mktemp("kvq_model") / "test_ctd_kvq_model")
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror",
           "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"),
           os.path.join(ROOT, "tests", "cpp", "test_ctd_kvq_model.cpp"), "-o", exe,
           "-L", PKG, "-lctdk", "-L", os.path.join(CUDA, "lib64"), "-lcudart",
           "-Wl,-rpath," + PKG, "-Wl,-rpath," + os.path.join(CUDA, "lib64")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-4000:]
    return exe


def test_compiles(program):
    assert os.path.exists(program)


@pytest.mark.gpu
def test_cases_pass_on_gpu(program):
    res = subprocess.run([program], capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stdout[-6000:] + res.stderr[-2000:]
    assert " 0 failed" in res.stdout
