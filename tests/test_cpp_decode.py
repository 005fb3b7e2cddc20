"""The C++ host adapter's answering path (Rotary, KvCache, paged_attention of include/te_b200.hpp): it compiles everywhere, and
its test program passes on a GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.join(ROOT, "torch-engine_b200")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _build(out):
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(CUDA, "include"),
                    os.path.join(ROOT, "tests", "cpp", "decode_test.cpp"), "-o", out, "-L" + LIBDIR, "-lte_b200", "-L" + os.path.join(CUDA, "lib64"), "-lcudart",
                    "-Wl,-rpath," + LIBDIR, "-Wl,-rpath," + os.path.join(CUDA, "lib64")], check=True, capture_output=True, text=True)


def test_decode_program_compiles_and_links(tmp_path):
    from torch_engine_b200 import lib
    lib.load()
    _build(str(tmp_path / "decode_test"))


@pytest.mark.gpu
def test_decode_program_passes_on_gpu(tmp_path):
    exe = str(tmp_path / "decode_test")
    _build(exe)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "All decode checks passed." in r.stdout
