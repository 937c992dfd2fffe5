"""The paged cache's classes of the C++ layer: tests/cpp/test_paged.cpp."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build(tmp_path):
    out, lib = str(tmp_path / "test_paged"), os.path.join(ROOT, "vkllama_b200")
    subprocess.check_call(["/usr/bin/g++", "-std=c++17", "-O2", "-mf16c", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "test_paged.cpp"),
                           "-o", out, "-L", lib, "-lvkllama_b200", "-Wl,-rpath," + lib])
    return out


def test_paged_classes_compile_and_link(tmp_path):
    assert os.path.exists(build(tmp_path))


@pytest.mark.gpu
def test_paged_classes_serve_sequences(tmp_path):
    r = subprocess.run([build(tmp_path)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "PASS" in r.stdout, r.stdout + r.stderr
