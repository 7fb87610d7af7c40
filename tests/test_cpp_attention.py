"""tests/cpp/attention_consumer.cpp: a C++ program on ltx25::Ops' attention members, built with the
host compiler and run in a fresh process. Without a GPU it stops at init."""
import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "vpipe-ltx-2.5_amd")


def build(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    exe = str(tmp_path / "attention_consumer")
    r = subprocess.run(
        [cxx, "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
         "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(PKG, "csrc"),
         os.path.join(ROOT, "tests", "cpp", "attention_consumer.cpp"), "-o", exe, "-L" + PKG,
         "-lltx25_qlinear", "-L/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath," + PKG,
         "-Wl,-rpath,/opt/rocm/lib"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return exe


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device path")
def test_attention_consumer_stops_at_init_without_a_device(tmp_path):
    r = subprocess.run([build(tmp_path)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 3 and r.stdout.startswith("NODEV:"), r.stdout + r.stderr


@pytest.mark.gpu
def test_attention_consumer_on_the_gpu(tmp_path):
    exe = build(tmp_path)
    print("[gpu] C++ consumer of ltx25::Ops' attention members", flush=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.rstrip().endswith("OK"), r.stdout + r.stderr
