"""The paged key / value cache without a GPU: the arithmetic that shares out the
attention's work, refusals that need no device, and the C++ surface (whose step runs
on the GPU)."""
import os
import shutil
import subprocess

import pytest
import torch

import dcpp_b200

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.dirname(dcpp_b200.LIB_PATH)


def test_work_is_shared_out_exactly(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    exe = str(tmp_path / "kv_sched_test")
    subprocess.check_call([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I",
                           os.path.join(ROOT, "diffusers-cpp_b200", "csrc"), "-I", os.path.join(ROOT, "include"),
                           os.path.join(ROOT, "tests", "cpp", "kv_sched_test.cu"), "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_cache_refuses_tensors_it_cannot_describe():
    k = torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16)
    for a, b in ((k, k), (k, None), (k, k.half()), (k[0], k[0]), (k, k[:1])):
        with pytest.raises(dcpp_b200.DcppError) as e:
            dcpp_b200.KVCache(a, b)
        assert e.value.status == 1


def test_geometry_alone_needs_no_device():
    c = dcpp_b200.KVCache(n_blocks=7, block_size=32)
    assert (c.n_blocks, c.c.block_size, c.device) == (7, 32, None)


@pytest.fixture(scope="module")
def kv_test(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    dcpp_b200.lib()  # the library must be built
    exe = str(tmp_path_factory.mktemp("cpp") / "kv_test")
    subprocess.check_call([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"),
                           os.path.join(ROOT, "tests", "cpp", "kv_test.cpp"), "-L", LIBDIR, "-ldcpp_b200",
                           f"-Wl,-rpath,{LIBDIR}", "-o", exe])
    return exe


def test_entry_points_refuse_a_null_context(kv_test):
    r = subprocess.run([kv_test, "cpu"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr


@pytest.mark.gpu
def test_step_through_the_cpp_surface(kv_test):
    r = subprocess.run([kv_test, "gpu"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
