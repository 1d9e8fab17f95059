"""The choice between the paged attention's forms, on the host."""
import os
import shutil
import subprocess

import pytest
import torch

import dcpp_b200
from kv_util import Batch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_forms_stay_in_proportion_to_the_gpu(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    exe = str(tmp_path / "kv_form_test")
    subprocess.check_call([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I",
                           os.path.join(ROOT, "diffusers-cpp_b200", "csrc"), "-I", os.path.join(ROOT, "include"),
                           os.path.join(ROOT, "tests", "cpp", "kv_form_test.cu"), "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("batch,prompt,live", [(300, 500, 1.0), (74, 500, 1.0), (1500, 1, 0.05), (148, 1, 0.5)])
def test_mixed_step_of_many_requests(ctx, batch, prompt, live):
    """Short requests, most with one new token or none and one with a prompt: on both
    sides of the choice."""
    g = torch.Generator().manual_seed(batch)
    new = (torch.rand(batch, generator=g) < live).int().tolist()
    new[batch // 2] = prompt
    cached = torch.randint(0, 250, (batch,), generator=g).tolist()
    s = Batch(new, cached, 8, 4, 16, torch.bfloat16, seed=batch)
    cache = dcpp_b200.KVCache(s.k, s.v)
    ws = torch.full((ctx.kv_attention_workspace(cache, s.heads, s.max_new),), 255, dtype=torch.uint8, device="cuda")
    ctx.kv_attention(cache, s.q, s.cu_new, s.seq_lens, s.table, s.max_new, ws, s.out)
    ctx.synchronize()
    s.check()
