"""Sizes, histories and launch chains of the paged-cache operators that the per-operator tests do not meet."""
from __future__ import annotations

import math
import subprocess
import sys

import pytest
import torch

from conftest import ROOT
from test_gpu_paged import BF, FP, HF

pytestmark = pytest.mark.gpu


def in_a_new_process(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_plan_sizes_before_any_larger_plan(fa):
    """Around the 48 KB of shared memory that a kernel has without asking for more, in a process that asked for none."""
    in_a_new_process("""
import torch, flash_attn_metal_cpp_b200 as fa
for n in (6127, 6128, 6143, 6144):
    one = torch.ones(n, dtype=torch.int32, device='cuda')
    free = torch.arange(n, dtype=torch.int32, device='cuda')
    table = torch.zeros((n, 1), dtype=torch.int32, device='cuda')
    lens, cu, slots, pos, end = fa.plan_pages(one * 0, one, table, free, 16, n)
    torch.cuda.synchronize()
    fa._flash_attn_metal.check_status()
    assert torch.equal(cu, torch.arange(n + 1, device='cuda')) and torch.equal(slots, free.long() * 16)
    assert torch.equal(table[:, 0], free) and torch.equal(lens, one) and int(end) == n and not pos.any()
""")


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_empty_cache_with_a_wide_table(fa, cuda_device, dtype):
    """A cache without pages: every request is empty, whatever the table's width."""
    kc = torch.zeros((0, 16, 2, 64), dtype=dtype, device=cuda_device)
    q = torch.randn((3, 8, 64), device=cuda_device).to(dtype)
    lens = torch.zeros(3, dtype=torch.int32, device=cuda_device)
    for columns in (10, 20, 100):
        table = torch.zeros((3, columns), dtype=torch.int32, device=cuda_device)
        o, lse = fa.paged_forward(q, kc, kc, table, lens, 0.125, return_lse=True)
        torch.cuda.synchronize()
        fa.check_status()
        assert (o == 0).all() and (lse == -math.inf).all()
