"""Sizes, histories and launch chains of the paged-cache operators that the per-operator tests do not meet."""
from __future__ import annotations

import subprocess
import sys

import pytest

from conftest import ROOT

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
