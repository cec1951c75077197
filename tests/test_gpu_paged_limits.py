"""Sizes, histories and launch chains of the paged-cache operators that the per-operator tests do not meet."""
from __future__ import annotations

import math
import subprocess
import sys

import pytest
import torch

import paged_reference as ref
from conftest import ROOT
from test_gpu_paged import BF, FP, HF, Batch

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


# ------------------------------------------------------------- angle tables
def store_at(fa, dev, max_position, theta, d=256):
    x = torch.ones((1, 1, d), dtype=BF, device=dev)
    kc = torch.zeros((1, 16, 1, d), dtype=BF, device=dev)
    fa.store_kv(x, x, kc, kc.clone(), torch.zeros(1, dtype=torch.int64, device=dev), rope_theta=theta,
                positions=torch.tensor([max_position - 1], dtype=torch.int32, device=dev), max_position=max_position)
    return kc


def test_growing_positions_do_not_pile_up_tables(fa, cuda_device):
    """A max_position that follows the sequence: what the tables take stays within a few times the last one."""
    theta, d, first, steps = 12321.0, 256, 20000, 60
    store_at(fa, cuda_device, 8, theta)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for i in range(steps):
        kc = store_at(fa, cuda_device, first + i, theta)
        inv = torch.tensor([theta ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64, device=cuda_device)
        ang = (first + i - 1) * inv
        want = torch.cat([ang.cos() - ang.sin(), ang.sin() + ang.cos()])
        # angle tables in float32, two products and a sum, one rounding
        assert ((kc[0, 0, 0].double() - want).abs() <= ref.U[BF] * want.abs() + 8 * 2.0 ** -24).all()
    torch.cuda.synchronize()
    fa.check_status()
    one = (first + steps) * (d // 2) * 4 * 2
    assert before - torch.cuda.mem_get_info()[0] <= 4 * one


def test_tables_survive_a_failed_enlargement(fa, cuda_device):
    store_at(fa, cuda_device, 64, 23432.0)
    with pytest.raises(RuntimeError, match="cudaMalloc"):
        store_at(fa, cuda_device, 1 << 30, 23432.0)
    torch.cuda.synchronize()
    x = torch.ones((1, 1, 256), dtype=BF, device=cuda_device)
    kc = torch.zeros((1, 16, 1, 256), dtype=BF, device=cuda_device)
    vc, slots = kc.clone(), torch.zeros(1, dtype=torch.int64, device=cuda_device)
    pos = torch.full((1,), 63, dtype=torch.int32, device=cuda_device)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fa.store_kv(x, x, kc, vc, slots, positions=pos, rope_theta=23432.0, max_position=64)
    g.replay()
    torch.cuda.synchronize()
    fa.check_status()
    assert torch.equal(kc, store_at(fa, cuda_device, 64, 23432.0))


# ------------------------------------------------------------------ scratch
def test_scratch_of_single_tokens_over_a_wide_table(fa, cuda_device):
    """A call without cu_seqlens_q asks for no scratch of the routes that only several tokens a request take."""
    b = Batch(cuda_device, [40] * 64, hq=32, hk=8, d=128, dtype=BF, width=16384)
    b.run(fa)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    o = b.run(fa)
    torch.cuda.synchronize()
    peak = torch.cuda.max_memory_allocated() - before
    # runs of the few-rows kernel: two partial units of 16 rows for each of 296 blocks, and their records
    most = 296 * (2 * 16 * (128 * 4 + 8) + 64) + o.numel() * 2 + (1 << 20)
    assert peak <= most, (peak, most)


# ------------------------------------------------------------- empty caches
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


# ------------------------------------------- prefix, cut own keys, join, merge
def chain(dev, dtype, qlens, seed):
    """8 requests behind a prefix of 2000 keys (read once), own keys of 1 to 1500 cut in runs."""
    lens = [1500, 1, 64, 777, 1200, 385, 20, 3] if qlens is None else [1500, 4, 64, 777, 1200, 385, 20, 3]
    return Batch(dev, lens, qlens=qlens, hq=32, hk=8, d=128, dtype=dtype, prefix=2000, page=16, seed=seed)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("qlens", [None, [2, 4, 1, 0, 3, 1, 1, 2]])
def test_prefix_beside_cut_own_keys(fa, cuda_device, dtype, qlens):
    b = chain(cuda_device, dtype, qlens, 0)
    n0 = fa.launch_count()
    b.run(fa, qlens is not None)
    assert fa.launch_count() - n0 == 4  # prefix, own keys, join of runs, merge
    b.check(fa, "chain", causal=qlens is not None)
    b.check(fa, "chain, window", causal=qlens is not None, window=(1700, -1))
    b.check(fa, "chain, cap", causal=qlens is not None, cap=20.0, out_dtype=dtype)
    first = b.run(fa, qlens is not None, return_lse=True)
    for _ in range(5):
        again = b.run(fa, qlens is not None, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_prefix_beside_cut_own_keys_captured(fa, cuda_device):
    """Two graphs of the chain replay on two streams at once while lengths and queries change."""
    batches = [chain(cuda_device, dtype, None, seed) for seed, dtype in enumerate((BF, HF))]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in batches]
    for b in batches:
        b.run(fa)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(b.run(fa, out_dtype="float32"))
        graphs.append(g)
    for lens in (batches[0].lens, [1, 1, 1, 1, 1200, 0, 20, 3], [1400, 0, 33, 700, 64, 300, 1, 2]):
        for b in batches:
            b.lens = lens
            b.seq.copy_(torch.tensor(lens, dtype=torch.int32))
            b.q.copy_(torch.randn(b.q.shape, device=cuda_device).to(b.q.dtype))
        torch.cuda.synchronize()
        for _ in range(10):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        fa.check_status()
        for b, o in zip(batches, outs):
            w, _, tol, _ = b.want(out_dtype=FP)
            ref.assert_attention(o, w, tol, f"{lens}")


# ------------------------------------------------------------ sizes, first calls
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("d", [136, 160, 192, 256])
@pytest.mark.parametrize("opts", [{}, dict(cap=50.0), dict(window=(100, -1))])
def test_wide_heads_with_many_rows(fa, cuda_device, dtype, d, opts):
    for prefix in (0, 300):
        b = Batch(cuda_device, [300, 129, 64], qlens=[150, 129, 33], d=d, hq=8, hk=2, dtype=dtype, prefix=prefix)
        b.check(fa, f"d {d}", causal=True, **opts)


@pytest.mark.parametrize("call", ["one", "few", "many", "prefix", "fp32"])
def test_first_call_of_a_process_is_captured(fa, call):
    """`initialize()` is enough before a capture: no kernel has to have run before."""
    in_a_new_process(f"""
import sys
sys.path.insert(0, 'tests')
import torch, paged_reference as ref
from test_gpu_paged import Batch, BF, FP
import flash_attn_metal_cpp_b200 as pkg
pkg.initialize()
fa = pkg._flash_attn_metal
kw = dict(one=dict(lens=[900, 40], d=128), few=dict(lens=[900, 40], qlens=[3, 2], d=64), many=dict(lens=[300, 90], qlens=[100, 90], d=128),
          prefix=dict(lens=[900, 40, 3, 60, 1, 2, 3, 4], d=128, hq=32, hk=8, prefix=2000), fp32=dict(lens=[900, 40], d=64))['{call}']
b = Batch(torch.device('cuda', 0), dtype=FP if '{call}' == 'fp32' else BF, **kw)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    o = b.run(fa, True)
    lens, cu, slots, pos, end = fa.plan_pages(b.seq, b.seq * 0 + 1, b.table.clone(), b.seq, 16, len(b.lens))
    fa.store_kv(torch.ones((len(b.lens), *b.k_cache.shape[2:]), dtype=b.q.dtype, device='cuda'),
                torch.ones((len(b.lens), *b.k_cache.shape[2:]), dtype=b.q.dtype, device='cuda'), b.k_cache.clone(), b.v_cache.clone(), slots * 0 - 1)
g.replay()
torch.cuda.synchronize()
w, _, tol, _ = b.want(True)
ref.assert_attention(o, w, tol, 'first')
""")


# -------------------------------------------------------- offsets above 32 bits
def moved_up(b, elements):
    """The batch with its pages at the end of caches of more than `elements` elements."""
    n, *shape = b.k_cache.shape
    total = elements // math.prod(shape) + n + 1

    def up(c):
        big = torch.empty((total, *shape), dtype=c.dtype, device=c.device)
        big[-n:] = c
        return big

    b.k_cache, b.v_cache = up(b.k_cache), up(b.v_cache)
    b.table[b.table >= 0] += total - n
    b.prefix_table += total - n
    return b


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("kw", [dict(lens=[300, 449, 65]), dict(lens=[300, 449, 65], width=400), dict(lens=[300, 129, 260], qlens=[200, 129, 33]),
                                dict(lens=[50, 9, 0] + [30] * 37, prefix=805)])
def test_pages_behind_32_bits_of_elements(fa, cuda_device, dtype, kw):
    b = moved_up(Batch(cuda_device, hq=8, hk=2, d=128, dtype=dtype, **kw), 1 << 32)
    causal = any(n != 1 for n in b.qlens)
    o = b.run(fa, causal, out_dtype="float32")
    torch.cuda.synchronize()
    fa.check_status()
    w, _, tol, _ = b.want(causal, out_dtype=FP)
    ref.assert_attention(o, w, tol, "far pages")


@pytest.mark.parametrize("d,slots", [(128, 1 << 22), (2, 1 << 31)])
def test_slots_behind_32_bits(fa, cuda_device, d, slots):
    """Rows stored where the element offset passes 2^32, and slot numbers above 2^31."""
    hk = 8 if d == 128 else 1
    pages = slots // 1024 + 1
    kc, vc = (torch.zeros((pages, 1024, hk, d), dtype=HF, device=cuda_device) for _ in range(2))
    k, v = (torch.randn((3, hk, d), device=cuda_device).to(HF) for _ in range(2))
    at = torch.tensor([pages * 1024 - 1, 5, pages * 1024 - 700], device=cuda_device)
    fa.store_kv(k, v, kc, vc, at)
    torch.cuda.synchronize()
    fa.check_status()
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c[at // 1024, at % 1024], x)
        assert int(c[-1].count_nonzero()) == 2 * hk * d and int(c[0].count_nonzero()) == hk * d and not c[1:-1].any()
