"""A NaN that a query row sees reaches the row's output and LSE on every path of the paged attention, and no other row."""
from __future__ import annotations

import math

import pytest
import torch

import paged_reference as ref
from test_gpu_paged import BF, FP, HF, Batch

pytestmark = pytest.mark.gpu

# What decides the path: lengths, query tokens (None = one each), columns of the table, prefix, head_dim. The first
# request holds the NaN.
PATHS = {
    "uncut": dict(lens=[60, 33, 20], d=128),
    "clusters": dict(lens=[300, 449, 65], d=64),
    "runs": dict(lens=[3000, 40, 700], d=128, width=400),
    "few tokens": dict(lens=[60, 33, 20], qlens=[4, 1, 3], d=64),
    "few tokens in runs": dict(lens=[3000, 40, 700], qlens=[4, 1, 3], d=64, width=400),
    "many tokens": dict(lens=[300, 129, 260], qlens=[200, 129, 33], d=128),
    "many tokens in parts": dict(lens=[300, 129, 260], qlens=[70, 129, 33], d=64, width=4000),
    "prefix beside one token": dict(lens=[50, 9, 0] + [30] * 37, d=128, prefix=805),
    "prefix beside runs": dict(lens=[900, 9, 0] + [30] * 37, d=128, prefix=805),
    "prefix of many tokens": dict(lens=[90, 70, 64], qlens=[90, 1, 64], d=64, prefix=300),
}


def poisoned(dev, path, dtype, where):
    """A batch with a NaN in a query row, in a key of the first request, or in a key of the prefix."""
    b = Batch(dev, hq=8, hk=2, dtype=dtype, **PATHS[path])
    if where == "query":
        b.q[b.starts[1] - 1, 5, 3] = math.nan
    else:
        page, key = (b.prefix_table, b.prefix // 2) if where == "prefix key" else (b.table[0], b.lens[0] // 2)
        b.k_cache[int(page[key // b.page]), key % b.page, 1, 2] = math.nan
    return b


def cases(fn):
    for name, values in (("path,where", [(p, w) for p in PATHS for w in ("query", "key", "prefix key")
                                         if w != "prefix key" or "prefix" in PATHS[p]]),
                         ("dtype", [BF, HF, FP])):
        fn = pytest.mark.parametrize(name, values)(fn)
    return fn


def check_output(fa, b, **kw):
    """O of every row: NaN where the definition's is, else within its tolerance."""
    causal = any(n != 1 for n in b.qlens)
    o, lse = b.run(fa, causal, out_dtype="float32", return_lse=True, softcap=kw.get("cap", 0.0), alibi_slopes=kw.get("slopes"))
    torch.cuda.synchronize()
    fa.check_status()
    w, w_lse, tol, lse_tol = b.want(causal, out_dtype=FP, **kw)
    assert w.isnan().any() and not w.isnan().all()
    assert torch.equal(o.isnan(), w.isnan())
    ref.assert_attention(o, w, tol, "rows without NaN")
    return lse, w_lse, lse_tol


@cases
def test_nan_reaches_the_output(fa, cuda_device, path, where, dtype):
    check_output(fa, poisoned(cuda_device, path, dtype, where))


@cases
@pytest.mark.parametrize("cap", [30.0, 400.0])
def test_nan_under_a_cap(fa, cuda_device, path, where, dtype, cap):
    check_output(fa, poisoned(cuda_device, path, dtype, where), cap=cap)


@cases
def test_nan_reaches_the_lse(fa, cuda_device, path, where, dtype):
    # fp16 with slopes, bf16 with a cap: other scores in front of the same end of a row
    kw = {BF: dict(cap=30.0), FP: {}, HF: dict(slopes=torch.tensor([2.0 ** -(i + 1) for i in range(8)], device=cuda_device))}[dtype]
    got, want, tol = check_output(fa, poisoned(cuda_device, path, dtype, where), **kw)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf())
    fin = want.isfinite()
    assert ((got.double() - want).abs() <= tol)[fin].all()
