"""Paged-cache operators without a GPU: the module's names, refusals that come before any device
call, the C struct's layout, and the 64-bit reference against the framework's own oracle."""
from __future__ import annotations

import ctypes
import math
import os
import shutil
import subprocess
import sys

import numpy as np
import pytest
import torch

import paged_reference as ref
from conftest import ROOT
from fa_ctypes import LIB_PATH
from oracle import attention_oracle as orc


class PagedParams(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("batch_size", "total_q", "max_seqlen_q", "num_heads_q", "num_heads_k",
                                               "head_dim", "page_size", "num_pages", "max_pages")] + [
        ("softmax_scale", ctypes.c_float), ("softcap", ctypes.c_float), ("is_causal", ctypes.c_int32),
        ("window_left", ctypes.c_int32), ("window_right", ctypes.c_int32), ("dtype", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32), ("prefix_len", ctypes.c_uint32), ("prefix_pages", ctypes.c_uint32),
        ("q_stride", ctypes.c_int64 * 2), ("o_stride", ctypes.c_int64 * 2), ("new_k_stride", ctypes.c_int64 * 2),
        ("new_v_stride", ctypes.c_int64 * 2), ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3),
        ("table_stride", ctypes.c_int64), ("alibi_slopes", ctypes.c_void_p)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB_PATH)
    lib.fa_paged_workspace_size.restype = ctypes.c_size_t
    lib.fa_last_error.restype = ctypes.c_char_p
    for n in ("fa_paged_params_init", "fa_paged_workspace_size"):
        getattr(lib, n).argtypes = [ctypes.POINTER(PagedParams)]
    lib.fa_paged_forward.argtypes = [ctypes.POINTER(PagedParams)] + [ctypes.c_void_p] * 10 + [ctypes.c_size_t, ctypes.c_void_p]
    lib.fa_store_kv.argtypes = ([ctypes.POINTER(PagedParams)] + [ctypes.c_void_p] * 8 +
                                [ctypes.c_uint32, ctypes.c_float] + [ctypes.c_void_p] * 3)
    return lib


def params(lib, **kw):
    p = PagedParams()
    lib.fa_paged_params_init(ctypes.byref(p))
    base = dict(batch_size=2, total_q=2, num_heads_q=4, num_heads_k=2, head_dim=64, page_size=16, num_pages=8, max_pages=4)
    for k, v in {**base, **kw}.items():
        setattr(p, k, v)
    return p


def test_layout_matches_header(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    names = [f[0] for f in PagedParams._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(
        ['#include "fa_b200.h"', "#include <stdio.h>", "#include <stddef.h>", "int main(void) {",
         '  printf("size %zu\\n", sizeof(fa_paged_params));'] +
        [f'  printf("{n} %zu\\n", offsetof(fa_paged_params, {n}));' for n in names] + ["  return 0;", "}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = dict(ln.split() for ln in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert ctypes.sizeof(PagedParams) == int(out.pop("size"))
    assert {n: getattr(PagedParams, n).offset for n in names} == {n: int(v) for n, v in out.items()}


def test_defaults(lib):
    p = PagedParams()
    p.softcap = 3.0
    lib.fa_paged_params_init(ctypes.byref(p))
    assert (p.window_left, p.window_right, p.out_dtype, p.softcap, p.dtype) == (-1, -1, -1, 0.0, 0)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=3), 1, b"dtype"), (dict(out_dtype=5), 1, b"out_dtype"), (dict(head_dim=0), 2, b"head_dim"),
    (dict(head_dim=257), 2, b"head_dim"), (dict(num_heads_k=3), 1, b"multiple"), (dict(num_heads_k=0), 1, b"multiple"),
    (dict(page_size=0), 1, b"page_size"), (dict(num_pages=1 << 31), 1, b"out of range"), (dict(softcap=-1.0), 1, b"softcap"),
    (dict(softcap=math.nan), 1, b"softcap"), (dict(softmax_scale=math.inf), 1, b"finite"),
    (dict(prefix_len=17, prefix_pages=1), 1, b"prefix"), (dict(table_stride=-1), 1, b"strides")])
def test_forward_refuses_parameters(lib, kw, code, text):
    p = params(lib, **kw)
    assert lib.fa_paged_workspace_size(ctypes.byref(p)) == 0
    assert lib.fa_paged_forward(ctypes.byref(p), *([256] * 10), 1 << 40, None) == code
    assert text in lib.fa_last_error()


def test_forward_refuses_pointers_and_scratch(lib):
    p = params(lib)
    need = lib.fa_paged_workspace_size(ctypes.byref(p))
    assert need > 0

    def call(ws=256, size=need, **null):
        names = ["q", "k", "v", "table", "lens", "cu", "prefix", "o", "lse"]
        return lib.fa_paged_forward(ctypes.byref(p), *[None if n in null else 256 for n in names], ws, size, None)

    for n in ("q", "k", "v", "table", "lens", "o"):
        assert call(**{n: True}) == 1 and b"NULL" in lib.fa_last_error()
    assert call(ws=None) == 1 and b"workspace" in lib.fa_last_error()
    assert call(size=need - 1) == 1 and b"workspace" in lib.fa_last_error()
    assert call(ws=16) == 1 and b"aligned" in lib.fa_last_error()
    p.total_q = 0  # nothing to do
    assert call(ws=None, size=0, q=True, o=True) == 0


def test_store_refuses(lib):
    p = params(lib)

    def call(k=256, q=None, qo=None, pos=None, cos=None, sin=None, rows=0, theta=0.0):
        return lib.fa_store_kv(ctypes.byref(p), k, 256, 256, 256, 256, pos, cos, sin, rows, theta, q, qo, None)

    for kw, text in ((dict(k=None), b"NULL"), (dict(q=256), b"q_out"), (dict(cos=256, pos=256), b"go together"),
                     (dict(pos=256), b"rope_theta"), (dict(theta=1e4), b"positions"),
                     (dict(pos=256, theta=math.inf), b"rope_theta")):
        assert call(**kw) == 1 and text in lib.fa_last_error(), kw


def test_plan_refuses(lib):
    lib.fa_plan_pages.argtypes = ([ctypes.c_uint32] * 5 + [ctypes.c_void_p] * 5 + [ctypes.c_int64] +
                                  [ctypes.c_void_p] * 6)

    def call(batch=2, page=16, ptrs=(8,) * 4, table=8, outs=(8,) * 4, end=16):
        return lib.fa_plan_pages(batch, page, 4, 4, 4, *ptrs, table, 4, *outs, end, None)

    assert call(batch=8193) == 2 and b"8192" in lib.fa_last_error()
    assert call(page=0) == 1
    assert call(ptrs=(None, 8, 8, 8)) == 1 and b"NULL" in lib.fa_last_error()
    assert call(end=8) == 1 and b"overlap" in lib.fa_last_error()


def test_module_refuses_other_than_cuda_tensors():
    import flash_attn_metal_cpp_b200 as pkg

    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    for fn, args in ((pkg.paged_forward, (x, x, x, x, x)), (pkg.shared_prefix_forward, (x, x, x, x, 0, x, x)),
                     (pkg.store_kv, (x, x, x, x, x)), (pkg.plan_pages, (x, x, x, x, 16, 4)),
                     (pkg.paged_forward, (np.zeros((2, 4, 64), np.float16),) * 5)):
        with pytest.raises(RuntimeError, match="Paged cache error: .* must be a CUDA torch tensor"):
            fn(*args)


def test_reference_agrees_with_the_oracle():
    g = torch.Generator().manual_seed(1)
    lens, page, hq, hk, d = [37, 20], 8, 4, 2, 16
    kc, vc = (torch.randn((12, page, hk, d), generator=g) for _ in range(2))
    order = torch.randperm(12, generator=g).to(torch.int32)
    table = torch.full((2, 5), -1, dtype=torch.int32)
    table[0, :5], table[1, :3] = order[:5], order[5:8]
    q = torch.randn((57, hq, d), generator=g)
    o, lse, _, _ = ref.attention(q, kc, vc, table, lens, 0.25, True, [0, 37, 57])
    for i, n in enumerate(lens):
        k, v = (ref.rows_of(c, table[i], n).float().numpy()[None] for c in (kc, vc))
        rows = slice(0, 37) if i == 0 else slice(37, 57)
        w, wl = orc.attention_ref(q[rows].numpy()[None], k, v, causal=True, softmax_scale=0.25, return_lse=True)
        np.testing.assert_allclose(o[rows].numpy(), w[0], atol=2e-6)
        np.testing.assert_allclose(lse[:, rows].numpy(), wl[0], atol=2e-6)
    # a prefix is the same keys put in front
    p, _, _, _ = ref.attention(q[37:], kc, vc, table[1:], [4], 0.25, True, [0, 20], prefix_table=table[1], prefix_len=16)
    full, _, _, _ = ref.attention(q[37:], kc, vc, torch.cat([table[1:, :2], table[1:, :3]], 1), [20], 0.25, True, [0, 20])
    assert torch.allclose(p[-4:], full[-4:], atol=1e-12)


def test_plan_reference():
    table, lens, cu, slots, pos, end = ref.plan([3, 4], [2, 1], [[9, -1, -1], [7, -1, -1]], [1, 2, 3], 4, 5)
    assert table == [[9, 1, -1], [7, 2, -1]] and lens == [5, 5] and cu == [0, 2, 3] and end == 2
    assert slots == [39, 4, 8, -1, -1] and pos == [3, 4, 4, 0, 0]


def test_module_loads_the_operators_on_first_use():
    """The module and the package import without torch; the first paged name loads its extension and torch."""
    code = ("import sys, flash_attn_metal_cpp_b200 as p, _flash_attn_metal as m\n"
            "assert 'torch' not in sys.modules\n"
            "assert not hasattr(m, 'no_such_name') and not hasattr(p, 'no_such_name')\n"
            "assert m.store_kv is p.store_kv and m.plan_pages is p.plan_pages and 'torch' in sys.modules\n"
            "from flash_attn_metal_cpp_b200 import paged_forward, shared_prefix_forward\n"
            "assert paged_forward.__module__ == '_flash_attn_paged'\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)
