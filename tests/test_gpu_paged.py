"""Paged-cache operators on the GPU against their 64-bit definition (tests/paged_reference.py):
plan_pages, store_kv, paged_forward, shared_prefix_forward, and a run of them together."""
from __future__ import annotations

import math

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


class Batch:
    """A cache with the requests' pages scattered over it; every slot that no request owns is NaN."""

    def __init__(self, dev, lens, qlens=None, hq=8, hk=2, d=64, page=16, dtype=BF, prefix=0, seed=0, layout="NPHD",
                 spare_rows=0, width=None, scale_q=1.0):
        g = torch.Generator(device=dev).manual_seed(1000 + seed)
        self.dev, self.lens, self.page, self.prefix = dev, list(lens), page, prefix
        self.qlens = [1] * len(lens) if qlens is None else list(qlens)
        counts = [-(-n // page) for n in lens]
        n_pages = sum(counts) + -(-prefix // page) + 3
        order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)

        def cache():
            base = torch.randn((n_pages, page, hk, d), generator=g, device=dev).to(dtype)
            if layout == "NHPD":
                base = base.transpose(1, 2).contiguous().transpose(1, 2)
            elif layout == "paired":  # K and V pages side by side in one tensor
                both = torch.zeros((n_pages, 2, page, hk, d), dtype=dtype, device=dev)
                both[:, 1] = base
                base = both[:, 1]
            elif layout == "odd":  # rows at element strides that no vector load can take
                wide = torch.zeros((n_pages, page, hk, d + 1), dtype=dtype, device=dev)
                wide[..., :d] = base
                base = wide[..., :d]
            return base

        self.k_cache, self.v_cache = cache(), cache()
        own = torch.zeros((n_pages, page), dtype=torch.bool, device=dev)
        p_pages = -(-prefix // page)
        self.prefix_table = order[:p_pages].contiguous()
        width = max([1, *counts]) if width is None else width
        self.table = torch.full((len(lens), width), -5, dtype=torch.int32, device=dev)
        at = p_pages
        for i, c in enumerate(counts):
            self.table[i, :c] = order[at:at + c]
            at += c
            for j in range(c):
                own[self.table[i, j].long(), :min(page, lens[i] - j * page)] = True
        for j in range(p_pages):
            own[self.prefix_table[j].long(), :min(page, prefix - j * page)] = True
        self.k_cache.masked_fill_(~own[..., None, None], math.nan)
        self.v_cache.masked_fill_(~own[..., None, None], math.nan)
        self.starts = [0]
        for n in self.qlens:
            self.starts.append(self.starts[-1] + n)
        self.q = (torch.randn((self.starts[-1] + spare_rows, hq, d), generator=g, device=dev) * scale_q).to(dtype)
        self.cu = torch.tensor(self.starts, dtype=torch.int32, device=dev)
        self.seq = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        self.scale = 1.0 / math.sqrt(d)

    def run(self, fa, causal=False, use_cu=None, **kw):
        use_cu = any(n != 1 for n in self.qlens) if use_cu is None else use_cu
        if use_cu:
            kw.update(cu_seqlens_q=self.cu, max_seqlen_q=max([1, *self.qlens]))
        kw.setdefault("softmax_scale", self.scale)
        if self.prefix:
            return fa.shared_prefix_forward(self.q, self.k_cache, self.v_cache, self.prefix_table, self.prefix, self.table,
                                            self.seq, is_causal=causal, **kw)
        return fa.paged_forward(self.q, self.k_cache, self.v_cache, self.table, self.seq, is_causal=causal, **kw)

    def want(self, causal=False, **kw):
        kw.setdefault("scale", self.scale)
        return ref.attention(self.q, self.k_cache, self.v_cache, self.table, self.lens, causal=causal, starts=self.starts,
                             prefix_table=self.prefix_table, prefix_len=self.prefix, **kw)

    def check(self, fa, what, causal=False, cap=0.0, window=None, slopes=None, scale=None, out_dtype=FP, use_cu=None):
        extra = {} if scale is None else {"softmax_scale": scale}
        o, lse = self.run(fa, causal, use_cu, softcap=cap, window_size=window, out_dtype=str(out_dtype), return_lse=True,
                          alibi_slopes=slopes, **extra)
        torch.cuda.synchronize()
        fa.check_status()
        assert o.dtype == out_dtype and lse.shape == (self.q.shape[1], self.q.shape[0])
        extra = {} if scale is None else {"scale": scale}
        w, w_lse, tol, lse_tol = self.want(causal, cap=cap, window=window, slopes=slopes, out_dtype=out_dtype, **extra)
        ref.assert_attention(o, w, tol, what)
        n = self.starts[-1]
        a, b = lse[:, :n].double(), w_lse[:, :n]
        # (a request with no rows leaves no column, every other column is set)
        assert torch.equal(a.isinf(), b.isinf()), f"{what}: rows without keys"
        fin = ~b.isinf()
        assert ((a - b).abs() <= lse_tol[:, :n])[fin].all(), f"{what}: lse off by {float((a - b).abs()[fin].max()):.2e}"


EDGE_LENS = [1, 15, 16, 17, 63, 64, 65, 130, 300, 0, 1025]


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("heads", [(8, 8), (8, 2), (8, 1), (32, 2), (40, 1), (6, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_single_tokens(fa, cuda_device, dtype, heads, d):
    b = Batch(cuda_device, EDGE_LENS, hq=heads[0], hk=heads[1], d=d, dtype=dtype)
    b.check(fa, f"{dtype} {heads} d{d}")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 48, 64, 128, 256])
def test_page_sizes(fa, cuda_device, dtype, page):
    b = Batch(cuda_device, [1, 47, 300, 511, 129], page=page, d=128, dtype=dtype)
    b.check(fa, f"page {page}")
    c = Batch(cuda_device, [70, 300, 200], qlens=[70, 33, 150], page=page, d=128, dtype=dtype)
    c.check(fa, f"page {page} chunks", causal=True)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("d", [8, 32, 40, 59, 80, 96, 111, 160, 256])
def test_head_dims(fa, cuda_device, dtype, d):
    b = Batch(cuda_device, [5, 64, 333], qlens=[2, 1, 7], d=d, hq=4, hk=2, dtype=dtype)
    b.check(fa, f"d {d}", causal=True)


@pytest.mark.parametrize("layout", ["NHPD", "paired", "odd"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("qlens", [[1, 1, 1], [90, 1, 200]])
def test_cache_strides(fa, cuda_device, layout, dtype, qlens):
    b = Batch(cuda_device, [100, 17, 400], qlens=qlens, d=64, dtype=dtype, layout=layout)
    b.check(fa, layout, causal=True)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("qlens", [[1, 2, 3, 4, 5, 6], [8, 0, 16, 1, 0, 9], [40, 1, 130, 0, 257, 33],
                                   [600, 1, 0, 0, 300, 256]])
@pytest.mark.parametrize("heads", [(8, 8), (8, 2), (16, 1)])
def test_several_tokens(fa, cuda_device, dtype, qlens, heads):
    lens = [max(n, x) for n, x in zip([700, 5, 300, 64, 1000, 257], qlens)]
    b = Batch(cuda_device, lens, qlens=qlens, hq=heads[0], hk=heads[1], d=128, dtype=dtype)
    b.check(fa, "causal", causal=True)
    b.check(fa, "full")


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("qlens", [None, [3, 1, 2, 4], [70, 1, 200, 64]])
@pytest.mark.parametrize("opts", [dict(cap=30.0), dict(cap=0.5), dict(window=(100, -1)), dict(window=(0, 0)),
                                  dict(window=(-1, 5)), dict(window=(63, 2), cap=20.0), "alibi", dict(scale=-0.2),
                                  dict(scale=0.0), "all"])
def test_scores_and_masks(fa, cuda_device, dtype, qlens, opts):
    b = Batch(cuda_device, [90, 1, 777, 64], qlens=qlens, hq=8, hk=2, d=64, dtype=dtype, scale_q=3.0)
    slopes = torch.tensor([2.0 ** -(i + 1) for i in range(8)], device=cuda_device)
    if opts == "alibi":
        opts = dict(slopes=slopes)
    elif opts == "all":
        opts = dict(slopes=slopes, cap=15.0, window=(200, -1))
    b.check(fa, str(opts), causal=True, **opts)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("qlens", [[5, 3, 1], [70, 40, 90]])
def test_more_tokens_than_keys(fa, cuda_device, dtype, qlens):
    """Rows whose position lies before the first key see nothing under a causal mask."""
    for prefix in (0, 20):
        b = Batch(cuda_device, [2, 0, 30], qlens=qlens, d=64, dtype=dtype, prefix=prefix)
        b.check(fa, "short", causal=True)
        b.check(fa, "short", causal=True, window=(3, -1))
        b.check(fa, "short full")


def test_large_scores(fa, cuda_device):
    """Scores far apart (one key takes all the weight) and a cap that flattens them."""
    for dtype in (BF, HF, FP):
        b = Batch(cuda_device, [300, 65], hq=8, hk=2, d=128, dtype=dtype, scale_q=20.0)
        b.check(fa, "large")
        b.check(fa, "large capped", cap=5.0)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("far", [9.0, 13.0, 17.0])
@pytest.mark.parametrize("qlens", [[1], [64]])
def test_many_small_weights(fa, cuda_device, dtype, far, qlens):
    """One key far above the others, whose value is 0: the output is what thousands of small weights add up to."""
    for prefix in (0, 4000):
        b = Batch(cuda_device, [20000], qlens=qlens, hq=8, hk=1, d=64, dtype=dtype, prefix=prefix, page=64)
        b.k_cache.zero_()
        b.v_cache.fill_(1.0)
        b.q.zero_()
        b.q[..., 0] = 8.0
        page, slot = int(b.table[0, 3]), 11
        b.k_cache[page, slot, :, 0] = far
        b.v_cache[page, slot] = 0.0
        b.check(fa, f"far {far}")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hk", [1, 8])
def test_one_long_request(fa, cuda_device, dtype, hk):
    b = Batch(cuda_device, [20011], hq=8, hk=hk, d=128, page=64, dtype=dtype)
    b.check(fa, "long")
    b.check(fa, "long windowed", window=(3000, -1))


def test_many_short_requests(fa, cuda_device):
    lens = [(i * 37) % 90 for i in range(700)]
    for dtype in (BF, FP):
        b = Batch(cuda_device, lens, hq=4, hk=2, d=64, dtype=dtype, width=64)
        b.check(fa, "short")


# Tables narrow enough that a cluster of 2, 4 or 8 blocks shares a unit's tiles (many requests, heads and
# columns leave fewer blocks a unit): requests of no key, of one, of fewer tiles than blocks.
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("heads", [(16, 16), (8, 2), (15, 1), (3, 3)])
@pytest.mark.parametrize("d", [40, 64, 128, 160, 256])
@pytest.mark.parametrize("copies", [1, 3])
def test_narrow_tables(fa, cuda_device, dtype, heads, d, copies):
    lens = [1, 0, 33, 64, 65, 130, 300, 449] * copies
    b = Batch(cuda_device, lens, hq=heads[0], hk=heads[1], d=d, dtype=dtype)
    b.check(fa, f"{dtype} {heads} d{d}")
    slopes = torch.linspace(0.02, 0.5, heads[0], dtype=torch.float32, device=cuda_device)
    b.check(fa, "window, slopes", window=(70, 0), slopes=slopes)
    b.check(fa, "cap", cap=15.0, out_dtype=dtype)


@pytest.mark.parametrize("dtype", [HF, FP])
@pytest.mark.parametrize("lens", [[512], [225], [0], [1, 2, 640, 3]])
def test_narrow_tables_few_requests(fa, cuda_device, dtype, lens):
    for width in (None, 60):
        b = Batch(cuda_device, lens, hq=8, hk=8, d=64, dtype=dtype, spare_rows=2, width=width)
        b.check(fa, f"{lens} width {width}")
        c = Batch(cuda_device, lens, hq=8, hk=2, d=128, dtype=dtype, prefix=130, width=width)
        c.check(fa, f"{lens} width {width}, short prefix")
        first = c.run(fa, return_lse=True)
        again = c.run(fa, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype", [BF, FP])
def test_narrow_tables_captured(fa, cuda_device, dtype):
    """Clusters in two captured graphs that replay side by side while the lengths change."""
    batches = [Batch(cuda_device, [300, 449, 65], hq=8, hk=4, d=d, dtype=dtype, seed=d) for d in (64, 128)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in batches]
    for b in batches:
        b.run(fa)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(b.run(fa, out_dtype="float32"))
        graphs.append(g)
    for lens in ([300, 449, 65], [1, 0, 64], [33, 448, 0]):
        for b in batches:
            b.lens = lens
            b.seq.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        fa.check_status()
        for b, o in zip(batches, outs):
            w, _, tol, _ = b.want(out_dtype=FP)
            ref.assert_attention(o, w, tol, f"{lens}")


def test_window_leaves_old_pages_unread(fa, cuda_device):
    """Pages wholly before the window may have been given away: their entries and slots hold anything."""
    for qlens in ([1, 1], [5, 2], [100, 40]):
        for dtype in (BF, HF, FP):
            b = Batch(cuda_device, [500, 333], qlens=qlens, hq=4, hk=2, d=64, dtype=dtype)
            for i, (n, m) in enumerate(zip(b.lens, qlens)):
                first = max(0, n - m - 77)
                b.table[i, :first // b.page] = -1
                page, slot = int(b.table[i, first // b.page]), first % b.page
                b.k_cache[page, :slot] = math.nan
                b.v_cache[page, :slot] = math.nan
            o = b.run(fa, True, window_size=(77, -1), out_dtype="float32")
            torch.cuda.synchronize()
            fa.check_status()
            for i, (n, m) in enumerate(zip(b.lens, qlens)):
                b.table[i, :max(0, n - m - 77) // b.page] = b.table[i, max(0, n - m - 77) // b.page]
            w, _, tol, _ = b.want(True, window=(77, -1), out_dtype=FP)
            ref.assert_attention(o, w, tol, f"{dtype} {qlens}")


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("out_dtype", [BF, HF, FP])
def test_output_types(fa, cuda_device, dtype, out_dtype):
    for qlens in (None, [64, 100, 70]):
        b = Batch(cuda_device, [64, 200, 77], qlens=qlens, dtype=dtype, d=128)
        b.check(fa, "type", causal=True, out_dtype=out_dtype)


@pytest.mark.parametrize("qlens", [[1, 1, 1], [3, 2, 1], [60, 0, 130]])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_rows_behind_the_last_sequence_are_left(fa, cuda_device, qlens, dtype):
    for prefix in (0, 300):
        b = Batch(cuda_device, [100, 50, 200], qlens=qlens, d=64, dtype=dtype, spare_rows=70, prefix=prefix)
        out = torch.full(b.q.shape, 7.0, dtype=dtype, device=cuda_device)
        b.run(fa, True, use_cu=True, out=out)
        torch.cuda.synchronize()
        fa.check_status()
        assert (out[b.starts[-1]:] == 7.0).all()
        w, _, tol, _ = b.want(True)
        ref.assert_attention(out, w, tol, "rows")


def test_strided_q_and_out(fa, cuda_device):
    for dtype in (BF, FP):
        for qlens in ([1, 1], [50, 80]):
            b = Batch(cuda_device, [100, 300], qlens=qlens, hq=8, hk=2, d=64, dtype=dtype)
            n = b.q.shape[0]
            fused = torch.randn((n, 12, 64), device=cuda_device).to(dtype)
            fused[:, 2:10] = b.q
            b.q = fused[:, 2:10]
            wide = torch.full((n, 8, 96), 3.0, dtype=dtype, device=cuda_device)
            b.run(fa, True, out=wide[..., :64])
            torch.cuda.synchronize()
            w, _, tol, _ = b.want(True)
            ref.assert_attention(wide[..., :64], w, tol, "strided")
            assert (wide[..., 64:] == 3.0).all()


def test_bad_pages_and_lengths_are_reported(fa, cuda_device):
    """Indexes outside the cache are skipped by the kernels and reported; the other requests stay right."""
    for dtype in (BF, FP):
        for qlens in ([1, 1, 1], [70, 60, 40]):
            for what in ("page", "big page", "length", "negative"):
                b = Batch(cuda_device, [100, 90, 300], qlens=qlens, d=64, dtype=dtype)
                w, _, tol, _ = b.want(True)
                if what == "page":
                    b.table[1, 2] = -1
                elif what == "big page":
                    b.table[1, 0] = 1 << 30
                elif what == "length":
                    b.table[1, 6:] = 0
                    b.seq[1] = 100000
                else:
                    b.seq[1] = -4
                o = b.run(fa, True, use_cu=True)
                torch.cuda.synchronize()
                with pytest.raises(RuntimeError, match="outside its cache"):
                    fa.check_status()
                fa.check_status()  # cleared
                for i in (0, 2):
                    s = slice(b.starts[i], b.starts[i + 1])
                    ref.assert_attention(o[s], w[s], tol[s], what)


@pytest.mark.parametrize("d", [8, 16, 40, 56, 64, 72, 88, 104, 120, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_head_dims_of_prompt_chunks(fa, cuda_device, d, dtype):
    b = Batch(cuda_device, [300, 129, 40], qlens=[200, 129, 33], d=d, hq=4, hk=2, dtype=dtype)
    b.check(fa, f"d {d}", causal=True)
    b.check(fa, f"d {d} capped", causal=True, cap=20.0)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("cap", [1e-30, 1e-3, 300.0, 1e4, 1e30])
@pytest.mark.parametrize("qlens", [None, [100, 60]])
def test_caps_of_any_size(fa, cuda_device, dtype, cap, qlens):
    """A cap far above the scores changes nothing, one far below makes the weights equal."""
    b = Batch(cuda_device, [150, 70], qlens=qlens, d=64, dtype=dtype)
    o = b.run(fa, softcap=cap, out_dtype="float32")
    torch.cuda.synchronize()
    exact_cap = 0.0 if cap > 1e6 else cap
    w, _, tol, _ = b.want(out_dtype=FP, cap=exact_cap)
    if 256 < cap <= 1e6:  # 2^-20 cap is the reference's allowance; beyond 256 the kernels are relatively exact
        w0, _, tol0, _ = b.want(out_dtype=FP)
        ref.assert_attention(o, w, tol0 + (w - w0).abs() * 2.0 ** -10, "cap")
    else:
        ref.assert_attention(o, w, tol, "cap")


@pytest.mark.parametrize("hint", [1, 3, 1000])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_max_seqlen_is_only_a_hint(fa, cuda_device, hint, dtype):
    b = Batch(cuda_device, [300, 90, 200], qlens=[150, 1, 70], d=64, dtype=dtype)
    o = fa.paged_forward(b.q, b.k_cache, b.v_cache, b.table, b.seq, b.scale, True, cu_seqlens_q=b.cu, max_seqlen_q=hint)
    p = fa.paged_forward(b.q, b.k_cache, b.v_cache, b.table, b.seq, b.scale, True, cu_seqlens_q=b.cu)
    torch.cuda.synchronize()
    fa.check_status()
    w, _, tol, _ = b.want(True)
    ref.assert_attention(o, w, tol, "hint")
    ref.assert_attention(p, w, tol, "no hint")


def test_offsets_out_of_order_are_reported(fa, cuda_device):
    """Offsets that fall, overlap or leave q give unspecified rows, no access outside q and a report."""
    for dtype in (BF, FP):
        for n in (1, 60):
            b = Batch(cuda_device, [100, 90, 300], qlens=[n, n, n], d=64, dtype=dtype, width=64)
            for cu in ([0, 3 * n, 0, 3 * n], [0, n, 5 * n, 3 * n], [-7, n, 2 * n, 1 << 30], [2 * n, n, 0, 3 * n]):
                fa.paged_forward(b.q, b.k_cache, b.v_cache, b.table, b.seq, b.scale, True, max_seqlen_q=n,
                                 cu_seqlens_q=torch.tensor(cu, dtype=torch.int32, device=cuda_device))
                torch.cuda.synchronize()
                with pytest.raises(RuntimeError, match="outside its cache"):
                    fa.check_status()
            b.check(fa, "after", causal=True, use_cu=True)


def test_broadcast_heads_and_unaligned_rows(fa, cuda_device):
    for qlens in ([1, 1], [70, 50]):
        b = Batch(cuda_device, [300, 90], qlens=qlens, hq=4, hk=1, d=64, dtype=BF)
        b.k_cache, b.v_cache = (c.expand(-1, -1, 2, -1) for c in (b.k_cache, b.v_cache))  # one row for two KV heads
        b.check(fa, "broadcast heads", causal=True)
        b = Batch(cuda_device, [300, 90], qlens=qlens, hq=4, hk=2, d=64, dtype=BF)
        flat = torch.zeros(b.q.numel() + 1, dtype=BF, device=cuda_device)
        flat[1:] = b.q.flatten()
        b.q = flat[1:].view(b.q.shape)
        b.check(fa, "unaligned q", causal=True)
        out = torch.zeros(b.q.numel() + 1, dtype=BF, device=cuda_device)[1:].view(b.q.shape)
        b.q = b.q.clone()
        b.run(fa, True, out=out)
        w, _, tol, _ = b.want(True)
        ref.assert_attention(out, w, tol, "unaligned out")


def test_wide_tables(fa, cuda_device):
    """A table with room for a million tokens a request, as a graph for any length has."""
    for dtype in (BF, FP):
        for qlens in (None, [40, 100, 64]):
            b = Batch(cuda_device, [50, 300, 64], qlens=qlens, d=64, dtype=dtype, width=65536)
            b.check(fa, "wide", causal=True)


# -------------------------------------------------------------- shared prefix
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("prefix", [1, 16, 100, 128, 1037])
@pytest.mark.parametrize("heads", [(8, 2), (8, 8), (16, 1)])
def test_shared_prefix(fa, cuda_device, dtype, prefix, heads):
    b = Batch(cuda_device, [1, 16, 0, 40, 129, 300, 7], hq=heads[0], hk=heads[1], d=128, dtype=dtype, prefix=prefix)
    b.check(fa, f"prefix {prefix}")


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("qlens", [[4] * 9, [1, 0, 3, 2, 7, 1, 1, 5, 2], [100, 0, 1, 30, 64, 2, 2, 2, 200]])
@pytest.mark.parametrize("opts", [{}, dict(cap=25.0), dict(window=(400, -1)), dict(window=(20, -1)), "alibi"])
def test_shared_prefix_several_tokens(fa, cuda_device, dtype, qlens, opts):
    lens = [max(n, m) for n, m in zip([4, 9, 100, 30, 64, 2, 17, 5, 250], qlens)]
    b = Batch(cuda_device, lens, qlens=qlens, hq=8, hk=2, d=64, dtype=dtype, prefix=519, page=32)
    if opts == "alibi":
        opts = dict(slopes=torch.tensor([2.0 ** -(i + 1) for i in range(8)], device=cuda_device))
    b.check(fa, str(opts), causal=True, **opts)


@pytest.mark.parametrize("d", [40, 59, 96, 256])
@pytest.mark.parametrize("page", [3, 8, 256])
def test_shared_prefix_odd_sizes(fa, cuda_device, d, page):
    for dtype in (BF, FP):
        b = Batch(cuda_device, [1, 30, 77], hq=12, hk=3, d=d, dtype=dtype, prefix=401, page=page)
        b.check(fa, "odd")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("opts", [{}, dict(cap=25.0), dict(cap=400.0), dict(window=(2500, -1)), dict(window=(50, -1)),
                                  dict(window=(-1, 3)), "alibi", dict(scale=-0.1)])
@pytest.mark.parametrize("qlens", [None, [1, 3, 2, 0, 4, 1]])
def test_prefix_shared_beside_single_tokens(fa, cuda_device, dtype, d, opts, qlens):
    """Prefixes long enough to be computed once for the batch while its own keys take the few-rows kernel."""
    n = 40 if qlens is None else 6
    prefix = 32e6 / (n * 2 * d * 4) // 1 + 3
    lens = [max((i * 29) % 90, 4) for i in range(n)]
    b = Batch(cuda_device, lens, qlens=qlens, hq=6, hk=2, d=d, dtype=dtype, prefix=int(prefix), page=48)
    if opts == "alibi":
        opts = dict(slopes=torch.tensor([2.0 ** -(i + 3) for i in range(6)], device=cuda_device))
    b.check(fa, str(opts), causal=qlens is not None, **opts)


def test_shared_prefix_large_batch(fa, cuda_device):
    b = Batch(cuda_device, [(i * 13) % 60 + 1 for i in range(150)], hq=16, hk=2, d=128, dtype=BF, prefix=3000, page=64)
    b.check(fa, "batch")


def test_empty_prefix_is_paged_forward(fa, cuda_device):
    b = Batch(cuda_device, [33, 70], d=64)
    o = fa.shared_prefix_forward(b.q, b.k_cache, b.v_cache, b.prefix_table, 0, b.table, b.seq, b.scale)
    assert torch.equal(o, b.run(fa))


# ------------------------------------------------------------------ planning
def _plan_case(dev, cached, new, page, rows, width, n_free, begin, seed=0):
    g = torch.Generator().manual_seed(seed)
    held = [min(-(-c // page), width) for c in cached]
    ids = torch.randperm(sum(held) + n_free + 5, generator=g).tolist()
    table = [[-9] * width for _ in cached]
    at = 0
    for i, h in enumerate(held):
        table[i][:h] = ids[at:at + h]
        at += h
    free = ids[at:at + n_free]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    return table, free, t(cached), t(new), t(table).reshape(len(cached), width), t(free), (
        None if begin is None else t([begin]))


@pytest.mark.parametrize("cached,new,page,rows", [
    ([0], [1], 16, 1), ([15, 16, 17, 0, 31], [1, 1, 1, 1, 1], 16, 5), ([0, 0, 5], [0, 0, 0], 4, 3),
    ([3, 0, 100, 7], [50, 1, 0, 9], 8, 70), (list(range(300)), [1] * 300, 16, 300),
    ([i % 40 for i in range(1500)], [(i * 7) % 5 for i in range(1500)], 3, 3100), ([5000, 12], [2500, 4000], 64, 6500),
    ([1, 2], [3, 4], 1, 7), ([i % 90 for i in range(8192)], [1] * 8192, 32, 8200)])
@pytest.mark.parametrize("begin", [None, 3])
def test_plan_pages(fa, cuda_device, cached, new, page, rows, begin):
    width = max(-(-(c + n) // page) for c, n in zip(cached, new)) + 2
    n_free = sum(-(-(c + n) // page) for c, n in zip(cached, new)) + 4
    table, free, c, n, tb, f, b = _plan_case(cuda_device, cached, new, page, rows, width, n_free, begin)
    got = fa.plan_pages(c, n, tb, f, page, rows, free_begin=b)
    torch.cuda.synchronize()
    fa.check_status()
    want = ref.plan(cached, new, table, free, page, rows, begin or 0)
    for g, w in zip((tb, *got), want):
        assert g.cpu().tolist() == (w if isinstance(w, list) else [w])


def test_plan_pages_runs_out(fa, cuda_device):
    """A free list, a table row or a token buffer that is too short: -1, reported, the rest as usual."""
    for cached, new, rows, width, n_free, begin in (([5, 9, 30], [20, 20, 3], 43, 8, 4, 0), ([5, 9], [20, 60], 80, 4, 30, 0),
                                                    ([0, 0], [9, 9], 10, 4, 20, 0), ([5], [20], 20, 8, 4, 4)):
        table, free, c, n, tb, f, b = _plan_case(cuda_device, cached, new, 8, rows, width, n_free, begin)
        got = fa.plan_pages(c, n, tb, f, 8, rows, free_begin=b)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="free list"):
            fa.check_status()
        want = ref.plan(cached, new, table, free, 8, rows, begin)
        for g, w in zip((tb, *got), want):
            assert g.cpu().tolist() == (w if isinstance(w, list) else [w])


def test_plan_pages_empty_batch(fa, cuda_device):
    z = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    f = torch.arange(4, dtype=torch.int32, device=cuda_device)
    lens, cu, slots, pos, end = fa.plan_pages(z, z, torch.zeros((0, 3), dtype=torch.int32, device=cuda_device), f, 16, 5)
    torch.cuda.synchronize()
    assert cu.tolist() == [0] and slots.tolist() == [-1] * 5 and pos.tolist() == [0] * 5 and end.tolist() == [0]
    assert lens.numel() == 0


# -------------------------------------------------------------- cache append
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("d,hk,hq", [(64, 2, 8), (128, 1, 5), (128, 8, 32), (16, 3, 0), (40, 2, 4), (59, 2, 3), (256, 2, 2)])
@pytest.mark.parametrize("rope", ["theta", "tables", None])
def test_store_kv(fa, cuda_device, dtype, d, hk, hq, rope):
    if rope == "theta" and d % 2:
        pytest.skip("rope_theta needs an even head_dim")
    g = torch.Generator(device=cuda_device).manual_seed(d + hk)
    t, page, n_pages = 77, 16, 9

    def rnd(*s):
        return torch.randn(s, generator=g, device=cuda_device).to(dtype)

    kc, vc = rnd(n_pages, page, hk, d), rnd(n_pages, hk, page, d).transpose(1, 2)
    k, fused = rnd(t, hk, d), rnd(t, hq + hk + 1, d)
    v, q = fused[:, :hk], fused[:, hk:hk + hq] if hq else None
    slots = torch.randperm(n_pages * page, generator=g, device=cuda_device)[:t]
    slots[[3, 40]] = -1
    pos = torch.randint(0, 5000, (t,), generator=g, device=cuda_device, dtype=torch.int32)
    kw = {}
    theta = 10000.0
    if rope == "theta":
        kw = dict(positions=pos, rope_theta=theta, max_position=5000)
    elif rope == "tables":
        inv = torch.tensor([theta ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device=cuda_device)
        ang = torch.arange(5000, device=cuda_device).double()[:, None] * inv
        kw = dict(positions=pos, cos=ang.cos().float().contiguous(), sin=ang.sin().float().contiguous())
    want_k, want_v = kc.double(), vc.double()
    turned = ref.rotate(k, pos, theta) if rope else k.double()
    keep = slots >= 0
    want_k[slots[keep] // page, slots[keep] % page] = turned[keep]
    want_v[slots[keep] // page, slots[keep] % page] = v[keep].double()
    out = fa.store_kv(k, v, kc, vc, slots, q=q, **kw)
    torch.cuda.synchronize()
    fa.check_status()
    assert torch.equal(vc.double(), want_v)
    # angles in float32 (half a step of 1), two products and a sum: 4 steps of 2^-24 on |a| + |b|; one rounding
    big = max(float(k.abs().max()), float(q.abs().max()) if hq else 0.0)
    u = ref.U[dtype]

    def close(got, want):
        return ((got.double() - want).abs() <= u * want.abs() + 8 * 2.0 ** -24 * big).all()

    assert close(kc, want_k)
    if hq:
        assert close(out, ref.rotate(q, pos, theta) if rope else q.double())
    else:
        assert out is None
    if rope is None:
        assert torch.equal(kc.double(), want_k)


def test_store_kv_bad_slots_and_positions(fa, cuda_device):
    for d in (64, 40):
        kc = torch.zeros((2, 16, 1, d), dtype=BF, device=cuda_device)
        vc = kc.clone()
        x = torch.ones((3, 1, d), dtype=BF, device=cuda_device)
        fa.store_kv(x, x, kc, vc, torch.tensor([32, 1 << 40, 4], device=cuda_device))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside its cache"):
            fa.check_status()
        assert float(kc.sum()) == d and (kc[0, 4] == 1).all() and (vc[0, 4] == 1).all()
        fa.store_kv(x, x, kc, vc, torch.tensor([0, 1, 2], device=cuda_device), rope_theta=1e4, max_position=8,
                    positions=torch.tensor([7, 8, -1], dtype=torch.int32, device=cuda_device))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside its cache"):
            fa.check_status()
        assert (kc[0, 1] == 1).all() and (kc[0, 2] == 1).all()  # kept as they were given


def test_rotation_equals_forward(fa, cuda_device):
    """A cache filled with rotated keys gives what forward gives with RoPE of the whole sequence."""
    s, hq, hk, d = 200, 8, 2, 128
    g = torch.Generator(device=cuda_device).manual_seed(3)
    q, k, v = (torch.randn((1, s, h, d), generator=g, device=cuda_device).to(HF) for h in (hq, hk, hk))
    want = fa.forward(q, k, v, 1 / math.sqrt(d), True, rope_theta=1e4, out_dtype="float32")
    kc, vc = (torch.zeros((20, 16, hk, d), dtype=HF, device=cuda_device) for _ in range(2))
    ids = torch.randperm(20, generator=g, device=cuda_device).to(torch.int32)
    table = torch.full((1, 14), -1, dtype=torch.int32, device=cuda_device)
    zero = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    lens, cu, slots, pos, _ = fa.plan_pages(zero, zero + s, table, ids, 16, s)
    qr = fa.store_kv(k[0], v[0], kc, vc, slots, q=q[0], positions=pos, rope_theta=1e4, max_position=s)
    got = fa.paged_forward(qr, kc, vc, table, lens, 1 / math.sqrt(d), True, cu_seqlens_q=cu, out_dtype="float32")
    torch.cuda.synchronize()
    fa.check_status()
    # both round the rotated q and k to fp16 and P to fp16: the framework's bar for this path
    assert float((got - want[0]).abs().max()) <= 2e-3


# ------------------------------------------------------------- steps together
def _serve(fa, dev, dtype, steps, prefix, seed=0, stream=None):
    """Prompts, then single-token steps; returns the outputs of every step and the tokens' K, V, q."""
    g = torch.Generator(device=dev).manual_seed(seed)
    hq, hk, d, page, n = 8, 2, 64, 16, 5
    kc, vc = (torch.full((200, page, hk, d), math.nan, dtype=dtype, device=dev) for _ in range(2))
    order = torch.randperm(200, generator=g, device=dev).to(torch.int32)
    p_pages = -(-prefix // page)
    ptab, free = order[:p_pages].contiguous(), order[p_pages:].contiguous()

    def rnd(t, h):
        return torch.randn((t, h, d), generator=g, device=dev).to(dtype)

    if prefix:
        kp, vp = rnd(prefix, hk), rnd(prefix, hk)
        at = torch.arange(prefix, device=dev)
        fa.store_kv(kp, vp, kc, vc, ptab.long()[at // page] * page + at % page)
    table = torch.full((n, 12), -1, dtype=torch.int32, device=dev)
    cached = torch.zeros(n, dtype=torch.int32, device=dev)
    begin = torch.zeros(1, dtype=torch.int32, device=dev)
    log = []
    for step in range(steps):
        new = torch.tensor([7, 30, 1, 16, 45] if step == 0 else [1] * n, dtype=torch.int32, device=dev)
        rows = 99 if step == 0 else n
        lens, cu, slots, pos, begin = fa.plan_pages(cached, new, table, free, page, rows, free_begin=begin)
        q, k, v = rnd(rows, hq), rnd(rows, hk), rnd(rows, hk)
        fa.store_kv(k, v, kc, vc, slots)
        kw = dict(softmax_scale=d ** -0.5, is_causal=True, cu_seqlens_q=cu if step == 0 else None, max_seqlen_q=45)
        if prefix:
            o = fa.shared_prefix_forward(q, kc, vc, ptab, prefix, table, lens, **kw)
        else:
            o = fa.paged_forward(q, kc, vc, table, lens, **kw)
        log.append((q, o, cu.clone(), lens.clone(), table.clone(), kc.clone(), vc.clone()))
        cached = lens
    return log, ptab


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("prefix", [0, 90])
def test_serving_steps(fa, cuda_device, dtype, prefix):
    log, ptab = _serve(fa, cuda_device, dtype, 4, prefix)
    torch.cuda.synchronize()
    fa.check_status()
    for q, o, cu, lens, table, kc, vc in log:
        starts, n = cu.tolist(), cu.tolist()[-1]
        w, _, tol, _ = ref.attention(q[:n], kc, vc, table, lens.tolist(), 64 ** -0.5, True, starts, prefix_table=ptab,
                                     prefix_len=prefix)
        ref.assert_attention(o[:n], w, tol, "step")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("prefix", [0, 700])
def test_captured_step_follows_the_lengths(fa, cuda_device, dtype, prefix):
    """One captured decoding step, replayed while lengths, tables and tokens change; two graphs at once."""
    b = Batch(cuda_device, [40, 300, 1, 99], hq=8, hk=2, d=128, dtype=dtype, prefix=prefix, width=64, page=16)
    c = Batch(cuda_device, [500, 3, 64, 10], hq=8, hk=2, d=128, dtype=dtype, prefix=prefix, width=64, page=16, seed=5)
    graphs, outs = [], []
    for x in (b, c):
        x.run(fa)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(x.run(fa))
        graphs.append(gr)
    for _ in range(2):
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        fa.check_status()
        for x, o in zip((b, c), outs):
            w, _, tol, _ = x.want()
            ref.assert_attention(o, w, tol, "replay")
        # other lengths on the same pages, another q
        b.lens = [33, 7, 1, 80]
        b.seq.copy_(torch.tensor(b.lens, dtype=torch.int32))
        b.q.copy_(torch.randn_like(b.q.float()).to(dtype))
    # replays on two streams at once, each graph with scratch of its own
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    s1.wait_stream(torch.cuda.current_stream())
    s2.wait_stream(torch.cuda.current_stream())
    keep = []
    for _ in range(20):
        for gr, s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for x, o in zip((b, c), outs):
        w, _, tol, _ = x.want()
        ref.assert_attention(o, w, tol, "two streams")
    del keep


def test_captured_serving_step(fa, cuda_device):
    """Planning, append and attention of a decoding step in one graph; each replay is the next step."""
    n, page, hq, hk, d, dev = 4, 16, 8, 2, 64, cuda_device
    kc, vc = (torch.full((40, page, hk, d), math.nan, dtype=HF, device=dev) for _ in range(2))
    table = torch.full((n, 8), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(40, device=dev).to(torch.int32)
    cached, new = torch.zeros(n, dtype=torch.int32, device=dev), torch.ones(n, dtype=torch.int32, device=dev)
    begin = torch.zeros(1, dtype=torch.int32, device=dev)
    q, k, v = (torch.empty((n, h, d), dtype=HF, device=dev) for h in (hq, hk, hk))

    def step():
        lens, _, slots, pos, end = fa.plan_pages(cached, new, table, free, page, n, free_begin=begin)
        qr = fa.store_kv(k, v, kc, vc, slots, q=q, positions=pos, rope_theta=1e4, max_position=256)
        o = fa.paged_forward(qr, kc, vc, table, lens, d ** -0.5)
        cached.copy_(lens)
        begin.copy_(end)
        return qr, o

    def reset():
        cached.copy_(torch.tensor([0, 15, 16, 31], dtype=torch.int32))
        begin.zero_()
        table.fill_(-1)
        for t in (kc, vc):
            t.fill_(math.nan)
        # what the requests hold already
        zero = torch.zeros(n, dtype=torch.int32, device=dev)
        _, _, slots, _, end = fa.plan_pages(zero, cached, table, free, page, 62, free_begin=begin)
        x = torch.randn((62, hk, d), device=dev).half()
        fa.store_kv(x, x, kc, vc, slots)
        begin.copy_(end)

    for t in (q, k, v):
        t.normal_()
    reset()
    step()
    torch.cuda.synchronize()
    reset()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        qr, o = step()
    reset()
    for i in range(20):
        for t in (q, k, v):
            t.normal_()
        g.replay()
        torch.cuda.synchronize()
        fa.check_status()
        lens = cached.tolist()
        assert lens == [x + i + 1 for x in (0, 15, 16, 31)]
        w, _, tol, _ = ref.attention(qr, kc, vc, table, lens, d ** -0.5)
        ref.assert_attention(o, w, tol, f"step {i}")


def test_an_error_does_not_reach_the_next_call(fa, cuda_device):
    x = torch.ones((1, 1, 256), dtype=FP, device=cuda_device)
    kc = torch.zeros((1, 16, 1, 256), dtype=FP, device=cuda_device)
    slots, pos = (torch.zeros(1, dtype=t, device=cuda_device) for t in (torch.int64, torch.int32))
    with pytest.raises(RuntimeError, match="cudaMalloc"):  # tables of 2^30 positions
        fa.store_kv(x, x, kc, kc.clone(), slots, positions=pos, rope_theta=77.0, max_position=1 << 30)
    q = torch.randn((1, 32, 2, 160), device=cuda_device)  # CUDA-core forward
    fa.forward(q, q, q, 0.1)
    fa.store_kv(x, x, kc, kc.clone(), slots)
    torch.cuda.synchronize()


def test_two_streams_eager(fa, cuda_device):
    bs = [Batch(cuda_device, [700, 90, 4000], hq=8, hk=2, d=128, dtype=BF, prefix=p, seed=i, page=64)
          for i, p in enumerate((0, 900))]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (b, s) in enumerate(zip(bs, streams)):
            with torch.cuda.stream(s):
                got[i].append(b.run(fa))
    torch.cuda.synchronize()
    for b, outs in zip(bs, got):
        w, _, tol, _ = b.want()
        for o in outs:
            ref.assert_attention(o, w, tol, "stream")


def test_results_repeat_exactly(fa, cuda_device):
    b = Batch(cuda_device, [9000, 100, 1, 2500], hq=8, hk=2, d=128, dtype=BF, page=64)
    c = Batch(cuda_device, [90, 100, 1, 250], hq=8, hk=2, d=128, dtype=BF, page=64, prefix=4000)
    for x in (b, c):
        first = x.run(fa)
        for _ in range(5):
            assert torch.equal(x.run(fa), first)


def test_capture_with_unbuilt_angles_is_refused(fa, cuda_device):
    kc = torch.zeros((2, 16, 1, 64), dtype=BF, device=cuda_device)
    vc, x = kc.clone(), torch.ones((1, 1, 64), dtype=BF, device=cuda_device)
    slots = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    pos = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="before the stream is captured"):
            fa.store_kv(x, x, kc, vc, slots, positions=pos, rope_theta=12345.0, max_position=64)
    fa.store_kv(x, x, kc, vc, slots, positions=pos, rope_theta=12345.0, max_position=64)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        fa.store_kv(x, x, kc, vc, slots, positions=pos, rope_theta=12345.0, max_position=64)


def test_refusals_on_cuda_tensors(fa, cuda_device):
    b = Batch(cuda_device, [20, 30], hq=4, hk=2, d=64)
    ok = (b.q, b.k_cache, b.v_cache, b.table, b.seq, b.scale)

    def bad(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            fa.paged_forward(*args, **kw)

    def swap(i, x):
        return ok[:i] + (x,) + ok[i + 1:]

    bad("dimensions", *swap(0, b.q[0]))
    bad("one dtype", *swap(0, b.q.float()))
    bad("head_dim", *swap(0, b.q[..., :32]))
    bad("unit innermost", *swap(0, b.q.transpose(0, 2).contiguous().transpose(0, 2)))
    bad("one row per request", *swap(0, b.q[:1]))
    bad("broadcast", *swap(0, b.q[:1, :1].expand(2, 4, 64)))
    bad("one shape", *swap(2, b.v_cache[:-1]))
    bad("one dtype", *swap(2, b.v_cache.half()))
    bad("int32", *swap(3, b.table.long()))
    bad("one row per request", *swap(3, b.table[:1]))
    bad("int32", *swap(4, b.seq.long()))
    bad("must be a CUDA torch tensor", *swap(4, b.seq.cpu()))
    bad("positive multiple", *swap(0, torch.zeros((2, 3, 64), dtype=BF, device=cuda_device)))
    bad("entries", *ok, cu_seqlens_q=b.seq)
    bad("softcap", *ok, softcap=-1.0)
    bad("softcap", *ok, softcap=math.inf)
    bad("finite", *swap(5, math.nan))
    bad("left, right", *ok, window_size=(1,))
    bad("one float32 slope", *ok, alibi_slopes=torch.ones(3, device=cuda_device))
    bad("out_dtype", *ok, out_dtype="int8")
    bad("wrong shape", *ok, out=b.q[:1])
    bad("wrong dtype", *ok, out=b.q.float())
    bad("overlaps itself", *ok, out=torch.zeros((2, 1, 64), dtype=BF, device=cuda_device).expand(2, 4, 64))
    with pytest.raises(RuntimeError, match="beyond the pages"):
        fa.shared_prefix_forward(b.q, b.k_cache, b.v_cache, b.prefix_table, 1, b.table, b.seq, b.scale)
    x = torch.zeros((2, 2, 64), dtype=BF, device=cuda_device)
    slots = torch.zeros(2, dtype=torch.int64, device=cuda_device)
    for match, kw in (("need cos/sin", dict(positions=b.seq)), ("need positions", dict(rope_theta=1e4, max_position=4)),
                      ("max_position", dict(positions=b.seq, rope_theta=1e4)),
                      ("go together", dict(positions=b.seq, cos=torch.zeros((4, 32), device=cuda_device))),
                      ("tokens, num_heads_q", dict(q=b.q[:1]))):
        with pytest.raises(RuntimeError, match=match):
            fa.store_kv(x, x, b.k_cache, b.v_cache, slots, **kw)
    with pytest.raises(RuntimeError, match="int64"):
        fa.store_kv(x, x, b.k_cache, b.v_cache, slots.int())
    with pytest.raises(RuntimeError, match="overlaps itself"):
        fa.store_kv(x, x, b.k_cache[:1].expand(3, -1, -1, -1), b.v_cache[:3], slots)
    i = b.seq
    with pytest.raises(RuntimeError, match="page_size"):
        fa.plan_pages(i, i, b.table, i, 0, 4)
    with pytest.raises(RuntimeError, match="must not overlap"):
        fa.plan_pages(i, i, b.table[:1].expand(2, -1), i, 16, 4)
    with pytest.raises(RuntimeError, match="at most 8192"):
        z = torch.zeros(8193, dtype=torch.int32, device=cuda_device)
        fa.plan_pages(z, z, z[:, None], z, 16, 4)


def test_empty_calls(fa, cuda_device):
    b = Batch(cuda_device, [20, 30], hq=4, hk=2, d=64)
    assert fa.paged_forward(b.q[:0], b.k_cache, b.v_cache, b.table[:0], b.seq[:0]).shape == (0, 4, 64)
    # a cache or table without a page: every request is empty
    o, lse = fa.paged_forward(b.q, b.k_cache[:0], b.v_cache[:0], b.table[:, :0], b.seq * 0, 1.0, return_lse=True)
    torch.cuda.synchronize()
    fa.check_status()
    assert (o == 0).all() and (lse == -math.inf).all()
    x = torch.zeros((0, 2, 64), dtype=BF, device=cuda_device)
    assert fa.store_kv(x, x, b.k_cache, b.v_cache, torch.zeros(0, dtype=torch.int64, device=cuda_device)) is None
