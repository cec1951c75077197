"""Workloads of the paged-cache operators: page planning, cache append, attention over a paged
cache, and attention for a batch that shares a prefix.

Every case is one call of a serving step. `run` takes what `prepare` made through one operator,
either as plain torch operations in 32 bits or (where `own` is true) through the package.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decoding step of a full serving batch: every request gets one token.
        dict(name="plan_decode", op="plan", requests=256, cached_lo=1, cached_hi=32768, new_lo=1, new_hi=1,
             page=16, lens_seed=1, pad=0),
        # Prompts of mixed lengths admitted at once, some of them continuing a conversation.
        dict(name="plan_prompts", op="plan", requests=48, cached_lo=0, cached_hi=4096, new_lo=17, new_hi=4096,
             page=16, lens_seed=2, pad=333),
        # Cache append of one decoding step, padded to a fixed batch as a captured step is.
        dict(name="store_decode", op="store", tokens=250, pad=6, hq=32, hkv=8, dim=128, page=16, dtype="bf16",
             theta=500000.0),
        # Cache append of a prompt batch, an odd number of tokens.
        dict(name="store_prompts", op="store", tokens=30001, pad=0, hq=32, hkv=8, dim=128, page=64,
             dtype="bf16", theta=500000.0),
        # Few short conversations, one KV head per query head: latency counts.
        dict(name="decode_short", op="paged", requests=4, cached_lo=90, cached_hi=512, new_lo=1, new_hi=1,
             hq=16, hkv=16, dim=64, page=16, dtype="fp16", lens_seed=3, cap=0.0, window=-1, causal=False),
        # Full-precision decoding at the smallest model's shape.
        dict(name="decode_fp32", op="paged", requests=8, cached_lo=200, cached_hi=1024, new_lo=1, new_hi=1,
             hq=8, hkv=8, dim=64, page=16, dtype="fp32", lens_seed=4, cap=0.0, window=-1, causal=False),
        # A serving batch of very different lengths, grouped heads.
        dict(name="decode_ragged", op="paged", requests=64, cached_lo=64, cached_hi=32768, new_lo=1, new_hi=1,
             hq=32, hkv=8, dim=128, page=64, dtype="bf16", lens_seed=5, cap=0.0, window=-1, causal=False),
        # Capped scores with a sliding window.
        dict(name="decode_capped", op="paged", requests=33, cached_lo=1, cached_hi=8192, new_lo=1, new_hi=1,
             hq=32, hkv=8, dim=128, page=32, dtype="fp16", lens_seed=6, cap=30.0, window=4095, causal=False),
        # Prompt chunks appended to conversations of several thousand tokens.
        dict(name="prefill_chunks", op="paged", requests=4, cached_lo=1000, cached_hi=8192, new_lo=300,
             new_hi=2048, hq=32, hkv=8, dim=128, page=16, dtype="bf16", lens_seed=7, cap=0.0, window=-1,
             causal=True),
        # A small batch behind one instruction text.
        dict(name="prefix_small", op="prefix", requests=16, prefix=2011, cached_lo=0, cached_hi=200, new_lo=1,
             new_hi=1, hq=32, hkv=8, dim=128, page=16, dtype="bf16", lens_seed=8, cap=0.0, window=-1,
             causal=False),
        # Four proposed tokens a request to verify behind a long text, eight heads on one KV head.
        dict(name="prefix_verify", op="prefix", requests=24, prefix=50001, cached_lo=0, cached_hi=1000,
             new_lo=4, new_hi=4, hq=8, hkv=1, dim=128, page=64, dtype="fp16", lens_seed=9, cap=0.0, window=-1,
             causal=True),
        # Many samples drawn from one long context.
        dict(name="prefix_large", op="prefix", requests=256, prefix=32768, cached_lo=0, cached_hi=2048,
             new_lo=1, new_hi=1, hq=64, hkv=8, dim=128, page=128, dtype="bf16", lens_seed=10, cap=0.0,
             window=-1, causal=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(max(lo, 0) + 1), math.log(hi + 1)))) - 1)))


def draw(rng):
    """One more case of the listed ranges."""
    op = rng.choice(["plan", "store", "paged", "paged", "prefix", "prefix"])
    seed = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        prompts = rng.random() < 0.5
        n = _log_int(rng, 1, 48 if prompts else 256)
        return dict(op=op, requests=n, cached_lo=0, cached_hi=_log_int(rng, 16, 32768),
                    new_lo=1, new_hi=4096 if prompts else 1, page=page,
                    lens_seed=seed, pad=rng.choice([0, rng.randrange(1, 400)]))
    hq, hkv = rng.choice([(32, 8), (8, 1), (16, 16), (64, 8), (8, 8), (32, 32), (12, 4)])
    dim = rng.choice([64, 128, 128])
    if op == "store":
        return dict(op=op, tokens=_log_int(rng, 1, 16000), pad=rng.choice([0, rng.randrange(1, 64)]), hq=hq, hkv=hkv,
                    dim=dim, page=page, dtype=rng.choice(["bf16", "fp16", "fp32"]), theta=rng.choice([10000.0, 500000.0]))
    cap = rng.choice([0.0, 0.0, 50.0, 30.0])
    window = rng.choice([-1, -1, rng.randrange(64, 8192)])
    if op == "paged":
        dtype = rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"])
        kind = rng.choice(["one", "few", "chunk"]) if dtype != "fp32" else rng.choice(["one", "few"])
        n = _log_int(rng, 1, {"one": 64, "few": 32, "chunk": 4}[kind])
        top = {"one": 16384, "few": 8192, "chunk": 4096}[kind] if dtype != "fp32" else 2048
        new = {"one": 1, "few": 8, "chunk": 1024}[kind]
        return dict(op=op, requests=n, cached_lo=0, cached_hi=_log_int(rng, 16, top), new_lo=1,
                    new_hi=new, hq=hq, hkv=hkv, dim=dim, page=page,
                    dtype=dtype, lens_seed=seed, cap=cap, window=window, causal=kind != "one")
    n = _log_int(rng, 2, 128)
    few = rng.random() < 0.3 and n <= 32
    return dict(op=op, requests=n, prefix=_log_int(rng, 256, 32768), cached_lo=0, cached_hi=_log_int(rng, 16, 1024),
                new_lo=1, new_hi=4 if few else 1, hq=hq, hkv=hkv, dim=dim, page=page,
                dtype=rng.choice(["bf16", "fp16"]), lens_seed=seed, cap=cap, window=-1, causal=few)


def _lens(case):
    """(cached, new) token counts of every request; they belong to the case, not to the inputs' seed."""
    rng = random.Random(case["lens_seed"])
    cached = [_log_int(rng, case["cached_lo"], case["cached_hi"]) for _ in range(case["requests"])]
    new = [_log_int(rng, case["new_lo"], case["new_hi"]) for _ in range(case["requests"])]
    return cached, new


def _pages(n, page):
    return (n + page - 1) // page


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    return {"plan": _prepare_plan, "store": _prepare_store, "paged": _prepare_attention,
            "prefix": _prepare_attention}[case["op"]](case, dev, g)


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _prepare_plan(case, dev, g):
    cached, new = _lens(case)
    page = case["page"]
    held = [_pages(c, page) for c in cached]
    after = [_pages(c + n, page) for c, n in zip(cached, new)]
    width = max(after) + 3
    total = sum(after) + 64
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    used = sum(held)
    # The table as the last step left it: held pages, anything behind them.
    table = torch.full((len(cached), width), -7, dtype=torch.int32, device=dev)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    return dict(case=case, cached=_i32(cached, dev), new=_i32(new, dev), table=table, free=order[used:].contiguous(),
                begin=torch.zeros(1, dtype=torch.int32, device=dev), rows=sum(new) + case["pad"])


def _prepare_store(case, dev, g):
    t, dt, page = case["tokens"], _TYPES[case["dtype"]], case["page"]
    n_pages = _pages(t, page) + 9
    shape = (n_pages, page, case["hkv"], case["dim"])
    rows = t + case["pad"]

    def rnd(*s):
        return torch.randn(*s, generator=g, device=dev).to(dt)

    slots = torch.full((rows,), -1, dtype=torch.int64, device=dev)
    slots[:t] = torch.randperm(n_pages * page, generator=g, device=dev)[:t]
    if t > 512:  # prompts fill whole pages in order, on pages anywhere
        where = torch.randperm(n_pages, generator=g, device=dev)
        at = torch.arange(t, device=dev)
        slots[:t] = where[at // page] * page + at % page
    positions = torch.zeros(rows, dtype=torch.int32, device=dev)
    positions[:t] = torch.randint(0, 65536, (t,), generator=g, device=dev, dtype=torch.int32)
    return dict(case=case, k_cache=rnd(*shape), v_cache=rnd(*shape), k=rnd(rows, case["hkv"], case["dim"]),
                v=rnd(rows, case["hkv"], case["dim"]), q=rnd(rows, case["hq"], case["dim"]), slots=slots,
                positions=positions, valid=t)


def _prepare_attention(case, dev, g):
    cached, new = _lens(case)
    page, dt = case["page"], _TYPES[case["dtype"]]
    lens = [c + n for c, n in zip(cached, new)]
    counts = [_pages(n, page) for n in lens]
    p_pages = _pages(case.get("prefix", 0), page)
    n_pages = sum(counts) + p_pages + 5
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32, device=dev)
    at = p_pages
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)

    def rnd(*s):
        return torch.randn(*s, generator=g, device=dev).to(dt)

    shape = (n_pages, page, case["hkv"], case["dim"])
    return dict(case=case, q=rnd(starts[-1], case["hq"], case["dim"]), k_cache=rnd(*shape), v_cache=rnd(*shape),
                table=table, lens=_i32(lens, dev), cu=_i32(starts, dev), prefix_table=order[:p_pages].contiguous(),
                host_lens=lens, host_starts=starts, max_new=max(new), scale=1.0 / math.sqrt(case["dim"]))


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "store": _own_store, "paged": _own_paged, "prefix": _own_prefix}[op](state)
    return {"plan": _plain_plan, "store": _plain_store, "paged": _plain_attention, "prefix": _plain_attention}[op](state)


def _own_plan(s):
    import flash_attn_metal_cpp_b200 as fa

    out = fa.plan_pages(s["cached"], s["new"], s["table"], s["free"], s["case"]["page"], s["rows"], free_begin=s["begin"])
    return (*out, s["table"])


def _own_store(s):
    import flash_attn_metal_cpp_b200 as fa

    q = fa.store_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], q=s["q"], positions=s["positions"],
                    rope_theta=s["case"]["theta"], max_position=65536)
    return s["k_cache"], s["v_cache"], q


def _extras(s):
    c = s["case"]
    return dict(cu_seqlens_q=None if c["new_hi"] == 1 else s["cu"], max_seqlen_q=s["max_new"],
                softcap=c["cap"], window_size=None if c["window"] < 0 else (c["window"], -1))


def _own_paged(s):
    import flash_attn_metal_cpp_b200 as fa

    return fa.paged_forward(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["scale"], s["case"]["causal"],
                            **_extras(s))


def _own_prefix(s):
    import flash_attn_metal_cpp_b200 as fa

    return fa.shared_prefix_forward(s["q"], s["k_cache"], s["v_cache"], s["prefix_table"], s["case"]["prefix"], s["table"],
                                    s["lens"], s["scale"], s["case"]["causal"], **_extras(s))


def _plain_plan(s):
    page, table, free = s["case"]["page"], s["table"], s["free"]
    cached, new = s["cached"].long(), s["new"].long()
    held = (cached + page - 1) // page
    after = (cached + new + page - 1) // page
    need = after - held
    ends = s["begin"].long() + need.cumsum(0)
    first = ends - need
    cols = torch.arange(table.shape[1], device=table.device)
    fresh = (cols >= held[:, None]) & (cols < after[:, None])
    pick = (first[:, None] + cols - held[:, None]).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[pick], table))
    cu = torch.zeros(new.numel() + 1, dtype=torch.int64, device=table.device)
    cu[1:] = new.cumsum(0)
    t = torch.arange(s["rows"], device=table.device)
    inside = t < cu[-1]
    req = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=new.numel() - 1)
    pos = torch.where(inside, cached[req] + t - cu[req], torch.zeros_like(t))
    slot = table[req, pos // page].long() * page + pos % page
    slots = torch.where(inside, slot, torch.full_like(slot, -1))
    return (cached + new).int(), cu.int(), slots, pos.int(), ends[-1:].int(), table


def _rotate(x, positions, theta):
    half = x.shape[-1] // 2
    freq = theta ** (-torch.arange(half, dtype=torch.float64, device=x.device) * 2 / x.shape[-1])
    ang = positions.double()[:, None] * freq
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)


def _plain_store(s):
    n, theta = s["valid"], s["case"]["theta"]
    rows = s["slots"][:n]
    kc, vc = s["k_cache"], s["v_cache"]
    kc.view(-1, *kc.shape[2:])[rows] = _rotate(s["k"][:n], s["positions"][:n], theta)
    vc.view(-1, *vc.shape[2:])[rows] = s["v"][:n]
    return kc, vc, _rotate(s["q"], s["positions"], theta)


def _gather(cache, pages, n):
    return cache[pages].reshape(-1, *cache.shape[2:])[:n].float()


def _plain_part(q, k, v, pos, first, case, scale):
    """Unnormalised attention of q [T, Hq, D] at positions pos over keys at first, first + 1, ...:
    (sum of exp times v, sum of exp, maximum) a row."""
    t, hq, d = q.shape
    n, hkv = k.shape[0], k.shape[1]
    qs = q.float().reshape(t, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
    x = qs @ k.permute(1, 2, 0) * scale
    if case["cap"] > 0:
        x = case["cap"] * torch.tanh(x / case["cap"])
    rel = first + torch.arange(n, device=q.device) - pos[:, None]
    hide = torch.zeros(t, n, dtype=torch.bool, device=q.device)
    if case["causal"]:
        hide |= rel > 0
    if case["window"] >= 0:
        hide |= rel < -case["window"]
    x = x.reshape(hkv, hq // hkv, t, n).masked_fill(hide, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    o = e.reshape(hkv, -1, n) @ v.permute(1, 0, 2)
    return (o.reshape(hq, t, d).transpose(0, 1), e.sum(-1).reshape(hq, t).t()[..., None],
            m.reshape(hq, t).t()[..., None])


def _plain_attention(s):
    case, q = s["case"], s["q"]
    prefix = case.get("prefix", 0)
    out = torch.empty_like(q)
    starts, lens = s["host_starts"], s["host_lens"]
    base = None
    if prefix:
        own_pos = torch.cat([torch.arange(prefix + n - (b - a), prefix + n, device=q.device)
                             for n, a, b in zip(lens, starts, starts[1:])])
        kp, vp = _gather(s["k_cache"], s["prefix_table"], prefix), _gather(s["v_cache"], s["prefix_table"], prefix)
        g = case["hq"] // case["hkv"]
        parts = [_plain_part(q[:, h * g:(h + 1) * g], kp[:, h:h + 1], vp[:, h:h + 1], own_pos, 0, case, s["scale"])
                 for h in range(case["hkv"])]
        base = [torch.cat(p, 1) for p in zip(*parts)]
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        pages = s["table"][i, :_pages(n, case["page"])]
        k, v = _gather(s["k_cache"], pages, n), _gather(s["v_cache"], pages, n)
        pos = torch.arange(prefix + n - (b - a), prefix + n, device=q.device)
        o, l, m = _plain_part(q[a:b], k, v, pos, prefix, case, s["scale"])
        if base is not None:
            o0, l0, m0 = (x[a:b] for x in base)
            top = torch.maximum(m, m0)
            o = o * torch.exp(m - top) + o0 * torch.exp(m0 - top)
            l = l * torch.exp(m - top) + l0 * torch.exp(m0 - top)
        out[a:b] = (o / l).to(out.dtype)
    return out


# ------------------------------------------------------------------ 64-bit values
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "store":
        n, half = s["valid"], case["dim"] // 2
        inv = torch.tensor([case["theta"] ** (-2.0 * i / case["dim"]) for i in range(half)], dtype=torch.float64,
                           device=s["q"].device)

        def turn(x, p):
            z = torch.complex(x[..., :half].double(), x[..., half:].double())
            z = z * torch.polar(torch.ones_like(inv), p.double()[:, None] * inv)[:, None]
            return torch.cat([z.real, z.imag], -1)

        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        at = s["slots"][:n]
        page = case["page"]
        k_cache[at // page, at % page] = turn(s["k"][:n], s["positions"][:n])
        v_cache[at // page, at % page] = s["v"][:n].double()
        return k_cache, v_cache, turn(s["q"], s["positions"])
    # Attention: all keys of a request side by side, one softmax in 64 bits.
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    prefix = case.get("prefix", 0)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i, n in enumerate(s["host_lens"]):
        a, b = s["host_starts"][i], s["host_starts"][i + 1]
        where = torch.arange(n, device=out.device)
        idx = s["table"][i].long()[where // page] * page + where % page
        if prefix:
            p = torch.arange(prefix, device=out.device)
            idx = torch.cat([s["prefix_table"].long()[p // page] * page + p % page, idx])
        key_at = torch.arange(prefix + n, device=out.device)
        row_at = prefix + n - (b - a) + torch.arange(b - a, device=out.device)
        seen = torch.ones(b - a, prefix + n, dtype=torch.bool, device=out.device)
        if case["causal"]:
            seen &= key_at[None] <= row_at[:, None]
        if case["window"] >= 0:
            seen &= key_at[None] >= row_at[:, None] - case["window"]
        for h in range(hkv):
            k = s["k_cache"].view(-1, hkv, case["dim"])[idx, h].double()
            v = s["v_cache"].view(-1, hkv, case["dim"])[idx, h].double()
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            x = torch.einsum("thd,nd->htn", s["q"][a:b, heads].double(), k) * s["scale"]
            if case["cap"] > 0:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            w = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
            out[a:b, heads] = torch.einsum("htn,nd->thd", w, v)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "plan":
        cached, new = _lens(case)
        page = case["page"]
        fresh = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        rows = sum(new) + case["pad"]
        # lengths in and out, new pages read and written, slot and position a token
        return {"bytes": 16 * len(cached) + 8 * fresh + 12 * rows, "flops": 4 * rows}
    el = _BYTES[case["dtype"]]
    if case["op"] == "store":
        rows, heads = case["tokens"], case["hq"] + 2 * case["hkv"]
        return {"bytes": 2 * rows * heads * case["dim"] * el + 12 * rows,
                "flops": 3 * rows * (case["hq"] + case["hkv"]) * case["dim"]}
    cached, new = _lens(case)
    prefix, w = case.get("prefix", 0), case["window"]
    keys, pairs = prefix, 0
    for c, n in zip(cached, new):
        first = max(0, prefix + c - w) if w >= 0 else 0   # first key the first row sees
        keys += c + n - max(0, first - prefix)
        for j in range(n):
            lo = max(0, prefix + c + j - w) if w >= 0 else 0
            hi = prefix + c + (j + 1 if case["causal"] else n)
            pairs += hi - lo
    rows = sum(new)
    return {"bytes": 2 * keys * case["hkv"] * case["dim"] * el + 2 * rows * case["hq"] * case["dim"] * el,
            "flops": 4 * pairs * case["hq"] * case["dim"]}
