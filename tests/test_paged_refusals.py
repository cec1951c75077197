"""Refusals of the paged-cache operators that need no device. Every call here is refused: none may reach a kernel."""
from __future__ import annotations

import ctypes

import pytest

from test_paged_api import lib  # noqa: F401  (fixture)

# 4 requests, 6 free pages, 10 rows: every array by itself, 4096 bytes apart.
PLAN = ["cached", "fresh", "free_pages", "free_begin", "table", "seq_lens", "cu", "slots", "positions", "free_end"]
SIZES = dict(cached=16, fresh=16, free_pages=24, free_begin=4, seq_lens=16, cu=20, slots=80, positions=40, free_end=4)
OUTPUTS = ["seq_lens", "cu", "slots", "positions", "free_end"]


@pytest.mark.parametrize("out", OUTPUTS)
@pytest.mark.parametrize("other", list(SIZES))
def test_plan_refuses_arrays_that_overlap(lib, out, other):  # noqa: F811
    if out == other:
        pytest.skip("one array")
    lib.fa_plan_pages.argtypes = ([ctypes.c_uint32] * 5 + [ctypes.c_void_p] * 5 + [ctypes.c_int64] +
                                  [ctypes.c_void_p] * 6)
    at = {n: 1 << 20 | i << 12 for i, n in enumerate(PLAN)}

    def call(**moved):
        p = {**at, **moved}
        return lib.fa_plan_pages(4, 16, 4, 6, 10, *(p[n] for n in PLAN[:5]), 0, *(p[n] for n in PLAN[5:]), None)

    # the same address, and the last element of one on the first of the other
    for where in (at[other], at[other] + SIZES[other] - 4, at[other] - SIZES[out] + 4):
        assert call(**{out: where}) == 1
        text = lib.fa_last_error()
        assert b"must not overlap" in text and out.encode() in text and other.encode() in text
