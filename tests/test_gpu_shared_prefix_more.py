"""Shared prefixes where test_gpu_shared_prefix does not reach: many short runs over
e4m3 pools, scales that are not positive.

Tolerances are those of test_gpu_shared_prefix (its `check`).
"""
from __future__ import annotations

import math

import pytest
import torch
from test_gpu_paged_gqa import BF, FP8
from test_gpu_shared_prefix import KINDS, batch, check, enough, ints, make, mods  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------
# short runs
# --------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,each", [(256, 3), (128, 5), (256, 15), (384, 3)])
def test_short_runs_of_scaled_queries(mods, tokens, each):
    """Many prefixes of one to three tiles with no more than 128 rows, e4m3 pools and bf16 queries
    of very different magnitudes: a CTA takes several of them one after the other, and each
    row's power of two is its own run's."""
    _lib, dec, paged = mods
    page, H, H_kv = 64, 64, 8
    table, P, lens, shared, starts = batch([(tokens, [(7 * i + 50 * j) % 90 for j in range(each)]) for i in range(64)], page, tokens)
    q, k, v = make(P, len(lens), H, H_kv, 128, page, BF, FP8, 5, 0.05, 0.03)
    g = torch.Generator(device="cuda").manual_seed(each)
    q = (q.float() * torch.randint(-30, 2, (len(lens), H, 1, 1), device="cuda", generator=g).float().exp2()).to(BF)
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, shared_groups=starts, k_scale=0.05, v_scale=0.03, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, 0.05, 0.03, what="short runs", sample=200)
    for _ in range(20):
        assert torch.equal(o, paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, shared_groups=starts, k_scale=0.05, v_scale=0.03))


# --------------------------------------------------------------------------
# scales
# --------------------------------------------------------------------------
@pytest.mark.parametrize("H,H_kv,D,qdt,kvdt", KINDS)
@pytest.mark.parametrize("sm_scale", [0.37, 0.0, -0.11, 1e-40, 2.0 ** -126, math.nan])
def test_any_scale(mods, H, H_kv, D, qdt, kvdt, sm_scale):
    """Scores may be scaled by anything, as without the prefix: a shared length that ends inside a tile
    has masked tokens, whose weight is nothing whatever the scale."""
    _lib, dec, paged = mods
    page, tokens = 16, 144
    n = enough(tokens, H, H_kv)
    table, P, lens, shared, _ = batch([(tokens, ([0, 1, 90] + [9] * n)[:n])], page, 7)
    q, k, v = make(P, n, H, H_kv, D, page, qdt, kvdt, 3)
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, sm_scale=sm_scale, return_lse=True)
    assert _lib.device_status() == (0, 0)
    if math.isnan(sm_scale):
        assert o.isnan().all() and lse.isnan().all()
    elif sm_scale < 0:
        check(o, lse, -q, k, v, table, lens, scale=-sm_scale, what="negative")
    else:
        check(o, lse, q, k, v, table, lens, scale=sm_scale, what=f"scale {sm_scale}")
    if not sm_scale > 0 and (H > H_kv or kvdt == FP8):     # the same kernel as without it
        a, b = paged.paged_decode(q, k, v, table, ints(lens), sm_scale=sm_scale, return_lse=True)
        assert torch.allclose(o, a, 0, 0, equal_nan=True) and torch.allclose(lse, b, 0, 0, equal_nan=True)


def test_scales_whose_product_vanishes(mods):
    """sm_scale and k_scale are positive, their product is not."""
    _lib, dec, paged = mods
    table, P, lens, shared, _ = batch([(144, [9] * 140)], 16, 7)
    q, k, v = make(P, 140, 12, 4, 128, 16, BF, FP8, 3)
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, sm_scale=1e-30, k_scale=1e-30, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, scale=0.0, what="product")
