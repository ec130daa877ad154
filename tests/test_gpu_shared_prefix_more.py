"""Shared prefixes where test_gpu_shared_prefix does not reach: many short runs over
e4m3 pools, scales that are not positive, and that shared pages are read once at all.

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


# --------------------------------------------------------------------------
# what is shared is read through one row
# --------------------------------------------------------------------------
@pytest.mark.parametrize("H,H_kv,D,qdt,kvdt", KINDS)
@pytest.mark.parametrize("page,tokens", [(16, 144), (64, 960), (256, 2048)])
def test_others_rows_are_not_read(mods, H, H_kv, D, qdt, kvdt, page, tokens):
    """Where sequences share, only one row names the shared pages: the others' entries may be anything.
    With one sequence fewer nothing is shared, and the missing entries are reported."""
    _lib, dec, paged = mods
    n = enough(tokens, H, H_kv)
    own = ([0, 1, 90, 130] + [9] * n)[:n]
    table, P, lens, shared, _ = batch([(tokens, own)], page, 7)
    q, k, v = make(P, n, H, H_kv, D, page, qdt, kvdt, 3)
    lens[0] = tokens - 1                 # the first sequence is too short to be the one that is read
    bare = table.clone()
    bare[2:, :tokens // page] = -1
    o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="one row")
    paged.paged_decode(q[:-1], k, v, bare[:-1].contiguous(), ints(lens[:-1]), shared_lens=shared)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 302)


def test_others_rows_of_several_groups_are_not_read(mods):
    _lib, dec, paged = mods
    page, groups = 32, [(960, [5, 0, 70] * 20), (320, [1] * 40), (64, []), (512, [33] * 50)]
    table, P, lens, shared, starts = batch(groups, page, 3)
    q, k, v = make(P, len(lens), 8, 2, 128, page, BF, BF, 5)
    bare, at = table.clone(), starts.tolist()
    for i, (tokens, _) in enumerate(groups):
        bare[at[i] + 1:at[i + 1], :tokens // page] = -1
    o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, shared_groups=starts, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="groups")
