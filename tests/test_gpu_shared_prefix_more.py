"""Shared prefixes where test_gpu_shared_prefix does not reach: many short runs over
e4m3 pools.

Tolerances are those of test_gpu_shared_prefix (its `check`).
"""
from __future__ import annotations

import pytest
import torch
from test_gpu_paged_gqa import BF, FP8
from test_gpu_shared_prefix import batch, check, ints, make, mods  # noqa: F401  (a fixture)

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
