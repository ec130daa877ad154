"""Shared prefixes where test_gpu_shared_prefix does not reach: many short runs over
e4m3 pools, scales that are not positive, and that shared pages are read once at all.

Tolerances are those of test_gpu_shared_prefix (its `check`).
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from test_gpu_paged_gqa import BF, FP8, HF
from test_gpu_shared_prefix import KINDS, batch, check, ints, make, mods  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def enough(tokens, H, H_kv, D, kvdt, short=0):
    """Sequences from which on a prefix of `tokens` tokens is shared: 2048 tiles saved, where a pass
    of 128 rows, those of `short` sequences that do not hold it among them, costs as much as 2 of a
    sequence's own tiles of 64 KB, or 4 of 32."""
    G, cost = H // H_kv, 2 if D == 128 and kvdt != FP8 else 4
    saved = lambda n: (n * -(-G // 16) - -(-(n + short) * G // 128) * cost) * -(-tokens // 128) * H_kv      # noqa: E731
    return next(n for n in range(2, 10000) if saved(n) >= 2048)


# --------------------------------------------------------------------------
# short runs
# --------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,each", [(256, 6), (128, 8), (256, 15), (384, 6)])
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
    n = enough(tokens, H, H_kv, D, kvdt)
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
    table, P, lens, shared, _ = batch([(144, [9] * 400)], 16, 7)
    q, k, v = make(P, 400, 12, 4, 128, 16, BF, FP8, 3)
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
    With one sequence fewer nothing is shared, and the missing entries are reported; so with one
    more that is too short to share."""
    _lib, dec, paged = mods
    n = enough(tokens, H, H_kv, D, kvdt)
    own = ([1, 0, 90, 130] + [9] * n)[:n]
    table, P, lens, shared, _ = batch([(tokens, own)], page, 7)
    q, k, v = make(P, n, H, H_kv, D, page, qdt, kvdt, 3)
    bare = table.clone()
    bare[1:, :tokens // page] = -1
    o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="one row")
    paged.paged_decode(q[:-1], k, v, bare[:-1].contiguous(), ints(lens[:-1]), shared_lens=shared)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 302)
    lens[2] = tokens - 1
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, return_lse=True)
    check(o, lse, q, k, v, table, lens, what="one too short")
    assert _lib.device_status() == (0, 0)
    paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 302)


def test_others_rows_of_several_groups_are_not_read(mods):
    _lib, dec, paged = mods
    page, groups = 32, [(960, [5, 0, 70] * 40), (320, [1] * 80), (64, []), (512, [33] * 90)]
    table, P, lens, shared, starts = batch(groups, page, 3)
    q, k, v = make(P, len(lens), 8, 2, 128, page, BF, BF, 5)
    bare, at = table.clone(), starts.tolist()
    for i, (tokens, _) in enumerate(groups):
        bare[at[i] + 1:at[i + 1], :tokens // page] = -1
    o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, shared_groups=starts, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="groups")


# --------------------------------------------------------------------------
# enough sequences that the device shares
# --------------------------------------------------------------------------
@pytest.mark.parametrize("H,H_kv,D,qdt,kvdt", KINDS)
@pytest.mark.parametrize("page,tokens", [(16, 16), (16, 144), (64, 128), (64, 960), (256, 2048)])
def test_just_enough(mods, H, H_kv, D, qdt, kvdt, page, tokens):
    """As few sequences as share: one page, tiles and a rest, several items of 256 rows; the sequences'
    own tokens from none on, some shorter than the prefix, the first among them."""
    _lib, dec, paged = mods
    r = np.random.RandomState(page + tokens)
    ks, vs = (0.05, 0.03) if kvdt == FP8 else (1.0, 1.0)
    n = enough(tokens, H, H_kv, D, kvdt, short=3) + 3
    own = [0, 1, page, 129] + r.randint(0, 40, n).tolist()
    table, P, lens, shared, _ = batch([(tokens, own[:n])], page, 7)
    lens[0], lens[n // 2], lens[n - 1] = 0, tokens - 1, tokens // 2
    q, k, v = make(P, n, H, H_kv, D, page, qdt, kvdt, 3)
    bare = table.clone()                 # the second sequence's row is the one that is read
    bare[2:, :tokens // page] = torch.where(ints(lens[2:] >= tokens).bool().unsqueeze(1), -1, table[2:, :tokens // page])
    o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, k_scale=ks, v_scale=vs, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, ks, vs, what=f"{tokens} shared by {n}")
    assert torch.equal(o, paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, k_scale=ks, v_scale=vs))


@pytest.mark.parametrize("kvdt", [BF, FP8])
def test_lengths_that_do_not_fit_a_large_batch(mods, kvdt):
    """Shared lengths inside a page, longer than the table or negative, sequences shorter than the
    prefix, starts in disorder, where what is left is still shared."""
    _lib, dec, paged = mods
    page, B = 64, 420
    table, P, lens, shared, _ = batch([(640, [10, 0, 100, 33, 5] + [7] * (B - 5))], page, 3)
    assert B - 20 >= enough(640, 8, 2, 128, kvdt, short=20)
    q, k, v = make(P, B, 8, 2, 128, page, BF, kvdt, 5)
    bare = table.clone()
    bare[7:, :10] = -1                   # the first seven hold it in what follows, or do not
    for s in (640, 641, 703):
        o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=ints([s]), return_lse=True)
        assert _lib.device_status() == (0, 0)
        check(o, lse, q, k, v, table, lens, what=f"shared {s}")
    for s in (2 ** 31 - 1, 639, 65, 0, -5):
        o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=ints([s]), return_lse=True)
        check(o, lse, q, k, v, table, lens, what=f"shared {s}")
    for short in ([0, 640, 740, 673, 645], [0, 0, 740, 1, 645], [300, 639, 0, 128, 640], [0, 0, 0, 0, 0], [5, 639, 70, 64, 1]):
        short = np.array(short + [647] * (B - 5))
        o, lse = paged.paged_decode(q, k, v, bare, ints(short), shared_lens=shared, return_lse=True)
        assert _lib.device_status() == (0, 0)
        check(o, lse, q, k, v, table, short, what=f"lengths {short}")
    for starts in ([0, B, 3], [-7, 2, 900], [4, 9, B], [5, 5, 5], [1, 410, B + 1]):
        o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=ints([640, 640]), shared_groups=ints(starts), return_lse=True)
        check(o, lse, q, k, v, table, lens, what=f"starts {starts}")
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("D,page,kvdt", [(128, 16, BF), (64, 32, HF), (128, 64, FP8), (128, 256, BF)])
def test_stale_and_missing_pages_of_a_large_batch(mods, D, page, kvdt):
    """NaN in pages of nobody never counts; shared entries outside the pool are reported and their tokens
    left out for all, in every tile of the prefix and in its last, partial one."""
    _lib, dec, paged = mods
    pages = 4 if page == 256 else 384 // page + 3
    tokens = pages * page
    table, P, lens, shared, _ = batch([(tokens, [5, 0, 100] + [7] * 500)], page, 3, spare=9)
    assert len(lens) >= enough(tokens, 8, 2, D, kvdt)
    q, k, v = make(P, len(lens), 8, 2, D, page, HF if kvdt == HF else BF, kvdt, 5)
    used = torch.zeros(P, dtype=torch.bool, device="cuda")
    used[table[table >= 0].long()] = True
    nan = torch.full((1,), math.nan, device="cuda").to(kvdt)
    for pool in (k, v):
        raw = pool.view(torch.uint8) if kvdt == FP8 else pool
        raw[~used] = nan.view(torch.uint8) if kvdt == FP8 else nan
    bare = table.clone()
    bare[1:, :pages] = -1
    o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="stale")
    for gone in ([1, pages - 1], list(range(pages))):
        if gone == list(range(pages)):
            lens = np.maximum(lens, tokens + 1)          # something is left of each
        bare[0] = table[0]
        bare[0, gone] = torch.tensor([P, -1] * len(gone), dtype=torch.int32, device="cuda")[:len(gone)]
        o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, return_lse=True)
        assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 302)
        rest = [i for i in range(table.shape[1]) if i not in gone]
        check(o, lse, q, k, v, table[:, rest].contiguous(), lens - len(gone) * page, what="missing")


def test_large_scores_of_a_large_batch(mods):
    """Scores of far more than exp's range: the maxima move and nothing overflows."""
    _lib, dec, paged = mods
    page, B = 32, 120
    table, P, lens, shared, _ = batch([(2048, [40] * B)], page, 3)
    for kvdt, qdt in ((BF, BF), (HF, HF), (FP8, BF), (FP8, HF)):
        assert B >= enough(2048, 8, 2, 128, kvdt)
        q, k, v = make(P, B, 8, 2, 128, page, qdt, kvdt, 5)
        q = (q.float() * torch.linspace(0.01, 40, B, device="cuda").view(-1, 1, 1, 1)).to(qdt)
        k[table[0, :64].long()] = (k[table[0, :64].long()].float() * torch.linspace(0.1, 2, 64, device="cuda").view(-1, 1, 1, 1)).to(kvdt)
        bare = table.clone()
        bare[1:, :64] = -1
        o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, return_lse=True)
        assert _lib.device_status() == (0, 0)
        check(o, lse, q, k, v, table, lens, what=f"{kvdt}")


@pytest.mark.parametrize("H,H_kv,D,qdt,kvdt", [(8, 2, 128, BF, BF), (40, 2, 64, BF, BF), (12, 4, 128, BF, FP8), (64, 1, 128, HF, HF)])
def test_too_little_for_any_lengths(mods, H, H_kv, D, qdt, kvdt):
    """Tables in which too little can be shared: the decode without a prefix, bit for bit; and one sequence
    alone however long."""
    _lib, dec, paged = mods
    for tokens, own, page in ((512, [30, 0, 300, 7], 64), (40000, [9], 64)):
        table, P, lens, shared, _ = batch([(tokens, own)], page, 5)
        q, k, v = make(P, len(lens), H, H_kv, D, page, qdt, kvdt, 3)
        a = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, return_lse=True)
        b = paged.paged_decode(q, k, v, table, ints(lens), return_lse=True)
        assert _lib.device_status() == (0, 0)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_bound_on_what_can_be_saved(mods):
    """As narrow a table as shares, and as few sequences: what the host may skip is never shared."""
    _lib, dec, paged = mods
    for kvdt, H, H_kv, page, tokens in ((BF, 8, 2, 128, 1024), (FP8, 8, 2, 128, 1024), (BF, 64, 1, 128, 4096)):
        n = enough(tokens, H, H_kv, 128, kvdt)
        table, P, lens, shared, _ = batch([(tokens, [0] * n)], page, 5)
        table = table[:, :tokens // page].contiguous()
        q, k, v = make(P, n, H, H_kv, 128, page, BF, kvdt, 3)
        bare = table.clone()
        bare[1:] = -1
        o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, return_lse=True)
        assert _lib.device_status() == (0, 0)
        check(o, lse, q, k, v, table, lens, what="narrow")


@pytest.mark.parametrize("H,H_kv,D,page,qdt,kvdt,tokens,n", [
    # more query heads of a K/V head than an item has rows; as many as that; the largest pages; one head
    (300, 1, 128, 64, BF, BF, 1024, 21), (300, 1, 128, 32, BF, FP8, 2048, 30), (512, 2, 64, 16, HF, HF, 1040, 16), (8, 2, 128, 4096, BF, BF, 8192, 30),
    (8, 4, 128, 4096, HF, FP8, 4096, 40), (2, 2, 64, 1024, HF, HF, 4096, 200), (1, 1, 128, 128, BF, BF, 2048, 140)])
def test_heads_and_pages(mods, H, H_kv, D, page, qdt, kvdt, tokens, n):
    _lib, dec, paged = mods
    ks, vs = (0.05, 0.03) if kvdt == FP8 else (1.0, 1.0)
    assert n >= enough(tokens, H, H_kv, D, kvdt)
    table, P, lens, shared, _ = batch([(tokens, [(37 * i) % 200 for i in range(n)])], page, n)
    q, k, v = make(P, n, H, H_kv, D, page, qdt, kvdt, 3, ks, vs)
    bare = table.clone()
    bare[1:, :tokens // page] = -1
    o, lse = paged.paged_decode(q, k, v, bare, ints(lens), shared_lens=shared, k_scale=ks, v_scale=vs, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, ks, vs, what="heads and pages", sample=12)


def test_the_largest_batch(mods):
    """8192 sequences in 64 groups, queries that are a view of other strides."""
    _lib, dec, paged = mods
    page, B = 16, 8192
    table, P, lens, shared, starts = batch([(16 * (1 + i % 20), [(5 * i + j) % 40 for j in range(128)]) for i in range(64)], page, 1)
    q, k, v = make(P, B, 4, 1, 128, page, BF, BF, 3)
    bare, at = table.clone(), starts.tolist()
    for i in range(64):
        bare[at[i] + 1:at[i + 1], :1 + i % 20] = -1
    strided = q.transpose(0, 1).contiguous().transpose(0, 1)
    o, lse = paged.paged_decode(strided, k, v, bare, ints(lens), shared_lens=shared, shared_groups=starts, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="largest batch", sample=100)
    odd = torch.empty(q.numel() + 1, dtype=BF, device="cuda")[1:].view(q.shape).copy_(q)     # 2 bytes off
    assert torch.equal(o, paged.paged_decode(odd, k, v, bare, ints(lens), shared_lens=shared, shared_groups=starts))
