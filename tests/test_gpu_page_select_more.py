"""Page selection over long tables with heads of 128, and page lists that are the same
for all heads of a sequence.

Chosen pages are whole numbers, compared exactly with the definition
(test_gpu_page_select's `choose`).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_page_select import BF, FP8, HF, _gen, choose, ints, mods, pages_of, spread  # noqa: F401  (mods is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,B,H,H_kv,pages,width", [(128, 2, 4, 2, 700, 800), (128, 2, 8, 2, 4096, 4096), (128, 1, 2, 1, 8192, 8192), (128, 2, 2, 2, 20000, 24576),
                                                    (128, 24, 16, 8, 900, 1000), (64, 24, 8, 8, 1500, 1500), (128, 70, 4, 4, 300, 24576)])
def test_choice_over_long_tables(mods, D, B, H, H_kv, pages, width):
    """Full clusters, one CTA an item with the longest first, and tables far wider than what is held."""
    _lib, dec, paged = mods
    r = np.random.RandomState(pages)
    lens = [pages * 16 - 5, pages * 8 + 1] + r.randint(0, pages * 16, max(0, B - 2)).tolist()
    lens = lens[:B]
    table, P = pages_of(lens, 16, 9, width=width)
    q, bounds = _gen((B, H, 1, D), 1, BF), spread(P, H_kv, D, BF, 2)
    for count, first, last in ((1, 0, 1), (128, 1, 2), (pages - 1, 0, 0)):
        got = paged.select_pages(q, bounds, table, ints(lens), count, page_size=16, first=first, last=last)
        want = choose(q, bounds, table, lens, 16, count, first, last)
        assert torch.equal(got.pages, want[0]) and torch.equal(got.lens, want[1]), count
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("pages", [600, 5000])
def test_choice_among_equals_of_long_heads(mods, pages):
    """Pages of few different scores, far more of each than can be ranked; one far above the rest."""
    _lib, dec, paged = mods
    table, P = pages_of([pages * 16], 16, 4)
    r = np.random.RandomState(0)
    for kind in range(3):
        lo, hi = -r.randint(0, 2, (P, 1, 128)) * 1.0, r.randint(0, 2, (P, 1, 128)) * 1.0
        if kind == 0:
            lo[:], hi[:] = -1, 1
        if kind == 2:
            hi[int(table[0, 17]), 0, 3] = 2.0 ** 90
        bounds = torch.from_numpy(np.stack([lo, hi], 2)).to(BF).cuda()
        q = torch.from_numpy(r.randint(-1, 2, (1, 3, 1, 128)) * 1.0).to(BF).cuda()
        for count in (1, 250, pages // 2, pages - 1):
            got = paged.select_pages(q, bounds, table, ints([pages * 16]), count, page_size=16, first=0, last=0)
            want = choose(q, bounds, table, [pages * 16], 16, count, 0, 0)
            assert torch.equal(got.pages, want[0]) and torch.equal(got.lens, want[1]), (kind, count)


@pytest.mark.parametrize("H,H_kv,D,qdt,kvdt", [(8, 4, 128, BF, BF), (32, 8, 64, HF, HF), (8, 8, 128, HF, FP8), (40, 2, 128, BF, FP8), (6, 6, 64, HF, HF), (8, 2, 128, BF, HF)])
def test_equal_lists_are_the_table(mods, H, H_kv, D, qdt, kvdt):
    """One list for all heads of a sequence gives the bits of the decode over its table row: the work is
    numbered and cut alike."""
    _lib, dec, paged = mods
    lens = [0, 1, 31, 32, 33, 700, 3001, 129, 0, 64]
    table, P = pages_of(lens, 32, 3)
    q = _gen((len(lens), H, 1, D), 1, qdt)
    k, v = (_gen((P, H_kv, 32, D), 2 + i).to(kvdt) for i in range(2))
    n = ints(lens)
    # scales other than 1: the same kernel for 16-bit pools of one query head each
    a = paged.paged_decode(q, k, v, table, n, k_scale=0.5, v_scale=2.0, return_lse=True)
    b = paged.paged_decode(q, k, v, table.unsqueeze(1).repeat(1, H_kv, 1), n.unsqueeze(1).repeat(1, H_kv), k_scale=0.5, v_scale=2.0, return_lse=True)
    assert _lib.device_status() == (0, 0)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("T,H_kv,D,dt", [(700, 4, 128, FP8), (4000, 4, 128, FP8), (3000, 8, 128, BF), (10000, 2, 64, HF), (14100, 3, 64, FP8), (14300, 5, 128, BF), (9000, 7, 64, BF)])
def test_bounds_of_prompts(mods, T, H_kv, D, dt):
    """Packed prompts of every cut of rows and heads over the CTAs, pages begun before among them."""
    from test_gpu_page_select import bounds_after, packed
    _lib, dec, paged = mods
    r = np.random.RandomState(T)
    new = r.multinomial(T - 40, [1 / 20] * 20)
    slots, P = packed(r.randint(0, 90, 20), new, 32, T, pad=40)
    k = _gen((P, H_kv, 32, D), 1).to(dt)
    bounds = _gen((P, H_kv, 2, D), 2).to(HF if dt == FP8 else dt)
    want = bounds_after(k, slots, bounds)
    paged.page_bounds(k, ints(slots), bounds)
    assert torch.equal(bounds.double(), want)
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("kvdt,D,H_kv,page", [(BF, 128, 2, 4096), (FP8, 64, 1, 4096), (HF, 64, 3, 1024)])
def test_large_pages(mods, kvdt, D, H_kv, page):
    """Bounds of runs far longer than a CTA's rows, choice and decode of the largest pages."""
    from test_gpu_page_select import bounds_after, check_lists, packed
    _lib, dec, paged = mods
    held, new = [0, page - 1, 5, page], [2 * page + 3, 2, page, 1]
    slots, P = packed(held, new, page, 3, pad=3)
    k, v = (_gen((P, H_kv, page, D), 1 + i).to(kvdt) for i in range(2))
    bounds = _gen((P, H_kv, 2, D), 50).to(HF if kvdt == FP8 else kvdt)
    want = bounds_after(k, slots, bounds)
    paged.page_bounds(k, ints(slots), bounds)
    assert torch.equal(bounds.double(), want)
    lens = (np.array(held) + new).tolist()
    table, _ = pages_of(lens, page, 3)
    bounds, q = spread(P, H_kv, D, BF, 7), _gen((4, 4 * H_kv, 1, D), 9, HF if kvdt == HF else BF)
    strided = q.transpose(0, 1).contiguous().transpose(0, 1)
    chosen = paged.select_pages(strided, bounds, table, ints(lens), 2, page_size=page)
    want = choose(q, bounds, table, lens, page, 2, 1, 1)
    assert torch.equal(chosen.pages, want[0]) and torch.equal(chosen.lens, want[1])
    o, lse = paged.paged_decode(q, k, v, chosen.pages, chosen.lens, return_lse=True)
    check_lists(o, lse, q, k, v, chosen.pages, chosen.lens.cpu().numpy(), what="large pages")
    assert _lib.device_status() == (0, 0)
