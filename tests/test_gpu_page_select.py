"""Page bounds, page selection and decode over page lists of each K/V head,
against the formulas in 64 bits.

Bounds are choices of stored values, compared bit for bit (by value); chosen
pages are whole numbers, compared exactly: the kernel sums in 64 bits, as the
formula here does, and random scores differ by far more than 2^-45 of them.
The decode's tolerance is that of the paged grouped decode (test_gpu_paged_gqa).
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from test_gpu_paged_gqa import BF, FP8, HF, _gen, check, pages_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    from pallas_flash import _lib
    from pallas_flash.kernels import decoding, paged
    _lib.device_status()
    return _lib, decoding, paged


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a)).int().cuda()


def wide(t):
    return t.view(torch.uint8).view(t.dtype).double() if t.dtype == FP8 else t.double()


# --------------------------------------------------------------------------
# bounds
# --------------------------------------------------------------------------
def packed(held, new, page, seed, pad=0):
    """Slots of a step's new tokens, as the page plan makes them, and the pages' number."""
    held, new = np.asarray(held), np.asarray(new)
    table, P = pages_of(held + new, page, seed)
    table = table.cpu().numpy()
    slots = []
    for b in range(len(held)):
        at = held[b] + np.arange(new[b])
        slots += (table[b, at // page].astype(np.int64) * page + at % page).tolist()
    return np.array(slots + [-1] * pad, np.int64), P


def bounds_after(k, slots, bounds):
    """The definition: rows named, and what was there where row 0 is not among them."""
    page, out = k.shape[2], bounds.double()
    rows = {}
    for s in slots:
        if 0 <= s < k.shape[0] * page:
            rows.setdefault(int(s) // page, []).append(int(s) % page)
    for p, r in rows.items():
        x = wide(k[p])[:, r]
        lo, hi = x.amin(1), x.amax(1)
        if 0 not in r:
            lo, hi = torch.minimum(lo, out[p, :, 0]), torch.maximum(hi, out[p, :, 1])
        out[p, :, 0], out[p, :, 1] = lo, hi
    return out


@pytest.mark.parametrize("kvdt", [BF, HF, FP8])
@pytest.mark.parametrize("D,H_kv,page", [(128, 3, 16), (64, 2, 64), (128, 1, 256), (64, 5, 32)])
def test_bounds(mods, kvdt, D, H_kv, page):
    """Single tokens, prompts, pages begun before, at their edges, padding rows; nothing else is written."""
    _lib, dec, paged = mods
    steps = [([0, 1, page - 1, page, 5 * page + 3, 0, 7], [1, 1, 1, 1, 1, 0, 1]),
             ([0, 3, page - 1, page, 2], [3 * page, page - 3, 2, page + 1, 1]),
             ([5], [1]), ([0] * 70, [1] * 70), ([0], [7 * page + 5])]
    for i, (held, new) in enumerate(steps):
        slots, P = packed(held, new, page, i, pad=i)
        k = _gen((P, H_kv, page, D), i).to(kvdt)
        bounds = _gen((P, H_kv, 2, D), 50 + i).to(HF if kvdt == FP8 else kvdt)
        want = bounds_after(k, slots, bounds)
        paged.page_bounds(k, ints(slots), bounds)
        assert torch.equal(bounds.double(), want), (i, held, new)
        paged.page_bounds(k, ints(slots), bounds)          # the same rows again change nothing
        assert torch.equal(bounds.double(), want)
    assert _lib.device_status() == (0, 0)


def test_bounds_of_special_values(mods):
    """Infinities are values, a NaN stays one; every finite e4m3 value has its bound in f16."""
    _lib, dec, paged = mods
    k = _gen((2, 1, 16, 64), 1, BF)
    k[0, 0, 3, 5], k[0, 0, 4, 6], k[1, 0, 0, 7] = math.inf, -math.inf, math.nan
    bounds = paged.empty_bounds(k)
    paged.page_bounds(k, ints(np.arange(32)), bounds)
    assert bounds[0, 0, 1, 5] == math.inf and bounds[0, 0, 0, 6] == -math.inf
    nan = torch.isnan(bounds)
    assert nan[1, 0, :, 7].all() and int(nan.sum()) == 2
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    codes = codes[(codes & 127) != 127].repeat(9)[:2 * 16 * 64]
    k = codes.view(2, 1, 16, 64).contiguous().view(FP8)
    bounds = paged.empty_bounds(k)
    paged.page_bounds(k, ints(np.arange(32)), bounds)
    assert torch.equal(bounds.double(), bounds_after(k, np.arange(32), bounds))


def test_bounds_of_bad_slots(mods):
    """A slot past the pool is reported and left out; negative ones and an empty batch write nothing."""
    _lib, dec, paged = mods
    k = _gen((3, 2, 32, 128), 2, HF)
    bounds = _gen((3, 2, 2, 128), 3, HF)
    before = bounds.clone()
    paged.page_bounds(k, ints([-1] * 50), bounds)
    paged.page_bounds(k, ints(np.zeros(0)), bounds)
    assert torch.equal(bounds, before) and _lib.device_status() == (0, 0)
    # page 1 is named by two runs here, which no plan makes: its bounds are either's
    paged.page_bounds(k, ints([96, 32, 33, 2 ** 31 - 1, -5, 34]), bounds)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 309)
    assert torch.equal(bounds[[0, 2]], before[[0, 2]])
    slots = [96, 32, 33, 34, 2 ** 31 - 1, -5, 70, 97]
    want = bounds_after(k, slots, before)
    paged.page_bounds(k, ints(slots), bounds)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 309)
    assert torch.equal(bounds.double(), want)


# --------------------------------------------------------------------------
# choice
# --------------------------------------------------------------------------
def choose(q, bounds, table, lens, page, count, first, last):
    """The definition, page by page."""
    (B, H, _, D), H_kv = q.shape, bounds.shape[1]
    G, P = H // H_kv, bounds.shape[0]
    pages = torch.full((B, H_kv, count), -1, dtype=torch.int32)
    out = torch.zeros((B, H_kv), dtype=torch.int32)
    table = table.cpu()
    for b, n in enumerate(np.minimum(np.maximum(np.asarray(lens), 0), table.shape[1] * page).tolist()):
        live = -(-n // page)
        good = [i for i in range(live) if 0 <= int(table[b, i]) < P]
        at = table[b, good].long().cuda()
        for g in range(H_kv):
            x = bounds[at, g].double().unsqueeze(1) * q[b, g * G:(g + 1) * G, 0].double().unsqueeze(1)
            score = x.amax(2).sum((1, 2)).tolist()
            keep = set(range(live)) if live <= count else set(range(first)) | set(range(live - last, live))
            keep &= set(good)
            order = sorted((i for i in range(len(good)) if good[i] not in keep), key=lambda i: (-score[i], i))
            if live > count:
                keep |= {good[i] for i in order[:count - len(keep)]}
            chosen = sorted(keep)
            pages[b, g, :len(chosen)] = table[b, chosen]
            out[b, g] = sum(min(page, n - i * page) for i in chosen)
    return pages.cuda(), out.cuda()


def spread(P, H_kv, D, dtype, seed):
    """Bounds of random pages."""
    c, w = _gen((P, H_kv, 1, D), seed), _gen((P, H_kv, 2, D), seed + 1).abs()
    return (0.5 * c + torch.tensor([[-1.0], [1.0]], device="cuda") * w).to(dtype)


@pytest.mark.parametrize("H,H_kv,D,page,qdt,bdt", [(32, 8, 128, 64, BF, BF), (6, 2, 64, 16, HF, HF), (5, 5, 128, 32, BF, HF), (40, 2, 64, 128, HF, BF),
                                                   (128, 1, 128, 16, BF, BF)])
@pytest.mark.parametrize("count,first,last", [(1, 0, 0), (1, 0, 1), (7, 1, 2), (40, 0, 4), (40, 20, 20)])
def test_choice(mods, H, H_kv, D, page, qdt, bdt, count, first, last):
    """Lengths from none to far more than are chosen, at the edges of pages and of `count`."""
    _lib, dec, paged = mods
    lens = [0, 1, page, page + 1, count * page - 1, count * page, count * page + 1, 60 * page, 61 * page - 3, 300 * page + 5]
    table, P = pages_of(lens, page, 3)
    q, bounds = _gen((len(lens), H, 1, D), 5, qdt), spread(P, H_kv, D, bdt, 6)
    got = paged.select_pages(q, bounds, table, ints(lens), count, page_size=page, first=first, last=last)
    pages, n = choose(q, bounds, table, lens, page, count, first, last)
    assert torch.equal(got.lens, n)
    assert torch.equal(got.pages, pages)
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("pages,width", [(1, 1), (63, 64), (65, 65), (129, 200), (700, 700), (5000, 6000), (24576, 24576)])
def test_choice_widths(mods, pages, width):
    """One CTA to a full cluster, few pages to as many as a call takes."""
    _lib, dec, paged = mods
    lens = [pages * 16 - 5, max(1, pages // 2) * 16, 3]
    table, P = pages_of(lens, 16, 9, width=width)
    q, bounds = _gen((3, 4, 1, 64), 1, BF), spread(P, 2, 64, BF, 2)
    for count in (1, 30, pages):
        got = paged.select_pages(q, bounds, table, ints(lens), count, page_size=16, first=0, last=1)
        want = choose(q, bounds, table, lens, 16, count, 0, 1)
        assert torch.equal(got.pages, want[0]) and torch.equal(got.lens, want[1]), count
    assert _lib.device_status() == (0, 0)


def test_choice_among_equals(mods):
    """Equal scores: the lowest index.  All equal, two values, zeros of both signs, and one
    outlier that leaves all the others in one bin."""
    _lib, dec, paged = mods
    page, n = 16, 3000
    table, P = pages_of([n * page], page, 4)
    r = np.random.RandomState(0)
    for kind in range(5):
        x = torch.zeros(n, dtype=torch.float64)
        if kind == 1:
            x[r.permutation(n)[:1500]] = 1
        if kind == 2:
            x[::2] = -0.0
        if kind == 3:
            x = torch.from_numpy(r.randint(0, 40, n) / 64.0)
            x[77] = 2.0 ** 100
        if kind == 4:
            x = torch.from_numpy(2.0 ** -(r.randint(0, 120, n).astype(np.float64)))
        bounds = torch.zeros((P, 1, 2, 64), dtype=BF, device="cuda")
        bounds[table[0].long(), 0, 1, 0] = x.to(BF).cuda()
        q = torch.zeros((1, 2, 1, 64), dtype=BF, device="cuda")
        q[..., 0] = 1
        for count in (1, 500, 1499, 2999):
            got = paged.select_pages(q, bounds, table, ints([n * page]), count, page_size=page, first=0, last=0)
            want = choose(q, bounds, table, [n * page], page, count, 0, 0)
            assert torch.equal(got.pages, want[0]) and torch.equal(got.lens, want[1]), (kind, count)


@pytest.mark.parametrize("dt", [BF, HF])
def test_choice_over_the_types_range(mods, dt):
    """Subnormal bounds and queries, and the largest ones: the sums see every bit of them."""
    _lib, dec, paged = mods
    page, n = 16, 400
    table, P = pages_of([n * page], page, 4)
    tiny = torch.finfo(dt).smallest_normal * 2.0 ** (-7 if dt == BF else -10)
    for size, qs in ((tiny, 1.0), (tiny, tiny), (torch.finfo(dt).max / 2, 1.0), (torch.finfo(dt).max / 2, torch.finfo(dt).max / 2), (tiny, torch.finfo(dt).max / 2)):
        r = np.random.RandomState(1)
        lo = r.randint(1, 3, (P, 1, 64)) * -1.0 * size if size != tiny else r.randint(-9, 1, (P, 1, 64)) * size
        hi = r.randint(1, 3, (P, 1, 64)) * 1.0 * size if size != tiny else r.randint(1, 9, (P, 1, 64)) * size
        bounds = torch.from_numpy(np.stack([lo, hi], 2)).to(dt).cuda()
        q = torch.from_numpy(r.randint(-2, 3, (1, 2, 1, 64)) * 0.5 * qs if qs != tiny else r.randint(-3, 4, (1, 2, 1, 64)) * qs).to(dt).cuda()
        got = paged.select_pages(q, bounds, table, ints([n * page]), 33, page_size=page)
        want = choose(q, bounds, table, [n * page], page, 33, 1, 1)
        assert torch.equal(got.pages, want[0]), (size, qs)


def test_choice_with_bad_entries(mods):
    """Entries outside the pool are never chosen, whether first, last or between."""
    _lib, dec, paged = mods
    page, lens = 16, [50 * 16 - 3, 50 * 16, 4 * 16]
    table, P = pages_of(lens, page, 4)
    table[0, 0], table[0, 49], table[1, 5:45], table[2, 3] = P, -1, -7, 2 ** 31 - 1
    q, bounds = _gen((3, 4, 1, 128), 1, HF), spread(P, 2, 128, HF, 2)
    got = paged.select_pages(q, bounds, table, ints(lens), 12, page_size=page, first=2, last=2)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 310)
    want = choose(q, bounds, table, lens, page, 12, 2, 2)
    assert torch.equal(got.pages, want[0]) and torch.equal(got.lens, want[1])


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_choice_of_values_that_are_not_finite(mods, value):
    """Any choice is allowed, but it is a list of the sequence's pages with its length."""
    _lib, dec, paged = mods
    page, n = 16, 500
    table, P = pages_of([n * page, n * page], page, 4)
    bounds = spread(P, 2, 64, BF, 2)
    bounds[::3, 0, 1, 5] = value
    bounds[::7, 1, 0, 9] = -value
    q = _gen((2, 4, 1, 64), 1, BF)
    q[1, 0, 0, 3] = value
    got = paged.select_pages(q, bounds, table, ints([n * page, n * page]), 37, page_size=page)
    assert (got.lens == 37 * page).all()
    for b in range(2):
        at = {int(p): i for i, p in enumerate(table[b].tolist())}
        for g in range(2):
            order = [at[int(p)] for p in got.pages[b, g].tolist()]
            assert order == sorted(set(order)) and order[0] == 0 and order[-1] == n - 1


# --------------------------------------------------------------------------
# decode over lists
# --------------------------------------------------------------------------
def lists_of(lens, page, H_kv, seed, width=None):
    """A list of random pages for each (sequence, K/V head): lens [B][H_kv]."""
    lens = np.asarray(lens)
    need = -(-lens // page)
    P = int(need.max()) * 2 + 3
    width = max(1, int(need.max())) if width is None else width
    r = np.random.RandomState(seed)
    lists = np.full(lens.shape + (width,), -1, np.int32)
    for b in range(lens.shape[0]):
        for g in range(H_kv):
            lists[b, g, :need[b, g]] = r.permutation(P)[:need[b, g]]
    return ints(lists), P


def check_lists(o, lse, q, k, v, lists, lens, k_scale=1.0, v_scale=1.0, what=""):
    """Each K/V head as a batch of its own."""
    B, H, _, D = q.shape
    H_kv = k.shape[1]
    G = H // H_kv
    for g in range(H_kv):
        s = slice(g * G, (g + 1) * G)
        check(o[:, s].contiguous(), lse[:, s], q[:, s].contiguous(), k[:, g:g + 1].contiguous(), v[:, g:g + 1].contiguous(), lists[:, g], np.asarray(lens)[:, g],
              None, k_scale, v_scale, f"{what} head {g}")


@pytest.mark.parametrize("H,H_kv,D,page,qdt,kvdt", [
    (8, 4, 128, 64, BF, BF), (32, 8, 64, 16, HF, HF), (40, 2, 128, 256, BF, BF), (8, 8, 128, 64, HF, FP8), (40, 4, 128, 16, HF, FP8), (20, 1, 128, 128, BF, FP8),
    # the query-head kernel: a query head each, other 16-bit type, e4m3 heads of 64
    (4, 4, 128, 32, BF, BF), (6, 6, 64, 16, HF, HF), (8, 2, 128, 64, BF, HF), (8, 4, 64, 32, BF, FP8)])
def test_lists(mods, H, H_kv, D, page, qdt, kvdt):
    """Lists of different lengths for the heads of one sequence, empty ones among them."""
    _lib, dec, paged = mods
    r = np.random.RandomState(H)
    some = [0, 1, page - 1, page, page + 1, 127, 128, 129, 257, 700, 3001]
    lens = np.array([[some[r.randint(len(some))] for _ in range(H_kv)] for _ in range(9)] + [[0] * H_kv])
    lists, P = lists_of(lens, page, H_kv, 3)
    ks, vs = (0.05, 0.03) if kvdt == FP8 else (1.0, 1.0)
    q = _gen((10, H, 1, D), 1, qdt)
    k, v = (_gen((P, H_kv, page, D), 2 + i, torch.float32, 1 / s).to(kvdt) for i, s in enumerate((ks, vs)))
    o, lse = dec.pallas_flash_decoding(q, k, v, kv_lens=ints(lens), page_table=lists, return_lse=True, k_scale=ks, v_scale=vs)
    assert _lib.device_status() == (0, 0)
    check_lists(o, lse, q, k, v, lists, lens, ks, vs, "lists")
    # one list for all heads: the same bits as the table of the sequences
    same = lists[:, :1].expand(-1, H_kv, -1).contiguous()
    n = ints(lens[:, 0])
    a = paged.paged_decode(q, k, v, same, n.unsqueeze(1).expand(-1, H_kv).contiguous(), return_lse=True, k_scale=ks, v_scale=vs)
    check_lists(*a, q, k, v, same, np.repeat(lens[:, :1], H_kv, 1), ks, vs, "one list")


@pytest.mark.parametrize("B,H,H_kv,D,kvdt", [(1, 32, 8, 128, BF), (64, 16, 8, 64, BF), (300, 16, 8, 128, FP8), (2, 2, 1, 128, HF)])
def test_list_batches(mods, B, H, H_kv, D, kvdt):
    _lib, dec, paged = mods
    r = np.random.RandomState(B)
    lens = r.randint(0, 2049, (B, H_kv))
    lists, P = lists_of(lens, 32, H_kv, 3)
    q = _gen((B, H, 1, D), 1, HF if kvdt == HF else BF)
    k, v = (_gen((P, H_kv, 32, D), 2 + i).to(kvdt) for i in range(2))
    o, lse = paged.paged_decode(q, k, v, lists, ints(lens), return_lse=True)
    assert _lib.device_status() == (0, 0)
    check_lists(o, lse, q, k, v, lists, lens, what="batch")


# --------------------------------------------------------------------------
# a serving step
# --------------------------------------------------------------------------
@pytest.mark.parametrize("kvdt,D", [(BF, 128), (FP8, 128), (HF, 64)])
def test_a_step_with_selection(mods, kvdt, D):
    """Plan, append (which keeps the bounds), select and decode, captured once and replayed:
    bounds, choice and outputs are those of the cache's contents at each step."""
    from pallas_flash.ops.rotary import rotary_frequencies
    _lib, dec, paged = mods
    B, H, H_kv, page, count = 4, 8, 2, 16, 6
    ks, vs = (0.05, 0.03) if kvdt == FP8 else (1.0, 1.0)
    qdt = HF if kvdt == HF else BF
    cache = paged.DevicePagedKVCache(B, H_kv, D, num_pages=80, page_size=page, max_seq_len=640, dtype=kvdt, k_scale=ks, v_scale=vs, bounds=True)
    f = rotary_frequencies(D)
    split = lambda x: (x[:, :H], x[:, H:H + H_kv], x[:, H + H_kv:])    # noqa: E731
    prompt = [40, 0, 300, 15]
    x = _gen((360, H + 2 * H_kv, D), 1, qdt)
    cache.append(*split(x), cache.plan(ints(prompt), num_tokens=360), f)
    new = torch.ones(B, dtype=torch.int32, device="cuda")
    x = torch.zeros((B, H + 2 * H_kv, D), dtype=qdt, device="cuda")
    state = (cache.page_table, cache.kv_lens, cache.free_ring, cache.cursor, cache.bounds)
    saved = [t.clone() for t in state]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = cache.append(*split(x), cache.plan(new, num_tokens=B), f)
        chosen = cache.select(q, count, first=1, last=2)
        o, lse = cache.decode(q, pages=chosen, return_lse=True)
    for t, s in zip(state, saved):
        t.copy_(s)
    held = list(prompt)
    for n in range(20):
        x.copy_(_gen(x.shape, 100 + n, qdt))
        graph.replay()
        held = [m + 1 for m in held]
        for b in range(B):
            for i in range(-(-held[b] // page)):
                p, rows = int(cache.page_table[b, i]), min(page, held[b] - i * page)
                y = wide(cache.k_pool[p])[:, :rows]
                assert torch.equal(cache.bounds[p].double(), torch.stack([y.amin(1), y.amax(1)], 1)), (n, b, i)
        want = choose(q.unsqueeze(2), cache.bounds, cache.page_table, held, page, count, 1, 2)
        assert torch.equal(chosen.pages, want[0]) and torch.equal(chosen.lens, want[1])
        check_lists(o, lse, q.unsqueeze(2), cache.k_pool, cache.v_pool, chosen.pages, chosen.lens.cpu().numpy(), ks, vs, f"step {n}")
    assert _lib.device_status() == (0, 0)
    # every page chosen is the whole cache
    a = cache.decode(q, pages=cache.select(q, 40), return_lse=True)
    check(*a, q.unsqueeze(2), cache.k_pool, cache.v_pool, cache.page_table, held, None, ks, vs, "all pages")


def test_streams_and_graphs(mods):
    """Two captured selections replayed at once on two streams, and calls on a stream of their own."""
    _lib, dec, paged = mods
    lens = [900, 40, 3000]
    table, P = pages_of(lens, 16, 4)
    n = ints(lens)
    sets = []
    for i in range(2):
        q, bounds = _gen((3, 8, 1, 128), i, BF), spread(P, 2, 128, BF, 10 + i)
        k, v = _gen((P, 2, 16, 128), 20 + i, BF), _gen((P, 2, 16, 128), 30 + i, BF)
        first = paged.select_pages(q, bounds, table, n, 9, page_size=16)
        want = [t.clone() for t in (*first, *paged.paged_decode(q, k, v, *first, return_lse=True))]
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            s = paged.select_pages(q, bounds, table, n, 9, page_size=16)
            got = (*s, *paged.paged_decode(q, k, v, *s, return_lse=True))
        sets.append((graph, stream, got, want, (q, bounds, k, v)))
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, stream, *_ in sets:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for graph, stream, got, want, _ in sets:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert _lib.device_status() == (0, 0)


def test_refusals(mods):
    _lib, dec, paged = mods
    q, bounds = _gen((2, 4, 1, 64), 1, BF), torch.zeros((5, 2, 2, 64), dtype=BF, device="cuda")
    table, n = torch.zeros((2, 3), dtype=torch.int32, device="cuda"), ints([5, 6])
    k = torch.zeros((5, 2, 16, 64), dtype=BF, device="cuda")
    good = dict(count=2, page_size=16)
    for a, kw in [((q[:, :3], bounds, table, n), good), ((q.float(), bounds, table, n), good), ((q, bounds[:, :, :1], table, n), good),
                  ((q, bounds.float(), table, n), good), ((q, bounds, table.long(), n), good), ((q, bounds, table, n[:1]), good),
                  ((q, bounds, table.t().contiguous().t(), n), good), ((q, bounds.cpu(), table, n), good), ((q, bounds, table.cpu(), n), good),
                  ((q, bounds, table, n), dict(count=0, page_size=16)), ((q, bounds, table, n), dict(count=2, page_size=16, first=2)),
                  ((q, bounds, table, n), dict(count=2, page_size=16, first=-1))]:
        with pytest.raises(ValueError):
            paged.select_pages(*a, **kw)
    for kw in (dict(count=2, page_size=24), dict(count=2, page_size=8)):
        with pytest.raises(_lib.PuError):
            paged.select_pages(q, bounds, table, n, **kw)
    with pytest.raises(_lib.PuError):
        paged.select_pages(q, bounds, torch.zeros((2, 24577), dtype=torch.int32, device="cuda"), n, 2, page_size=16)
    slots = ints([0, 1])
    for a in [(k, slots.long(), bounds), (k, slots, bounds.half()), (k[:4], slots, bounds), (k.float(), slots, bounds), (k.transpose(0, 1), slots, bounds),
              (k, slots.cpu(), bounds), (k, ints([0, 1, 2, 3])[::2], bounds), (k.to(FP8), slots, bounds)]:
        with pytest.raises(ValueError):
            paged.page_bounds(*a)
    lists = torch.zeros((2, 2, 3), dtype=torch.int32, device="cuda")
    for t, m in [(lists[:, :1].contiguous(), n), (lists, n), (lists.long(), n.view(2, 1).repeat(1, 2)), (lists, torch.zeros((2, 3), dtype=torch.int32, device="cuda"))]:
        with pytest.raises(ValueError):
            paged.paged_decode(q, k, k, t, m)
    cache = paged.DevicePagedKVCache(2, 2, 64, num_pages=5, page_size=16, max_seq_len=48)
    with pytest.raises(ValueError):
        cache.select(q, 2)
