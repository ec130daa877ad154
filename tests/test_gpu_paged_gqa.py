"""Paged decode with grouped heads and e4m3 pools (pu_decode_paged_gqa), and the
serving step it belongs to, against the formula in 64 bits.

Tolerance of an output, element by element: half a step of bf16 (2^-8 of the
value), plus what the weights p_j = exp(s_j - lse) are off by, times
A = sum_j p_j |v_j|:
  - each p is rounded once to its operand type: 2^-8 for bf16, 2^-11 for f16,
    and for e4m3 pools three parts of 4 bits, 2^-12;
  - a score is off by e = 2^-24 (D + 16) scale sum_i |q_i k_i| (fp32 sums) plus,
    for e4m3 pools, 2^-17 max|q| scale sum_i |k_i| (what the parts of q leave
    of elements far below the largest);
    with ex2 (2 ulp) and the sums of p, 2 e + 2^-19 relative.
  - a p below its type's smallest step may vanish: at most 2^-25 of the
    largest for f16 and 2^-26 for e4m3 each.
lse is off by at most the largest e plus 2^-19.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def mods(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    from pallas_flash import _lib
    from pallas_flash.kernels import decoding, paged
    _lib.device_status()
    return _lib, decoding, paged


def _gen(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def pages_of(lens, page, seed, spare=2, width=None):
    """A page table with pages in random order."""
    r = np.random.RandomState(seed)
    need = -(-np.asarray(lens) // page)
    P = int(need.sum()) + spare
    order = r.permutation(P).astype(np.int32)
    width = max(1, int(need.max())) if width is None else width
    table = np.full((len(lens), width), -1, np.int32)
    table[np.arange(width)[None] < need[:, None]] = order[:need.sum()]
    return torch.from_numpy(table).cuda(), P


def dense(pool, table, b, n, scale):
    """Keys or values [H_kv, n, D] fp64 of sequence b."""
    page = pool.shape[2]
    at = table[b, :-(-n // page)].long()
    x = pool.view(torch.uint8)[at].view(pool.dtype).double() if pool.dtype == FP8 else pool[at].double()
    return x.transpose(0, 1).flatten(1, 2)[:, :n] * scale


def check(o, lse, q, k_pool, v_pool, table, lens, scale=None, k_scale=1.0, v_scale=1.0, what=""):
    B, H, _, D = q.shape
    H_kv = k_pool.shape[1]
    G = H // H_kv
    scale = 1 / math.sqrt(D) if scale is None else scale
    f8 = k_pool.dtype == FP8
    rnd = 2.0 ** -12 if f8 else 2.0 ** -8 if k_pool.dtype == torch.bfloat16 else 2.0 ** -11
    lost = 2.0 ** -26 if f8 else 0.0 if k_pool.dtype == torch.bfloat16 else 2.0 ** -25
    assert o.dtype == torch.bfloat16 and o.shape == q.shape and lse.shape == (B, H)
    for b, n in enumerate(np.asarray(lens).tolist()):
        if n == 0:
            assert (o[b] == 0).all() and (lse[b] == -math.inf).all(), f"{what}: empty sequence {b}"
            continue
        k, v = dense(k_pool, table, b, n, k_scale), dense(v_pool, table, b, n, v_scale)
        x = q[b, :, 0].double().view(H_kv, G, D)
        s = scale * x @ k.transpose(1, 2)
        e = 2.0 ** -24 * (D + 16) * scale * (x.abs() @ k.abs().transpose(1, 2))
        if f8:
            e = e + 2.0 ** -17 * scale * x.abs().amax(-1, keepdim=True) * k.abs().sum(-1).unsqueeze(1)
        l = torch.logsumexp(s, -1, keepdim=True)
        p = (s - l).exp()
        want = (p @ v).reshape(H, D)
        tol = 2.0 ** -8 * want.abs() + ((p * (rnd + 2 * e + 2.0 ** -19) + lost * p.amax(-1, keepdim=True)) @ v.abs()).reshape(H, D)
        err = (o[b, :, 0].double() - want).abs()
        assert (err <= tol).all(), f"{what}: sequence {b} of {n}, worst {float((err / tol).max()):.2f} of the tolerance"
        off = (lse[b].double() - l.reshape(H)).abs()
        assert (off <= e.amax(-1).reshape(H) + 2.0 ** -19 + 2.0 ** -23 * l.reshape(H).abs()).all(), f"{what}: lse of sequence {b}"


def make(B, H, H_kv, D, page, lens, qdt, kvdt, seed=0, k_scale=1.0, v_scale=1.0, width=None):
    table, P = pages_of(lens, page, seed, width=width)
    q = _gen((B, H, 1, D), seed + 1, qdt)
    k = _gen((P, H_kv, page, D), seed + 2, torch.float32, 1 / k_scale).to(kvdt)
    v = _gen((P, H_kv, page, D), seed + 3, torch.float32, 1 / v_scale).to(kvdt)
    return q, k, v, table, torch.tensor(np.asarray(lens), dtype=torch.int32, device="cuda")


BF, HF = torch.bfloat16, torch.float16
CASES = [
    # H, H_kv, D, page, q, cache
    (8, 4, 128, 64, BF, BF), (32, 8, 128, 16, HF, HF), (6, 2, 128, 32, BF, BF), (16, 1, 128, 128, HF, HF),
    (40, 2, 128, 256, BF, BF), (33, 1, 128, 64, HF, HF), (16, 2, 64, 16, BF, BF), (10, 5, 64, 64, HF, HF),
    (24, 1, 64, 512, BF, BF), (8, 8, 128, 64, BF, FP8), (8, 2, 128, 16, HF, FP8), (20, 1, 128, 128, BF, FP8),
    (64, 8, 128, 32, HF, FP8),
    # the query-head kernel: other 16-bit type, e4m3 heads of 64, scales on a 16-bit cache
    (8, 2, 128, 64, BF, HF), (8, 2, 64, 16, HF, BF), (8, 4, 64, 32, BF, FP8),
]


@pytest.mark.parametrize("H,H_kv,D,page,qdt,kvdt", CASES)
def test_lengths(mods, H, H_kv, D, page, qdt, kvdt):
    """Lengths from none to several thousand, at the edges of pages and tiles."""
    _lib, dec, paged = mods
    lens = [0, 1, page - 1, page, page + 1, 127, 128, 129, 255, 256, 257, 700, 5000, 0, 3001]
    ks, vs = (0.05, 0.03) if kvdt == FP8 else (1.0, 1.0)
    q, k, v, table, n = make(len(lens), H, H_kv, D, page, lens, qdt, kvdt, 7, ks, vs)
    o, lse = dec.pallas_flash_decoding(q, k, v, kv_lens=n, page_table=table, return_lse=True, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, None, ks, vs, "lengths")
    # the same bits again, and without the lse
    again = dec.pallas_flash_decoding(q, k, v, kv_lens=n, page_table=table, k_scale=ks, v_scale=vs)
    assert torch.equal(o, again)


@pytest.mark.parametrize("B,length", [(1, 1), (1, 130), (1, 60000), (2, 33333), (3, 127), (150, 300), (500, 129)])
@pytest.mark.parametrize("D,kvdt", [(128, BF), (64, BF), (128, FP8)])
def test_batches(mods, B, length, D, kvdt):
    """Few long sequences (many CTAs on one) to many short ones (many on one CTA)."""
    _lib, dec, paged = mods
    r = np.random.RandomState(B)
    lens = [length] if B == 1 else r.randint(length // 2, length + 1, B)
    ks, vs = (0.02, 0.02) if kvdt == FP8 else (1.0, 1.0)
    q, k, v, table, n = make(B, 8, 2, D, 32, lens, BF, kvdt, 3, ks, vs)
    o, lse = paged.paged_decode(q, k, v, table, n, return_lse=True, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, None, ks, vs, "batch")


def test_matches_dense_grouped_decode(mods):
    """The dense grouped kernel on the cache that the pages describe: both
    within their rounding of the same values."""
    _lib, dec, paged = mods
    B, H, H_kv, N, D, page = 2, 16, 4, 2000, 128, 64
    q, k, v = (_gen(s, i, HF) for i, s in enumerate([(B, H, 1, D), (B, H_kv, N, D), (B, H_kv, N, D)]))
    lens = [2000, 777]
    cache = paged.PagedKVCache.from_dense(k, v, lens, page_size=page, shuffle_seed=5)
    o, lse = cache.decode(q, return_lse=True)
    check(o, lse, q, cache.k_pool, cache.v_pool, cache.page_table, lens)
    od, ld = dec.pallas_flash_decoding(q, k, v, kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), return_lse=True)
    assert (o.float() - od.float()).abs().max() <= 2.0 ** -8 * od.float().abs().max() + 2.0 ** -11 * 4
    assert (lse - ld).abs().max() <= 2.0 ** -16


@pytest.mark.parametrize("D,kvdt", [(128, BF), (64, HF), (128, FP8)])
def test_stale_values_never_count(mods, D, kvdt):
    """NaN in rows behind a length, in pages of nobody and in pages of others."""
    _lib, dec, paged = mods
    lens, page = [5, 130, 64, 1, 300], 64
    q, k, v, table, n = make(5, 8, 2, D, page, lens, HF if kvdt == HF else BF, kvdt, 11)
    nan = torch.full((1,), math.nan, device="cuda").to(kvdt)
    for pool in (k, v):
        raw = pool.view(torch.uint8) if kvdt == FP8 else pool
        mark = nan.view(torch.uint8) if kvdt == FP8 else nan
        keep = raw.clone()
        raw[:] = mark
        for b, m in enumerate(lens):
            for i in range(-(-m // page)):
                pg, rows = int(table[b, i]), min(page, m - i * page)
                raw[pg, :, :rows] = keep[pg, :, :rows]
    o, lse = paged.paged_decode(q, k, v, table, n, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="stale")


@pytest.mark.parametrize("D,page,kvdt", [(128, 16, BF), (64, 32, BF), (128, 64, FP8)])
def test_invalid_entries_are_left_out(mods, D, page, kvdt):
    """Entries outside the pool are reported and their tokens left out: a page
    inside a tile, a whole tile, a whole sequence."""
    _lib, dec, paged = mods
    lens = [400, 400, page, 300]
    q, k, v, table, n = make(4, 4, 2, D, page, lens, BF, kvdt, 13, 1.0, 1.0)
    P = k.shape[0]
    bad = table.clone()
    drop = {0: [1], 1: list(range(0, 256 // page)), 2: [0]}
    marks = [P, -1, P + 12345, -(1 << 31), (1 << 31) - 1]
    for b, entries in drop.items():
        for i, e in enumerate(entries):
            bad[b, e] = marks[i % len(marks)]
    o, lse = paged.paged_decode(q, k, v, bad, n, return_lse=True)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 302)
    assert (o[2] == 0).all() and (lse[2] == -math.inf).all()
    for b in (0, 1, 3):
        # the sequence without those tokens, packed into a table of its own
        rest = [e for e in range(-(-lens[b] // page)) if e not in drop.get(b, [])]
        m = sum(min(page, lens[b] - e * page) for e in rest)
        check(o[b:b + 1], lse[b:b + 1], q[b:b + 1], k, v, table[b:b + 1, rest], [m], what=f"invalid {b}")


@pytest.mark.parametrize("kvdt", [BF, HF, FP8])
def test_growing_scores_and_long_tails(mods, kvdt):
    """Scores that keep growing along the sequence (the maximum moves in every
    tile), and one token that outweighs each of 20000 others by 2^14 while
    they outweigh it together."""
    _lib, dec, paged = mods
    D, page, H, H_kv, n = 128, 64, 4, 2, 20000
    qdt = HF if kvdt == HF else BF
    table, P = pages_of([n, n], page, 1)
    q = torch.zeros((2, H, 1, D), device="cuda")
    q[..., 0] = math.sqrt(D)
    k = torch.zeros((P, H_kv, page, D), device="cuda")
    v = _gen((P, H_kv, page, D), 5) * 0.5 + 1.0
    pos = torch.arange(n, device="cuda")
    at = table[:, pos // page].long()
    k[at[0], :, pos % page, 0] = (pos.float() / n * 20.0).view(-1, 1)
    k[at[1], :, pos % page, 0] = 0.0
    k[at[1][7], :, 7 % page, 0] = 14 * math.log(2.0)
    v[at[1][7], :, 7 % page] = -1.0
    q, k, v = q.to(qdt), k.to(kvdt), v.to(kvdt)
    lens = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    o, lse = paged.paged_decode(q, k, v, table, lens, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, [n, n], what="tails")


def test_every_e4m3_code(mods):
    """One token of each finite code as key and as value."""
    _lib, dec, paged = mods
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(FP8)
    codes = codes[torch.isfinite(codes.float())]
    n, D, page = len(codes), 128, 16
    table, P = pages_of([n, 1], page, 1)
    k = torch.zeros((P, 1, page, D), device="cuda").to(FP8)
    v = torch.zeros((P, 1, page, D), device="cuda").to(FP8)
    for i in range(n):
        pg, r = int(table[0, i // page]), i % page
        k.view(torch.uint8)[pg, 0, r, :4] = codes[i].view(torch.uint8)
        v.view(torch.uint8)[pg, 0, r] = codes.view(torch.uint8)[(i + torch.arange(D, device="cuda")) % n]
    for qdt in (BF, HF):
        q = _gen((2, 8, 1, D), 3, qdt)
        o, lse = paged.paged_decode(q, k, v, table, torch.tensor([n, 1], dtype=torch.int32, device="cuda"),
                                    return_lse=True, k_scale=0.004)
        check(o, lse, q, k, v, table, [n, 1], None, 0.004, 1.0, f"codes {qdt}")


@pytest.mark.parametrize("qdt,power", [(BF, 120), (BF, -120), (HF, 11), (HF, -14)])
def test_queries_of_any_size(mods, qdt, power):
    """e4m3 pools: queries near both ends of their type's range, with a k_scale that
    brings the scores back (a power of two: nothing is rounded by it)."""
    _lib, dec, paged = mods
    lens = [1, 129, 700]
    q, k, v, table, n = make(3, 8, 2, 128, 32, lens, torch.float32, FP8, 11)
    q = (q.clamp(-4, 4) * 2.0 ** power).to(qdt)
    assert torch.isfinite(q).all()
    ks = 2.0 ** -power
    o, lse = paged.paged_decode(q, k, v, table, n, return_lse=True, k_scale=ks)
    torch.cuda.synchronize()
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, None, ks, 1.0, f"2^{power}")


def test_layouts_and_clamps(mods):
    """A strided and an unaligned q, a table wider than needed, lengths behind
    the table and below zero, any scale."""
    _lib, dec, paged = mods
    lens, page = [200, 90], 64
    q, k, v, table, n = make(2, 8, 2, 128, page, lens, BF, BF, 17, width=9)
    want = paged.paged_decode(q, k, v, table, n, sm_scale=0.3, return_lse=True)
    check(*want, q, k, v, table, lens, 0.3)
    off = torch.empty(q.numel() + 1, dtype=BF, device="cuda")[1:].view(q.shape).copy_(q)
    strided = torch.zeros((2, 1, 8, 128), dtype=BF, device="cuda").transpose(1, 2).copy_(q)
    for x in (off, strided):
        assert torch.equal(paged.paged_decode(x, k, v, table, n, sm_scale=0.3), want[0])
    few = table[:, :2].contiguous()
    over = paged.paged_decode(q, k, v, few, torch.tensor([1 << 20, -7], dtype=torch.int32, device="cuda"), return_lse=True)
    check(*over, q, k, v, few, [128, 0])
    assert _lib.device_status() == (0, 0)


def test_offsets_behind_32_bits(mods):
    """A pool of more than 2^32 bytes and 2^31 elements, its last pages in use."""
    _lib, dec, paged = mods
    H_kv, page, D = 8, 256, 128
    P = (1 << 31) // (H_kv * page * D) + 40
    lens = [900, 3000]
    q = _gen((2, 16, 1, D), 1, BF)
    k = torch.empty((P, H_kv, page, D), dtype=BF, device="cuda")
    v = torch.empty_like(k)
    need = [-(-n // page) for n in lens]
    table = torch.full((2, max(need)), -1, dtype=torch.int32, device="cuda")
    at = P - 1
    for b in range(2):
        for i in range(need[b]):
            table[b, i] = at
            k[at], v[at] = _gen((H_kv, page, D), at, BF), _gen((H_kv, page, D), at + 1, BF)
            at -= 1
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    o, lse = paged.paged_decode(q, k, v, table, n, return_lse=True)
    check(o, lse, q, k, v, table, lens, what="far pages")
    # and written there
    T = 5
    x = _gen((T, 16 + 2 * H_kv, D), 3, BF)
    slots = torch.tensor([(P - 1) * page + 7, (P - 2) * page + 255, -1, (P - 3) * page, (P - 4) * page + 100],
                         dtype=torch.int32, device="cuda")
    f = torch.ones(64, dtype=torch.float64, device="cuda")
    paged.qk_norm_rope_append(x[:, :16], x[:, 16:24], x[:, 24:], f, torch.zeros(T, dtype=torch.int32, device="cuda"), slots, k, v)
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            assert torch.equal(k[s // page, :, s % page], x[t, 16:24]) and torch.equal(v[s // page, :, s % page], x[t, 24:])


def test_two_graphs_at_once(mods):
    """Two captured decodes replayed on two streams at the same time, beside an
    eager one: none sees another's scratch."""
    _lib, dec, paged = mods
    sets, graphs, outs = [], [], []
    for i in range(2):
        s = make(3, 16, 2, 128, 64, [3000 + i, 50, 9000], BF, BF, 40 + i)
        sets.append(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(paged.paged_decode(s[0], s[1], s[2], s[3], s[4], return_lse=True))
        graphs.append(g)
    want = [paged.paged_decode(*s, return_lse=True) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = paged.paged_decode(*sets[0], return_lse=True)
    torch.cuda.synchronize()
    for got, w in zip(outs + [eager], want + [want[0]]):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
    assert _lib.device_status() == (0, 0)


def test_threads_and_streams(mods):
    """Decodes of different shapes from several host threads, each on its own
    stream with its own scratch."""
    import threading
    _lib, dec, paged = mods
    shapes = [(3, 16, 2, 128, 64, [3000, 50, 9000], BF, BF), (20, 8, 2, 64, 16, list(range(0, 400, 20)), HF, HF),
              (2, 8, 8, 128, 32, [700, 10000], BF, FP8), (1, 32, 4, 128, 64, [20000], HF, HF)]
    sets = [make(*a[:8], seed=70 + i) for i, a in enumerate(shapes)]
    want = [paged.paged_decode(*x, return_lse=True) for x in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(40):
                o, lse = paged.paged_decode(*sets[i], return_lse=True)
                if not (torch.equal(o, want[i][0]) and torch.equal(lse, want[i][1])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not bad and _lib.device_status() == (0, 0)


def test_shared_pages(mods):
    """Sequences that share their first pages (a common prompt)."""
    _lib, dec, paged = mods
    lens, page = [300, 420, 256], 64
    q, k, v, table, n = make(3, 8, 2, 128, page, lens, BF, BF, 80, width=8)
    table[1, :4] = table[0, :4]
    table[2, :4] = table[0, :4]
    o, lse = paged.paged_decode(q, k, v, table, n, return_lse=True)
    check(o, lse, q, k, v, table, lens, what="shared")
    assert _lib.device_status() == (0, 0)


# ---------------------------------------------------------------------------
# norm, rotation and cache write
# ---------------------------------------------------------------------------
def _turned(x, w, f, pos, eps=1e-6):
    """Norm and rotation (halves) of x [T, H, D] in 64 bits, and |a| + |b| of each pair."""
    x = x.double()
    R = 2 * f.numel()
    n = x if w is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    t = (pos.double().unsqueeze(-1) * f).unsqueeze(1)
    a, b, c = n[..., :R // 2], n[..., R // 2:R], n[..., R:]
    m = a.abs() + b.abs()
    return torch.cat([a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin(), c], -1), torch.cat([m, m, c.abs()], -1)


@pytest.mark.parametrize("H,H_kv,D,R,page,dt,pool", [
    (8, 2, 128, 128, 64, BF, BF), (5, 5, 64, 32, 16, HF, HF), (16, 1, 128, 64, 128, BF, HF), (4, 2, 96, 96, 32, torch.float32, BF),
    (8, 8, 128, 128, 32, BF, FP8), (6, 3, 64, 64, 16, HF, FP8), (3, 1, 16, 16, 4096, torch.float32, FP8)])
@pytest.mark.parametrize("T", [1, 77, 900])
def test_append(mods, H, H_kv, D, R, page, dt, pool, T):
    """q, keys and values of packed tokens in scattered slots; padding rows and
    all other places of the pools stay as they were.  Tolerance of a 16-bit
    pool: half a step and 32 roundings of 2^-24 of the pair (the norm's and
    rotation's bound).  An e4m3 pool: half a step there is 2^-4 of the value,
    or 2^-10 below its normal range, plus the same 32 roundings."""
    _lib, dec, paged = mods
    P = -(-T // page) + 3
    ks, vs = (0.011, 0.03) if pool == FP8 else (1.0, 1.0)
    r = np.random.RandomState(T)
    slots = r.permutation(P * page)[:T].astype(np.int32)
    slots[r.rand(T) < 0.1] = -1 - r.randint(0, 3)
    x = _gen((T, (H + 2 * H_kv) * D), 1, dt, 2.0)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in x.split([H * D, H_kv * D, H_kv * D], -1))
    wq, wk = (1 + 0.1 * _gen((D,), s) for s in (2, 3))
    f = torch.pow(torch.tensor(1e4, dtype=torch.float64), -torch.arange(0, R, 2, dtype=torch.float64) / R).cuda()
    pos = torch.from_numpy(r.randint(0, 100000, T)).cuda()
    before = [_gen((P, H_kv, page, D), s).to(pool) for s in (5, 6)]
    kp, vp = (t.clone() for t in before)
    got = paged.qk_norm_rope_append(q, k, v, f, pos, torch.from_numpy(slots).cuda(), kp, vp, q_weight=wq, k_weight=wk,
                                    k_scale=ks, v_scale=vs)
    assert _lib.device_status() == (0, 0)
    U = 2.0 ** -24
    yq, mq = _turned(q, wq, f, pos)
    # below a type's smallest normal value (f16: 2^-14) its steps no longer
    # shrink with the value: half the smallest one, tiny * eps / 2 (f16: 2^-25)
    small = torch.finfo(dt).tiny * torch.finfo(dt).eps / 2
    tol = torch.finfo(dt).eps / 2 * yq.abs() + 32 * U * mq
    off = (got.double() - yq).abs()
    assert (yq[off > tol].abs() < torch.finfo(dt).tiny).all() and (off <= tol + small).all()
    yk, mk = _turned(k, wk, f, pos)
    live = torch.from_numpy(slots >= 0).cuda()
    at = torch.from_numpy(slots[slots >= 0]).long().cuda()
    raw = lambda t: t.view(torch.uint8) if pool == FP8 else t    # noqa: E731
    for p, old, y, m, c in ((kp, before[0], yk, mk, ks), (vp, before[1], v.double(), v.double().abs(), vs)):
        place = raw(p)[at // page, :, at % page]
        place = place.view(FP8).double() if pool == FP8 else place.double()
        want, mag = y[live] / c, m[live] / c
        if pool == FP8:
            want = want.clamp(-448, 448)
            tol = torch.maximum(2.0 ** -4 * want.abs(), torch.tensor(2.0 ** -10, device="cuda", dtype=torch.float64)) + 34 * U * mag
        else:
            tol = torch.finfo(pool).eps / 2 * want.abs() + 32 * U * mag + torch.finfo(pool).tiny * torch.finfo(pool).eps
        assert ((place - want).abs() <= tol).all()
        rest = torch.ones(p.shape[0] * page, dtype=torch.bool, device="cuda")
        rest[at] = False
        flat = lambda t: raw(t).transpose(1, 2).reshape(-1, H_kv, D)   # noqa: E731
        assert torch.equal(flat(p)[rest].view(torch.uint8), flat(old)[rest].view(torch.uint8))


def test_append_reports_slots_past_the_pool(mods):
    _lib, dec, paged = mods
    x = _gen((3, 4, 64), 1, BF)
    kp = torch.zeros((2, 1, 16, 64), dtype=BF, device="cuda")
    vp = torch.zeros_like(kp)
    f = torch.ones(32, dtype=torch.float64, device="cuda")
    slots = torch.tensor([32, 5, (1 << 31) - 1], dtype=torch.int32, device="cuda")
    q = paged.qk_norm_rope_append(x[:, :2], x[:, 2:3], x[:, 3:], f, torch.zeros(3, dtype=torch.int32, device="cuda"), slots, kp, vp)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 306)
    assert torch.equal(q, x[:, :2]) and torch.equal(vp[0, 0, 5], x[1, 3])
    assert (kp != 0).any(-1).sum() == 1


def test_append_axes_and_interleaved(mods):
    """Positions with axes, neighbouring pairs: the training form's own values."""
    from pallas_flash.ops.rotary import qk_norm_rope, rotary_frequencies
    _lib, dec, paged = mods
    T, H, H_kv, D = 50, 6, 2, 64
    x = _gen((T, H + 2 * H_kv, D), 1, BF)
    w = 1 + 0.1 * _gen((D,), 2)
    f = rotary_frequencies(D)
    pos = torch.randint(0, 500, (3, T), device="cuda", dtype=torch.int32)
    kp = torch.zeros((4, H_kv, 16, D), dtype=BF, device="cuda")
    vp = torch.zeros_like(kp)
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    for inter in (False, True):
        q = paged.qk_norm_rope_append(x[:, :H], x[:, H:H + H_kv], x[:, H + H_kv:], f, pos, slots, kp, vp, q_weight=w, k_weight=w,
                                      sections=(8, 12, 12), interleaved=inter)
        t = x.transpose(0, 1).unsqueeze(0)
        qr, kr = qk_norm_rope(t[:, :H], t[:, H:H + H_kv], f, pos, q_weight=w, k_weight=w, sections=(8, 12, 12), interleaved=inter)
        assert torch.equal(q, qr[0].transpose(0, 1))
        flat = kp.transpose(1, 2).reshape(-1, H_kv, D)
        assert torch.equal(flat[:T], kr[0].transpose(0, 1))


# ---------------------------------------------------------------------------
# the serving step
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kvdt", [BF, FP8])
@pytest.mark.parametrize("captured", [False, True])
def test_serving_chain(mods, kvdt, captured):
    """Prompts, then steps of one token with a sequence that ends and one that
    takes its place: plan, norm + rotation + cache write, decode, against
    attention over everything appended so far in 64 bits.  The decode's
    tolerance applies to the cache as it was stored."""
    from pallas_flash.ops.rotary import rotary_frequencies
    _lib, dec, paged = mods
    B, H, H_kv, D, page = 4, 8, 2, 128, 16
    ks, vs = (0.05, 0.03) if kvdt == FP8 else (1.0, 1.0)
    cache = paged.DevicePagedKVCache(B, H_kv, D, num_pages=60, page_size=page, max_seq_len=400, dtype=kvdt, k_scale=ks, v_scale=vs)
    f = rotary_frequencies(D)
    wq, wk = (1 + 0.1 * _gen((D,), s) for s in (2, 3))
    kw = dict(q_weight=wq, k_weight=wk)
    r = np.random.RandomState(0)
    new = torch.tensor([100, 0, 17, 250], dtype=torch.int32, device="cuda")
    T = 367 + 5
    x = _gen((T, H + 2 * H_kv, D), 1, BF)
    plan = cache.plan(new, num_tokens=T)
    cache.append(x[:, :H], x[:, H:H + H_kv], x[:, H + H_kv:], plan, f, **kw)
    seqs = {b: x[(plan.seq_ids == b)] for b in range(B)}
    lens = [100, 0, 17, 250]

    one = torch.ones(B, dtype=torch.int32, device="cuda")
    release = torch.zeros(B, dtype=torch.bool, device="cuda")
    xs = torch.zeros((B, H + 2 * H_kv, D), dtype=BF, device="cuda")

    def step():
        p = cache.plan(one, num_tokens=B, release=release)
        q = cache.append(xs[:, :H], xs[:, H:H + H_kv], xs[:, H + H_kv:], p, f, **kw)
        return cache.decode(q, return_lse=True) + (q,)

    if captured:
        saved = [t.clone() for t in (cache.page_table, cache.kv_lens, cache.free_ring, cache.cursor)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for t, s in zip((cache.page_table, cache.kv_lens, cache.free_ring, cache.cursor), saved):
            t.copy_(s)
    for i in range(24):
        xs.copy_(_gen((B, H + 2 * H_kv, D), 100 + i, BF))
        release.zero_()
        if i == 9:
            release[3] = True
        if captured:
            graph.replay()
        else:
            out = step()
        for b in range(B):
            if i == 9 and b == 3:
                seqs[b], lens[b] = xs[b:b + 1].clone(), 1
            else:
                seqs[b], lens[b] = torch.cat([seqs[b], xs[b:b + 1]]), lens[b] + 1
        assert cache.kv_lens.tolist() == lens
        o, lse, q = out
        check(o, lse, q.unsqueeze(2), cache.k_pool, cache.v_pool, cache.page_table, lens, None, ks, vs, f"step {i}")
    assert _lib.device_status() == (0, 0)
    # what is stored is what was appended
    half = 2.0 ** -4 if kvdt == FP8 else 2.0 ** -8
    for b in range(B):
        k = dense(cache.k_pool, cache.page_table, b, lens[b], ks).transpose(0, 1)
        v = dense(cache.v_pool, cache.page_table, b, lens[b], vs).transpose(0, 1)
        want, m = _turned(seqs[b][:, H:H + H_kv], wk, f, torch.arange(lens[b], device="cuda"))
        for got, w, mag, c in ((k, want, m, ks), (v, seqs[b][:, H + H_kv:].double(), None, vs)):
            mag = w.abs() if mag is None else mag
            assert ((got - w).abs() <= half * w.abs() + (2.0 ** -10 * c if kvdt == FP8 else 0) + 34 * 2.0 ** -24 * mag).all()


@pytest.mark.parametrize("B,H,H_kv,D,kvdt", [(1024, 65, 1, 64, BF), (2100, 32, 8, 128, BF), (1100, 64, 4, 128, FP8)])
def test_batches_of_many_heads(mods, B, H, H_kv, D, kvdt):
    """More than 65535 (sequence, head) pairs: the tensor-core kernel counts per CTA."""
    _lib, dec, paged = mods
    assert B * H > 65535
    lens = np.random.RandomState(B).randint(0, 40, B)
    lens[[0, 17, B - 1]] = [300, 0, 129]
    ks, vs = (0.02, 0.02) if kvdt == FP8 else (1.0, 1.0)
    q, k, v, table, n = make(B, H, H_kv, D, 16, lens, BF, kvdt, 3, ks, vs)
    o, lse = paged.paged_decode(q, k, v, table, n, return_lse=True, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, None, ks, vs, "many heads")


def test_captured_decodes_clear_what_they_count_in(mods, monkeypatch):
    """Captured decodes of every kernel on scratch full of garbage: each replay clears the
    counters that it needs (4 bytes for a sequence's head or an SM) and no more, and is right."""
    _lib, dec, paged = mods
    q, k, v, table, n = make(3, 16, 4, 128, 64, [900, 5, 3000], BF, BF, 21)
    k8, v8 = k.to(FP8), v.to(FP8)
    dk, dv = _gen((3, 16, 500, 128), 1, BF), _gen((3, 16, 500, 128), 2, BF)
    calls = [lambda: paged.paged_decode(q, k, v, table, n, return_lse=True),
             lambda: paged.paged_decode(q, k8, v8, table, n, return_lse=True),
             lambda: paged.paged_decode(q.half(), k, v, table, n, return_lse=True),       # the query-head kernel
             lambda: paged.paged_decode(q[:, :4], k, v, table, n, return_lse=True),       # a K/V head each
             lambda: dec.pallas_flash_decoding(q, dk, dv, return_lse=True),
             lambda: dec.pallas_flash_decoding(q, dk[:, :4], dv[:, :4], return_lse=True)]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    get, held = dec.DecodeWorkspace.get, []
    monkeypatch.setattr(dec.DecodeWorkspace, "get", lambda *a: held.append(get(*a)) or held[-1])
    for i, call in enumerate(calls):
        want = [t.clone() for t in call()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for _ in range(3):
            held[-1].fill_(255)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i
            assert 0 < int((held[-1][:1 << 18] == 0).sum()) <= 4 * max(3 * 16, sms), i
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("kvdt", [BF, FP8])
def test_layers_share_a_plan(mods, kvdt):
    """A model of several layers plans a step once: every layer writes to the plan's slots
    in pools of its own and decodes over the one table, all in one captured graph."""
    from pallas_flash.ops.rotary import rotary_frequencies
    _lib, dec, paged = mods
    L, B, H, H_kv, D, page, P = 3, 3, 8, 2, 128, 16, 40
    ks, vs = (0.05, 0.03) if kvdt == FP8 else (1.0, 1.0)
    pools = [[torch.zeros((P, H_kv, page, D), device="cuda").to(kvdt) for _ in range(2)] for _ in range(L)]
    table = torch.full((B, 12), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    ring = torch.arange(P, dtype=torch.int32, device="cuda")
    cursor = torch.tensor([0, P], dtype=torch.int64, device="cuda")
    f = rotary_frequencies(D)
    ws = [[1 + 0.1 * _gen((D,), 10 * i + s) for s in range(2)] for i in range(L)]

    def step(new, xs, T):
        plan = paged.plan_append(table, lens, new, ring, cursor, page_size=page, num_tokens=T, inplace=True)
        qs = [paged.qk_norm_rope_append(x[:, :H], x[:, H:H + H_kv], x[:, H + H_kv:], f, plan.positions, plan.slots, *pools[i],
                                        q_weight=ws[i][0], k_weight=ws[i][1], k_scale=ks, v_scale=vs) for i, x in enumerate(xs)]
        return qs, plan

    prompts = torch.tensor([33, 0, 100], dtype=torch.int32, device="cuda")
    x0 = [_gen((140, H + 2 * H_kv, D), 30 + i, BF) for i in range(L)]
    _, plan = step(prompts, x0, 140)
    seqs = [[x[plan.seq_ids == b] for b in range(B)] for x in x0]
    one = torch.ones(B, dtype=torch.int32, device="cuda")
    xs = [torch.zeros((B, H + 2 * H_kv, D), dtype=BF, device="cuda") for _ in range(L)]
    state = (table, lens, ring, cursor)
    saved = [t.clone() for t in state]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qs, _ = step(one, xs, B)
        outs = [paged.paged_decode(q.unsqueeze(2), *pools[i], table, lens, return_lse=True, k_scale=ks, v_scale=vs)
                for i, q in enumerate(qs)]
    for t, s in zip(state, saved):
        t.copy_(s)
    held = [33, 0, 100]
    for n in range(20):
        for i in range(L):
            xs[i].copy_(_gen(xs[i].shape, 1000 + 10 * n + i, BF))
            seqs[i] = [torch.cat([s, xs[i][b:b + 1]]) for b, s in enumerate(seqs[i])]
        graph.replay()
        held = [m + 1 for m in held]
        assert lens.tolist() == held
        for i in range(L):
            check(outs[i][0], outs[i][1], qs[i].unsqueeze(2), *pools[i], table, held, None, ks, vs, f"step {n} layer {i}")
    assert _lib.device_status() == (0, 0)
    half = 2.0 ** -4 if kvdt == FP8 else 2.0 ** -8
    for i in range(L):
        for b in range(B):
            k = dense(pools[i][0], table, b, held[b], ks).transpose(0, 1)
            want, m = _turned(seqs[i][b][:, H:H + H_kv], ws[i][1], f, torch.arange(held[b], device="cuda"))
            assert ((k - want).abs() <= half * want.abs() + (2.0 ** -10 * ks if kvdt == FP8 else 0) + 34 * 2.0 ** -24 * m).all()
