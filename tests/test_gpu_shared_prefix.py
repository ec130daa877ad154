"""Paged decode of sequences that share their first pages (pu_decode_paged_shared)
against the formula in 64 bits.

The tolerance is that of the paged grouped decode (test_gpu_paged_gqa), element
by element: half a step of bf16 plus what the weights p are off by times
A = sum_j p_j |v_j|.  A weight of a shared token is rounded once to the operands'
type: 2^-8 for bf16, 2^-11 for f16 and for e4m3 pools (own tokens there: three
parts, 2^-12).  Small weights vanish below 2^-25 of f16's largest.  Scores are fp32
sums; with e4m3 pools the own tokens' queries are off by 2^-17 of the head's largest
element, the shared tokens' (f16 times a power of two) by less.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from test_gpu_paged_gqa import BF, FP8, HF, _gen, dense

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


def enough(tokens, H, H_kv):
    """Sequences from which on a prefix of `tokens` tokens is shared."""
    return -(-1024 // (-(-tokens // 128) * H_kv * -(-(H // H_kv) // 16)))


def check(o, lse, q, k_pool, v_pool, table, lens, k_scale=1.0, v_scale=1.0, scale=None, what="", sample=60):
    B, H, _, D = q.shape
    H_kv = k_pool.shape[1]
    G = H // H_kv
    scale = 1 / math.sqrt(D) if scale is None else scale
    f8 = k_pool.dtype == FP8
    rnd = 2.0 ** -8 if k_pool.dtype == BF else 2.0 ** -11
    lost = 0.0 if k_pool.dtype == BF else 2.0 ** -25
    assert o.dtype == BF and o.shape == q.shape and lse.shape == (B, H)
    some = np.random.RandomState(B).permutation(B)[:sample].tolist() + [0, B - 1]
    for b, n in enumerate(np.asarray(lens).tolist()):
        if b not in some:
            continue
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
        assert (off <= e.amax(-1).reshape(H) + 2.0 ** -19 + 2.0 ** -22 * l.reshape(H).abs()).all(), f"{what}: lse of sequence {b}"


def batch(groups, page, seed, spare=2):
    """groups: (shared tokens, own tokens of each sequence).  A table with pages in random order, and
    lengths, shared lengths and group starts."""
    r = np.random.RandomState(seed)
    tails = [n for _, own in groups for n in own]
    pre = [s // page for s, _ in groups]
    P = sum(pre) + sum(-(-n // page) for n in tails) + spare
    order = r.permutation(P).astype(np.int32).tolist()
    width = 1 + max(p + -(-n // page) for p, (_, own) in zip(pre, groups) for n in (list(own) or [0]))
    rows, lens = [], []
    for p, (s, own) in zip(pre, groups):
        head = [order.pop() for _ in range(p)]
        for n in own:
            row = head + [order.pop() for _ in range(-(-n // page))]
            rows.append(row + [-1] * (width - len(row)))
            lens.append(p * page + n)
    starts = np.cumsum([0] + [len(own) for _, own in groups])
    return ints(np.array(rows)), P, np.array(lens), ints([s for s, _ in groups]), ints(starts)


def make(P, B, H, H_kv, D, page, qdt, kvdt, seed, ks=1.0, vs=1.0):
    q = _gen((B, H, 1, D), seed, qdt)
    return (q, *(_gen((P, H_kv, page, D), seed + 1 + i, torch.float32, 1 / s).to(kvdt) for i, s in enumerate((ks, vs))))


KINDS = [(8, 2, 128, BF, BF), (6, 6, 128, HF, HF), (40, 2, 64, BF, BF), (5, 1, 64, HF, HF), (12, 4, 128, BF, FP8), (8, 8, 128, HF, FP8)]


@pytest.mark.parametrize("H,H_kv,D,qdt,kvdt", KINDS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_prefixes(mods, H, H_kv, D, qdt, kvdt, page):
    """Prefixes of one page, of whole tiles and between, few rows to several items of 256, own
    tokens from none on."""
    _lib, dec, paged = mods
    r = np.random.RandomState(page)
    ks, vs = (0.05, 0.03) if kvdt == FP8 else (1.0, 1.0)
    for i, (tokens, n) in enumerate([(page, 3), (768, 1), (1024 + page, 40), (512, 140 // (H // H_kv) + 1), (page * 3, 600 // (H // H_kv))]):
        table, P, lens, shared, _ = batch([(tokens, [0, 1, page, 129][:n] + r.randint(0, 300, max(0, n - 4)).tolist())], page, i)
        q, k, v = make(P, len(lens), H, H_kv, D, page, qdt, kvdt, 7 * i, ks, vs)
        o, lse = dec.pallas_flash_decoding(q, k, v, kv_lens=ints(lens), page_table=table, shared_lens=shared, k_scale=ks, v_scale=vs, return_lse=True)
        assert _lib.device_status() == (0, 0)
        check(o, lse, q, k, v, table, lens, ks, vs, what=f"{tokens} shared by {n}")
        again = dec.pallas_flash_decoding(q, k, v, kv_lens=ints(lens), page_table=table, shared_lens=shared, k_scale=ks, v_scale=vs)
        assert torch.equal(o, again)


@pytest.mark.parametrize("H,H_kv,D,qdt,kvdt", KINDS)
@pytest.mark.parametrize("page,tokens", [(16, 16), (16, 144), (64, 128), (64, 960), (256, 2048)])
def test_shared(mods, H, H_kv, D, qdt, kvdt, page, tokens):
    """As few sequences as share, and one fewer: one page, tiles and a rest, several items of 256 rows;
    the sequences' own tokens from none on, one sequence shorter than the prefix."""
    _lib, dec, paged = mods
    r = np.random.RandomState(page + tokens)
    ks, vs = (0.05, 0.03) if kvdt == FP8 else (1.0, 1.0)
    n = enough(tokens, H, H_kv)
    own = [0, 1, page, 129] + r.randint(0, 40, max(0, n - 4)).tolist()
    table, P, lens, shared, _ = batch([(tokens, own[:n])], page, 7)
    lens[n // 2] = max(0, tokens - 1)
    q, k, v = make(P, n, H, H_kv, D, page, qdt, kvdt, 3, ks, vs)
    for m in (n, max(1, n - 1)):
        args = q[:m], k, v, table[:m].contiguous(), ints(lens[:m])
        o, lse = paged.paged_decode(*args, shared_lens=shared, k_scale=ks, v_scale=vs, return_lse=True)
        assert _lib.device_status() == (0, 0)
        check(o, lse, args[0], k, v, args[3], lens[:m], ks, vs, what=f"{tokens} shared by {m}")
        assert torch.equal(o, paged.paged_decode(*args, shared_lens=shared, k_scale=ks, v_scale=vs))


@pytest.mark.parametrize("H,H_kv,D,qdt,kvdt", KINDS)
def test_groups(mods, H, H_kv, D, qdt, kvdt):
    """Several prefixes, groups without one, empty groups, sequences in no group."""
    _lib, dec, paged = mods
    page = 32
    # 7680 tokens shared by 160 sequences: 9600 tiles of a K/V head
    groups = [(96, [5, 0, 70]), (0, [3, 200]), (7680, list(range(160))), (64, []), (320, [1] * 9), (512, [0])]
    table, P, lens, shared, starts = batch(groups, page, 3)
    q, k, v = make(P, len(lens), H, H_kv, D, page, qdt, kvdt, 5)
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, shared_groups=starts, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="groups")
    # the first and last group's sequences in no group
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared[1:5].contiguous(), shared_groups=starts[1:6].contiguous(), return_lse=True)
    check(o, lse, q, k, v, table, lens, what="some in no group")
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=torch.zeros_like(shared), shared_groups=starts, return_lse=True)
    check(o, lse, q, k, v, table, lens, what="nothing shared")
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("groups", [64])
def test_many_groups(mods, groups):
    _lib, dec, paged = mods
    page = 16
    table, P, lens, shared, starts = batch([(16 * (1 + i % 60), [i, 3 * i, 0, 5, 1, 17][:1 + i % 6]) for i in range(groups)], page, 3)
    q, k, v = make(P, len(lens), 8, 2, 128, page, BF, BF, 5)
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, shared_groups=starts, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="many groups")


@pytest.mark.parametrize("kvdt", [BF, FP8])
def test_lengths_that_do_not_fit(mods, kvdt):
    """Shared lengths inside a page, longer than the table or negative, sequences shorter than the
    prefix (an empty slot of a padded batch first), starts in disorder: the result stays that of the
    plain decode."""
    _lib, dec, paged = mods
    page = 64
    more = [7] * 140                     # so that 640 tokens are shared
    table, P, lens, shared, _ = batch([(640, [10, 0, 100, 33, 5] + more)], page, 3)
    B = len(lens)
    assert B >= enough(640, 8, 2)
    q, k, v = make(P, B, 8, 2, 128, page, BF, kvdt, 5)
    for s in (639, 641, 65, 63, 0, -5):
        o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=ints([s]), return_lse=True)
        check(o, lse, q, k, v, table, lens, what=f"shared {s}")
    for short in ([0, 640, 740, 673, 645], [0, 0, 740, 1, 645], [300, 639, 0, 128, 640], [0, 0, 0, 0, 0], [5, 639, 70, 64, 1]):
        short = np.array(short + [647] * (B - 5))
        o, lse = paged.paged_decode(q, k, v, table, ints(short), shared_lens=shared, return_lse=True)
        check(o, lse, q, k, v, table, short, what=f"lengths {short}")
    low = np.minimum(lens, 639)           # none holds the prefix
    o, lse = paged.paged_decode(q, k, v, table, ints(low), shared_lens=shared, return_lse=True)
    check(o, lse, q, k, v, table, low, what="none holds it")
    # longer than any sequence: nothing is shared
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=ints([2 ** 31 - 1]), return_lse=True)
    check(o, lse, q, k, v, table, lens, what="too long")
    for starts in ([0, B, 3], [-7, 2, 900], [4, 1, B], [5, 5, 5], [1, 140, B + 1]):
        o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=ints([640, 640]), shared_groups=ints(starts), return_lse=True)
        check(o, lse, q, k, v, table, lens, what=f"starts {starts}")
    # an empty slot whose row names no page
    table[0] = -1
    o, lse = paged.paged_decode(q, k, v, table, ints([0] + lens[1:].tolist()), shared_lens=shared, return_lse=True)
    check(o, lse, q, k, v, table, [0] + lens[1:].tolist(), what="empty slot")
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("D,page,kvdt", [(128, 16, BF), (64, 32, HF), (128, 64, FP8)])
def test_stale_and_missing_pages(mods, D, page, kvdt):
    """NaN in pages of nobody never counts; table entries outside the pool are reported and their
    tokens left out for all."""
    _lib, dec, paged = mods
    table, P, lens, shared, _ = batch([(384 + page, [5, 0, 100] + [7] * 180)], page, 3, spare=9)
    assert len(lens) >= enough(384 + page, 8, 2)
    q, k, v = make(P, len(lens), 8, 2, D, page, HF if kvdt == HF else BF, kvdt, 5)
    used = torch.zeros(P, dtype=torch.bool, device="cuda")
    used[table[table >= 0].long()] = True
    nan = torch.full((1,), math.nan, device="cuda").to(kvdt)
    for pool in (k, v):
        raw = pool.view(torch.uint8) if kvdt == FP8 else pool
        raw[~used] = nan.view(torch.uint8) if kvdt == FP8 else nan
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="stale")
    bad = table.clone()
    gone = [1, 3]
    bad[:, 1], bad[:, 3] = P, -1
    o, lse = paged.paged_decode(q, k, v, bad, ints(lens), shared_lens=shared, return_lse=True)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 302)
    rest = [i for i in range(table.shape[1]) if i not in gone]
    check(o, lse, q, k, v, table[:, rest].contiguous(), lens - 2 * page, what="missing")


def test_large_scores(mods):
    """Scores of far more than exp's range: the maxima move and nothing overflows."""
    _lib, dec, paged = mods
    page = 32
    table, P, lens, shared, _ = batch([(2048, [40] * 70)], page, 3)
    for kvdt, qdt in ((BF, BF), (HF, HF), (FP8, BF)):
        q, k, v = make(P, len(lens), 8, 2, 128, page, qdt, kvdt, 5)
        q = (q.float() * torch.linspace(0.01, 40, len(lens), device="cuda").view(-1, 1, 1, 1)).to(qdt)
        # keys grow along the prefix, so that the maximum keeps moving
        k[table[0, :64].long()] = (k[table[0, :64].long()].float() * torch.linspace(0.1, 2, 64, device="cuda").view(-1, 1, 1, 1)).to(kvdt)
        o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, return_lse=True)
        check(o, lse, q, k, v, table, lens, what=f"{kvdt}")
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("B,tokens,H,H_kv", [(64, 33000, 32, 8), (200, 5000, 16, 1), (2, 20000, 4, 2)])
def test_long_prefixes(mods, B, tokens, H, H_kv):
    _lib, dec, paged = mods
    page = 64
    r = np.random.RandomState(B)
    table, P, lens, shared, _ = batch([(tokens // page * page, r.randint(0, 500, B))], page, 3)
    q, k, v = make(P, B, H, H_kv, 128, page, BF, BF, 5)
    o, lse = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, return_lse=True)
    assert _lib.device_status() == (0, 0)
    check(o, lse, q, k, v, table, lens, what="long")


def test_other_types_are_the_plain_decode(mods):
    _lib, dec, paged = mods
    table, P, lens, shared, _ = batch([(128, [5, 0, 100])], 64, 3)
    for H, D, qdt, kvdt in ((8, 128, HF, BF), (8, 64, BF, FP8)):
        q, k, v = make(P, 3, H, 2, D, 64, qdt, kvdt, 5)
        a = paged.paged_decode(q, k, v, table, ints(lens), shared_lens=shared, return_lse=True)
        b = paged.paged_decode(q, k, v, table, ints(lens), return_lse=True)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_shared_document(mods):
    """One sequence's pages shared by others in a device cache: append, decode in a captured step,
    give the pages up, release."""
    from pallas_flash.ops.rotary import rotary_frequencies
    _lib, dec, paged = mods
    B, H, H_kv, D, page = 5, 8, 2, 128, 16
    cache = paged.DevicePagedKVCache(B, H_kv, D, num_pages=60, page_size=page, max_seq_len=400)
    f = rotary_frequencies(D)
    split = lambda x: (x[:, :H], x[:, H:H + H_kv], x[:, H + H_kv:])    # noqa: E731
    x = _gen((200, H + 2 * H_kv, D), 1, BF)
    cache.append(*split(x), cache.plan(ints([192, 0, 0, 0, 0]), num_tokens=200), f)
    others = torch.tensor([1, 2, 4], device="cuda")
    cache.share(0, others, 192)
    shared, groups = ints([192]), ints([0, 5])
    new = ints([1, 1, 1, 0, 1])
    x = torch.zeros((5, H + 2 * H_kv, D), dtype=BF, device="cuda")
    pick = torch.tensor([0, 1, 2, 2, 3], device="cuda")     # rows of the packed batch, sequence 3 has none
    state = (cache.page_table, cache.kv_lens, cache.free_ring, cache.cursor)
    saved = [t.clone() for t in state]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = cache.append(*split(x), cache.plan(new, num_tokens=5), f)[pick]
        o, lse = cache.decode(q, shared_lens=shared, shared_groups=groups, return_lse=True)
    for t, s in zip(state, saved):
        t.copy_(s)
    held = [192, 192, 192, 0, 192]
    for n in range(20):
        x.copy_(_gen(x.shape, 100 + n, BF))
        graph.replay()
        held = [m + a for m, a in zip(held, (1, 1, 1, 0, 1))]
        assert cache.kv_lens.tolist() == held
        check(o, lse, q.unsqueeze(2), cache.k_pool, cache.v_pool, cache.page_table, held, what=f"step {n}")
    cache.unshare(others, 192)
    assert cache.kv_lens.tolist() == [212, 20, 20, 0, 20]
    cache.plan(ints([0] * 5), num_tokens=0, release=torch.ones(5, dtype=torch.bool, device="cuda"))
    assert _lib.device_status() == (0, 0)
    head, tail = cache.cursor.tolist()
    assert tail - head == 60 and sorted(cache.free_ring.tolist()) == list(range(60))


def test_streams_and_graphs(mods):
    """Two captured calls replayed at once on two streams: each has a workspace of its own."""
    _lib, dec, paged = mods
    table, P, lens, shared, _ = batch([(1024, [40, 0, 700] + [9] * 70)], 32, 3)
    n, sets = ints(lens), []
    for i in range(2):
        q, k, v = make(P, len(lens), 8, 2, 128, 32, BF, BF, 5 + 10 * i)
        want = [t.clone() for t in paged.paged_decode(q, k, v, table, n, shared_lens=shared, return_lse=True)]
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            got = paged.paged_decode(q, k, v, table, n, shared_lens=shared, return_lse=True)
        sets.append((graph, stream, got, want, (q, k, v)))
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
    table, P, lens, shared, _ = batch([(128, [5, 0, 100])], 64, 3)
    q, k, v = make(P, 3, 8, 2, 128, 64, BF, BF, 5)
    n = ints(lens)
    lists = table.unsqueeze(1).repeat(1, 2, 1)
    for kw in (dict(shared_lens=shared.long()), dict(shared_lens=shared.view(1, 1)), dict(shared_lens=ints([1] * 65), shared_groups=ints([0] * 66)),
               dict(shared_lens=ints([64, 64])), dict(shared_lens=shared, shared_groups=ints([0])), dict(shared_groups=ints([0, 3])),
               dict(shared_lens=shared.cpu()), dict(shared_lens=shared, shared_groups=torch.tensor([0, 3], device="cuda")),
               dict(shared_lens=ints([64, 1, 64])[::2], shared_groups=ints([0, 1, 2]))):
        with pytest.raises(ValueError):
            paged.paged_decode(q, k, v, table, n, **kw)
    with pytest.raises(ValueError):
        paged.paged_decode(q, k, v, lists, n.view(3, 1).repeat(1, 2), shared_lens=shared)
    with pytest.raises(ValueError):
        dec.pallas_flash_decoding(q, _gen((3, 2, 64, 128), 1, BF), _gen((3, 2, 64, 128), 2, BF), shared_lens=shared)
    cache = paged.DevicePagedKVCache(2, 2, 64, num_pages=5, page_size=16, max_seq_len=48)
    for tokens in (15, 64, -16):
        with pytest.raises(ValueError):
            cache.share(0, torch.tensor([1], device="cuda"), tokens)
        with pytest.raises(ValueError):
            cache.unshare(torch.tensor([1], device="cuda"), tokens)
