"""Page tables, slots and positions made on the device (pu_page_plan) against
a loop over sequences and tokens.  Every result is a whole number and has to
be equal."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    from pallas_flash import _lib
    from pallas_flash.kernels import paged
    _lib.device_status()
    return _lib, paged


def oracle(table, lens, new, ring, cursor, page, T, release):
    """The plan, token by token; `ring` is written like the kernel's."""
    B, width = table.shape
    P = len(ring)
    head, tail = int(cursor[0]), int(cursor[1])
    left = tail - head
    out = np.full_like(table, -1)
    slots, pos, seq = np.full(T, -1), np.zeros(T, int), np.full(T, -1)
    cu, lens_out = [], []
    free = [int(ring[(head + i) % P]) for i in range(left)]
    asked, row, back, refused = 0, 0, [], set()
    for b in range(B):
        gone = release is not None and bool(release[b])
        old = [int(e) for e in table[b, :-(-int(lens[b]) // page)]]
        base = 0 if gone else int(lens[b])
        kept = [] if gone else old
        if gone:
            back += old
        n = max(int(new[b]), 0)
        cu.append(min(row, T))
        pages = list(kept)
        fits = base + n <= width * page and row + n <= T
        more = -(-(base + n) // page) - len(kept) if fits else 0
        ok = fits and (more == 0 or asked + more <= left)
        if ok:
            pages += free[asked:asked + more]
        else:
            refused.add("fit" if not fits else "free")
        asked += more
        out[b, :len(pages)] = pages
        lens_out.append(base + n if ok else base)
        for i in range(n):
            if row + i < T:
                pos[row + i], seq[row + i] = base + i, b
                if ok:
                    slots[row + i] = pages[(base + i) // page] * page + (base + i) % page
        row += n
    cu.append(min(row, T))
    used = sum(1 for b in range(B) for _ in range((out[b] >= 0).sum())) - \
        sum(-(-int(lens[b]) // page) for b in range(B) if not (release is not None and release[b]))
    for i, e in enumerate(back):
        ring[(tail + i) % P] = e
    return dict(slots=slots, positions=pos, seq_ids=seq, cu_new=np.array(cu), kv_lens=np.array(lens_out),
                cursor=np.array([head + used, tail + len(back)]), page_table=out, refused=refused)


def state(B, width, page, held, spare, seed, head=None):
    r = np.random.RandomState(seed)
    lens = np.asarray(held, np.int32)
    have = -(-lens // page)
    P = int(have.sum()) + spare
    order = r.permutation(P).astype(np.int32)
    table = np.full((B, width), -1, np.int32)
    table[np.arange(width)[None] < have[:, None]] = order[:have.sum()]
    ring = np.full(P, -9, np.int32)
    head = r.randint(0, 5 * P) if head is None else head
    ring[(head + np.arange(spare)) % P] = order[have.sum():]
    return table, lens, ring, np.array([head, head + spare], np.int64)


def check(paged, st, new, page, T, release=None, inplace=False):
    table, lens, ring, cursor = st
    t = [torch.from_numpy(a.copy()).cuda() for a in (table, lens, ring, cursor)]
    rel = None if release is None else torch.from_numpy(np.asarray(release, bool)).cuda()
    ring64 = ring.copy()
    want = oracle(table, lens, new, ring64, cursor, page, T, release)
    plan = paged.plan_append(t[0], t[1], torch.tensor(np.asarray(new), dtype=torch.int32, device="cuda"), t[2], t[3],
                             page_size=page, num_tokens=T, release=rel, inplace=inplace)
    for n in ("slots", "positions", "seq_ids", "cu_new", "kv_lens", "cursor", "page_table"):
        np.testing.assert_array_equal(getattr(plan, n).cpu().numpy(), want[n], err_msg=n)
    np.testing.assert_array_equal(t[2].cpu().numpy(), ring64, err_msg="ring")
    if inplace:
        assert plan.page_table is t[0] and plan.kv_lens is t[1] and plan.cursor is t[3]
    else:
        assert torch.equal(t[0].cpu(), torch.from_numpy(table)) and torch.equal(t[1].cpu(), torch.from_numpy(lens))
    return plan, want, (plan.page_table.cpu().numpy(), plan.kv_lens.cpu().numpy(), t[2].cpu().numpy(), plan.cursor.cpu().numpy())


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("B,width,page,most,per,pad", [
    (1, 1, 16, 0, 1, 0), (1, 3000, 16, 40000, 1, 0), (5, 7, 32, 200, 24, 3), (64, 40, 64, 2000, 1, 0),
    (33, 600, 16, 4000, 400, 11), (1024, 9, 16, 100, 1, 5), (2500, 5, 16, 60, 9, 0), (3, 2, 4096, 4000, 3000, 100),
    (8192, 2, 16, 20, 3, 1)])
def test_plan(mods, B, width, page, most, per, pad, inplace):
    _lib, paged = mods
    r = np.random.RandomState(B + width)
    held = r.randint(0, most + 1, B)
    new = np.ones(B, int) if per == 1 else r.randint(0, per + 1, B)
    new = np.minimum(new, width * page - held)
    st = state(B, width, page, held, int((-(-(held + new) // page)).sum()) + 3, B)
    _, want, _ = check(paged, st, new, page, int(new.sum()) + pad, inplace=inplace)
    assert not want["refused"] and _lib.device_status() == (0, 0)


@pytest.mark.parametrize("inplace", [False, True])
def test_release_and_reuse(mods, inplace):
    """Several steps with released sequences: their pages come back at the
    tail, wrap around the ring and are handed out by later calls."""
    _lib, paged = mods
    B, width, page = 9, 12, 16
    r = np.random.RandomState(3)
    st = state(B, width, page, r.randint(0, 60, B), 25, 7)
    for step in range(30):
        release = r.rand(B) < 0.35
        base = np.where(release, 0, st[1])
        new = np.minimum(r.randint(0, 40, B), width * page - base)
        # keep within the free pages
        left = int(st[3][1] - st[3][0])
        for b in range(B):
            more = -(-(base[b] + new[b]) // page) - -(-base[b] // page)
            if more > left:
                new[b] = 0
                more = 0
            left -= more
        _, want, st = check(paged, st, new, page, int(new.sum()) + step % 3, release, inplace)
        assert not want["refused"]
        live = st[0][st[0] >= 0]
        free = st[2][(st[3][0] + np.arange(st[3][1] - st[3][0])) % len(st[2])]
        assert sorted(np.concatenate([live, free])) == list(range(len(st[2])))    # every page in one place
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("inplace", [False, True])
def test_refusals(mods, inplace):
    """What does not fit stays as it is, its rows get no slot, the rest is served,
    and the device status says so."""
    _lib, paged = mods
    page, width = 16, 4
    st = state(4, width, page, [20, 60, 0, 33], 3, 1)
    # sequence 1 would exceed its table row
    _, want, _ = check(paged, st, [1, 10, 5, 2], page, 18, inplace=inplace)
    assert want["refused"] == {"fit"}
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 307)
    # three free pages: sequences 2 and 3 ask for more than what is left
    _, want, _ = check(paged, st, [20, 2, 40, 15], page, 77, inplace=inplace)
    assert want["refused"] == {"free"}
    assert _lib.device_status() == (_lib.PU_ERR_WORKSPACE, 308)
    # no page is needed: served although nothing is free
    none = state(2, width, page, [20, 5], 0, 1)
    _, want, _ = check(paged, none, [3, 11], page, 14, inplace=inplace)
    assert not want["refused"] and _lib.device_status() == (0, 0)
    # the batch's rows end inside a sequence
    _, want, _ = check(paged, st, [4, 1, 9, 1], page, 9, inplace=inplace)
    assert want["refused"] == {"fit"}
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 307)
    # negative counts are none
    _, want, _ = check(paged, st, [-5, 1, 0, -1], page, 2, inplace=inplace)
    assert not want["refused"] and _lib.device_status() == (0, 0)


def test_bad_state_is_reported(mods):
    """A cursor that describes no ring, a length past the table, a kept page
    outside the pool: nothing is read or written out of place."""
    _lib, paged = mods
    page, width = 16, 4
    table, lens, ring, cursor = state(2, width, page, [20, 5], 6, 2)
    t = lambda a: torch.from_numpy(np.asarray(a).copy()).cuda()   # noqa: E731
    new = torch.tensor([20, 1], dtype=torch.int32, device="cuda")
    for bad in ([-3, 2], [0, len(ring) + 1], [7, 2]):
        plan = paged.plan_append(t(table), t(lens), new, t(ring), t(np.array(bad, np.int64)), page_size=page, num_tokens=21)
        assert plan.slots[:20].tolist() == [-1] * 20 and plan.slots[20] >= 0
        assert _lib.device_status()[0] != 0
    plan = paged.plan_append(t(table), t(np.array([2000, 5], np.int32)), torch.tensor([1, 1], dtype=torch.int32, device="cuda"),
                             t(ring), t(cursor), page_size=page, num_tokens=2)
    assert plan.slots[0] == -1 and plan.slots[1] >= 0 and plan.kv_lens.tolist() == [64, 6]
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 307)
    wrong = table.copy()
    wrong[1, 0] = 1 << 20
    plan = paged.plan_append(t(wrong), t(lens), torch.tensor([0, 2], dtype=torch.int32, device="cuda"), t(ring), t(cursor),
                             page_size=page, num_tokens=2)
    assert plan.slots.tolist() == [-1, -1]
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 307)
    # a ring that already holds every page cannot take a released one back
    full = state(1, width, page, [20], 0, 2)
    ring_all = np.arange(2, dtype=np.int32)
    plan = paged.plan_append(t(full[0]), t(full[1]), torch.tensor([0], dtype=torch.int32, device="cuda"), t(ring_all),
                             t(np.array([0, 2], np.int64)), page_size=page, num_tokens=0,
                             release=torch.ones(1, dtype=torch.bool, device="cuda"))
    assert plan.kv_lens.tolist() == [0] and plan.cursor.tolist() == [0, 2]
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 308)


def test_captured_in_place(mods):
    """A captured step replayed many times: state advances on the device alone."""
    _lib, paged = mods
    B, width, page = 6, 20, 16
    table, lens, ring, cursor = state(B, width, page, [0, 15, 16, 17, 31, 40], 40, 4, head=70)
    t = [torch.from_numpy(a.copy()).cuda() for a in (table, lens, ring, cursor)]
    new = torch.ones(B, dtype=torch.int32, device="cuda")
    release = torch.zeros(B, dtype=torch.bool, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = paged.plan_append(t[0], t[1], new, t[2], t[3], page_size=page, num_tokens=B, release=release, inplace=True)
    want_state = (table, lens, ring, cursor)
    for step in range(50):
        gone = np.zeros(B, bool)
        if step in (10, 25):
            gone[step % B] = True
        release.copy_(torch.from_numpy(gone))
        graph.replay()
        r = want_state[2].copy()
        want = oracle(want_state[0], want_state[1], [1] * B, r, want_state[3], page, B, gone)
        want_state = (want["page_table"], want["kv_lens"].astype(np.int32), r, want["cursor"])
        np.testing.assert_array_equal(plan.slots.cpu().numpy(), want["slots"])
    np.testing.assert_array_equal(t[0].cpu().numpy(), want_state[0])
    np.testing.assert_array_equal(t[3].cpu().numpy(), want_state[3])
    assert _lib.device_status() == (0, 0)


@pytest.mark.parametrize("inplace", [False, True])
def test_refused_releases_lose_no_page(mods, inplace):
    """Where the ring cannot take what is released (a cursor that describes no ring,
    more free and released pages than there are), sequences keep their pages and
    lengths, get no new tokens, and the status says so; the others are served."""
    _lib, paged = mods
    page, width, B = 16, 6, 4
    table, lens, ring, cursor = state(B, width, page, [40, 33, 0, 20], 5, 3, head=7)
    t = lambda a: torch.from_numpy(np.asarray(a).copy()).cuda()   # noqa: E731
    P = len(ring)
    release = torch.tensor([True, False, False, True], device="cuda")
    new = torch.tensor([10, 3, 0, 0], dtype=torch.int32, device="cuda")
    # free: 5 of 13; with a tail that claims 9, the 5 released pages no longer fit
    for bad in ([-3, 2], [0, P + 1], [7, 2], [7, 7 + 9]):
        a = [t(x) for x in (table, lens, ring, np.array(bad, np.int64))]
        plan = paged.plan_append(a[0], a[1], new, a[2], a[3], page_size=page, num_tokens=14, release=release, inplace=inplace)
        got = plan.page_table.cpu().numpy()
        np.testing.assert_array_equal(got, table)                 # sequence 1's tokens fit its last page
        assert plan.kv_lens.tolist() == [40, 36, 0, 20], bad
        assert plan.slots[:10].tolist() == [-1] * 10 and (plan.slots[10:13] >= 0).all() and plan.slots[13] == -1
        assert plan.seq_ids.tolist() == [0] * 10 + [1] * 3 + [-1]
        assert plan.positions[:13].tolist() == list(range(40, 50)) + [33, 34, 35]
        assert plan.cursor.tolist() == bad
        np.testing.assert_array_equal(a[2].cpu().numpy(), ring)
        assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 308), bad
    # a ring that holds every page has those of the row already: the row is emptied
    a = [t(x) for x in (np.array([[1, 0, -1]], np.int32), np.array([20], np.int32), np.arange(2, dtype=np.int32), np.array([4, 6], np.int64))]
    plan = paged.plan_append(a[0], a[1], torch.tensor([5], dtype=torch.int32, device="cuda"), a[2], a[3], page_size=page, num_tokens=5,
                             release=torch.ones(1, dtype=torch.bool, device="cuda"), inplace=inplace)
    assert plan.kv_lens.tolist() == [5] and plan.page_table.tolist() == [[0, -1, -1]] and plan.cursor.tolist() == [5, 6]
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 308)


@pytest.mark.parametrize("inplace", [False, True])
def test_release_returns_pages_of_the_pool_only(mods, inplace):
    """Entries of a released row that name no page (a length past the pages it holds, a
    damaged table) are reported and never become free pages; the others come back in
    order.  Rows over several of a warp's segments, beside sound ones."""
    _lib, paged = mods
    page, width, B = 16, 1400, 5
    r = np.random.RandomState(5)
    held = np.array([1300 * 16 - 3, 50, 16, 700 * 16, 900], np.int32)
    table, lens, ring, cursor = state(B, width, page, held, 9, 5, head=3)
    P = len(ring)
    for b, at in ((0, [0, 5, 511, 512, 513, 1024, 1299]), (2, [0]), (3, [])):
        table[b, at] = r.choice([-1, P, P + 7, -(1 << 31), (1 << 31) - 1], len(at))
    gone = np.array([1, 0, 1, 1, 0], bool)
    new = np.array([20, 2, 0, 3, 1], np.int32)
    t = lambda a: torch.from_numpy(np.asarray(a).copy()).cuda()   # noqa: E731
    a = [t(x) for x in (table, lens, ring, cursor)]
    plan = paged.plan_append(a[0], a[1], t(new), a[2], a[3], page_size=page, num_tokens=26, release=t(gone), inplace=inplace)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 307)
    back = [int(e) for b in (0, 2, 3) for e in table[b, :-(-int(held[b]) // page)] if 0 <= e < P]
    head, tail = (int(c) for c in cursor)
    want_ring = ring.copy()
    for i, e in enumerate(back):
        want_ring[(tail + i) % P] = e
    np.testing.assert_array_equal(a[2].cpu().numpy(), want_ring)
    free = [int(ring[(head + i) % P]) for i in range(9)]
    want = table.copy()
    want[[0, 2, 3]] = -1
    want[0, :2], want[3, 0] = free[:2], free[2]
    np.testing.assert_array_equal(plan.page_table.cpu().numpy(), want)
    assert plan.kv_lens.tolist() == [20, 52, 0, 3, 901]
    assert plan.cursor.tolist() == [head + 3, tail + len(back)]
    assert (plan.slots >= 0).all()
    # every place that is free now names a page of the pool
    at = (int(plan.cursor[0]) + np.arange(int(plan.cursor[1] - plan.cursor[0]))) % P
    got = a[2].cpu().numpy()[at]
    assert ((got >= 0) & (got < P)).all()


def test_refused_after_release(mods):
    """A sequence that is released and then does not fit is left empty, its pages back."""
    _lib, paged = mods
    page, width = 16, 2
    st = state(2, width, page, [20, 5], 4, 1)
    for inplace in (False, True):
        _, want, after = check(paged, st, [40, 2], page, 42, [True, False], inplace)
        assert want["refused"] == {"fit"} and after[1].tolist() == [0, 7] and (after[0][0] == -1).all()
        assert after[3][1] - st[3][1] == 2
        assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 307)


def test_pages_are_counted_in_sequence_order(mods):
    """A sequence refused for want of pages keeps its claim within the call: later ones that
    need a page are refused as well, those that need none are served."""
    _lib, paged = mods
    page = 16
    st = state(4, 8, page, [16, 16, 5, 16], 2, 1)
    _, want, after = check(paged, st, [1, 40, 2, 1], page, 44)
    assert want["refused"] == {"free"} and after[1].tolist() == [17, 16, 7, 16]
    assert _lib.device_status() == (_lib.PU_ERR_WORKSPACE, 308)
