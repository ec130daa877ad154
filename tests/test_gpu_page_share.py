"""Sequences that begin with pages of another one in a device cache: what share,
unshare and a release may do to them, against a model of the cache's state.

Everything here is whole numbers, compared exactly.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE = 16


@pytest.fixture(scope="module")
def mods(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    from pallas_flash import _lib
    from pallas_flash.kernels import paged
    _lib.device_status()
    return _lib, paged


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a)).int().cuda()


def make(paged, B, num_pages=200, max_seq_len=640):
    return paged.DevicePagedKVCache(B, 1, 64, num_pages=num_pages, page_size=PAGE, max_seq_len=max_seq_len)


def plan(cache, new, release=None):
    B = cache.kv_lens.shape[0]
    r = None if release is None else torch.tensor([b in release for b in range(B)], device="cuda")
    return cache.plan(ints(new), num_tokens=int(np.sum(new)), release=r)


def rows(cache):
    """Each sequence's pages."""
    t, n = cache.page_table.cpu().numpy(), cache.kv_lens.cpu().numpy()
    return [t[b, :-(-int(n[b]) // PAGE)].tolist() for b in range(len(n))]


def free(cache):
    head, tail = cache.cursor.tolist()
    ring = cache.free_ring.cpu().numpy()
    return [int(ring[i % len(ring)]) for i in range(head, tail)]


# --------------------------------------------------------------------------
# what must not happen
# --------------------------------------------------------------------------
def test_release_returns_no_shared_page(mods):
    """A sequence that shares pages is released as it is: its source's pages do not become free, and
    nobody is handed one of them."""
    _lib, paged = mods
    cache = make(paged, 4, num_pages=12)
    plan(cache, [100, 0, 0, 0])
    cache.share(0, torch.tensor([1, 2], device="cuda"), 96)
    plan(cache, [0, 20, 0, 0])
    before = rows(cache)
    assert before[1][:6] == before[2] == before[0][:6]
    plan(cache, [0, 0, 0, 0], release=[1, 2])
    assert _lib.device_status() == (0, 0)
    assert cache.kv_lens.tolist() == [100, 0, 0, 0] and (cache.page_table[1:] == -1).all()
    assert sorted(free(cache) + before[0]) == list(range(12))
    plan(cache, [0, 0, 80, 0])
    assert _lib.device_status() == (0, 0)
    assert not set(rows(cache)[2]) & set(before[0])


def test_a_source_stays_while_others_hold_its_pages(mods):
    _lib, paged = mods
    cache = make(paged, 4)
    plan(cache, [100, 0, 0, 0])
    cache.share(0, torch.tensor([1, 2], device="cuda"), 64)
    before, room = rows(cache), len(free(cache))
    # not released, nor grown, while 2 holds its pages; 1 is released, 3 grows
    p = plan(cache, [5, 0, 0, 7], release=[0, 1])
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 311)
    assert cache.kv_lens.tolist() == [100, 0, 64, 7] and p.slots[:5].tolist() == [-1] * 5 and (p.slots[5:] >= 0).all()
    assert rows(cache)[0] == before[0] and rows(cache)[2] == before[2] and len(free(cache)) == room - 1
    # with the last of them in the same call it is
    plan(cache, [0] * 4, release=[0, 2])
    assert _lib.device_status() == (0, 0)
    assert cache.kv_lens.tolist() == [0, 0, 0, 7]
    assert sorted(free(cache) + rows(cache)[3]) == list(range(200))
    assert (cache.shared_lens == 0).all() and (cache.sources == -1).all()


def test_share_of_what_cannot_be(mods):
    """Receivers that hold something, a source that holds too little or is its own receiver, sequences out of
    range: reported, and nothing changes; the others of the call are served, once each."""
    _lib, paged = mods
    cache = make(paged, 6)
    plan(cache, [70, 0, 3, 0, 0, 0])
    state = lambda: [t.clone() for t in (cache.page_table, cache.kv_lens, cache.shared_lens, cache.sources)]    # noqa: E731
    for source, to, tokens in ((0, [2], 64), (0, [0], 64), (0, [1], 80), (1, [3], 16), (2, [1], 16), (0, [6], 16), (0, [-7], 16), (0, [2 ** 40], 16)):
        before = state()
        cache.share(source, torch.tensor(to, device="cuda"), tokens)
        assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 311), (source, to)
        assert all(torch.equal(a, b) for a, b in zip(before, state()))
    cache.share(0, torch.tensor([3, 2, 3, 3, -1], device="cuda"), 48)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 311)
    assert cache.kv_lens.tolist() == [70, 0, 3, 48, 0, 48] and cache.sources.tolist() == [-1, -1, -1, 0, -1, 0]
    assert rows(cache)[3] == rows(cache)[5] == rows(cache)[0][:3]
    cache.share(0, torch.tensor([4], device="cuda"), 0)              # nothing
    cache.share(0, torch.tensor([], dtype=torch.int64, device="cuda"), 16)
    cache.share(0, [], 16)
    cache.share(-6, torch.tensor([False, True, False, False, False, False], device="cuda"), 64)
    assert _lib.device_status() == (0, 0) and cache.kv_lens.tolist() == [70, 64, 3, 48, 0, 48]
    for bad in (lambda: cache.share(6, [1], 16), lambda: cache.share(-7, [1], 16), lambda: cache.share(0, [1.0], 16), lambda: cache.share(0, [1], 17),
                lambda: cache.unshare([1], 16.5)):
        with pytest.raises(ValueError):
            bad()


def test_unshare_of_what_is_not_shared(mods):
    _lib, paged = mods
    cache = make(paged, 5)
    plan(cache, [100, 0, 40, 0, 0])
    cache.share(0, torch.tensor([1], device="cuda"), 64)
    plan(cache, [0, 30, 0, 0, 0])                                   # 64 shared and 30 of its own
    cache.share(1, torch.tensor([3], device="cuda"), 80)            # both kinds
    cache.share(1, torch.tensor([4], device="cuda"), 32)            # the first's alone
    assert cache.sources.tolist() == [-1, 0, -1, 1, 0] and _lib.device_status() == (0, 0)
    before = rows(cache)
    for who, tokens in (([2], 16), ([0], 64), ([4], 48), ([1], 64)):
        cache.unshare(torch.tensor(who, device="cuda"), tokens)
        assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 311), who
        assert rows(cache) == before
    # 3 gives up a part, then all; then 1 may
    cache.unshare(torch.tensor([3, 3], device="cuda"), 32)
    assert rows(cache)[3] == before[3][2:] and cache.shared_lens.tolist() == [0, 64, 0, 48, 32]
    cache.unshare(torch.tensor([3], device="cuda"), 48)
    cache.unshare(torch.tensor([1], device="cuda"), 64)
    assert _lib.device_status() == (0, 0)
    assert rows(cache) == [before[0], before[1][4:], before[2], [], before[4]]
    plan(cache, [0] * 5, release=[0, 1])                            # 4 still holds 0's
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 311)
    assert cache.kv_lens.tolist() == [100, 0, 40, 0, 32]


def test_a_sequence_that_was_emptied_by_hand_holds_nothing(mods):
    _lib, paged = mods
    cache = make(paged, 4)
    plan(cache, [50, 0, 0, 0])
    cache.share(0, [1], 32)
    plan(cache, [0, 20, 0, 0])
    cache.share(1, [2], 48)
    cache.kv_lens[2] = 0
    cache.unshare([1], 32)
    assert _lib.device_status() == (0, 0) and cache.kv_lens.tolist() == [50, 20, 0, 0]
    cache.share(0, [2], 16)              # and may begin anew
    plan(cache, [0] * 4, release=[1])
    assert _lib.device_status() == (0, 0) and cache.kv_lens.tolist() == [50, 0, 16, 0]


def test_chains(mods):
    """Pages shared on: a release waits for all that hold them, through others too."""
    _lib, paged = mods
    cache = make(paged, 4)
    plan(cache, [50, 0, 0, 0])
    cache.share(0, [1], 32)
    plan(cache, [0, 40, 0, 0])
    cache.share(1, [2], 64)
    plan(cache, [0, 0, 20, 0])
    cache.share(2, [3], 80)
    assert _lib.device_status() == (0, 0) and cache.sources.tolist() == [-1, 0, 1, 2]
    for release in ([0, 1, 2], [0], [1, 2], [0, 2]):
        plan(cache, [0] * 4, release=release)
        assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 311), release
        assert cache.kv_lens.tolist() == [50, 72, 84, 80], release
    # all that stands in the way of 3 and 2 is taken out in one call
    cache.unshare([3], 80)
    cache.unshare([1, 2], 32)
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 311)      # 2 shares 32 of its 64 still, 1 stays
    assert cache.kv_lens.tolist() == [50, 72, 52, 0] and cache.shared_lens.tolist() == [0, 32, 32, 0]
    plan(cache, [0] * 4, release=[0, 1, 2, 3])
    assert _lib.device_status() == (0, 0)
    assert sorted(free(cache)) == list(range(200))


def test_release_with_entries_that_are_no_pages(mods):
    """Gaps behind the shared part are left out of the ring, as without it."""
    _lib, paged = mods
    cache = make(paged, 3, max_seq_len=16 * 900, num_pages=2000)
    plan(cache, [16 * 600, 0, 0])
    cache.share(0, [1], 16 * 550)
    plan(cache, [0, 16 * 300, 0])
    cache.page_table[1, 700] = -1
    cache.page_table[1, 849] = 2000
    before, own = rows(cache), set(free(cache))
    plan(cache, [0, 0, 0], release=[1])
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 307)
    back = set(free(cache)) - own
    assert back == {p for p in before[1][550:] if 0 <= p < 2000} and len(back) == 298
    assert rows(cache)[0] == before[0] and len(free(cache)) == len(set(free(cache)))


# --------------------------------------------------------------------------
# a model of the state
# --------------------------------------------------------------------------
class Model:
    def __init__(self, B):
        self.B, self.lens, self.shared, self.source, self.rows = B, [0] * B, [0] * B, [-1] * B, [[] for _ in range(B)]

    def root(self, s, tokens):
        while self.shared[s] >= tokens:
            s = self.source[s]
        return s

    def share(self, source, to, tokens):
        bad, root = False, self.root(source, tokens)
        for b in dict.fromkeys(to):
            if b == source or self.lens[b] or self.lens[source] < tokens:
                bad = True
                continue
            self.lens[b] = self.shared[b] = tokens
            self.source[b], self.rows[b] = root, self.rows[source][:tokens // PAGE]
        return bad

    def held(self, leaves, who):
        """Of `who`, those whose pages a sequence holds that does not leave."""
        stay = set()
        while True:
            new = {self.source[b] for b in range(self.B) if self.shared[b] and not (leaves(b) and b not in stay)} & who
            if new == stay:
                return stay
            stay = new

    def unshare(self, who, tokens):
        who = set(who)
        stay = self.held(lambda b: b in who and self.shared[b] == tokens, who)
        bad = False
        for b in who:
            if b in stay or self.shared[b] < tokens:
                bad = True
                continue
            self.lens[b] -= tokens
            self.shared[b] -= tokens
            self.rows[b] = self.rows[b][tokens // PAGE:]
            if not self.shared[b]:
                self.source[b] = -1
        return bad

    def plan(self, new, release):
        release = set(release)
        stay = self.held(lambda b: b in release, release)
        for b in release - stay:
            self.lens[b] = self.shared[b] = 0
            self.source[b], self.rows[b] = -1, []
        for b in range(self.B):
            if b not in stay:
                self.lens[b] += new[b]
        return bool(stay)


@pytest.mark.parametrize("B,steps,seed", [(5, 120, 0), (12, 120, 1), (40, 60, 2), (1500, 20, 3)])
def test_random_steps(mods, B, steps, seed):
    """Random sharing, growth and release: lengths, rows and refusals are the model's, and every page is
    free once or one sequence's own."""
    _lib, paged = mods
    r = np.random.RandomState(seed)
    pages = 60 * B
    cache, m = make(paged, B, num_pages=pages, max_seq_len=PAGE * 200), Model(B)
    for step in range(steps):
        kind, some = r.randint(4), r.randint(0, B, 1 + r.randint(1 + B // 3)).tolist()
        if kind == 0:
            source = int(r.randint(B))
            tokens = PAGE * r.randint(1, 4)
            bad = m.share(source, some, tokens)
            cache.share(source, torch.tensor(some, device="cuda"), tokens)
        elif kind == 1:
            tokens = PAGE * r.randint(1, 3)
            bad = m.unshare(some, tokens)
            cache.unshare(torch.tensor(some, device="cuda"), tokens)
        else:
            new = np.where(r.rand(B) < 0.4, r.randint(0, 50, B), 0)
            new[[b for b in range(B) if m.lens[b] > PAGE * 40]] = 0
            release = some if kind == 3 else []
            kept = [list(x) for x in m.rows]
            bad = m.plan(new.tolist(), release)
            plan(cache, new, release if kind == 3 else None)
            for b, row in enumerate(rows(cache)):
                if m.rows[b]:
                    assert row[:len(kept[b])] == kept[b], (step, b)
                m.rows[b] = row
        assert _lib.device_status() == ((_lib.PU_ERR_INVALID_ARGUMENT, 311) if bad else (0, 0)), (step, kind)
        assert cache.kv_lens.tolist() == m.lens and cache.shared_lens.tolist() == m.shared and cache.sources.tolist() == m.source, (step, kind)
        assert rows(cache) == m.rows, (step, kind)
        own = [p for b in range(B) for p in m.rows[b][m.shared[b] // PAGE:]]
        assert sorted(own + free(cache)) == list(range(pages)), (step, kind)


def test_captured(mods):
    """A captured release guards what is shared after the capture, and a captured share replays."""
    _lib, paged = mods
    cache = make(paged, 4)
    state = (cache.page_table, cache.kv_lens, cache.free_ring, cache.cursor, cache.shared_lens, cache.sources)
    saved = [t.clone() for t in state]
    new, release, to = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.bool, device="cuda"), torch.tensor([2], device="cuda")
    step, share = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(step):
        cache.plan(new, num_tokens=200, release=release)
    with torch.cuda.graph(share):
        cache.share(0, to, 64)
    for t, s in zip(state, saved):
        t.copy_(s)
    new.copy_(ints([100, 0, 0, 0]))
    step.replay()
    share.replay()
    new.zero_()
    release[0] = True
    step.replay()
    assert _lib.device_status() == (_lib.PU_ERR_INVALID_ARGUMENT, 311)
    assert cache.kv_lens.tolist() == [100, 0, 64, 0]
    release[2] = True
    step.replay()
    assert _lib.device_status() == (0, 0)
    assert cache.kv_lens.tolist() == [0] * 4 and sorted(free(cache)) == list(range(200))
