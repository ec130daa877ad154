"""Argument errors of page sharing and of plans with shared pages, without a GPU: the
host checks come before any CUDA call (pointers here are never followed)."""
from __future__ import annotations

import pytest
import torch
from test_long_context_cpu import P, change, lib  # noqa: F401  (a fixture)


def test_page_share_arguments(lib):
    _lib, so = lib
    inv, uns = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED
    # table, max_pages, page_size, lens, shared, sources, sequences, n, source, tokens, B
    good = [P, 4, 16, P, P, P, P, 0, 1, 32, 3, None]
    for at, code in [({}, _lib.PU_OK), (dict(_0=None), inv), (dict(_3=None), inv), (dict(_4=None), inv), (dict(_5=None), inv), (dict(_6=None, _7=1), inv),
                     (dict(_6=None), _lib.PU_OK), (dict(_1=0), uns), (dict(_2=24), uns), (dict(_2=8), uns), (dict(_2=8192), uns), (dict(_7=-1), inv), (dict(_8=-1), _lib.PU_OK),
                     (dict(_8=-2), inv), (dict(_8=3), inv), (dict(_9=-16), inv), (dict(_9=17), inv), (dict(_9=80), inv), (dict(_9=0, _7=2), _lib.PU_OK), (dict(_10=0), uns),
                     (dict(_10=8193), uns)]:
        assert so.pu_page_share(*change(good, **at)) == code, at


def test_plan_arguments(lib):
    _lib, so = lib
    inv, uns = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED
    # table, max_pages, lens, new, release, ring, num_pages, cursor, page_size, slots, positions, seq_ids, cu, shared, sources, B, T
    good = [P, 4, P, P + 4096, P, P, 8, P, 16, P, P, P, P, P, P, 3, 5, None]
    for at, code in [(dict(_0=None), inv), (dict(_2=None), inv), (dict(_13=None), inv), (dict(_14=None), inv), (dict(_3=P + 8), inv), (dict(_8=24), uns), (dict(_15=8193), uns),
                     (dict(_9=None), inv), (dict(_16=-1), uns)]:
        assert so.pu_page_plan_shared(*change(good, **at)) == code, at


def test_python_checks():
    from pallas_flash.kernels import paged
    ints = lambda *a: torch.tensor(a, dtype=torch.int32)      # noqa: E731
    cache = paged.DevicePagedKVCache(3, 2, 64, num_pages=5, page_size=16, max_seq_len=48, device="cpu")
    assert cache.shared_lens.tolist() == [0, 0, 0] and cache.sources.tolist() == [-1, -1, -1]
    for bad in (lambda: cache.share(3, [1], 16), lambda: cache.share(0, [1], 15), lambda: cache.share(0, [1], 64), lambda: cache.unshare([1], -16),
                lambda: cache.share(0, [0.5], 16)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="CUDA"):
        cache.share(0, [1], 16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.plan_append(cache.page_table, cache.kv_lens, ints(1, 1, 1), cache.free_ring, cache.cursor, page_size=16, num_tokens=3, inplace=True)
