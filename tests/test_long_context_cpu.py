"""Argument errors of page bounds, page selection, decode over page lists of each
head and decode behind shared prefixes, without a GPU: the host checks come
before any CUDA call (pointers here are never followed)."""
from __future__ import annotations

import pytest
import torch

P = 1 << 12      # 16-byte aligned, never followed
BF, F16, F32, F8 = 0, 1, 2, 3


@pytest.fixture(scope="module")
def lib(built_lib):
    from pallas_flash import _lib
    return _lib, _lib.lib()


def change(good, **at):
    """Positional arguments with some replaced by position: _3=..."""
    a = list(good)
    for k, v in at.items():
        a[int(k[1:])] = v
    return a


def test_page_bounds_arguments(lib):
    _lib, so = lib
    inv, uns = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED
    # k_pool, kv_dtype, slots, bounds, num_pages, page_size, H_kv, D, num_tokens
    good = [P, BF, P, P, 8, 16, 2, 128, 5, None]
    for at, code in [(dict(_0=None), inv), (dict(_2=None), inv), (dict(_3=None), inv), (dict(_0=P + 8), inv), (dict(_3=P + 8), inv), (dict(_1=F32), uns),
                     (dict(_1=7), uns), (dict(_4=0), inv), (dict(_5=24), uns), (dict(_5=8), uns), (dict(_5=8192), uns), (dict(_4=1 << 31), uns), (dict(_6=0), uns),
                     (dict(_6=65536), uns), (dict(_7=96), uns), (dict(_8=-1), uns), (dict(_8=1 << 31), uns)]:
        assert so.pu_page_bounds(*change(good, **at)) == code, at
    # nothing to do, and checked all the same
    assert so.pu_page_bounds(*change(good, _2=None, _8=0)) == _lib.PU_OK
    assert so.pu_page_bounds(*change(good, _5=24, _8=0)) == uns


def test_select_pages_arguments(lib):
    _lib, so = lib
    inv, uns = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED
    # q, q_dtype, bounds, bounds_dtype, table, max_pages, num_pages, page_size, lens, pages, out_lens, count, first, last, B, H, H_kv, D
    good = [P, BF, P, F16, P, 4, 8, 16, P, P, P, 3, 1, 1, 2, 8, 2, 128, None]
    for at, code in [(dict(_0=None), inv), (dict(_2=None), inv), (dict(_4=None), inv), (dict(_8=None), inv), (dict(_9=None), inv), (dict(_10=None), inv),
                     (dict(_2=P + 8), inv), (dict(_1=F32), uns), (dict(_3=F8), uns), (dict(_3=F32), uns), (dict(_5=0), inv), (dict(_5=24577), uns), (dict(_6=0), inv),
                     (dict(_7=48), uns), (dict(_11=0), inv), (dict(_12=-1), inv), (dict(_13=-1), inv), (dict(_12=2, _13=2), inv), (dict(_11=1 << 40), uns),
                     (dict(_14=0), inv), (dict(_15=7), inv), (dict(_16=0), inv), (dict(_17=96), uns), (dict(_14=1 << 31), uns), (dict(_6=1 << 27, _15=64, _16=64), uns)]:
        assert so.pu_select_pages(*change(good, **at)) == code, at


def test_page_list_decode_arguments(lib):
    _lib, so = lib
    inv, uns, ws = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED, _lib.PU_ERR_WORKSPACE
    # q, q_dtype, k, v, kv_dtype, table, max_pages, num_pages, page_size, lens, o, lse, ws, bytes, B, H, H_kv, D, scales
    good = [P, BF, P, P, BF, P, 4, 8, 16, P, P, None, P, 1, 2, 8, 2, 128, 0.1, 1.0, 1.0, None]
    for at, code in [({}, ws), (dict(_5=None), inv), (dict(_9=None), inv), (dict(_10=None), inv), (dict(_10=P + 8), inv), (dict(_16=3), inv), (dict(_8=24), uns),
                     (dict(_17=80), uns), (dict(_19=0.0), inv), (dict(_20=-1.0), inv),
                     # the tensor core counts lists, the query-head kernel heads
                     (dict(_14=4096, _15=64, _16=2), ws), (dict(_14=4097, _15=64, _16=2), uns), (dict(_14=1024, _15=64, _16=8), ws), (dict(_14=1025, _15=64, _16=8), uns),
                     (dict(_14=1024, _15=64, _16=64), uns)]:
        assert so.pu_decode_paged_heads(*change(good, **at)) == code, at


def test_shared_prefix_arguments(lib):
    _lib, so = lib
    inv, uns, ws = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED, _lib.PU_ERR_WORKSPACE
    # q, q_dtype, k, v, kv_dtype, table, max_pages, num_pages, page_size, lens, shared, starts, groups, o, lse, ws, bytes, B, H, H_kv, D, scales
    good = [P, BF, P, P, BF, P, 4, 8, 16, P, P, P, 2, P, None, P, 1, 2, 8, 2, 128, 0.1, 1.0, 1.0, None]
    for at, code in [({}, ws), (dict(_0=None), inv), (dict(_5=None), inv), (dict(_9=None), inv), (dict(_10=None), inv), (dict(_11=None), inv), (dict(_11=None, _12=1), ws),
                     (dict(_12=0), inv), (dict(_12=65), inv), (dict(_12=64), ws), (dict(_13=None), inv), (dict(_13=P + 8), inv), (dict(_15=P + 8), inv), (dict(_15=None), ws),
                     (dict(_8=24), uns), (dict(_19=3), inv), (dict(_22=0.0), inv), (dict(_23=float("inf")), inv), (dict(_4=F16), uns), (dict(_4=F8), ws), (dict(_4=F8, _20=64), uns),
                     (dict(_20=64), ws), (dict(_17=8193), uns), (dict(_17=8192), ws), (dict(_18=65536), uns)]:
        assert so.pu_decode_paged_shared(*change(good, **at)) == code, at
    size = so.pu_decode_paged_shared_workspace_size
    assert size(2, 8, 2, 2, 128) > 0
    assert size(0, 8, 2, 2, 128) == size(2, 7, 2, 2, 128) == size(2, 8, 2, 0, 128) == 0
    # room for every item's record, and more for more sequences
    assert size(512, 8, 2, 2, 128) - size(256, 8, 2, 2, 128) >= 2 * 4 * 256 * 130 * 4


def test_python_checks_come_first():
    """Host tensors and wrong shapes are refused before the library is asked."""
    from pallas_flash.kernels import decoding, paged
    k = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16)
    bounds = paged.empty_bounds(k)
    assert bounds.shape == (5, 2, 2, 64) and bounds.dtype == k.dtype
    assert paged.empty_bounds(k.to(torch.float8_e4m3fn)).dtype == torch.float16
    slots, table, lens = torch.zeros(3, dtype=torch.int32), torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.page_bounds(k, slots, bounds)
    with pytest.raises(ValueError, match="CUDA"):
        paged.select_pages(q, bounds, table, lens, 2, page_size=16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.paged_decode(q, k, k, table, lens)
    with pytest.raises(ValueError, match="H_kv"):
        paged.paged_decode(q, k, k, torch.zeros((2, 2, 3), dtype=torch.int32), lens)
    with pytest.raises(ValueError, match="each K/V head"):
        paged.paged_decode(q, k, k, torch.zeros((2, 3, 3), dtype=torch.int32), lens)
    for bad in (torch.zeros((5, 2, 1, 64), dtype=torch.bfloat16), bounds.float(), bounds[0], torch.zeros((5, 2, 2, 80), dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            paged.page_bounds(k, slots, bad)
    with pytest.raises(ValueError, match="paged cache"):
        decoding.pallas_flash_decoding(q, k, k, shared_lens=lens)
    with pytest.raises(ValueError, match="kv_lens"):
        decoding.pallas_flash_decoding(q, k, k, page_table=table, shared_lens=lens)


def test_sharing_arguments():
    """The checks of shared_lens and shared_groups, on the host."""
    from pallas_flash.kernels.paged import _check_shared
    cpu = torch.device("cpu")
    ints = lambda *a: torch.tensor(a, dtype=torch.int32)      # noqa: E731
    _check_shared(ints(5), None, False, cpu)
    _check_shared(ints(5, 6), ints(0, 1, 2), False, cpu)
    for shared, groups, lists in [(ints(5), None, True), (ints(5).long(), None, False), (ints(5).view(1, 1), None, False), (ints(), None, False), (ints(5, 6), None, False),
                                  (ints(5, 6), ints(0, 1), False), (ints(5, 6), ints(0, 1, 2).long(), False), (ints(*range(65)), ints(*range(66)), False),
                                  (ints(5, 6, 7)[::2], ints(0, 1, 2), False)]:
        with pytest.raises(ValueError):
            _check_shared(shared, groups, lists, cpu)


def test_packed_calls_are_the_entry_points(lib):
    """pu_call_packed takes the same arguments in the same order: every refusal comes back alike, for each
    argument changed in turn."""
    import struct
    _lib, so = lib
    scale = [0.1, 1.0, 1.0]
    cases = [(_lib.DECODE_PAGED_GQA, so.pu_decode_paged_gqa, _lib.pack_decode, [P, BF, P, P, BF, P, 4, 8, 16, P, P, 0, P, 1, 2, 8, 2, 128] + scale + [0]),
             (_lib.DECODE_PAGED_HEADS, so.pu_decode_paged_heads, _lib.pack_decode, [P, BF, P, P, BF, P, 4, 8, 16, P, P, 0, P, 1, 2, 8, 2, 128] + scale + [0]),
             (_lib.DECODE_PAGED_SHARED, so.pu_decode_paged_shared, _lib.pack_shared,
              [P, BF, P, P, BF, P, 4, 8, 16, P, P, P, 2, P, 0, P, 1, 2, 8, 2, 128] + scale + [0]),
             (_lib.PAGE_BOUNDS, so.pu_page_bounds, _lib.pack_bounds, [P, BF, P, P, 8, 16, 2, 96, 5, 0]),
             (_lib.SELECT_PAGES, so.pu_select_pages, _lib.pack_select, [P, BF, P, F16, P, 4, 8, 16, P, P, P, 3, 1, 1, 2, 8, 2, 96, 0])]
    for entry, call, pack, good in cases:
        seen = set()
        for i in range(len(good)):
            for v in ((0.0, -1.0) if isinstance(good[i], float) else (0, -1, 3, P + 8, 1 << 40)):
                a = list(good)
                a[i] = v
                if i in (1, 3, 4) and abs(v) >= 1 << 31:
                    continue                  # 32-bit arguments
                if good[i] == 1 and pack is not _lib.pack_bounds and pack is not _lib.pack_select:
                    continue                  # the workspace's bytes: as they are, every call is refused
                want = call(*a)
                text = so.pu_last_error()
                assert want in (_lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED, _lib.PU_ERR_WORKSPACE), (entry, i, v)
                assert so.pu_call_packed(entry, pack(*a)) == want and so.pu_last_error() == text, (entry, i, v)
                seen.add(text)
        assert len(seen) > 4
    assert so.pu_call_packed(5, struct.pack("<q", 0)) == _lib.PU_ERR_INVALID_ARGUMENT
    assert so.pu_call_packed(0, None) == _lib.PU_ERR_INVALID_ARGUMENT
