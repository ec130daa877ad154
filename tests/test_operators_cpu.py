"""Argument errors of the norm + rotation, page planning and grouped paged
decode entry points, without a GPU: the host checks come before any CUDA call
(pointers here are never followed)."""
from __future__ import annotations

import ctypes
import itertools
import re
from pathlib import Path

import pytest
import torch

P = 1 << 12      # 16-byte aligned, never followed
ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def lib(built_lib):
    from pallas_flash import _lib
    return _lib, _lib.lib()


def desc(**kw):
    """A valid description of 2 x 5 tokens, with changes."""
    from pallas_flash.ops import rotary
    f = dict(B=2, N=5, H=4, H_kv=2, D=64, dtype=0, R=64, inter=0, freq=P, f64=1, pos=P, pos64=0, pos_st=(0, 5, 1), axes=1,
             sizes=(32, 0, 0, 0), wq=P, wqd=2, wk=P, wkd=2, eps=1e-6, strides=(1280, 320, 64) * 7)
    f.update(kw)
    return rotary._DESC.pack(f["B"], f["N"], f["H"], f["H_kv"], f["D"], f["dtype"], f["R"], f["inter"], f["freq"], f["f64"], f["pos"],
                             f["pos64"], *f["pos_st"], f["axes"], *f["sizes"], f["wq"], f["wqd"], f["wk"], f["wkd"], f["eps"],
                             *f["strides"])


def test_description_matches_the_header():
    """The packed description has the header's fields in its order, 8 bytes each."""
    from pallas_flash.ops import rotary
    text = (ROOT / "include" / "pu_attn.h").read_text()
    body = re.search(r"typedef struct pu_qk_rope_desc \{(.*?)\} pu_qk_rope_desc;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    kinds = ""
    for line in body.split(";"):
        m = re.match(r"\s*(int64_t|double|const void\s*\*)\s*(.*)", line.strip(), re.S)
        if not m:
            continue
        for name in m.group(2).split(","):
            n = re.search(r"\[(\d+)\]", name)
            kinds += ("d" if m.group(1) == "double" else "q") * (int(n.group(1)) if n else 1)
    assert kinds == "q" * 24 + "d" + "q" * 21
    assert rotary._DESC.size == 8 * len(kinds)


BAD = [
    dict(B=0), dict(N=-1), dict(H=0), dict(H_kv=0), dict(D=0), dict(D=24), dict(D=144), dict(R=0), dict(R=80), dict(R=24),
    dict(dtype=3), dict(freq=0), dict(wqd=3), dict(wkd=9), dict(eps=-1.0), dict(eps=float("nan")), dict(axes=0), dict(axes=5),
    dict(axes=2, sizes=(16, 16, 0, 0), pos=0), dict(sizes=(31, 0, 0, 0)), dict(axes=2, sizes=(40, -8, 0, 0)),
    dict(B=1 << 20, N=1 << 20), dict(strides=(1280, 324, 64) * 7), dict(strides=(1280, 320, 60) * 7),
]


@pytest.mark.parametrize("change", BAD, ids=[str(i) for i in range(len(BAD))])
def test_descriptions_are_checked(lib, change):
    _lib, so = lib
    d = desc(**change)
    refused = (_lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED)
    assert so.pu_qk_norm_rope_fwd(d, P, P, P, P, None) in refused
    assert so.pu_last_error()
    assert so.pu_qk_norm_rope_bwd(d, P, P, P, P, P, P, P, P, P, 1 << 20, None) in refused
    one = dict(change) if "B" in change else dict(change, B=1)
    assert so.pu_qk_norm_rope_append(desc(**one), P, P, P, P, P, P, P, 0, 8, 16, 1.0, 1.0, None) in refused


def test_pointers_and_pools_are_checked(lib):
    _lib, so = lib
    inv, uns, ws = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED, _lib.PU_ERR_WORKSPACE
    d, d1 = desc(), desc(B=1)
    assert so.pu_qk_norm_rope_fwd(None, P, P, P, P, None) == inv
    for i in range(4):
        a = [P] * 4
        a[i] = None
        assert so.pu_qk_norm_rope_fwd(d, *a, None) == inv
        a[i] = P + 8
        assert so.pu_qk_norm_rope_fwd(d, *a, None) == inv
    assert so.pu_qk_norm_rope_bwd(d, P, P, P, P, None, None, None, None, None, 0, None) == inv
    assert so.pu_qk_norm_rope_bwd(d, P, P, None, P, P, P, None, None, None, 0, None) == inv
    assert so.pu_qk_norm_rope_bwd(d, P, P, P, P, None, P, P, None, P, 1 << 20, None) == inv      # a weight's gradient without its rows
    assert so.pu_qk_norm_rope_bwd(desc(wq=0), P, P, P, P, P, P, P, None, P, 1 << 20, None) == inv
    assert so.pu_qk_norm_rope_bwd(d, P, P, P, P, P, P, P, P, P, 16, None) == ws
    assert so.pu_qk_norm_rope_bwd(d, P, P, P, P, P, P, P, P, None, 1 << 20, None) == ws
    assert so.pu_qk_norm_rope_bwd_workspace_size(0) == 0 and so.pu_qk_norm_rope_bwd_workspace_size(128) > 0
    good = [P, P, P, P, P, P, P, 0, 8, 16, 1.0, 1.0, None]
    assert so.pu_qk_norm_rope_append(d, *good) == inv                  # B must be 1
    for at, bad, code in ((0, None, inv), (4, None, inv), (6, None, inv), (2, P + 2, inv), (5, P + 8, inv), (7, 2, uns), (8, 0, inv),
                          (9, 24, uns), (9, 8, uns), (9, 8192, uns), (8, 1 << 28, uns), (10, 0.0, inv), (11, float("inf"), inv)):
        a = list(good)
        a[at] = bad
        assert so.pu_qk_norm_rope_append(d1, *a) == code, (at, bad)


def test_page_plan_arguments(lib):
    _lib, so = lib
    inv, uns = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED
    Q = P + 4096
    #       table, out, width, lens, out, new, release, ring, pages, cursor, out, page, slots, pos, seq, cu, B, T, stream
    good = [P, Q, 4, P, Q, P, None, P, 8, P, Q, 16, P, P, P, P, 2, 3, None]
    for at in (0, 1, 3, 4, 5, 7, 9, 10, 12, 13, 14, 15):
        a = list(good)
        a[at] = None
        assert so.pu_page_plan(*a) == inv, at
    for at, bad, code in ((2, 0, uns), (2, 1 << 30, uns), (8, 0, inv), (11, 24, uns), (11, 8, uns), (16, 0, uns), (16, 8193, uns),
                          (17, -1, uns), (1, P, inv), (4, P, inv), (10, P, inv)):
        a = list(good)
        a[at] = bad
        assert so.pu_page_plan(*a) == code, (at, bad)


def test_grouped_paged_decode_arguments(lib):
    _lib, so = lib
    inv, uns, ws = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED, _lib.PU_ERR_WORKSPACE
    #       q, qdt, k, v, kvdt, table, width, pages, page, lens, o, lse, ws, bytes, B, H, H_kv, D, scale, ks, vs, stream
    good = [P, 0, P, P, 0, P, 4, 8, 16, P, P, None, P, 1 << 24, 2, 8, 2, 128, 0.1, 1.0, 1.0, None]
    for at, bad, code in ((0, None, inv), (2, None, inv), (5, None, inv), (9, None, inv), (10, None, inv), (12, None, ws), (13, 4096, ws),
                          (1, 2, uns), (1, 3, uns), (4, 2, uns), (6, 0, inv), (7, 0, inv), (8, 24, uns), (14, 0, inv), (15, 7, inv),
                          (16, 0, inv), (16, 3, inv), (17, 96, uns), (0, P + 8, inv), (3, P + 8, inv), (19, 0.0, inv),
                          (20, float("nan"), inv), (14, 40000, uns)):
        a = list(good)
        a[at] = bad
        assert so.pu_decode_paged_gqa(*a) == code, (at, bad)
    assert so.pu_decode_paged_gqa_workspace_size(2, 8, 3, 4, 16, 128) == 0
    assert so.pu_decode_paged_gqa_workspace_size(2, 8, 2, 4, 16, 128) > 0


def test_python_checks_come_first():
    """Host tensors and mismatched shapes are refused before the library is asked."""
    from pallas_flash.kernels.paged import DevicePagedKVCache, paged_decode, plan_append, qk_norm_rope_append
    from pallas_flash.ops.rotary import qk_norm_rope, rotary_frequencies
    z = torch.zeros
    f = z(32, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(z(1, 2, 3, 64), z(1, 1, 3, 64), f)
    with pytest.raises(ValueError, match="does not match"):
        qk_norm_rope(z(1, 2, 3, 64), z(1, 1, 4, 64), f)
    with pytest.raises(ValueError, match="B, H, N, D"):
        qk_norm_rope(z(2, 3, 64), z(1, 3, 64), f)
    with pytest.raises(ValueError, match="multiple of 16"):
        rotary_frequencies(40, device="cpu")
    i32 = lambda *s: z(*s, dtype=torch.int32)     # noqa: E731
    cursor = z(2, dtype=torch.int64)
    for bad in (dict(kv_lens=i32(3)), dict(new_lens=z(2)), dict(cursor=i32(2)), dict(page_table=z(2, 4)), dict(free_ring=z(8)),
                dict(release=z(2)), dict()):
        a = dict(page_table=i32(2, 4), kv_lens=i32(2), new_lens=i32(2), free_ring=i32(8), cursor=cursor)
        rel = bad.pop("release", None)
        a.update(bad)
        with pytest.raises(ValueError):
            plan_append(*a.values(), page_size=16, num_tokens=2, release=rel)
    with pytest.raises(ValueError):
        paged_decode(z(2, 4, 1, 64).half(), z(8, 2, 16, 64).half(), z(8, 2, 16, 64).half(), i32(2, 4), i32(2))
    with pytest.raises(ValueError, match="T, H, D"):
        qk_norm_rope_append(z(3, 4, 64), z(3, 2, 64), z(2, 2, 64), f, i32(3), i32(3), z(8, 2, 16, 64), z(8, 2, 16, 64))
    with pytest.raises(ValueError, match="page_size"):
        DevicePagedKVCache(1, 1, 64, num_pages=4, page_size=24, max_seq_len=64, device="cpu")


def test_sections_and_positions_are_checked():
    from pallas_flash.ops.rotary import _check_angles
    dev = torch.device("cpu")
    f = torch.zeros(32, dtype=torch.float64)
    pos = lambda *s: torch.zeros(*s, dtype=torch.int32)     # noqa: E731
    ok = _check_angles(f, pos(2, 5), None, 64, (2, 5), dev)
    assert ok[1:] == (64, (0, 5, 1), 1, (32, 0, 0, 0))
    assert _check_angles(f, pos(5), None, 64, (2, 5), dev)[2] == (0, 0, 1)
    assert _check_angles(f, pos(3, 2, 5), (8, 12, 12), 64, (2, 5), dev)[2:] == ((10, 5, 1), 3, (8, 12, 12, 0))
    assert _check_angles(f, pos(3, 5), (8, 12, 12), 64, (2, 5), dev)[2] == (5, 0, 1)
    assert _check_angles(f, pos(3, 5), (8, 12, 12), 64, (5,), dev)[2] == (5, 1)
    assert _check_angles(f, None, None, 64, (2, 5), dev)[2] == (0, 0, 0)
    for args in ((f, pos(2, 6), None, 64), (f, pos(5, 2), None, 64), (f, pos(2, 5), (8, 12, 12), 64), (f, None, (16, 16), 64),
                 (f, pos(3, 2, 5), (8, 12, 13), 64), (f, pos(3, 2, 5), (8, 12, 20, -8, 0), 64), (f, torch.zeros(2, 5), None, 64),
                 (f, pos(2, 5), None, 32), (torch.zeros(12, dtype=torch.float64), pos(2, 5), None, 64), (f.half(), pos(2, 5), None, 64),
                 (f, pos(1, 2, 5), (), 64)):
        with pytest.raises(ValueError):
            _check_angles(*args, (2, 5), dev)
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_grouped_paged_decode_alignment_and_page_counts(lib):
    """An output or workspace off a 16-byte boundary, and page counts whose products pass 64 bits."""
    _lib, so = lib
    inv, uns = _lib.PU_ERR_INVALID_ARGUMENT, _lib.PU_ERR_UNSUPPORTED
    good = [P, 0, P, P, 0, P, 4, 8, 16, P, P, None, P, 1 << 24, 2, 8, 2, 128, 0.1, 1.0, 1.0, None]
    for at, bad, code in ((10, P + 8, inv), (12, P + 8, inv), (6, (1 << 60) + 1, uns), (7, (1 << 60) + 1, uns), (7, 1 << 28, uns)):
        a = list(good)
        a[at] = bad
        assert so.pu_decode_paged_gqa(*a) == code, (at, bad)


@pytest.mark.parametrize("shape,stride", [
    ((2, 4, 8, 32), (1024, 1, 64, 1)), ((2, 4, 8, 32), (1024, 256, 1, 1)), ((2, 4, 8, 32), (0, 256, 32, 1)),
    ((2, 4, 8, 32), (1024, 32, 128, 1)), ((2, 4, 8, 32), (1024, 1, 4, 32)), ((1, 4, 1, 32), (7, 32, 1, 1)),
    ((2, 40, 1, 32), (0, 1, 1, 1)), ((2, 4, 64, 16), (0, 0, 1, 1)),
])
def test_gradients_have_dense_rows(shape, stride):
    """Whatever the input's strides (windows that overlap, expanded heads), a
    gradient has its own element for each and rows on 16-byte boundaries."""
    from pallas_flash.ops.rotary import _grad_like
    t = torch.empty(1 << 14, dtype=torch.float16).as_strided(shape, stride)
    g = _grad_like(t)
    assert g.shape == t.shape and g.stride(-1) == 1
    assert all(n == 1 or s % 8 == 0 for n, s in zip(shape[:-1], g.stride()))
    seen = torch.zeros(g.untyped_storage().nbytes() // 2, dtype=torch.int32)
    seen.as_strided(g.shape, g.stride()).add_(1)
    assert int(seen.sum()) == g.numel() and int(seen.max()) == 1


class _Library:
    """Stands in for libpu_attn.so: keeps what its entry points were given."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        if name.endswith("workspace_size"):
            return lambda *a: 256
        return lambda *a: self.calls.__setitem__(name, a) or 0


@pytest.fixture
def host_rotary(monkeypatch):
    """ops.rotary on host tensors, with the library's calls recorded."""
    import contextlib
    from pallas_flash import _lib
    from pallas_flash.ops import rotary
    so = _Library()
    check = rotary._check_qk

    class OnGpu:
        """A tensor's shape, type and device, as one on a GPU."""
        is_cuda = True

        def __init__(self, t):
            self.t = t

        def __getattr__(self, name):
            return getattr(self.t, name)

        def dim(self):
            return self.t.dim()

    monkeypatch.setattr(rotary, "_check_qk", lambda q, k: check(OnGpu(q), OnGpu(k)))
    monkeypatch.setattr(_lib, "lib", lambda: so)
    monkeypatch.setattr(_lib, "on_device", lambda device: contextlib.nullcontext(0))
    rotary._bwd_bytes.cache_clear()
    yield rotary, so
    rotary._bwd_bytes.cache_clear()


def _addressed(pointer, strides, shape, dtype):
    """(first, last) byte that a [..] view of these strides reads at `pointer`."""
    last = sum((n - 1) * s for n, s in zip(shape, strides))
    return pointer, pointer + (last + 1) * dtype.itemsize


@pytest.mark.parametrize("sections", [None, (8, 12, 12)])
@pytest.mark.parametrize("hooked", [False, True])
def test_backward_addresses_the_saved_tensors(host_rotary, sections, hooked):
    """What the backward is told to read lies inside tensors that are there, and holds
    the positions, also where saved-tensor hooks gave copies with other strides back."""
    import contextlib
    rotary, so = host_rotary
    B, N, H, H_kv, D = 3, 4, 4, 2, 64
    x = torch.randn(B, N, (H + H_kv) * D, dtype=torch.bfloat16)
    q = x[..., :H * D].view(B, N, H, D).transpose(1, 2).detach().requires_grad_(True)
    k = x[..., H * D:].view(B, N, H_kv, D).transpose(1, 2).detach().requires_grad_(True)
    big = torch.arange(3 * B * 100, dtype=torch.int32).view(3, B, 100)
    pos = big[:, :, 10:10 + N] if sections else big[0, :, 10:10 + N]
    freq = torch.arange(64, dtype=torch.float64)[::2]
    w = torch.ones(2 * D)[::2].requires_grad_(True)
    held = []

    def give(t):
        held.append(t.detach().clone(memory_format=torch.contiguous_format))
        return held[-1]

    hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t, give) if hooked else contextlib.nullcontext()
    with hooks:
        y = rotary.qk_norm_rope(q, k, freq, pos, q_weight=w, k_weight=w, sections=sections)
        torch.autograd.grad(y, (q, k, w), tuple(torch.ones_like(t) for t in y))
    desc, pq, pk = so.calls["pu_qk_norm_rope_bwd"][:3]
    d = rotary._DESC.unpack(desc)
    known = held + [t.detach() for t in (q, k, freq, pos, w)]
    inside = lambda lo, hi: any(t.data_ptr() <= lo and hi <= t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
                                * t.element_size() for t in known)     # noqa: E731
    assert len(d) == 46 and d[10] != 0
    strides = d[12:15]
    shape = (3, B, N) if sections else (1, B, N)
    assert inside(*_addressed(d[10], strides, shape, torch.int32))
    at = lambda i: ctypes.c_int32.from_address(d[10] + 4 * sum(a * b for a, b in zip(i, strides))).value     # noqa: E731
    want = pos if sections else pos.expand(1, B, N)
    assert all(at(i) == int(want[i]) for i in itertools.product(*map(range, shape if sections else (1, B, N))))
    for p, st, heads in ((pq, d[25:28], H), (pk, d[28:31], H_kv)):
        assert inside(*_addressed(p, tuple(st) + (1,), (B, heads, N, D), torch.bfloat16))


def test_hooks_that_give_other_tensors_back_are_refused(host_rotary):
    """A saved tensor of another type or shape is refused before the library is asked."""
    rotary, so = host_rotary
    q, k = (torch.randn(2, h, 5, 64, dtype=torch.bfloat16, requires_grad=True) for h in (4, 2))
    w = torch.ones(64, requires_grad=True)
    f, pos = torch.ones(32, dtype=torch.float64), torch.zeros(2, 5, dtype=torch.int32)
    for which, other in ((torch.float32, lambda t: t[:32]), (torch.float32, lambda t: t.double()), (torch.bfloat16, lambda t: t.float()),
                         (torch.bfloat16, lambda t: t[:, :, 1:]), (torch.bfloat16, lambda t: t.to("meta"))):
        so.calls.clear()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: other(t) if t.dtype == which else t):
            y = rotary.qk_norm_rope(q, k, f, pos, q_weight=w)
            with pytest.raises((ValueError, TypeError)):
                torch.autograd.grad(y, (q, k, w), tuple(torch.ones_like(t) for t in y))
        assert "pu_qk_norm_rope_bwd" not in so.calls


@pytest.mark.parametrize("which", ["positions", "inv_freq", "q"])
def test_inputs_changed_before_the_backward_are_refused(host_rotary, which):
    rotary, so = host_rotary
    x = {"q": torch.randn(2, 4, 5, 64), "inv_freq": torch.ones(32, dtype=torch.float64), "positions": torch.zeros(2, 5, dtype=torch.int32)}
    k = torch.randn(2, 2, 5, 64, requires_grad=True)
    y = rotary.qk_norm_rope(x["q"], k, x["inv_freq"], x["positions"])
    x[which].add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y[1], k, torch.ones_like(k))
    assert "pu_qk_norm_rope_bwd" not in so.calls


def test_forward_mode_is_refused(host_rotary):
    """An input with a tangent is refused: the result would have none, which reads as
    a derivative of zero."""
    import torch.autograd.forward_ad as fwAD
    rotary, so = host_rotary
    f, w = torch.ones(32, dtype=torch.float64), torch.ones(64)
    pos = torch.zeros(2, 5, dtype=torch.int32)
    with fwAD.dual_level():
        for which in range(5):
            a = [torch.randn(2, 4, 5, 64), torch.randn(2, 2, 5, 64), f, w, w]
            a[which] = fwAD.make_dual(a[which], torch.ones_like(a[which]))
            for call in (rotary.qk_norm_rope, rotary.qk_norm_rope_forward):
                so.calls.clear()
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(a[0], a[1], a[2], pos, q_weight=a[3], k_weight=a[4])
                assert not so.calls
        q, k, v = (torch.randn(5, h, 64) for h in (4, 2, 2))
        from pallas_flash.kernels.paged import _refuse_tangents
        _refuse_tangents(q, k, v, None)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _refuse_tangents(q, k, fwAD.make_dual(v, v), None)
        # a tangent of an output's gradient
        q = torch.randn(2, 4, 5, 64, requires_grad=True)
        y, _ = rotary.qk_norm_rope(q, torch.randn(2, 2, 5, 64), f, pos)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, q, fwAD.make_dual(torch.ones_like(y), torch.ones_like(y)))
        so.calls.clear()
        # no tangent: served
        rotary.qk_norm_rope(torch.randn(2, 4, 5, 64), torch.randn(2, 2, 5, 64), f, pos)
        assert "pu_qk_norm_rope_fwd" in so.calls


def test_frequencies_that_want_a_gradient_are_refused(host_rotary):
    """There is none by the frequencies: asked for one, the call says so."""
    rotary, so = host_rotary
    q, k = torch.randn(2, 4, 5, 64, requires_grad=True), torch.randn(2, 2, 5, 64)
    f = torch.ones(32, dtype=torch.float64, requires_grad=True)
    for x in (q, q.detach()):
        with pytest.raises(ValueError, match="frequencies"):
            rotary.qk_norm_rope(x, k, f)
    assert not so.calls
    rotary.qk_norm_rope(q, k, f.detach())
    with torch.no_grad():
        rotary.qk_norm_rope(q, k, f)


def test_page_plan_in_place_counts(lib):
    """In place, the new counts may not lie where the lengths are written."""
    _lib, so = lib
    Q, B = P + 4096, 2
    a = [P, P, 4, P, P, Q, None, P, 8, P, P, 16, P, P, P, P, B, 3, None]
    for new in (P, P + 4, P - 4):
        assert so.pu_page_plan(*a[:5], new, *a[6:]) == _lib.PU_ERR_INVALID_ARGUMENT, new


def test_batch_limits_of_grouped_paged_decode(lib):
    """Up to 8192 sequences whatever their heads on the tensor core (what is refused
    then is the workspace); the query-head kernel counts 65535 heads of sequences."""
    _lib, so = lib
    uns, ws = _lib.PU_ERR_UNSUPPORTED, _lib.PU_ERR_WORKSPACE
    good = [P, 0, P, P, 0, P, 4, 8, 16, P, P, None, P, 1, 2, 8, 2, 128, 0.1, 1.0, 1.0, None]
    for B, H, H_kv, kv, D, code in ((1024, 64, 8, 0, 128, ws), (8192, 64, 8, 0, 128, ws), (8192, 64, 8, 3, 128, ws), (8193, 64, 8, 0, 128, uns),
                                    (16000, 4, 2, 0, 128, ws), (1024, 64, 8, 1, 128, uns), (1024, 64, 8, 3, 64, uns), (1, 1 << 20, 8, 0, 128, uns),
                                    (8192, 1 << 20, 1 << 19, 0, 64, uns)):
        a = list(good)
        a[4], a[14], a[15], a[16], a[17] = kv, B, H, H_kv, D
        assert so.pu_decode_paged_gqa(*a) == code, (B, H, H_kv, kv, D)
    assert so.pu_decode_paged_gqa_workspace_size(8192, 64, 8, 4, 16, 128) >= so.pu_decode_paged_gqa_workspace_size(1, 64, 8, 4, 16, 128)


def test_captured_scratch_clears_its_counters_only(monkeypatch):
    """A captured call's own scratch: as many zeroed bytes as its kernels count in, and
    the question whether a capture runs is asked of the device that was named."""
    from pallas_flash.kernels.decoding import DecodeWorkspace
    asked = []
    monkeypatch.setattr(DecodeWorkspace, "_capturing", staticmethod(lambda device: asked.append(device) or True))
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: empty(*a, **kw).fill_(255))
    for counters in (4, 592, 8192, 1 << 18, 1 << 19):
        buf = DecodeWorkspace.get(torch.device("cpu"), (1 << 18) + 4096, counters)
        used = min(counters, 1 << 18)
        assert buf.numel() >= (1 << 18) + 4096 and int((buf == 0).sum()) == used and not buf[:used].any()
    assert asked == [torch.device("cpu")] * 5
