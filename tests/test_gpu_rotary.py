"""Norm and rotation of queries and keys (pu_qk_norm_rope_fwd, _bwd) against
the formula in 64 bits.

Tolerances, element by element.  A result is rounded once to its type (half a
step: eps/2 of the value) after fp32 work: the sum of D squares is a chain of
at most 16 + 3 roundings of positive terms (halved by the root), the root 2
ulp, and about 14 more for the products, the sine and cosine (2 ulp) and the
angle (2^-25 of half a turn): under 32 roundings of 2^-24 of the pair's
magnitude |a| + |b|.  The gradient adds a dot product (19 roundings of the sum
of magnitudes) and four products: 48 roundings of its terms' magnitudes.  A
weight gradient sums rows one after the other: rows/8 + 64 roundings of the
sum of magnitudes cover the longest chain of these shapes.
"""
from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

from helpers import assert_close_grad, assert_close_o, to_np

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def rot(built_lib):
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    from pallas_flash import _lib
    from pallas_flash.ops import rotary
    _lib.device_status()
    return rotary


def _gen(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _turns(f, pos, sections, B, N):
    """cos, sin fp64 [B, 1, N, R/2]."""
    f = f.double()
    if pos is None:
        pos = torch.arange(N, device="cuda")
    if sections is None:
        t = pos.double().expand(B, N).unsqueeze(-1) * f
    else:
        parts, at = [], 0
        for a, n in enumerate(sections):
            parts.append(pos[a].double().expand(B, N).unsqueeze(-1) * f[at:at + n])
            at += n
        t = torch.cat(parts, -1)
    return t.cos().unsqueeze(1), t.sin().unsqueeze(1)


def _pairs(n, R, inter):
    return (n[..., 0:R:2], n[..., 1:R:2]) if inter else (n[..., :R // 2], n[..., R // 2:R])


def _join(a, b, rest, inter):
    y = torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)
    return torch.cat((y, rest), -1)


def _oracle(x, w, cos, sin, inter, eps):
    """(result, magnitude |a| + |b| of each value's pair) in 64 bits."""
    x = x.double()
    R = 2 * cos.shape[-1]
    n = x if w is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    a, b = _pairs(n, R, inter)
    y = _join(a * cos - b * sin, b * cos + a * sin, n[..., R:], inter)
    m = a.abs() + b.abs()
    return y, _join(m, m, n[..., R:].abs(), inter)


def _oracle_back(x, w, g, cos, sin, inter, eps):
    """(dx, magnitude of its terms, dw, magnitude of its terms) in 64 bits."""
    x, g = x.double(), g.double()
    R, D = 2 * cos.shape[-1], x.shape[-1]
    a, b = _pairs(g, R, inter)
    h = _join(a * cos + b * sin, b * cos - a * sin, g[..., R:], inter)
    m = _join(a.abs() + b.abs(), a.abs() + b.abs(), g[..., R:].abs(), inter)
    if w is None:
        return h, m, None, None
    w = w.double()
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    dx = r * (h * w - x * r * r * (h * w * x).mean(-1, keepdim=True))
    dxm = r * (m * w.abs() + x.abs() * r * r * (m * w.abs() * x.abs()).mean(-1, keepdim=True))
    return dx, dxm, (h * x * r).sum((0, 1, 2)), (m * x.abs() * r).sum((0, 1, 2))


def _close(got, want, mag, steps, what):
    half = torch.finfo(got.dtype).eps / 2
    # a result below the type's smallest normal value is off by up to half its smallest step
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    tol = half * want.abs() + steps * U * mag + tiny
    err = (got.double() - want).abs()
    bad = err > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((err / tol).max()):.2f} of the tolerance"


CASES = [
    # B, N, H, H_kv, D, R, dtype, weights, interleaved, sections
    (2, 33, 4, 2, 128, 128, torch.bfloat16, torch.float32, False, None),
    (1, 1, 1, 1, 64, 64, torch.float16, torch.float16, False, None),
    (3, 17, 5, 3, 96, 32, torch.float32, torch.float32, True, None),
    (2, 129, 7, 1, 80, 80, torch.bfloat16, torch.bfloat16, True, None),
    (1, 1000, 32, 8, 128, 64, torch.float16, torch.bfloat16, False, None),
    (2, 50, 16, 2, 64, 64, torch.bfloat16, torch.float32, False, (8, 12, 12)),
    (2, 31, 3, 2, 128, 96, torch.float32, torch.float32, True, (16, 0, 20, 12)),
    (1, 5, 9, 9, 16, 16, torch.float32, torch.float32, False, (8,)),
    (2, 40, 4, 4, 112, 48, torch.bfloat16, None, False, None),
    (4, 700, 40, 8, 128, 128, torch.bfloat16, torch.float32, False, None),
]


def _inputs(case, seed=0):
    B, N, H, H_kv, D, R, dt, wdt, inter, sections = case
    # heads beside each other in one projection, as a model has them
    x = _gen((B, N, (H + H_kv) * D), 1 + seed, dt, 2.0)
    q = x[..., :H * D].view(B, N, H, D).transpose(1, 2)
    k = x[..., H * D:].view(B, N, H_kv, D).transpose(1, 2)
    wq, wk = (None, None) if wdt is None else ((1 + 0.2 * _gen((D,), s)).to(wdt) for s in (2, 3))
    f = torch.pow(torch.tensor(1e4, dtype=torch.float64), -torch.arange(0, R, 2, dtype=torch.float64) / R).cuda()
    if sections is None:
        pos = torch.randint(0, 1 << 20, (B, N), device="cuda", dtype=torch.int32)
    else:
        pos = torch.randint(0, 5000, (len(sections), B, N), device="cuda", dtype=torch.int64)
    return q, k, wq, wk, f, pos, sections, inter


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_forward_and_backward(rot, case):
    B, N, H, H_kv, D, R, dt, wdt, inter, sections = case
    eps = 1e-5
    q, k, wq, wk, f, pos, sections, inter = _inputs(case)
    cos, sin = _turns(f, pos, sections, B, N)
    leaves = [t.detach().requires_grad_(True) for t in (q, k) + (() if wq is None else (wq, wk))]
    lq, lk = leaves[:2]
    lwq, lwk = leaves[2:] if wq is not None else (None, None)
    yq, yk = rot.qk_norm_rope(lq, lk, f, pos, q_weight=lwq, k_weight=lwk, eps=eps, sections=sections, interleaved=inter)
    assert yq.shape == q.shape and yk.shape == k.shape and yq.dtype == dt
    assert yq.is_contiguous() and yk.is_contiguous()
    gq, gk = _gen(q.shape, 11, dt), _gen(k.shape, 12, dt)
    grads = torch.autograd.grad((yq, yk), leaves, (gq, gk))
    for i, (x, w, g, y) in enumerate(((q, wq, gq, yq), (k, wk, gk, yk))):
        want, mag = _oracle(x, w, cos, sin, inter, eps)
        _close(y.detach(), want, mag, 32, f"output {i}")
        dx, dxm, dw, dwm = _oracle_back(x, w, g, cos, sin, inter, eps)
        assert grads[i].dtype == dt and grads[i].shape == x.shape
        _close(grads[i], dx, dxm, 48, f"gradient {i}")
        if w is not None:
            assert grads[2 + i].dtype == w.dtype
            rows = B * N * (H, H_kv)[i]
            _close(grads[2 + i], dw, dwm, rows / 8 + 64, f"weight gradient {i}")
    # the gradient of a projection's view keeps its heads beside each other
    assert N == 1 or H == 1 or grads[0].stride(1) == D


@pytest.mark.parametrize("inter", [False, True])
def test_gradient_against_differences(rot, inter):
    """Central differences of the kernel's own fp32 forward along a random
    direction.  Tolerance: the roundings of the two sums (32 of 2^-24 of the
    terms' magnitudes, over the step) and what the step itself leaves, twice
    its value in 64 bits."""
    B, N, H, H_kv, D, R = 1, 6, 2, 1, 64, 32
    case = (B, N, H, H_kv, D, R, torch.float32, torch.float32, inter, None)
    q, k, wq, wk, f, pos, _, _ = _inputs(case)
    gq, gk = _gen(q.shape, 21), _gen(k.shape, 22)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
    y = rot.qk_norm_rope(leaves[0], leaves[1], f, pos, q_weight=leaves[2], k_weight=leaves[3], interleaved=inter)
    grads = torch.autograd.grad(y, leaves, (gq, gk))
    cos, sin = _turns(f, pos, None, B, N)
    h = 2.0 ** -6

    def in64(q, k, wq, wk):
        return sum((_oracle(x, w, cos, sin, inter, 1e-6)[0] * g.double()).sum() for x, w, g in ((q, wq, gq), (k, wk, gk)))

    for which in range(4):
        d = _gen(leaves[which].shape, 30 + which)
        at = lambda s: [t.detach() + s * d if i == which else t.detach() for i, t in enumerate(leaves)]   # noqa: E731
        total, mags = [], 0.0
        for s in (h, -h):
            a = at(s)
            yq, yk = rot.qk_norm_rope_forward(a[0], a[1], f, pos, q_weight=a[2], k_weight=a[3], interleaved=inter)
            total.append((yq.double() * gq.double()).sum() + (yk.double() * gk.double()).sum())
            for x, w, g in ((a[0], a[2], gq), (a[1], a[3], gk)):
                mags += float((_oracle(x, w, cos, sin, inter, 1e-6)[1] * g.double().abs()).sum())
        got = float((total[0] - total[1]) / (2 * h))
        want = float((grads[which].double() * d.double()).sum())
        d64 = d.double()
        at64 = lambda s: [t.detach().double() + s * d64 if i == which else t.detach().double() for i, t in enumerate(leaves)]   # noqa: E731
        step = float((in64(*at64(h)) - in64(*at64(-h))) / (2 * h))
        tiny = h / 64
        exact = float((in64(*at64(tiny)) - in64(*at64(-tiny))) / (2 * tiny))
        assert abs(got - want) <= 32 * U * mags / (2 * h) + 2 * abs(step - exact) + 1e-5 * abs(want)


def test_far_positions(rot):
    """Angles stay exact to fp32 up to 2^31 - 1 (a position times a frequency in
    fp32 would be off by whole turns) and for negative positions."""
    D = 64
    pos = torch.tensor([0, 1, 131071, (1 << 24) + 1, (1 << 31) - 1, -1, -12345678], dtype=torch.int64, device="cuda")
    N = pos.numel()
    q, k = _gen((1, 2, N, D), 1), _gen((1, 1, N, D), 2)
    f = rot.rotary_frequencies(D, theta=1e4)
    y, _ = rot.qk_norm_rope(q, k, f, pos)
    # 64-bit angles carry 2^-53 of up to 2^31 turns: 2^-22 of a turn, about 2^-19 rad at the far end
    cos, sin = _turns(f, pos, None, 1, N)
    want, mag = _oracle(q, None, cos, sin, False, 0.0)
    tol = 32 * U * mag + (pos.abs().double() * 2.0 ** -51).view(1, 1, N, 1) * mag
    assert ((y.double() - want).abs() <= tol).all()
    y32, _ = rot.qk_norm_rope(q[:, :, 2:4].contiguous(), k[:, :, 2:4].contiguous(), f, pos[2:4].int())
    assert torch.equal(y32, y[:, :, 2:4])
    # frequencies held in fp32 are taken as those values
    y_f32, _ = rot.qk_norm_rope(q[:, :, :3].contiguous(), k[:, :, :3].contiguous(), f.float(), pos[:3])
    cos, sin = _turns(f.float(), pos[:3], None, 1, 3)
    want, mag = _oracle(q[:, :, :3], None, cos, sin, False, 0.0)
    _close(y_f32, want, mag, 32, "fp32 frequencies")


def test_strides_alignment_and_defaults(rot):
    """Views that the kernel reads in place, and ones that go through a copy;
    positions that are left out, shared by sequences or strided."""
    B, N, H, D = 2, 9, 3, 64
    f = rot.rotary_frequencies(D)
    w = 1 + 0.1 * _gen((D,), 5)
    base = _gen((B, H, N, D), 1, torch.bfloat16)
    k = _gen((B, 1, N, D), 2, torch.bfloat16)
    want = rot.qk_norm_rope(base, k, f, q_weight=w, k_weight=w)
    odd = torch.empty(base.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(B, H, N, D).copy_(base)
    assert odd.data_ptr() % 16
    wide = torch.zeros((B, H, N, D + 4), dtype=torch.bfloat16, device="cuda")
    wide[..., :D] = base
    turned = base.transpose(2, 3).contiguous().transpose(2, 3)
    every = torch.empty((B, N, 2 * H, D), dtype=torch.bfloat16, device="cuda").transpose(1, 2)[:, ::2]
    every.copy_(base)
    for q in (odd, wide[..., :D], turned, every):
        got = rot.qk_norm_rope(q, k, f, q_weight=w, k_weight=w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        leaf = q.detach().requires_grad_(True)
        y, _ = rot.qk_norm_rope(leaf, k, f, q_weight=w, k_weight=w)
        g = _gen((B, H, N, D), 8, torch.bfloat16)
        (dq,) = torch.autograd.grad(y, leaf, g)
        ref = base.detach().requires_grad_(True)
        yr, _ = rot.qk_norm_rope(ref, k, f, q_weight=w, k_weight=w)
        (dr,) = torch.autograd.grad(yr, ref, g)
        assert torch.equal(dq, dr)
    pos = torch.arange(N, device="cuda", dtype=torch.int32)
    for p in (pos, pos.long(), pos.expand(B, N), torch.arange(2 * N, device="cuda", dtype=torch.int32)[::2] // 2):
        got = rot.qk_norm_rope(base, k, f, p, q_weight=w, k_weight=w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_overlapping_windows(rot):
    """Rows that share elements (windows of one buffer): read as they are or
    through a copy, and a gradient of its own for every row."""
    B, H, N, D = 2, 4, 8, 32
    f = rot.rotary_frequencies(D)
    w = 1 + 0.1 * _gen((D,), 5)
    buf = _gen((4096,), 1, torch.bfloat16)
    k = _gen((B, 1, N, D), 2, torch.bfloat16)
    gq, gk = _gen((B, H, N, D), 3, torch.bfloat16), _gen((B, 1, N, D), 4, torch.bfloat16)
    for st in ((1024, 1, 64, 1), (1024, 256, 1, 1), (8, 16, 32, 1), (0, 8, 16, 1)):
        q = buf.as_strided((B, H, N, D), st)
        got = rot.qk_norm_rope_backward(gq, gk, q, k, f, q_weight=w, k_weight=w)
        want = rot.qk_norm_rope_backward(gq, gk, q.contiguous(), k, f, q_weight=w, k_weight=w)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), st
        leaf = buf.clone().requires_grad_(True)
        y, _ = rot.qk_norm_rope(leaf.as_strided((B, H, N, D), st), k, f, q_weight=w, k_weight=w)
        assert torch.equal(y, rot.qk_norm_rope(q.contiguous(), k, f, q_weight=w, k_weight=w)[0])
        (grad,) = torch.autograd.grad(y, leaf, gq)
        assert torch.isfinite(grad).all()


@pytest.mark.parametrize("H,H_kv,D", [(3, 1, 128), (5, 2, 64), (9, 7, 96)])
def test_no_epsilon(rot, H, H_kv, D):
    """eps = 0 with head counts that leave lanes without a row, whose 0 / 0 must reach
    no sum; the gradients of the weights are those of the rows that are there."""
    B, N = 2, 37
    f = rot.rotary_frequencies(64 if D == 128 else 32)
    q, k = _gen((B, H, N, D), 1, torch.bfloat16), _gen((B, H_kv, N, D), 2, torch.bfloat16)
    w = 1 + 0.2 * _gen((D,), 3)
    gq, gk = _gen(q.shape, 4, torch.bfloat16), _gen(k.shape, 5, torch.bfloat16)
    got = rot.qk_norm_rope_backward(gq, gk, q, k, f, q_weight=w, k_weight=w, eps=0.0)
    cos, sin = _turns(f, None, None, B, N)
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        dx, dxm, dw, dwm = _oracle_back(x, w, g, cos, sin, False, 0.0)
        _close(got[i], dx, dxm, 48, f"gradient {i}")
        _close(got[2 + i], dw, dwm, B * N * x.shape[1] / 8 + 64, f"weight gradient {i}")


@pytest.mark.parametrize("T", [2367, 2368, 2369, 3551, 3553, 5000])
def test_token_counts_around_a_round_of_warps(rot, T):
    """Counts at which the tokens behind the last full round are cut differently,
    in sequences shorter than a round: the same rows as alone."""
    B = 7 if T % 7 == 0 else 1
    H, H_kv, D = 6, 2, 128
    f = rot.rotary_frequencies(D)
    w = 1 + 0.2 * _gen((D,), 3)
    for b in {1, B}:
        n = T // b
        q, k = _gen((b, H, n, D), 1, torch.bfloat16), _gen((b, H_kv, n, D), 2, torch.bfloat16)
        gq, gk = _gen(q.shape, 4, torch.bfloat16), _gen(k.shape, 5, torch.bfloat16)
        pos = torch.randint(0, 1 << 20, (b, n), device="cuda", dtype=torch.int32)
        yq, yk = rot.qk_norm_rope_forward(q, k, f, pos, q_weight=w, k_weight=w)
        dq, dk, dwq, dwk = rot.qk_norm_rope_backward(gq, gk, q, k, f, pos, q_weight=w, k_weight=w)
        cos, sin = _turns(f, pos, None, b, n)
        for i, (x, g, y, d, dw) in enumerate(((q, gq, yq, dq, dwq), (k, gk, yk, dk, dwk))):
            want, mag = _oracle(x, w, cos, sin, False, 1e-6)
            _close(y, want, mag, 32, f"output {i}")
            dx, dxm, dwr, dwm = _oracle_back(x, w, g, cos, sin, False, 1e-6)
            _close(d, dx, dxm, 48, f"gradient {i}")
            _close(dw, dwr, dwm, T * x.shape[1] / 8 + 64, f"weight gradient {i}")


def test_broadcast_inputs_and_gradients(rot):
    """A key head expanded over the batch, and a gradient that is one value
    expanded over the output: sums of the rows' gradients."""
    B, N, H, D = 3, 20, 2, 64
    f, w = rot.rotary_frequencies(D), (1 + 0.1 * _gen((D,), 5)).requires_grad_(True)
    q = _gen((B, H, N, D), 1)
    k1 = _gen((1, 1, N, D), 2).requires_grad_(True)
    yq, yk = rot.qk_norm_rope(q, k1.expand(B, 1, N, D), f, q_weight=w, k_weight=w)
    dk, dw = torch.autograd.grad(yk.sum(), (k1, w))
    cos, sin = _turns(f, None, None, B, N)
    ones = torch.ones((B, 1, N, D), device="cuda")
    dx, dxm, dwr, dwm = _oracle_back(k1.detach().expand(B, 1, N, D), w.detach(), ones, cos, sin, False, 1e-6)
    _close(dk, dx.sum(0, keepdim=True), dxm.sum(0, keepdim=True), 60, "shared key")
    _close(dw, dwr, dwm, 100, "shared weight")     # the unused query output adds nothing
    assert torch.equal(dw, torch.autograd.grad(rot.qk_norm_rope(q, k1.expand(B, 1, N, D), f, q_weight=w, k_weight=w)[1].sum(), w)[0])


def test_partial_requirements(rot):
    """Only what asks for a gradient gets one; a second derivative is refused."""
    q, k = _gen((1, 2, 4, 32), 1), _gen((1, 1, 4, 32), 2)
    f = rot.rotary_frequencies(32)
    w = _gen((32,), 3).requires_grad_(True)
    yq, yk = rot.qk_norm_rope(q, k, f, q_weight=w, k_weight=None)
    assert yq.requires_grad
    (dw,) = torch.autograd.grad(yq.square().sum(), w)
    assert dw.shape == (32,) and torch.isfinite(dw).all()
    qa = q.clone().requires_grad_(True)
    y, _ = rot.qk_norm_rope(qa, k, f)
    (d,) = torch.autograd.grad(y.square().sum(), qa, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), qa)
    with torch.no_grad():
        assert not rot.qk_norm_rope(qa, k, f)[0].requires_grad


def test_values_out_of_range_stay_in_their_rows(rot):
    """NaN or infinity in one row reaches that row alone; without a norm, values
    behind the rotation are copied as they are; an all-zero row gives zeros and
    finite gradients."""
    N, D, R = 6, 64, 32
    f = rot.rotary_frequencies(R)
    w = 1 + 0.1 * _gen((D,), 4)
    q, k = _gen((1, 2, N, D), 1), _gen((1, 1, N, D), 2)
    clean, _ = rot.qk_norm_rope(q, k, f, q_weight=w)
    bad = q.clone()
    bad[0, 1, 2, 5] = math.nan
    bad[0, 0, 4, 40] = math.inf
    bad[0, 0, 5] = 0
    leaf = bad.clone().requires_grad_(True)
    y, _ = rot.qk_norm_rope(leaf, k, f, q_weight=w)
    hit = torch.zeros((1, 2, N), dtype=torch.bool, device="cuda")
    hit[0, 1, 2] = hit[0, 0, 4] = hit[0, 0, 5] = True
    assert torch.equal(y[~hit], clean[~hit])
    assert y[0, 1, 2].isnan().all() and (y[0, 0, 5] == 0).all()
    (d,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    rest = torch.ones_like(hit)
    rest[0, 1, 2] = rest[0, 0, 4] = False
    assert torch.isfinite(d[rest]).all()
    plain, _ = rot.qk_norm_rope(bad, k, f)
    assert plain[0, 0, 4, 40] == math.inf and torch.isfinite(plain[0, 0, 4, :R]).all()
    assert torch.equal(plain[0, 0, 4, R:], bad[0, 0, 4, R:])


def test_reproducible_and_captured(rot):
    """The same bits every time; captured into a graph with its backward and
    replayed on new inputs, also while another stream runs the same call."""
    case = (2, 300, 8, 2, 128, 128, torch.bfloat16, torch.float32, False, None)
    q, k, wq, wk, f, pos, _, _ = _inputs(case)
    gq, gk = _gen(q.shape, 11, q.dtype), _gen(k.shape, 12, k.dtype)
    kw = dict(q_weight=wq, k_weight=wk)
    first = rot.qk_norm_rope_forward(q, k, f, pos, **kw) + rot.qk_norm_rope_backward(gq, gk, q, k, f, pos, **kw)
    for _ in range(3):
        again = rot.qk_norm_rope_forward(q, k, f, pos, **kw) + rot.qk_norm_rope_backward(gq, gk, q, k, f, pos, **kw)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    sq, sk = q.clone(), k.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rot.qk_norm_rope_forward(sq, sk, f, pos, **kw) + rot.qk_norm_rope_backward(gq, gk, sq, sk, f, pos, **kw)
    other = _inputs(case, seed=50)
    sq.copy_(other[0])
    sk.copy_(other[1])
    graph.replay()
    with torch.cuda.stream(side):
        at_once = rot.qk_norm_rope_backward(gq, gk, q, k, f, pos, **kw)
    torch.cuda.synchronize()
    want = rot.qk_norm_rope_forward(other[0], other[1], f, pos, **kw) + \
        rot.qk_norm_rope_backward(gq, gk, other[0], other[1], f, pos, **kw)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert all(torch.equal(a, b) for a, b in zip(at_once, first[2:]))


def test_empty(rot):
    f = rot.rotary_frequencies(64)
    w = torch.ones(64, device="cuda").requires_grad_(True)
    q = torch.empty((2, 3, 0, 64), device="cuda", requires_grad=True)
    k = torch.empty((2, 1, 0, 64), device="cuda")
    yq, yk = rot.qk_norm_rope(q, k, f, q_weight=w, k_weight=w)
    assert yq.shape == q.shape and yk.shape == k.shape
    dq, dw = torch.autograd.grad(yq.sum(), (q, w))
    assert dq.shape == q.shape and (dw == 0).all()


def test_more_than_2_31_elements(rot):
    """Rows whose offsets pass 2^31 elements and 2^32 bytes: the last tokens equal
    the same tokens in a small call, forward and backward."""
    H, N, D = 20, 900_001, 128
    f, w = rot.rotary_frequencies(D), 1 + 0.1 * _gen((D,), 5)
    q = torch.empty((1, H, N, D), dtype=torch.bfloat16, device="cuda")
    q.random_(-8, 9)
    k = q[:, :1, :, :]
    pos = torch.arange(N, device="cuda", dtype=torch.int32)
    y, yk = rot.qk_norm_rope_forward(q, k, f, pos, q_weight=w, k_weight=w)
    dq, dk, dw, _ = rot.qk_norm_rope_backward(y, yk, q, k, f, pos, q_weight=w, k_weight=w)
    for at in (slice(0, 50), slice(N - 50, N)):
        a, b = (t[:, :, at].contiguous() for t in (q, k))
        ya, yb = rot.qk_norm_rope_forward(a, b, f, pos[at].contiguous(), q_weight=w, k_weight=w)
        assert torch.equal(ya, y[:, :, at]) and torch.equal(yb, yk[:, :, at])
        da, db, _, _ = rot.qk_norm_rope_backward(ya, yb, a, b, f, pos[at].contiguous(), q_weight=w, k_weight=w)
        assert torch.equal(da, dq[:, :, at]) and torch.equal(db, dk[:, :, at])
    assert torch.isfinite(dw).all()


def test_threads_and_streams(rot):
    """Calls from several host threads, each on its own stream."""
    import threading
    case = (2, 200, 8, 2, 128, 128, torch.bfloat16, torch.float32, False, None)
    sets = [_inputs(case, seed=60 + i) for i in range(4)]
    want = [rot.qk_norm_rope_forward(q, k, f, p, q_weight=wq, k_weight=wk) for q, k, wq, wk, f, p, _, _ in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        q, k, wq, wk, f, p, _, _ = sets[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                a = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
                y = rot.qk_norm_rope(a[0], a[1], f, p, q_weight=a[2], k_weight=a[3])
                torch.autograd.grad(y, a, y)
                if not all(torch.equal(u, v) for u, v in zip(y, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not bad


def test_training_chain(rot):
    """Projection -> norm and rotation -> causal attention -> gradients, against
    the same chain in 64 bits (the attention's own bar for outputs and
    gradients: bf16 products inside)."""
    from pallas_flash.ops.interface import pallas_flash_attention
    B, N, H, D = 2, 160, 3, 128
    x = _gen((B, N, 3 * H * D), 1, torch.bfloat16)
    wq, wk = ((1 + 0.1 * _gen((D,), s)) for s in (2, 3))
    f = rot.rotary_frequencies(D)
    do = _gen((B, H, N, D), 4, torch.bfloat16)

    def split(t):
        return [p.view(B, N, H, D).transpose(1, 2) for p in t.split(H * D, -1)]

    leaf = x.clone().requires_grad_(True)
    ws = [w.clone().requires_grad_(True) for w in (wq, wk)]
    q, k, v = split(leaf)
    q, k = rot.qk_norm_rope(q, k, f, q_weight=ws[0], k_weight=ws[1])
    o = pallas_flash_attention(q, k, v, causal=True)
    got = torch.autograd.grad(o, [leaf] + ws, do)

    leaf64 = x.double().requires_grad_(True)
    ws64 = [w.double().requires_grad_(True) for w in (wq, wk)]
    q, k, v = split(leaf64)
    cos, sin = _turns(f, None, None, B, N)
    q, k = (_oracle(t, w, cos, sin, False, 1e-6)[0] for t, w in ((q, ws64[0]), (k, ws64[1])))
    s = (q @ k.transpose(2, 3)) / math.sqrt(D)
    s = s.masked_fill(torch.ones(N, N, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    o64 = s.softmax(-1) @ v
    want = torch.autograd.grad(o64, [leaf64] + ws64, do.double())
    assert_close_o(to_np(o), to_np(o64), what="chain")
    for n, a, b in zip(("x", "wq", "wk"), got, want):
        assert_close_grad(to_np(a), to_np(b), what=n)


def test_saved_tensor_hooks(rot):
    """Gradients are the same where hooks copy the saved tensors (to the host and
    back, or to a dense tensor): views of positions, weights and inputs."""
    for sections in (None, (8, 12, 12)):
        B, N, H, H_kv, D = 3, 17, 4, 2, 64
        x = _gen((B, N, (H + H_kv) * D), 1, torch.bfloat16)
        q = x[..., :H * D].view(B, N, H, D).transpose(1, 2)
        k = x[..., H * D:].view(B, N, H_kv, D).transpose(1, 2)
        big = torch.randint(0, 10000, (3, B, 100), device="cuda", dtype=torch.int32)
        pos = big[:, :, 10:10 + N] if sections else big[1, :, 10:10 + N]
        f = rot.rotary_frequencies(2 * D).contiguous()[::2]
        w = (1 + 0.1 * _gen((2 * D,), 3))[::2]
        gq, gk = _gen((B, H, N, D), 4, torch.bfloat16), _gen((B, H_kv, N, D), 5, torch.bfloat16)

        def grads(hooks):
            a = [t.detach().requires_grad_(True) for t in (q, k, w, w)]
            with hooks:
                y = rot.qk_norm_rope(a[0], a[1], f, pos, q_weight=a[2], k_weight=a[3], sections=sections)
                return torch.autograd.grad(y, a, (gq, gk))

        import contextlib
        want = grads(contextlib.nullcontext())
        clone = lambda t: t.detach().clone(memory_format=torch.contiguous_format)     # noqa: E731
        for hooks in (torch.autograd.graph.saved_tensors_hooks(clone, lambda t: t), torch.autograd.graph.save_on_cpu()):
            got = grads(hooks)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), sections


def test_forward_mode_is_refused(rot):
    import torch.autograd.forward_ad as fwAD
    q, k = _gen((1, 2, 4, 32), 1), _gen((1, 1, 4, 32), 2)
    f = rot.rotary_frequencies(32)
    with fwAD.dual_level():
        for a, b in ((fwAD.make_dual(q, q), k), (q, fwAD.make_dual(k, k)), (fwAD.make_dual(q.clone().requires_grad_(True), q), k)):
            with pytest.raises(NotImplementedError):
                rot.qk_norm_rope(a, b, f)
        with pytest.raises(NotImplementedError):
            rot.qk_norm_rope(q, k, f, q_weight=fwAD.make_dual(q[0, 0, 0].clone(), q[0, 0, 1].clone()))
        leaf = q.clone().requires_grad_(True)
        y, _ = rot.qk_norm_rope(leaf, k, f)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, leaf, fwAD.make_dual(q, q))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: rot.qk_norm_rope(x, k, f)[0], (q,), (q,))


# 2 pi to 60 digits: turns of far positions are worked out in whole numbers
_TWO_PI = 2 * Fraction(314159265358979323846264338327950288419716939937510582097494, 10 ** 59)


def _sine_cosine(f, pos):
    """sin, cos [positions, pairs] in 64 bits of position * f, reduced to half a turn exactly."""
    s, c = [], []
    for p in pos.tolist():
        row = []
        for x in f.tolist():
            turn = Fraction(x) * p / _TWO_PI
            row.append(float((turn - round(turn)) * _TWO_PI))
        s.append([math.sin(a) for a in row])
        c.append([math.cos(a) for a in row])
    return (torch.tensor(t, dtype=torch.float64, device="cuda") for t in (s, c))


def _one_hot_turns(rot, f, pos, inter):
    """sin and cos that the kernels turn with, forward and backward: rows with a 1 as a
    pair's first value, and no norm, hold the pair's cosine and sine."""
    R, N = 2 * f.numel(), pos.numel()
    first = torch.arange(R // 2, device="cuda") * (2 if inter else 1)
    second = first + (1 if inter else R // 2)
    q = torch.zeros((1, 1, N, R), device="cuda")
    q[..., first] = 1
    y, _ = rot.qk_norm_rope_forward(q, q, f, pos, interleaved=inter)
    dq, _, _, _ = rot.qk_norm_rope_backward(q, None, q, q, f, pos, interleaved=inter)
    return (y[0, 0][:, second], y[0, 0][:, first]), (-dq[0, 0][:, second], dq[0, 0][:, first])


@pytest.mark.parametrize("inter", [False, True])
def test_small_angles_keep_their_precision(rot, inter):
    """Sines of small angles to 8 roundings of 2^-24 of themselves: the angle's
    conversion, constant and product (3), the fixed-point fraction (2^-64 of a turn in 2^-23
    of one), the series (2 and its last product's part)."""
    f = rot.rotary_frequencies(128, theta=1e6)
    pos = torch.tensor([1, 2, 3, 5, 8, 100, -1, -77], dtype=torch.int32, device="cuda")
    s, c = _sine_cosine(f, pos)
    for sine, cosine in _one_hot_turns(rot, f, pos, inter):
        assert ((sine.double() - s).abs() <= 8 * U * s.abs()).all()
        assert ((cosine.double() - c).abs() <= 8 * U).all()


@pytest.mark.parametrize("inter", [False, True])
def test_far_angles(rot, inter):
    """Sines and cosines at any int32 position, and beyond: 8 roundings of 2^-24 (the
    angle within its quarter turn, 3 of pi / 4; the series, 3), and what the fraction of
    a turn per position, 2^-64, comes to at the position."""
    f = rot.rotary_frequencies(64, theta=1e4)
    far = torch.tensor([(1 << 31) - 1, (1 << 31) - 12345, -(1 << 31), (1 << 30) + 7, 1 << 27, -((1 << 24) + 1)],
                       dtype=torch.int64, device="cuda")
    further = torch.tensor([(1 << 40) + 3, -(1 << 36) - 5], dtype=torch.int64, device="cuda")
    for pos in (far.int(), far, further):
        s, c = _sine_cosine(f, pos)
        tol = 8 * U + 2 * math.pi * pos.abs().double().view(-1, 1) * 2.0 ** -64
        for sine, cosine in _one_hot_turns(rot, f, pos, inter):
            assert ((sine.double() - s).abs() <= tol).all() and ((cosine.double() - c).abs() <= tol).all()


@pytest.mark.parametrize("B,N,H,H_kv,D,R,dt,inter", [
    (4, 700, 40, 8, 128, 128, torch.bfloat16, False), (2, 5000, 7, 3, 64, 32, torch.float16, True),
    (1, 9001, 5, 2, 96, 96, torch.float32, False), (3, 2369, 4, 1, 128, 64, torch.bfloat16, True),
    (7, 1016, 6, 2, 16, 16, torch.float32, False), (4, 4096, 32, 8, 128, 128, torch.bfloat16, False)])
def test_weight_gradients_miss_no_row(rot, B, N, H, H_kv, D, R, dt, inter):
    """Inputs and gradients of +-1 at position 0, without an epsilon: every row's norm
    is 1 (looked at first), so the weight gradients are sums of +-1 over the rows, whole
    numbers under 2^24 that fp32 adds without rounding in any order.  A row that is
    missing or counted twice changes every one of them."""
    rows = [B * N * h for h in (H, H_kv)]
    assert max(rows) < 1 << 20
    sign = lambda shape, s: (_gen(shape, s) > 0).to(dt) * 2 - 1     # noqa: E731
    x, g = sign((B, N, (H + H_kv) * D), 1), sign((B, N, (H + H_kv) * D), 2)
    heads = lambda t: [p.view(B, N, -1, D).transpose(1, 2) for p in t.split([H * D, H_kv * D], -1)]   # noqa: E731
    q, k = heads(x)
    gq, gk = heads(g)
    w = torch.ones(D, device="cuda")
    f = rot.rotary_frequencies(R)
    pos = torch.zeros(N, dtype=torch.int32, device="cuda")
    one = torch.ones((1, 1, 1, D), device="cuda")
    assert (rot.qk_norm_rope_forward(one, one, f, q_weight=w, eps=0.0)[0] == 1).all()
    _, _, dwq, dwk = rot.qk_norm_rope_backward(gq, gk, q, k, f, pos, q_weight=w, k_weight=w, eps=0.0, interleaved=inter)
    for got, a, b in ((dwq, q, gq), (dwk, k, gk)):
        want = (a.double() * b.double()).sum((0, 1, 2))
        assert torch.equal(got.double(), want)


def test_weight_gradient_behind_2_31_elements(rot):
    """The weight gradient of a call whose offsets pass 2^31 elements: sums of +-1 as above,
    whose partial sums stay far under 2^24 (18 million rows of random signs)."""
    H, N, D = 20, 900_001, 128
    q = torch.empty((1, H, N, D), dtype=torch.bfloat16, device="cuda")
    g = torch.empty_like(q)
    for i, t in enumerate((q, g)):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(i)
        t.random_(0, 2, generator=gen).mul_(2).sub_(1)
    w, f = torch.ones(D, device="cuda"), rot.rotary_frequencies(D)
    pos = torch.zeros(N, dtype=torch.int32, device="cuda")
    dw = rot.qk_norm_rope_backward(g, None, q, q[:, :1], f, pos, q_weight=w, eps=0.0)[2]
    want = torch.zeros(D, dtype=torch.int64, device="cuda")
    for h in range(H):
        want += (q[0, h] * g[0, h]).sum(0, dtype=torch.float32).long()      # +-1: exact in 32 bits under 2^24 rows
    assert torch.equal(dw.double(), want.double())


@pytest.mark.parametrize("B,N", [("7", "R/7"), ("7", "R/7+1"), ("2", "R-1"), ("3", "R"), ("2", "R+1"), ("3", "R+5"), ("4", "2*R-3"),
                                 ("R+9", "2"), ("2*R+3", "1"), ("3*R//5", "5"), ("R//3+1", "9")])
@pytest.mark.parametrize("H,H_kv,D", [(2, 1, 64), (6, 2, 128)])
def test_batches_over_rounds_of_warps(rot, B, N, H, H_kv, D):
    """Batches in which a warp takes a second and third whole token (R warps a round),
    in sequences shorter than, equal to and longer than a round: every row equals, bit
    for bit, the one of a call for its sequences alone, forward and backward, and those are
    the formula's."""
    R = torch.cuda.get_device_properties(0).multi_processor_count * 2 * 8
    B, N = int(eval(B, {"R": R})), int(eval(N, {"R": R}))
    assert B > 1 and B * N >= R - 7
    f = rot.rotary_frequencies(D)
    w = 1 + 0.2 * _gen((D,), 3)
    q, k = _gen((B, H, N, D), 1, torch.bfloat16), _gen((B, H_kv, N, D), 2, torch.bfloat16)
    gq, gk = _gen(q.shape, 4, torch.bfloat16), _gen(k.shape, 5, torch.bfloat16)
    pos = torch.randint(0, 1 << 20, (B, N), device="cuda", dtype=torch.int32)
    kw = dict(q_weight=w, k_weight=w)
    y = rot.qk_norm_rope_forward(q, k, f, pos, **kw)
    d = rot.qk_norm_rope_backward(gq, gk, q, k, f, pos, **kw)[:2]
    # sequences in groups of less than a round of tokens, so that each is one unit or a part of one
    step = max(1, (R // 2) // N)
    for b in range(0, B, step):
        s = slice(b, b + step)
        for n in range(0, N, R // 2):
            at = (s, slice(None), slice(n, n + R // 2))
            a = [t[at].contiguous() for t in (q, k, gq, gk)]
            p = pos[s, n:n + R // 2].contiguous()
            assert all(torch.equal(u, v[at]) for u, v in zip(rot.qk_norm_rope_forward(a[0], a[1], f, p, **kw), y)), (b, n)
            assert all(torch.equal(u, v[at]) for u, v in zip(rot.qk_norm_rope_backward(a[2], a[3], a[0], a[1], f, p, **kw)[:2], d)), (b, n)
    cos, sin = _turns(f, pos, None, B, N)
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        want, mag = _oracle(x, w, cos, sin, False, 1e-6)
        _close(y[i], want, mag, 32, f"output {i}")
        dx, dxm, _, _ = _oracle_back(x, w, g, cos, sin, False, 1e-6)
        _close(d[i], dx, dxm, 48, f"gradient {i}")


def test_training_chain_with_grouped_heads(rot):
    """Fewer key heads than query heads: normed and rotated as they are, then repeated
    for the attention, which takes one key head per query head; against the chain in 64 bits."""
    from pallas_flash.ops.interface import pallas_flash_attention
    B, N, H, H_kv, D = 2, 130, 6, 2, 128
    G = H // H_kv
    x = _gen((B, N, (H + 2 * H_kv) * D), 1, torch.bfloat16)
    wq, wk = ((1 + 0.1 * _gen((D,), s)) for s in (2, 3))
    f = rot.rotary_frequencies(D)
    do = _gen((B, H, N, D), 4, torch.bfloat16)

    def split(t):
        return [p.view(B, N, -1, D).transpose(1, 2) for p in t.split([H * D, H_kv * D, H_kv * D], -1)]

    leaf = x.clone().requires_grad_(True)
    ws = [w.clone().requires_grad_(True) for w in (wq, wk)]
    q, k, v = split(leaf)
    q, k = rot.qk_norm_rope(q, k, f, q_weight=ws[0], k_weight=ws[1])
    o = pallas_flash_attention(q, k.repeat_interleave(G, 1), v.repeat_interleave(G, 1), causal=True)
    got = torch.autograd.grad(o, [leaf] + ws, do)

    leaf64 = x.double().requires_grad_(True)
    ws64 = [w.double().requires_grad_(True) for w in (wq, wk)]
    q, k, v = split(leaf64)
    cos, sin = _turns(f, None, None, B, N)
    q, k = (_oracle(t, w, cos, sin, False, 1e-6)[0] for t, w in ((q, ws64[0]), (k, ws64[1])))
    s = (q @ k.repeat_interleave(G, 1).transpose(2, 3)) / math.sqrt(D)
    s = s.masked_fill(torch.ones(N, N, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    o64 = s.softmax(-1) @ v.repeat_interleave(G, 1)
    want = torch.autograd.grad(o64, [leaf64] + ws64, do.double())
    assert_close_o(to_np(o), to_np(o64), what="chain")
    for n, a, b in zip(("x", "wq", "wk"), got, want):
        assert_close_grad(to_np(a), to_np(b), what=n)
