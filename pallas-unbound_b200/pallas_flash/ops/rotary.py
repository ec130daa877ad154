"""Norms of queries and keys for each head with the position rotation in the
same pass — what a model does to q and k right before
`pallas_flash_attention`.  No counterpart in the reference, whose attention
takes q, k, v as they are (src/pallas_flash/ops/interface.py:20-27).

    inv_freq = rotary_frequencies(128, theta=1e6)            # kept by the program
    q, k = qk_norm_rope(q, k, inv_freq, positions, q_weight=wq, k_weight=wk)
    o = pallas_flash_attention(q, k, v, causal=True)

With fewer key heads than query heads, k and v are repeated in between
(`k.repeat_interleave(H // H_kv, 1)`): the attention takes a key head for each
query head, while the norm and rotation need each key head once.

For one row x of D values (one head of one token):
  n = x / sqrt(mean(x^2) + eps) * weight
  (a, b) = pair p of n  ->  (a cos t - b sin t, b cos t + a sin t),
  t = position * inv_freq[p]
Pair p is (p, p + R/2), or (2p, 2p + 1) with `interleaved`, where R = 2 *
len(inv_freq); the values behind R are normed and not rotated.  Everything is
fp32 inside and rounded once.  An angle is a 64-bit fraction of a turn: off by
|position| 2^-64 of a turn, and sines of small angles keep fp32's precision.

Differentiable by q, k and the weights (once, in reverse mode); the weights' gradients come
from fixed-order sums, the same bits every time.  Into a CUDA graph, capture
`qk_norm_rope_forward` and `qk_norm_rope_backward`: autograd inside a capture
waits for the streams of eager graphs that hold the same leaves.  Compute runs in
libpu_attn.so (pu_qk_norm_rope_fwd, pu_qk_norm_rope_bwd); there is no CPU
fallback.
"""
from __future__ import annotations

import functools
import struct
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _lib

__all__ = ["rotary_frequencies", "qk_norm_rope", "qk_norm_rope_forward", "qk_norm_rope_backward"]

_DT = {torch.bfloat16: _lib.PU_DTYPE_BF16, torch.float16: _lib.PU_DTYPE_F16,
       torch.float32: _lib.PU_DTYPE_F32}
_DESC = struct.Struct("=24qd21q")      # pu_qk_rope_desc
_NONE = (0, 0, 0)


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """theta^(-2p/R) for the R/2 pairs, fp64 on `device` (default: the current GPU)."""
    if rotary_dim < 16 or rotary_dim % 16:
        raise ValueError("rotary_dim must be a multiple of 16")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    p = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    return torch.pow(torch.tensor(float(theta), dtype=torch.float64), -p / rotary_dim).to(device)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t`, or a dense copy where a kernel cannot read its rows in 16-byte vectors
    (rows are a multiple of 16 elements)."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        unit, st, shape = 16 // t.element_size(), t.stride(), t.shape
        ok = st[-1] == 1
        for i in range(len(st) - 1):
            if st[i] % unit and shape[i] > 1:
                ok = False
        if ok:
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _refuse_tangents(*tensors) -> None:
    """Raises where an input carries a forward-mode tangent: the result would have
    none, which reads as a derivative of zero."""
    if getattr(forward_ad, "_current_level", 0) < 0:        # outside every dual level there are none
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("norm and rotation have no forward-mode derivative")


def _check_weight(w, D: int, device, name: str):
    if w is None:
        return None
    if w.shape != (D,) or w.dtype not in _DT or w.device != device:
        raise ValueError(f"{name} must be a bf16, fp16 or fp32 [{D}] tensor on {device}")
    return w.contiguous()


def _check_angles(inv_freq, positions, sections, D: int, lead: tuple, device):
    """Checks the rotation's arguments; returns (inv_freq, rotary size, position
    strides {axis, *lead}, axes, four section sizes)."""
    if inv_freq.dim() != 1 or inv_freq.dtype not in (torch.float64, torch.float32) or inv_freq.device != device:
        raise ValueError(f"inv_freq must be a fp64 or fp32 vector on {device}")
    pairs = inv_freq.numel()
    if pairs % 8 or not 8 <= pairs <= D // 2:
        raise ValueError(f"inv_freq must hold a multiple of 8 pairs, at most {D // 2}: got {pairs}")
    if sections is None:
        axes, sizes = 1, (pairs, 0, 0, 0)
    else:
        axes = len(sections)
        if not 1 <= axes <= 4 or any(int(n) != n or n < 0 for n in sections) or sum(sections) != pairs:
            raise ValueError(f"sections must be 1 to 4 sizes that add up to {pairs} pairs: got {tuple(sections)}")
        sizes = tuple(int(n) for n in sections) + (0,) * (4 - axes)
    if positions is None:
        if axes > 1:
            raise ValueError("sections need positions with an axis for each")
        return inv_freq.contiguous(), 2 * pairs, _NONE, axes, sizes
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != device:
        raise ValueError(f"positions must be int32 or int64 on {device}")
    shape, st = tuple(positions.shape), positions.stride()
    head = () if sections is None else (axes,)
    if shape == head + lead:
        full = st if head else (0,) + st
    elif len(lead) == 2 and shape == head + lead[1:]:       # the same for every sequence
        full = (st[0], 0, st[1]) if head else (0, 0, st[0])
    else:
        want = "[axes, ...]" if head else ""
        raise ValueError(f"positions {shape} do not match the tokens {lead} {want}")
    return inv_freq.contiguous(), 2 * pairs, full, axes, sizes


def _pack(B, N, H, H_kv, D, dtype, R, interleaved, inv_freq, positions, pos_st, axes, sizes, wq, wk, eps,
          q=_NONE, k=_NONE, v=_NONE, gq=_NONE, gk=_NONE, dq=_NONE, dk=_NONE) -> bytes:
    """pu_qk_rope_desc; the last seven are strides of {B, H, N}."""
    return _DESC.pack(
        B, N, H, H_kv, D, _DT[dtype], R, 1 if interleaved else 0,
        inv_freq.data_ptr(), 1 if inv_freq.dtype == torch.float64 else 0,
        0 if positions is None else positions.data_ptr(),
        1 if positions is not None and positions.dtype == torch.int64 else 0, *pos_st,
        axes, *sizes,
        0 if wq is None else wq.data_ptr(), 0 if wq is None else _DT[wq.dtype],
        0 if wk is None else wk.data_ptr(), 0 if wk is None else _DT[wk.dtype],
        eps, *q, *k, *v, *gq, *gk, *dq, *dk)


def _check_qk(q: torch.Tensor, k: torch.Tensor):
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k must be [B, H, N, D] and [B, H_kv, N, D]")
    B, H, N, D = q.shape
    if k.shape[0] != B or k.shape[2] != N or k.shape[3] != D:
        raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    if not q.is_cuda or k.device != q.device:
        raise ValueError("q and k must be CUDA tensors on one device")
    if q.dtype not in _DT or k.dtype != q.dtype:
        raise TypeError("q and k must share one dtype: bf16, fp16 or fp32")
    if D % 16 or not 16 <= D <= 128:
        raise ValueError(f"head size {D} (a multiple of 16 up to 128)")
    if H == 0 or k.shape[1] == 0:
        raise ValueError("q and k need at least one head")


def _description(q, k, inv_freq, positions, q_weight, k_weight, eps, sections, interleaved):
    """Checked arguments of a pass over [B, H, N, D] tensors, for _pack."""
    _check_qk(q, k)
    _refuse_tangents(q, k, inv_freq, q_weight, k_weight)
    B, H, N, D = q.shape
    dev = q.device
    wq, wk = _check_weight(q_weight, D, dev, "q_weight"), _check_weight(k_weight, D, dev, "k_weight")
    f, R, pos_st, axes, sizes = _check_angles(inv_freq, positions, sections, D, (B, N), dev)
    return (B, N, H, k.shape[1], D, q.dtype, R, interleaved, f, positions, pos_st, axes, sizes, wq, wk, float(eps))


def _forward(desc, q, k):
    B, N, H, H_kv, D = desc[:5]
    with _lib.on_device(q.device) as stream:
        q_out = torch.empty(B, H, N, D, dtype=q.dtype, device=q.device)
        k_out = torch.empty(B, H_kv, N, D, dtype=q.dtype, device=q.device)
        if B * N:
            q, k = _rows(q), _rows(k)
            _lib.check(_lib.lib().pu_qk_norm_rope_fwd(_pack(*desc, q.stride()[:3], k.stride()[:3]), q.data_ptr(),
                                                      k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), stream),
                       "pu_qk_norm_rope_fwd")
    return q_out, k_out


def qk_norm_rope_forward(q, k, inv_freq, positions=None, *, q_weight=None, k_weight=None, eps: float = 1e-6,
                         sections: Optional[Sequence[int]] = None, interleaved: bool = False):
    """`qk_norm_rope` without autograd (pu_qk_norm_rope_fwd on the current stream)."""
    return _forward(_description(q, k, inv_freq, positions, q_weight, k_weight, eps, sections, interleaved), q, k)


def _grad_like(t: torch.Tensor) -> torch.Tensor:
    """A gradient laid out like `t` (a projection's heads stay beside each other)."""
    g = torch.empty_like(t)
    return g if g.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


@functools.lru_cache(maxsize=64)
def _bwd_bytes(device: int, D: int) -> int:
    return int(_lib.lib().pu_qk_norm_rope_bwd_workspace_size(D))


def _backward(desc, gq, gk, q, k, want_wq: bool, want_wk: bool):
    B, N, H, H_kv, D = desc[:5]
    for g, t in ((gq, q), (gk, k)):
        if g is not None and (g.shape != t.shape or g.dtype != t.dtype or g.device != t.device):
            raise ValueError(f"an output gradient must match {tuple(t.shape)} {t.dtype} on {t.device}")
    _refuse_tangents(gq, gk)
    if gq is None and gk is None:
        return None, None, None, None
    wq, wk = desc[13], desc[14]
    dq = dk = dwq = dwk = ws = None
    with _lib.on_device(q.device) as stream:
        make = torch.empty_like if B * N else torch.zeros_like
        if gq is not None:
            dq = _grad_like(q)
            if want_wq and wq is not None:
                dwq = make(wq)
        if gk is not None:
            dk = _grad_like(k)
            if want_wk and wk is not None:
                dwk = make(wk)
        if B * N:
            q, k = _rows(q), _rows(k)
            gq, gk = (None if g is None else _rows(g) for g in (gq, gk))
            need = 0
            if dwq is not None or dwk is not None:
                need = _bwd_bytes(q.device.index, D)
                ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            st = lambda t: _NONE if t is None else t.stride()[:3]     # noqa: E731
            ptr = lambda t: None if t is None else t.data_ptr()       # noqa: E731
            _lib.check(_lib.lib().pu_qk_norm_rope_bwd(
                _pack(*desc, st(q), st(k), _NONE, st(gq), st(gk), st(dq), st(dk)), q.data_ptr(), k.data_ptr(),
                ptr(gq), ptr(gk), ptr(dq), ptr(dk), ptr(dwq), ptr(dwk), ptr(ws), need, stream), "pu_qk_norm_rope_bwd")
    return dq, dk, dwq, dwk


def qk_norm_rope_backward(gq, gk, q, k, inv_freq, positions=None, *, q_weight=None, k_weight=None,
                          eps: float = 1e-6, sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                          weight_grads: bool = True):
    """(dq, dk, dq_weight, dk_weight) from the inputs and the output gradients.

    A None output gradient gives None for that side; `weight_grads=False`
    leaves the weights' out.  Calls pu_qk_norm_rope_bwd on the current stream."""
    desc = _description(q, k, inv_freq, positions, q_weight, k_weight, eps, sections, interleaved)
    return _backward(desc, gq, gk, q, k, weight_grads, weight_grads)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, inv_freq, positions, eps, sections, interleaved):
        ctx.set_materialize_grads(False)
        # positions and frequencies stay here, as they were described: a saved-tensor
        # hook may give another tensor back, with other strides
        ctx.save_for_backward(q, k, q_weight, k_weight)
        desc = _description(q, k, inv_freq, positions, q_weight, k_weight, eps, sections, interleaved)
        ctx.desc, ctx.angles = desc[:13] + (None, None) + desc[15:], (inv_freq, positions)
        ctx.versions = [t._version for t in ctx.angles if t is not None]
        return _forward(desc, q, k)

    @staticmethod
    def backward(ctx, gq, gk):
        # (the decorator costs more than a small kernel; it only matters where a
        # graph of the gradients is kept)
        return _QkNormRope._once(ctx, gq, gk) if torch.is_grad_enabled() else _QkNormRope._grads(ctx, gq, gk)

    @staticmethod
    def _grads(ctx, gq, gk):
        q, k, wq, wk = ctx.saved_tensors
        need, desc, dev = ctx.needs_input_grad, ctx.desc, ctx.angles[0].device
        B, N, H, H_kv, D, dtype = desc[:6]
        if ctx.versions != [t._version for t in ctx.angles if t is not None]:
            raise RuntimeError("positions or inv_freq were changed in place since the forward")
        if q.shape != (B, H, N, D) or k.shape != (B, H_kv, N, D) or q.dtype != dtype or k.dtype != dtype \
                or q.device != dev or k.device != dev:
            raise ValueError("a saved tensor came back with another shape, type or device")
        if not (need[0] or need[2]):
            gq = None
        if not (need[1] or need[3]):
            gk = None
        wq, wk = _check_weight(wq, D, dev, "q_weight"), _check_weight(wk, D, dev, "k_weight")
        desc = desc[:13] + (wq, wk) + desc[15:]
        dq, dk, dwq, dwk = _backward(desc, gq, gk, q, k, need[2], need[3])
        return (dq if need[0] else None, dk if need[1] else None, dwq, dwk, None, None, None, None, None)

    _once = staticmethod(once_differentiable(lambda ctx, gq, gk: _QkNormRope._grads(ctx, gq, gk)))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, inv_freq: torch.Tensor,
                 positions: Optional[torch.Tensor] = None, *, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = False):
    """Norm and rotate every head of q [B,H,N,D] and k [B,H_kv,N,D].

    Returns dense (q, k) of the same shapes and dtype (bf16, fp16 or fp32), what
    `pallas_flash_attention` takes where H_kv == H (otherwise repeat k's heads
    first).  q and k may be strided views, such as a projection's [B,N,H,D]
    transposed: rows that start on 16-byte boundaries are read where they are,
    others through a copy.

      inv_freq   [R/2] fp64 or fp32 radians per position; R/2 a multiple of 8.  There
                 is no gradient by them: one that requires_grad is refused
      positions  int32 or int64 [N] or [B,N]; default 0..N-1
      q_weight, k_weight   [D] norm weights; None: that side is only rotated
      sections   sizes of 1 to 4 runs of pairs, one for each axis of
                 `positions` [axes,N] or [axes,B,N]: the first run turns with
                 axis 0 (time, say), the next with axis 1 (height), ...
    """
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise ValueError("the frequencies have no gradient: pass inv_freq.detach()")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad
                                    or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        return _QkNormRope.apply(q, k, q_weight, k_weight, inv_freq, positions, eps, sections, interleaved)
    return qk_norm_rope_forward(q, k, inv_freq, positions, q_weight=q_weight, k_weight=k_weight, eps=eps,
                                sections=sections, interleaved=interleaved)
