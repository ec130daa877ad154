"""Cases, plain forms and exact values of four operators around attention:

  rope    norms of queries and keys for each head with the position rotation
          in the same pass, forward and backward (a training step's share)
  append  the same for new tokens of a served batch, with keys and values
          written into their places of a paged cache
  plan    page table, slots and positions of a batch's next tokens, from
          lengths alone
  decode  attention of one new token over a paged cache with grouped heads

Formulas.  With a row x of D values (one head of one token), a weight w and
frequencies f_p of R/2 pairs:
  n = x / sqrt(mean(x^2) + eps) * w
  (a, b) = pair p of n  ->  (a cos t - b sin t, b cos t + a sin t),
  t = position * f_p; pair p is (p, p + R/2), or (2p, 2p + 1) interleaved;
  with sections (s0, s1, s2) the first s0 pairs take the position's first
  axis, the next s1 its second, and so on.  Values behind R stay.
  o = sum_j exp(s_j - lse) v_j,  s_j = q k_j / sqrt(D),  lse = log sum_j exp s_j
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
#: scales of an 8-bit cache
K_SCALE, V_SCALE = 0.02, 0.015


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # the attention input of a training step: 32 query heads over 8 key heads of 128, views of one projection
        {"name": "rope_train_4x4096", "op": "rope", "B": 4, "N": 4096, "H": 32, "H_kv": 8, "D": 128, "R": 128, "axes": 1,
         "interleaved": False, "type": "bf16", "weights": "f32"},
        # image and video tokens with time, height and width, heads of 64, a length that no tile divides
        {"name": "rope_axes_2x4999", "op": "rope", "B": 2, "N": 4999, "H": 16, "H_kv": 2, "D": 64, "R": 64, "axes": 3,
         "interleaved": False, "type": "f16", "weights": "f16"},
        # a small call: odd head count, a third of the head rotated in neighbouring pairs, 32-bit data
        {"name": "rope_partial_3x257", "op": "rope", "B": 3, "N": 257, "H": 5, "H_kv": 5, "D": 96, "R": 32, "axes": 1,
         "interleaved": True, "type": "f32", "weights": "f32"},
        # one served step of 64 sequences: latency
        {"name": "append_step_64", "op": "append", "B": 64, "per": 1, "held": 4000, "pad": 0, "H": 32, "H_kv": 8, "D": 128, "R": 128, "axes": 1,
         "page": 64, "type": "bf16", "weights": "bf16"},
        # prompts of a batch, packed, with padding rows behind the last sequence
        {"name": "append_prompts_17", "op": "append", "B": 17, "per": 1900, "held": 70, "pad": 37, "H": 16, "H_kv": 4, "D": 128, "R": 64, "axes": 1,
         "page": 32, "type": "f16", "weights": "f32"},
        # one served step of 256 sequences of up to 32768 tokens
        {"name": "plan_step_256", "op": "plan", "B": 256, "per": 1, "held": 30000, "pages": 2048, "page": 16, "pad": 0, "release": 7},
        # prompts of new requests beside running ones, slots that were released
        {"name": "plan_prompts_61", "op": "plan", "B": 61, "per": 2500, "held": 9000, "pages": 1024, "page": 64, "pad": 113, "release": 5},
        # one short conversation: latency
        {"name": "decode_short_1", "op": "decode", "B": 1, "lo": 1000, "hi": 1000, "H": 32, "H_kv": 8, "D": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # a ragged batch of long contexts
        {"name": "decode_ragged_8", "op": "decode", "B": 8, "lo": 4096, "hi": 131072, "H": 32, "H_kv": 8, "D": 128, "page": 64, "type": "f16", "cache": "f16"},
        # an 8-bit cache, sequences from empty to 32768 tokens
        {"name": "decode_e4m3_24", "op": "decode", "B": 24, "lo": 0, "hi": 32768, "H": 64, "H_kv": 8, "D": 128, "page": 32, "type": "bf16", "cache": "e4m3"},
        # many short sequences, heads of 64, small pages that end inside every tile
        {"name": "decode_many_256", "op": "decode", "B": 256, "lo": 0, "hi": 2048, "H": 16, "H_kv": 2, "D": 64, "page": 16, "type": "bf16", "cache": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "plan", "decode"])
    kv = rng.choice([1, 2, 3, 4, 8])
    H, D = kv * rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "rope":
        D = rng.choice([64, 80, 96, 128])
        B = rng.randint(1, 5)
        most = 4 * 4096 * 40 * 128 // (B * (H + kv) * D)
        axes = rng.choice([1, 1, 3])
        t = rng.choice(["bf16", "bf16", "f16"]) if rng.random() < 0.8 else "f32"
        return {"op": op, "B": B, "N": min(_spread(rng, 1, 16384), most * 2 // SIZES[t]), "H": H, "H_kv": kv, "D": D,
                "R": rng.choice([D, D, 32]), "axes": axes, "interleaved": rng.random() < 0.4, "type": t, "weights": rng.choice(["f32", t])}
    if op == "append":
        B = rng.randint(1, 100)
        return {"op": op, "B": B, "per": rng.choice([1, _spread(rng, 2, 2000 * 17 // max(17, B))]), "held": _spread(rng, 1, 5000), "pad": rng.choice([0, rng.randint(1, 50)]),
                "H": min(H, 32), "H_kv": kv if H <= 32 else 1, "D": D, "R": rng.choice([D, 32]), "axes": rng.choice([1, 3]), "page": page,
                "type": rng.choice(["bf16", "f16"]), "weights": rng.choice(["f32", "bf16"])}
    if op == "plan":
        B = _spread(rng, 1, 400)
        held = _spread(rng, 1, 12000)
        per = rng.choice([1, _spread(rng, 2, max(3, 120000 // B))])
        return {"op": op, "B": B, "per": per, "held": held, "pages": (held + per) // page + rng.randint(2, 400), "page": page, "pad": rng.choice([0, rng.randint(1, 200)]), "release": rng.choice([0, 3, 10])}
    t = rng.choice(["bf16", "f16"])
    cache = rng.choice([t, t, "e4m3"])
    kv, H = (kv, H) if H > kv else (kv, 4 * kv)
    hi = _spread(rng, 1, 131072)
    most = max(1, min(256, 600_000_000 // (hi * kv * D)))
    return {"op": op, "B": _spread(rng, 1, most), "lo": rng.choice([0, 1, hi]), "hi": hi, "H": H, "H_kv": kv, "D": D, "page": page, "type": t, "cache": cache}


# --------------------------------------------------------------------------
# lengths of a case (they follow from the case alone, so that its work does)
# --------------------------------------------------------------------------
def _lens(case):
    """Tokens held by each sequence of a decode case."""
    r = np.random.RandomState((case["B"] * 7919 + case["hi"] * 31 + case["D"]) % (1 << 31))
    return r.randint(case["lo"], case["hi"] + 1, case["B"])


def _growth(case):
    """(held, new, released) of each sequence of a plan or append case."""
    r = np.random.RandomState((case["B"] * 104729 + case["held"] * 17 + case["per"] * 3 + case["page"]) % (1 << 31))
    held = r.randint(0, case["held"] + 1, case["B"])
    new = np.ones(case["B"], np.int64) if case["per"] == 1 else r.randint(0, case["per"] + 1, case["B"])
    new[0] = max(new[0], 1)
    gone = np.zeros(case["B"], bool)
    if case.get("release"):
        gone[r.permutation(case["B"])[:max(1, case["B"] * case["release"] // 100)]] = True
    if "pages" in case:
        most = case["pages"] * case["page"]
        held = np.minimum(held, most)
        new = np.minimum(new, most - np.where(gone, 0, held))
    return held, new, gone


def _sections(case):
    """Pairs of each axis: a quarter for time, the rest shared by height and width."""
    pairs = case["R"] // 2
    if case["axes"] == 1:
        return None
    t = pairs // 4
    h = (pairs - t) // 2
    return (t, h, pairs - t - h)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, kind, scale=1.0):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).mul_(scale).to(TYPES[kind])


def _weight(g, D, kind):
    return (1.0 + 0.1 * torch.randn(D, device="cuda", generator=g)).to(TYPES[kind])


def _frequencies(R, theta=1e6):
    return torch.pow(torch.tensor(theta, dtype=torch.float64), -torch.arange(0, R, 2, dtype=torch.float64) / R).cuda()


def _positions(case, g, shape):
    """Positions of image and video tokens: (frame, row, column) of a grid, some way into a context."""
    n = shape[-1]
    i = torch.arange(n, device="cuda")
    side = max(1, math.isqrt(max(1, n // 4)))
    off = torch.randint(0, 30000, shape[1:-1] + (1,), device="cuda", generator=g)
    axes = torch.stack([i // (side * side), i // side % side, i % side])
    return (axes.reshape((3,) + (1,) * (len(shape) - 2) + (n,)) + off).to(torch.int32).contiguous()


def _prepare_rope(case, g):
    B, N, H, kv, D = (case[k] for k in ("B", "N", "H", "H_kv", "D"))
    x = _normal(g, (B, N, (H + kv) * D), case["type"], 2.0)
    q = x[..., :H * D].view(B, N, H, D).transpose(1, 2)
    k = x[..., H * D:].view(B, N, kv, D).transpose(1, 2)
    s = {"q": q.detach().requires_grad_(True), "k": k.detach().requires_grad_(True),
         "wq": _weight(g, D, case["weights"]).requires_grad_(True), "wk": _weight(g, D, case["weights"]).requires_grad_(True),
         "gq": _normal(g, (B, H, N, D), case["type"]), "gk": _normal(g, (B, kv, N, D), case["type"]),
         "f": _frequencies(case["R"]), "sections": _sections(case), "interleaved": case["interleaved"]}
    s["pos"] = _positions(case, g, (3, B, N)) if case["axes"] == 3 else \
        (torch.arange(N, device="cuda") + torch.randint(0, 100000, (B, 1), device="cuda", generator=g)).to(torch.int32)
    return s


def _prepare_append(case, g):
    H, kv, D, ps = (case[k] for k in ("H", "H_kv", "D", "page"))
    held, new, _ = _growth(case)
    T = int(new.sum()) + case["pad"]
    first = np.cumsum(-(-(held + new) // ps)) - (-(-(held + new) // ps))
    pages = max(1, int((-(-(held + new) // ps)).sum()))
    order = torch.randperm(pages, device="cuda", generator=g).cpu().numpy()
    seq = np.repeat(np.arange(case["B"]), new)
    pos = held[seq] + np.arange(len(seq)) - (np.cumsum(new) - new)[seq]
    slots = np.full(T, -1, np.int64)
    slots[:len(seq)] = order[first[seq] + pos // ps] * ps + pos % ps
    place = np.zeros(T, np.int64)
    place[:len(seq)] = pos
    x = _normal(g, (T, (H + 2 * kv) * D), case["type"], 2.0)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in x.split([H * D, kv * D, kv * D], -1))
    s = {"q": q, "k": k, "v": v, "slots": torch.from_numpy(slots).int().cuda(), "f": _frequencies(case["R"]),
         "wq": _weight(g, D, case["weights"]), "wk": _weight(g, D, case["weights"]), "sections": _sections(case),
         "k_pool": torch.zeros((pages, kv, ps, D), dtype=TYPES[case["type"]], device="cuda")}
    s["v_pool"] = torch.zeros_like(s["k_pool"])
    s["pos"] = _positions(case, g, (3, T)) if case["axes"] == 3 else torch.from_numpy(place).int().cuda()
    return s


def _prepare_plan(case, g):
    ps, B = case["page"], case["B"]
    held, new, gone = _growth(case)
    have, extra = -(-held // ps), -(-(np.where(gone, 0, held) + new) // ps)
    total = int(have.sum() + extra.sum()) + 64
    order = torch.randperm(total, device="cuda", generator=g).cpu().numpy()
    table = np.full((B, case["pages"]), -1, np.int32)
    inside = np.arange(case["pages"])[None] < have[:, None]
    table[inside] = order[:int(have.sum())]
    free = order[int(have.sum()):]
    # the free pages lie in a ring: it starts anywhere
    head = int(order[0]) + 3 * total
    ring = np.zeros(total, np.int32)
    ring[(head + np.arange(len(free))) % total] = free
    cuda = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(t).cuda()  # noqa: E731
    return {"table": cuda(table, torch.int32), "lens": cuda(held, torch.int32), "new": cuda(new, torch.int32),
            "release": cuda(gone, torch.bool) if case["release"] else None, "ring": cuda(ring, torch.int32),
            "cursor": torch.tensor([head, head + len(free)], dtype=torch.int64, device="cuda"),
            "page": ps, "tokens": int(new.sum()) + case["pad"]}


def _prepare_decode(case, g):
    B, H, kv, D, ps = (case[k] for k in ("B", "H", "H_kv", "D", "page"))
    lens = _lens(case)
    need = -(-lens // ps)
    pages = max(1, int(need.sum()))
    order = torch.randperm(pages, device="cuda", generator=g).int().cpu().numpy()
    width = max(1, int(need.max()))
    table = np.full((B, width), -1, np.int32)
    table[np.arange(width)[None] < need[:, None]] = order[:int(need.sum())]

    def pool():
        # made in parts: a whole pool in 32 bits would be twice its size again
        out = torch.empty((pages, kv, ps, D), dtype=torch.float8_e4m3fn if case["cache"] == "e4m3" else TYPES[case["cache"]], device="cuda")
        for part in out.split(max(1, (1 << 27) // (kv * ps * D))):
            x = torch.randn(part.shape, device="cuda", generator=g)
            part.copy_(x / K_SCALE if case["cache"] == "e4m3" else x)
        return out
    return {"q": _normal(g, (B, H, 1, D), case["type"]), "k_pool": pool(), "v_pool": pool(), "lens": torch.from_numpy(lens).int().cuda(),
            "table": torch.from_numpy(table).cuda(), "scales": (K_SCALE, V_SCALE) if case["cache"] == "e4m3" else (1.0, 1.0)}


def prepare(case, seed):
    s = globals()["_prepare_" + case["op"]](case, _gen(seed))
    s["op"] = case["op"]
    return s


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
def _angles(pos, f, sections):
    """cos and sin [..., R/2] of positions [...] or [axes, ...], angles in 64 bits."""
    if sections is None:
        t = pos.double().unsqueeze(-1) * f
    else:
        axis = torch.repeat_interleave(torch.arange(len(sections), device=f.device), torch.tensor(sections, device=f.device), output_size=f.numel())
        t = pos.double()[axis].movedim(0, -1) * f
    return t.cos().float(), t.sin().float()


def _turn(n, cos, sin, interleaved):
    """Rotates the pairs of n [..., D] in 32 bits."""
    R = 2 * cos.shape[-1]
    if interleaved:
        a, b = n[..., 0:R:2], n[..., 1:R:2]
        out = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = n[..., :R // 2], n[..., R // 2:R]
        out = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([out, n[..., R:]], -1)


def _normed(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _rope_back(x, w, g, cos, sin, interleaved):
    """Gradients of _turn(_normed(x, w)): by x and by w."""
    h = _turn(g.float(), cos, -sin, interleaved)
    x = x.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    u = x * r
    hw = h * w.float()
    dx = r * (hw - u * (hw * u).mean(-1, keepdim=True))
    return dx, (h * u).sum((0, 1, 2))


def _plain_rope(s):
    with torch.no_grad():
        cos, sin = (t.unsqueeze(1) for t in _angles(s["pos"], s["f"], s["sections"]))
        out = {}
        for n in ("q", "k"):
            x, w, g = s[n], s["w" + n], s["g" + n]
            out[n] = _turn(_normed(x, w), cos, sin, s["interleaved"]).to(x.dtype)
            dx, dw = _rope_back(x, w, g, cos, sin, s["interleaved"])
            out["d" + n], out["dw" + n] = dx.to(x.dtype), dw.to(w.dtype)
        return out


def _plain_append(s):
    cos, sin = (t.unsqueeze(1) for t in _angles(s["pos"], s["f"], s["sections"]))
    q = _turn(_normed(s["q"], s["wq"]), cos, sin, False).to(s["q"].dtype)
    k = _turn(_normed(s["k"], s["wk"]), cos, sin, False)
    ps = s["k_pool"].shape[2]
    live = s["slots"] >= 0
    at = s["slots"][live].long()
    s["k_pool"][at // ps, :, at % ps] = k[live].to(s["k_pool"].dtype)
    s["v_pool"][at // ps, :, at % ps] = s["v"][live].to(s["v_pool"].dtype)
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_plan(s):
    ps, table, T, P = s["page"], s["table"], s["tokens"], s["ring"].numel()
    held, new = s["lens"].long(), s["new"].long()
    gone = s["release"] if s["release"] is not None else torch.zeros_like(held, dtype=torch.bool)
    head, tail = s["cursor"][0], s["cursor"][1]
    base = torch.where(gone, 0, held)
    have, last = (base + ps - 1) // ps, (base + new + ps - 1) // ps
    need = last - have
    upto, start = need.cumsum(0), new.cumsum(0) - new
    freed = torch.where(gone, (held + ps - 1) // ps, 0)
    # rows: kept pages, then pages from the head of the ring, then nothing
    j = torch.arange(table.shape[1], device=table.device).unsqueeze(0)
    taken = s["ring"][(head + (upto - need).unsqueeze(1) + j - have.unsqueeze(1)) % P]
    rows = torch.where(j < have.unsqueeze(1), table, torch.where(j < last.unsqueeze(1), taken, -1)).int()
    # pages of released sequences go to the tail
    j_old = (j < freed.unsqueeze(1)).nonzero(as_tuple=True)
    s["ring"][(tail + (freed.cumsum(0) - freed)[j_old[0]] + j_old[1]) % P] = table[j_old]
    # tokens
    i = torch.arange(T, device=table.device)
    seq = torch.searchsorted(start + new, i, right=True)
    live = seq < held.numel()
    at = torch.where(live, seq, 0)
    pos = torch.where(live, base[at] + i - start[at], 0)
    slot = torch.where(live, rows[at, pos // ps].long() * ps + pos % ps, -1)
    return {"slots": slot.int(), "positions": pos.int(), "seq_ids": torch.where(live, seq, -1).int(),
            "cu_new": torch.cat([start, (start + new)[-1:]]).int(), "kv_lens": (base + new).int(),
            "cursor": torch.stack([head + upto[-1], tail + freed.sum()]), "page_table": rows, "ring": s["ring"]}


def _plain_decode(s):
    q, kp, vp, table, lens = s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"]
    (B, H, _, D), (kv, ps) = q.shape, kp.shape[1:3]
    rows = table.clamp(min=0).long()
    dense = lambda pool, scale: (pool[rows].float() * scale).transpose(1, 2).reshape(B, kv, -1, D)  # noqa: E731
    if kp.dtype == torch.float8_e4m3fn:
        kp, vp = kp.view(torch.uint8), vp.view(torch.uint8)
        dense = lambda pool, scale: (pool[rows].view(torch.float8_e4m3fn).float() * scale).transpose(1, 2).reshape(B, kv, -1, D)  # noqa: E731
    x = torch.matmul(q.float().reshape(B, kv, H // kv, D), dense(kp, s["scales"][0]).transpose(2, 3)) / math.sqrt(D)
    past = torch.arange(x.shape[-1], device=x.device) >= lens.view(-1, 1, 1, 1)
    x = x.masked_fill(past, -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-1e30)
    e = torch.exp(x - m)
    l = e.sum(-1, keepdim=True)
    o = torch.matmul(e, dense(vp, s["scales"][1])) / l.clamp(min=1e-30)
    return {"o": o.reshape(B, H, 1, D).to(torch.bfloat16), "lse": torch.where(l > 0, m + l.log(), -math.inf).reshape(B, H)}


# --------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------
def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pallas-unbound_b200")
    if at not in sys.path:
        sys.path.insert(0, at)


def _own_rope(s):
    from pallas_flash.ops.rotary import qk_norm_rope
    q, k = qk_norm_rope(s["q"], s["k"], s["f"], s["pos"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS,
                        sections=s["sections"], interleaved=s["interleaved"])
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _own_append(s):
    from pallas_flash.kernels.paged import qk_norm_rope_append
    q = qk_norm_rope_append(s["q"], s["k"], s["v"], s["f"], s["pos"], s["slots"], s["k_pool"], s["v_pool"],
                            q_weight=s["wq"], k_weight=s["wk"], eps=EPS, sections=s["sections"])
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _own_plan(s):
    from pallas_flash.kernels.paged import plan_append
    p = plan_append(s["table"], s["lens"], s["new"], s["ring"], s["cursor"], page_size=s["page"], num_tokens=s["tokens"], release=s["release"])
    return {"slots": p.slots, "positions": p.positions, "seq_ids": p.seq_ids, "cu_new": p.cu_new, "kv_lens": p.kv_lens,
            "cursor": p.cursor, "page_table": p.page_table, "ring": s["ring"]}


def _own_decode(s):
    from pallas_flash.kernels.decoding import pallas_flash_decoding
    o, lse = pallas_flash_decoding(s["q"], s["k_pool"], s["v_pool"], kv_lens=s["lens"], page_table=s["table"],
                                   k_scale=s["scales"][0], v_scale=s["scales"][1], return_lse=True)
    return {"o": o, "lse": lse}


def run(state):
    if own:
        _package()
        return globals()["_own_" + state["op"]](state)
    return globals()["_plain_" + state["op"]](state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    if case["op"] == "rope":
        rows, D = case["B"] * case["N"] * (case["H"] + case["H_kv"]), case["D"]
        # forward: x in, out; backward: x and the gradient in, the gradient out
        return {"bytes": 5 * rows * D * SIZES[case["type"]] + case["axes"] * case["B"] * case["N"] * 4, "flops": 25 * rows * D}
    if case["op"] == "append":
        T, D, size = int(_growth(case)[1].sum()), case["D"], SIZES[case["type"]]
        T += case["pad"]
        return {"bytes": 2 * T * (case["H"] + 2 * case["H_kv"]) * D * size + T * 4 * (1 + case["axes"]), "flops": 9 * T * (case["H"] + case["H_kv"]) * D}
    if case["op"] == "plan":
        held, new, _ = _growth(case)
        pages, T = int((-(-held // case["page"])).sum()), int(new.sum()) + case["pad"]
        return {"bytes": 4 * (pages + case["B"] * case["pages"] + 3 * T + 5 * case["B"]), "flops": 10 * T + 10 * case["B"]}
    lens = int(_lens(case).sum())
    per = case["H_kv"] * case["D"]
    return {"bytes": 2 * lens * per * SIZES[case["cache"]] + 4 * case["B"] * case["H"] * (case["D"] + 1), "flops": 4 * lens * case["H"] * case["D"]}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def _exact_rows(x, w, f, pos, sections, interleaved):
    """Norm and rotation of x [..., heads, D] with positions [...] or [axes, ...]: pairs as complex numbers."""
    R, places = 2 * f.numel(), []
    for p in range(f.numel()):
        axis = 0 if sections is None else sum(p >= sum(sections[:i + 1]) for i in range(len(sections)))
        places.append((pos if sections is None else pos[axis]).double() * f[p])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), torch.stack(places, -1)).unsqueeze(-2)
    n = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w
    if interleaved:
        z = torch.view_as_complex(n[..., :R].unflatten(-1, (R // 2, 2)).contiguous()) * turn
        y = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(n[..., :R // 2], n[..., R // 2:R]) * turn
        y = torch.cat((z.real, z.imag), -1)
    return torch.cat((y, n[..., R:]), -1)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "rope":
        out = {}
        for n in ("q", "k"):
            x, w = s[n].detach().double().requires_grad_(True), s["w" + n].detach().double().requires_grad_(True)
            y = _exact_rows(x.transpose(1, 2), w, s["f"], s["pos"], s["sections"], s["interleaved"]).transpose(1, 2)
            out["d" + n], out["dw" + n] = torch.autograd.grad(y, (x, w), s["g" + n].double())
            out[n] = y.detach()
        return out
    if case["op"] == "append":
        k = _exact_rows(s["k"].double(), s["wk"].double(), s["f"], s["pos"], s["sections"], False)
        pools = {n: torch.zeros(s["k_pool"].shape, dtype=torch.float64, device="cuda") for n in ("k_pool", "v_pool")}
        for n, x in (("k_pool", k), ("v_pool", s["v"].double())):
            flat = pools[n].transpose(1, 2).reshape(-1, case["H_kv"], case["D"])
            spare = torch.cat([flat, flat[:1]])  # rows without a slot go behind the last one
            spare[torch.where(s["slots"] < 0, len(flat), s["slots"]).long()] = x
            pools[n] = spare[:-1].reshape(-1, case["page"], case["H_kv"], case["D"]).transpose(1, 2)
        return {"q": _exact_rows(s["q"].double(), s["wq"].double(), s["f"], s["pos"], s["sections"], False), **pools}
    B, H, kv, D = (case[k] for k in ("B", "H", "H_kv", "D"))
    o = torch.zeros((B, H, 1, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case).tolist()):
        if n == 0:
            continue
        at = s["table"][b, :-(-n // case["page"])].tolist()
        for h in range(kv):
            k, v = (p.view(torch.uint8)[at, h].view(p.dtype).reshape(-1, D)[:n].double() * c for p, c in zip((s["k_pool"], s["v_pool"]), s["scales"]))
            heads = slice(h * (H // kv), (h + 1) * (H // kv))
            x = s["q"][b, heads, 0].double() @ k.T * D ** -0.5
            lse[b, heads] = torch.logsumexp(x, -1)
            o[b, heads, 0] = torch.softmax(x, -1) @ v
    return {"o": o, "lse": lse}
