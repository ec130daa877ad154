"""Cases, plain forms and exact values of four operators of serving long contexts
from a paged cache:

  bounds  elementwise minimum and maximum of each page's keys, brought up to
          date by the slots of a step's new tokens
  select  the pages that a cheap score picks for a query, for each K/V head
  sparse  attention of one new token over a page list of each K/V head
  shared  attention of one new token of sequences that hold the same first
          pages, those read once for all

Formulas.  lo_p and hi_p are the minimum and the maximum over the keys of page p
(vectors of D values, for each K/V head).  A page's score for the query heads h
of a K/V head is
  sum_h sum_d max(q_hd lo_pd, q_hd hi_pd),
an upper bound of what any of its keys scores, summed over the heads.  Chosen
are the first `first` and the last `last` pages of a sequence and the best of
the others, `count` in all, listed in the sequence's order; a sequence of no
more than `count` pages keeps all of them.
  o = sum_j exp(s_j - lse) v_j,  s_j = q k_j / sqrt(D),  lse = log sum_j exp s_j
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZES = {"f16": 2, "bf16": 2, "e4m3": 1}
#: scales of an 8-bit cache
K_SCALE, V_SCALE = 0.02, 0.015
#: no drawn case reads, computes or keeps more than the largest listed ones
MAX_BYTES, MAX_FLOPS, MAX_ELEMENTS = 1.05e9, 3.4e10, 1.2e9


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # one served step of 64 sequences: latency
        {"name": "bounds_step_64", "op": "bounds", "B": 64, "per": 1, "held": 4000, "pad": 0, "H_kv": 8, "D": 128, "page": 64, "cache": "bf16"},
        # prompts of a batch, packed, beside running sequences, into an 8-bit cache, with padding rows behind them
        {"name": "bounds_prompts_17", "op": "bounds", "B": 17, "per": 1900, "held": 700, "pad": 37, "H_kv": 4, "D": 128, "page": 32, "cache": "e4m3"},
        # one conversation of 32768 tokens: latency
        {"name": "select_one_1", "op": "select", "B": 1, "lo": 32768, "hi": 32768, "H": 32, "H_kv": 8, "D": 128, "page": 64, "count": 32, "first": 1, "last": 1, "type": "bf16"},
        # a ragged batch, sequences from empty to 131072 tokens, some of fewer pages than are chosen
        {"name": "select_ragged_24", "op": "select", "B": 24, "lo": 0, "hi": 131072, "H": 64, "H_kv": 8, "D": 128, "page": 32, "count": 128, "first": 1, "last": 2, "type": "f16"},
        # many short sequences, heads of 64, small pages
        {"name": "select_many_256", "op": "select", "B": 256, "lo": 0, "hi": 4096, "H": 16, "H_kv": 2, "D": 64, "page": 16, "count": 61, "first": 2, "last": 4, "type": "bf16"},
        # one conversation, 32 pages for each head: latency
        {"name": "sparse_one_1", "op": "sparse", "B": 1, "held": 512, "count": 32, "short": 0, "H": 32, "H_kv": 8, "D": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # a served batch, 4096 of 16384 tokens for each head
        {"name": "sparse_batch_64", "op": "sparse", "B": 64, "held": 256, "count": 64, "short": 3, "H": 32, "H_kv": 8, "D": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # an 8-bit cache, small pages that end inside every tile, some sequences that hold little or nothing
        {"name": "sparse_e4m3_48", "op": "sparse", "B": 48, "held": 512, "count": 99, "short": 30, "H": 40, "H_kv": 4, "D": 128, "page": 16, "type": "f16", "cache": "e4m3"},
        # four answers to one short question: latency
        {"name": "shared_four_4", "op": "shared", "groups": 1, "each": 4, "prefix": 1024, "tail": 200, "H": 32, "H_kv": 8, "D": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # 64 questions about one long document
        {"name": "shared_document_64", "op": "shared", "groups": 1, "each": 64, "prefix": 32768, "tail": 1000, "H": 32, "H_kv": 8, "D": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # three assistants' instructions before the conversations of each, an 8-bit cache
        {"name": "shared_groups_93", "op": "shared", "groups": 3, "each": 31, "prefix": 7000, "tail": 2500, "H": 64, "H_kv": 8, "D": 128, "page": 32, "type": "bf16", "cache": "e4m3"},
        # many sequences behind one instruction, heads of 64, small pages
        {"name": "shared_many_256", "op": "shared", "groups": 1, "each": 256, "prefix": 6144, "tail": 300, "H": 16, "H_kv": 2, "D": 64, "page": 16, "type": "f16", "cache": "f16"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS and _elements(case) <= MAX_ELEMENTS:
            return case


def _draw(rng):
    op = rng.choice(["bounds", "select", "sparse", "shared"])
    kv, D = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 128])
    H, page = kv * rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.choice([16, 32, 64, 128])
    t = rng.choice(["bf16", "f16"])
    cache = rng.choice([t, t, "e4m3"]) if D == 128 else t
    if op == "bounds":
        B = _spread(rng, 1, 200)
        return {"op": op, "B": B, "per": rng.choice([1, _spread(rng, 2, 32000 // B)]), "held": _spread(rng, 1, 5000), "pad": rng.choice([0, rng.randint(1, 50)]),
                "H_kv": kv, "D": D, "page": page, "cache": cache}
    if op == "select":
        hi = _spread(rng, 1, 131072)
        first, last = rng.randint(0, 3), rng.randint(1, 4)
        return {"op": op, "B": _spread(rng, 1, 300), "lo": rng.choice([0, 1, hi]), "hi": hi, "H": H, "H_kv": kv, "D": D, "page": page,
                "count": rng.randint(first + last, max(first + last + 1, _spread(rng, 8, 300))), "first": first, "last": last, "type": t}
    if op == "sparse":
        count = _spread(rng, 1, 256)
        return {"op": op, "B": _spread(rng, 1, 128), "held": count + _spread(rng, 1, 600), "count": count, "short": rng.choice([0, 5, 50]), "H": H, "H_kv": kv, "D": D,
                "page": page, "type": t, "cache": cache}
    return {"op": op, "groups": rng.choice([1, 1, 2, 4]), "each": _spread(rng, 1, 200), "prefix": _spread(rng, 16, 32768), "tail": _spread(rng, 1, 3000), "H": H, "H_kv": kv, "D": D,
            "page": page, "type": t, "cache": cache}


def _elements(case):
    """Elements of the largest array that a case keeps, or that its plain form makes."""
    if case["op"] == "bounds":
        return case["B"] * (case["held"] + case["per"]) * case["H_kv"] * case["D"]
    if case["op"] == "select":
        return 2 * case["B"] * -(-case["hi"] // case["page"]) * case["H_kv"] * case["D"]
    if case["op"] == "sparse":
        return case["B"] * case["held"] * case["page"] * case["H_kv"] * case["D"]
    B, H = case["groups"] * case["each"], case["H"]
    return max(B * H * case["prefix"], (B * case["tail"] + case["groups"] * case["prefix"]) * case["H_kv"] * case["D"])


# --------------------------------------------------------------------------
# lengths of a case (they follow from the case alone, so that its work does)
# --------------------------------------------------------------------------
def _random(case, *names):
    s = 17
    for n in names:
        s = (s * 1000003 + case[n]) % (1 << 31)
    return np.random.RandomState(s)


def _growth(case):
    """Tokens held and new tokens of each sequence of a bounds case."""
    r = _random(case, "B", "held", "per", "page")
    held = r.randint(0, case["held"] + 1, case["B"])
    new = np.ones(case["B"], np.int64) if case["per"] == 1 else r.randint(0, case["per"] + 1, case["B"])
    new[0] = max(new[0], 1)
    return held, new


def _held(case):
    """Tokens held by each sequence of a select case."""
    return _random(case, "B", "hi", "lo", "D").randint(case["lo"], case["hi"] + 1, case["B"])


def _chosen(case):
    """Tokens in the chosen pages of each sequence of a sparse case (every K/V head of it chooses as many pages):
    `short` percent of the sequences hold fewer pages than that, or nothing."""
    r = _random(case, "B", "held", "count", "short")
    full = case["count"] * case["page"]
    lens = full - r.randint(0, case["page"], case["B"])
    few = r.rand(case["B"]) * 100 < case["short"]
    return np.where(few, r.randint(0, full + 1, case["B"]), lens)


def _tails(case):
    """Tokens of each sequence of a shared case behind the prefix of its group, and the prefixes' lengths."""
    r = _random(case, "groups", "each", "prefix", "tail")
    own_tokens = r.randint(0, case["tail"] + 1, case["groups"] * case["each"])
    prefix = r.randint(case["prefix"] // 2, case["prefix"] + 1, case["groups"]) if case["groups"] > 1 else np.array([case["prefix"]])
    return own_tokens, prefix // case["page"] * case["page"]


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, kind):
    return torch.randn(shape, device="cuda", generator=g).to(TYPES[kind])


def _pool(case, g, pages):
    """Keys or values of all pages; made in parts, since a whole pool in 32 bits would be twice its size again."""
    kind = case["cache"]
    out = torch.empty((pages, case["H_kv"], case["page"], case["D"]), dtype=TYPES[kind], device="cuda")
    for part in out.split(max(1, (1 << 27) // out[0].numel())):
        x = torch.randn(part.shape, device="cuda", generator=g)
        part.copy_(x / K_SCALE if kind == "e4m3" else x)
    return out


def _scales(case):
    return (K_SCALE, V_SCALE) if case["cache"] == "e4m3" else (1.0, 1.0)


def _int(a):
    return torch.from_numpy(np.ascontiguousarray(a)).int().cuda()


def _table(need, order):
    """Rows of a page table: need[b] pages of each sequence, taken from `order` one after the other."""
    width = max(1, int(need.max()))
    table = np.full((len(need), width), -1, np.int32)
    table[np.arange(width)[None] < need[:, None]] = order[:int(need.sum())]
    return table


def _prepare_bounds(case, g):
    ps, (held, new) = case["page"], _growth(case)
    need = -(-(held + new) // ps)
    pages = int(need.sum()) + 3
    order = torch.randperm(pages, device="cuda", generator=g).cpu().numpy()
    table = _table(need, order)
    seq = np.repeat(np.arange(case["B"]), new)
    pos = held[seq] + np.arange(len(seq)) - (np.cumsum(new) - new)[seq]
    slots = np.full(len(seq) + case["pad"], -1, np.int64)
    slots[:len(seq)] = table[seq, pos // ps] * ps + pos % ps
    k = _pool(case, g, pages)
    # the pages' bounds before the step: over the rows held then; of pages not begun, what their last owner left
    rows = np.zeros(pages, np.int64)
    at = np.arange(table.shape[1])[None]
    live = at < need[:, None]
    rows[table[live]] = np.clip(held[:, None] - at * ps, 0, ps)[live]
    bounds = torch.empty((pages, case["H_kv"], 2, case["D"]), dtype=torch.float16 if case["cache"] == "e4m3" else k.dtype, device="cuda")
    step = max(1, (1 << 27) // k[0].numel())
    for i in range(0, pages, step):
        x = k[i:i + step].float()
        gone = (torch.arange(ps, device="cuda") >= torch.from_numpy(rows[i:i + step]).cuda()[:, None])[:, None, :, None]
        lo, hi = x.masked_fill(gone, math.inf).amin(2), x.masked_fill(gone, -math.inf).amax(2)
        none = torch.isinf(lo)
        old = torch.randn(lo.shape, device="cuda", generator=g)
        bounds[i:i + step, :, 0], bounds[i:i + step, :, 1] = torch.where(none, old - 9, lo), torch.where(none, old + 9, hi)
    return {"k_pool": k, "slots": _int(slots), "bounds": bounds, "page": ps}


def _prepare_select(case, g):
    lens = _held(case)
    need = -(-lens // case["page"])
    pages = max(1, int(need.sum()))
    order = torch.randperm(pages, device="cuda", generator=g).cpu().numpy()
    # keys of a page: normal around a centre of its own, the more of them the wider
    centre = torch.randn((pages, case["H_kv"], 1, case["D"]), device="cuda", generator=g)
    width = math.sqrt(2 * math.log(case["page"])) + 0.3 * torch.randn((pages, case["H_kv"], 2, case["D"]), device="cuda", generator=g).abs()
    bounds = (0.5 * centre + torch.tensor([[-1.0], [1.0]], device="cuda") * width).to(TYPES[case["type"]])
    return {"q": _normal(g, (case["B"], case["H"], 1, case["D"]), case["type"]), "bounds": bounds, "table": _int(_table(need, order)), "lens": _int(lens),
            "page": case["page"], "count": case["count"], "first": case["first"], "last": case["last"]}


def _prepare_sparse(case, g):
    B, kv, ps, held, count = (case[k] for k in ("B", "H_kv", "page", "held", "count"))
    lens = np.repeat(_chosen(case)[:, None], kv, 1)
    # each K/V head of a sequence has its own pages of those that the sequence holds, in order
    at = torch.rand((B, kv, held), device="cuda", generator=g).argsort(-1)[..., :count].sort(-1).values
    pages = torch.randperm(B * held, device="cuda", generator=g).view(B, 1, held).expand(B, kv, held).gather(-1, at)
    live = torch.arange(count, device="cuda") < torch.from_numpy(-(-lens // ps)).cuda()[..., None]
    return {"q": _normal(g, (B, case["H"], 1, case["D"]), case["type"]), "k_pool": _pool(case, g, B * held), "v_pool": _pool(case, g, B * held),
            "pages": torch.where(live, pages, -1).int().contiguous(), "lens": _int(lens), "scales": _scales(case)}


def _prepare_shared(case, g):
    ps, each, (own_tokens, prefix) = case["page"], case["each"], _tails(case)
    need, first = -(-own_tokens // ps), prefix // ps
    pages = int(need.sum() + first.sum()) + 1
    order = torch.randperm(pages, device="cuda", generator=g).cpu().numpy()
    mine = _table(need, order[int(first.sum()):])
    ahead = _table(first, order)
    table = np.full((len(need), int((np.repeat(first, each) + need).max()) + 1), -1, np.int32)
    for b in range(len(need)):
        n = first[b // each]
        table[b, :n] = ahead[b // each, :n]
        table[b, n:n + need[b]] = mine[b, :need[b]]
    s = {"q": _normal(g, (len(need), case["H"], 1, case["D"]), case["type"]), "k_pool": _pool(case, g, pages), "v_pool": _pool(case, g, pages), "table": _int(table),
         "lens": _int(own_tokens + np.repeat(prefix, each)), "shared": _int(prefix), "scales": _scales(case),
         "groups": _int(np.arange(case["groups"] + 1) * each) if case["groups"] > 1 else None}
    # the plain form's own sizes
    s["each"], s["most"], s["tail"] = each, max(1, int(first.max())), max(1, int(need.max()))
    return s


def prepare(case, seed):
    s = globals()["_prepare_" + case["op"]](case, _gen(seed))
    s["op"] = case["op"]
    return s


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
def _plain_bounds(s):
    k, ps, bounds = s["k_pool"], s["page"], s["bounds"]
    slots = s["slots"][s["slots"] >= 0].long()
    page, row = slots // ps, slots % ps
    if k.dtype == torch.float8_e4m3fn:
        x = k.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn).float()
    else:
        x = k[page, :, row].float()
    begun = torch.zeros(len(k), dtype=torch.bool, device=k.device)
    begun[page[row == 0]] = True
    at = torch.unique(page)
    place = torch.empty(len(k), dtype=torch.long, device=k.device)
    place[at] = torch.arange(len(at), device=k.device)
    to = place[page].view(-1, 1, 1).expand_as(x)
    old, fresh = bounds[at].float(), begun[at].view(-1, 1, 1)
    lo = torch.where(fresh, math.inf, old[:, :, 0]).scatter_reduce(0, to, x, "amin")
    hi = torch.where(fresh, -math.inf, old[:, :, 1]).scatter_reduce(0, to, x, "amax")
    bounds[at] = torch.stack([lo, hi], 2).to(bounds.dtype)
    return {"bounds": bounds}


def _plain_select(s):
    q, bounds, table, lens, ps, count = s["q"], s["bounds"], s["table"], s["lens"].long(), s["page"], s["count"]
    (B, H, _, D), kv, width = q.shape, bounds.shape[1], table.shape[1]
    # in 64 bits: pages next to the border differ by little
    x = q.double().view(B, kv, H // kv, D)
    weight = torch.cat([x.clamp(max=0).sum(2), x.clamp(min=0).sum(2)], -1)
    rows = bounds[table.clamp(min=0).long()].transpose(1, 2).reshape(B, kv, width, 2 * D).double()
    score = torch.matmul(rows, weight.unsqueeze(-1)).squeeze(-1)
    live = ((lens + ps - 1) // ps).view(B, 1, 1)
    j = torch.arange(width, device=q.device)
    score = torch.where((j < s["first"]) | (j >= live - s["last"]), math.inf, score)
    score = torch.where(j < live, score, -math.inf)
    best = torch.argsort(score, dim=-1, descending=True, stable=True)[..., :count]
    best = torch.where(best < live, best, width).sort(-1).values
    inside = best < width
    tokens = torch.where(inside, (lens.view(B, 1, 1) - best * ps).clamp(max=ps), 0).sum(-1)
    pages = torch.where(inside, table.unsqueeze(1).expand(B, kv, width).gather(-1, best.clamp(max=width - 1)).long(), -1)
    full = torch.full((B, kv, count), -1, dtype=torch.int32, device=q.device)
    full[..., :best.shape[-1]] = pages
    return {"pages": full, "lens": tokens.int()}


def _dense(pool, rows, scale):
    """Keys or values [..., tokens, D] in 32 bits of page rows [..., pages]; pool [pages, tokens, D]."""
    x = pool.view(torch.uint8)[rows].view(pool.dtype) if pool.dtype == torch.float8_e4m3fn else pool[rows]
    return (x.float() * scale).flatten(-3, -2)


def _softmax(x):
    """exp(x - m), its sum and m of the last axis; nothing counts where all of it is masked."""
    m = x.amax(-1, keepdim=True).clamp(min=-1e30)
    e = torch.exp(x - m)
    return e, e.sum(-1, keepdim=True), m


def _plain_sparse(s):
    q, kp, vp, pages, lens = s["q"], s["k_pool"], s["v_pool"], s["pages"], s["lens"]
    (B, H, _, D), (kv, ps) = q.shape, kp.shape[1:3]
    # pool rows of (page, head)
    rows = pages.clamp(min=0).long() * kv + torch.arange(kv, device=q.device).view(1, kv, 1)
    k, v = _dense(kp.flatten(0, 1), rows, s["scales"][0]), _dense(vp.flatten(0, 1), rows, s["scales"][1])
    x = torch.matmul(q.float().reshape(B, kv, H // kv, D), k.transpose(2, 3)) / math.sqrt(D)
    past = torch.arange(x.shape[-1], device=x.device) >= lens.view(B, kv, 1, 1)
    e, l, m = _softmax(x.masked_fill(past, -math.inf))
    o = torch.matmul(e, v) / l.clamp(min=1e-30)
    return {"o": o.reshape(B, H, 1, D).to(torch.bfloat16), "lse": torch.where(l > 0, m + l.log(), -math.inf).reshape(B, H)}


def _plain_shared(s):
    q, kp, vp, table, lens, each = s["q"], s["k_pool"], s["v_pool"], s["table"].long(), s["lens"].long(), s["each"]
    (B, H, _, D), (kv, ps) = q.shape, kp.shape[1:3]
    G, groups = H // kv, B // each
    head = torch.arange(kv, device=q.device).view(1, kv, 1)
    x = q.float().reshape(B, kv, G, D) / math.sqrt(D)
    prefix = s["shared"].long()

    def attend(x, at, n):
        """x [.., kv, rows, D] over pages at [.., pages], n tokens of them: e V, sum, maximum."""
        rows = at.clamp(min=0).unsqueeze(1) * kv + head
        z = torch.matmul(x, _dense(kp.flatten(0, 1), rows, s["scales"][0]).transpose(2, 3))
        e, l, m = _softmax(z.masked_fill(torch.arange(z.shape[-1], device=z.device) >= n.view(-1, 1, 1, 1), -math.inf))
        return torch.matmul(e, _dense(vp.flatten(0, 1), rows, s["scales"][1])), l, m

    # the prefix of a group, once for all of its sequences
    rows = x.reshape(groups, each, kv, G, D).transpose(1, 2).reshape(groups, kv, each * G, D)
    first = [t.reshape(groups, kv, each, G, -1).transpose(1, 2).reshape(B, kv, G, -1) for t in attend(rows, table[::each, :s["most"]], prefix)]
    # each sequence's own tokens
    ahead = prefix.repeat_interleave(each, output_size=B)
    j = (ahead // ps).unsqueeze(1) + torch.arange(s["tail"], device=q.device)
    second = attend(x, table.gather(1, j.clamp(max=table.shape[1] - 1)), lens - ahead)
    m = torch.maximum(first[2], second[2])
    a, b = torch.exp(first[2] - m), torch.exp(second[2] - m)
    l = a * first[1] + b * second[1]
    o = (a * first[0] + b * second[0]) / l.clamp(min=1e-30)
    return {"o": o.reshape(B, H, 1, D).to(torch.bfloat16), "lse": torch.where(l > 0, m + l.log(), -math.inf).reshape(B, H)}


# --------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------
def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pallas-unbound_b200")
    if at not in sys.path:
        sys.path.insert(0, at)


def _own_bounds(s):
    from pallas_flash.kernels.paged import page_bounds
    page_bounds(s["k_pool"], s["slots"], s["bounds"])
    return {"bounds": s["bounds"]}


def _own_select(s):
    from pallas_flash.kernels.paged import select_pages
    p = select_pages(s["q"], s["bounds"], s["table"], s["lens"], s["count"], page_size=s["page"], first=s["first"], last=s["last"])
    return {"pages": p.pages, "lens": p.lens}


def _own_sparse(s):
    from pallas_flash.kernels.decoding import pallas_flash_decoding
    o, lse = pallas_flash_decoding(s["q"], s["k_pool"], s["v_pool"], kv_lens=s["lens"], page_table=s["pages"],
                                   k_scale=s["scales"][0], v_scale=s["scales"][1], return_lse=True)
    return {"o": o, "lse": lse}


def _own_shared(s):
    from pallas_flash.kernels.decoding import pallas_flash_decoding
    o, lse = pallas_flash_decoding(s["q"], s["k_pool"], s["v_pool"], kv_lens=s["lens"], page_table=s["table"], shared_lens=s["shared"], shared_groups=s["groups"],
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
    kv, D, ps = case["H_kv"], case["D"], case["page"]
    if case["op"] == "bounds":
        held, new = _growth(case)
        tokens, row = int(new.sum()), kv * D
        touched = int((-(-(held + new) // ps) - held // ps)[new > 0].sum())
        begun = int((held % ps > 0)[new > 0].sum())      # bounds of pages begun before are read as well
        return {"bytes": tokens * row * SIZES[case["cache"]] + 4 * row * (touched + begun) + 4 * (tokens + case["pad"]), "flops": 2 * tokens * row}
    if case["op"] == "select":
        need = -(-_held(case) // ps)
        # a sequence that keeps all of its pages needs no scores
        scored = int(need[need > case["count"]].sum())
        return {"bytes": scored * (kv * 2 * D * 2 + 4) + case["B"] * (2 * case["H"] * D + kv * 4 * (case["count"] + 1) + 4), "flops": 4 * scored * kv * D}
    out = 4 * case["H"] * (D + 1)                        # q, o and lse of a sequence
    if case["op"] == "sparse":
        tokens = int(_chosen(case).sum()) * kv
        return {"bytes": 2 * tokens * D * SIZES[case["cache"]] + case["B"] * out + 4 * tokens // ps, "flops": 4 * tokens * (case["H"] // kv) * D}
    own_tokens, prefix = _tails(case)
    held = int(own_tokens.sum()) + int(prefix.sum())
    seen = int(own_tokens.sum()) + case["each"] * int(prefix.sum())
    return {"bytes": 2 * held * kv * D * SIZES[case["cache"]] + len(own_tokens) * out, "flops": 4 * seen * case["H"] * D}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def _wide(pool, at, head, n, scale):
    """The first n keys or values [n, D] of one head in the pages `at`."""
    return pool.view(torch.uint8)[at, head].view(pool.dtype).reshape(-1, pool.shape[3])[:n].double() * scale if pool.dtype == torch.float8_e4m3fn \
        else pool[at, head].reshape(-1, pool.shape[3])[:n].double() * scale


def _attend(q, k, v):
    """o [heads, D] and lse [heads] of q [heads, D] over keys and values [n, D], n > 0."""
    x = q.double() @ k.T * q.shape[-1] ** -0.5
    return torch.softmax(x, -1) @ v, torch.logsumexp(x, -1)


def exact(case, seed):
    s = prepare(case, seed)
    kv, D, ps = case["H_kv"], case["D"], case["page"]
    if case["op"] == "bounds":
        out = s["bounds"].double()
        slots = s["slots"].tolist()
        i = 0
        while i < len(slots) and slots[i] >= 0:
            page, row = divmod(slots[i], ps)
            n = 1
            while row + n < ps and i + n < len(slots) and slots[i + n] == slots[i] + n:
                n += 1
            x = s["k_pool"][page, :, row:row + n].double()
            if row > 0:
                x = torch.cat([x, out[page]], 1)
            out[page, :, 0], out[page, :, 1] = x.min(1).values, x.max(1).values
            i += n
        return {"bounds": out}
    if case["op"] == "select":
        pages = torch.full((case["B"], kv, case["count"]), -1, dtype=torch.int32, device="cuda")
        lens = torch.zeros((case["B"], kv), dtype=torch.int32, device="cuda")
        for b, n in enumerate(_held(case).tolist()):
            live = -(-n // ps)
            if live == 0:
                continue
            at = s["table"][b, :live].long()
            for h in range(kv):
                if live <= case["count"]:
                    keep = torch.arange(live, device="cuda")
                else:
                    x = s["bounds"][at, h].double().unsqueeze(1) * s["q"][b, h * (case["H"] // kv):(h + 1) * (case["H"] // kv), 0].double().unsqueeze(1)
                    score = x.amax(2).sum((1, 2))
                    score[:case["first"]] = math.inf
                    score[live - case["last"]:] = math.inf
                    keep = torch.sort(score, descending=True, stable=True).indices[:case["count"]].sort().values
                pages[b, h, :len(keep)] = at[keep].int()
                lens[b, h] = len(keep) * ps - (live * ps - n if int(keep[-1]) == live - 1 else 0)
        return {"pages": pages, "lens": lens}
    H = case["H"]
    B = s["q"].shape[0]
    o = torch.zeros((B, H, 1, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    if case["op"] == "sparse":
        lens = _chosen(case)
    else:
        own_tokens, prefix = _tails(case)
        lens = own_tokens + np.repeat(prefix, case["each"])
    if B * kv > 20000 or int(lens.sum()) * H * D > 1e12:
        return None
    rows = s["pages"] if case["op"] == "sparse" else s["table"].unsqueeze(1).expand(B, kv, -1)
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            continue
        for h in range(kv):
            at = rows[b, h, :-(-n // ps)].long()
            heads = slice(h * (H // kv), (h + 1) * (H // kv))
            k, v = (_wide(p, at, h, n, c) for p, c in zip((s["k_pool"], s["v_pool"]), s["scales"]))
            o[b, heads, 0], lse[b, heads] = _attend(s["q"][b, heads, 0], k, v)
    return {"o": o, "lse": lse}
