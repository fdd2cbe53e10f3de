"""What the operators between a decoder layer's projections are measured on: the rotation of queries and keys with their
norms, attention over a paged cache, and the care of the cache's pages.

`listed()` names the cases, `draw(rng)` makes further ones of the same ranges.  A case is a dict of plain values:

  op        "attention"  paged_attention over a plan the pass makes
            "rope"       qk_norm_rope; mode "plain": to new tensors; "append": keys and values go to the cache's pages;
                         "train": forward and backward through autograd
            "fork"       kv_fork of every prompt into `samples` requests, and kv_free of these
            "turnover"   kv_free of every `every`-th request and kv_extend of all: a new prompt in each freed one's place, none
                         for the others
            "compact"    kv_compact of a pool of which a share of `live` pages is in use
  dtype     "fp16" or "bf16"
  q_heads, kv_heads, dim, page   heads, head size, tokens of a page
  batch     attention: "NEWxCOUNT@LO-HI,...": COUNT requests that bring NEW tokens each and have LO to HI tokens cached already
  nhd       attention: pages hold [token, head, dim] instead of [head, token, dim]
  rows, rot, norm   rope: tokens, rotated dimensions of a head, with or without the norms
  layers, requests, lo, hi       pages: layers in a page, requests, tokens of a request
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def _attention(dtype, q_heads, kv_heads, dim, page, batch, nhd=False):
    return dict(op="attention", dtype=dtype, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, batch=batch, nhd=nhd)


def _rope(dtype, mode, rows, q_heads, kv_heads, dim, rot, norm, page=16):
    return dict(op="rope", dtype=dtype, mode=mode, rows=rows, q_heads=q_heads, kv_heads=kv_heads, dim=dim, rot=rot, norm=norm,
                page=page)


def _pages(op, dtype, layers, kv_heads, dim, page, requests, lo, hi, **more):
    return dict(op=op, dtype=dtype, layers=layers, kv_heads=kv_heads, dim=dim, page=page, requests=requests, lo=lo, hi=hi, **more)


def listed():
    cases = {
        # two requests decode their first tokens: launches are all there is
        "decode_first": _attention("fp16", 32, 32, 128, 16, "1x2@1-37"),
        # a busy server's decode step, ragged contexts, grouped heads: the cache is read once
        "decode_batch": _attention("bf16", 32, 8, 128, 16, "1x256@0-4095"),
        # a few requests far into long documents: the long axis has to fill the card
        "decode_long": _attention("fp16", 32, 8, 128, 64, "1x3@100001-131000"),
        # prompts join a decoding batch: four of 512 tokens, some over cached prefixes, and 64 single tokens
        "mixed_step": _attention("fp16", 32, 32, 128, 16, "512x4@0-1500,1x64@1-2000"),
        # a chunk of a long prompt over what is cached of it: the matrix cores
        "chunk_long": _attention("bf16", 32, 8, 128, 16, "2048x1@14336-14336"),
        # the rotation of a decode step, keys and values to the cache
        "rope_decode": _rope("fp16", "append", 256, 32, 8, 128, 128, False),
        # a prefill batch with norms
        "rope_prefill": _rope("bf16", "append", 2112, 32, 32, 128, 128, True),
        # four training sequences of 1024 tokens, forward and backward
        "rope_train": _rope("bf16", "train", 4096, 32, 8, 128, 128, True),
        # small heads of which half is rotated, an odd number of rows
        "rope_train_odd": _rope("fp16", "train", 1021, 12, 4, 64, 32, True),
        # sixteen prompts answered eight times each
        "fork_samples": _pages("fork", "bf16", 8, 8, 128, 16, 16, 17, 2000, samples=8),
        # a quarter of a batch has finished and makes room for new prompts
        "turnover": _pages("turnover", "fp16", 1, 8, 128, 16, 256, 1, 4000, every=4),
        # a pool half of whose pages are free, everywhere, is packed to its front
        "compact": _pages("compact", "bf16", 8, 8, 128, 16, 64, 100, 1000, live=0.5),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 5e14)


def draw(rng: random.Random):
    """A case of the ranges the listed ones stand for: 1 to 256 requests of 0 to 131072 cached tokens and chunks of 1 to 2048, 1 to
    64 query heads, pages of 8 to 128 tokens (odd ones among them); 1 to 8192 rotated rows; 1 to 256 requests in a pool."""
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    most = max(_cost(c) for c in listed())
    while True:
        dtype, dim = rng.choice(["fp16", "bf16"]), rng.choice([64, 128, 128])
        kv_heads, group = rng.choice([1, 2, 3, 4, 8, 8, 16, 32]), rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8])
        page = rng.choice([8, 16, 16, 16, 20, 32, 64, 128])
        family = rng.choice(["decode", "chunk", "mixed", "rope", "rope", "rope", "fork", "turnover", "compact"])
        if kv_heads * group > 64:
            continue
        if family in ("decode", "chunk", "mixed"):
            parts = []
            if family != "decode":
                hi = log(1, 16384)
                parts.append(f"{log(2, 2048)}x{log(1, 8)}@{rng.choice([0, hi, hi // 2])}-{hi}")
            if family != "chunk":
                hi = log(1, 131072)
                parts.append(f"1x{log(1, 256)}@{rng.choice([0, hi // 2])}-{hi}")
            case = _attention(dtype, kv_heads * group, kv_heads, dim, page, ",".join(parts), rng.random() < 0.25)
        elif family == "rope":
            dim = rng.choice([64, 96, 128, 128, 256])
            case = _rope(dtype, rng.choice(["plain", "append", "train", "train"]), log(1, 8192), kv_heads * group, kv_heads, dim,
                         rng.choice([dim, dim, dim // 2]), rng.random() < 0.6, page)
        else:
            lo = log(1, 1000)
            requests = log(4 if family == "turnover" else 1, 64 if family == "fork" else 256)
            case = _pages(family, dtype, log(1, 16), min(kv_heads, 16), dim, page, requests, lo, lo + log(1, 2500))
            case |= {"fork": dict(samples=log(1, 16)), "turnover": dict(every=rng.randint(2, 4)),
                     "compact": dict(live=round(rng.uniform(0.3, 0.95), 2))}[family]
            if family == "turnover":
                case["layers"] = 1
            if _pool_pages(case) * _page_bytes(case) > 2.6e9:
                continue
        if case["op"] == "attention" and _padded(case) > 3e9:
            continue
        if _cost(case) <= most:
            return case


# ---- sizes of a case ---------------------------------------------------------------------------------------

def _spread(n, lo, hi):
    """n lengths from lo to hi, the same for every seed (their order is the seed's)."""
    return [lo + (i * 2654435761 + 12345) % 4294967296 % (hi - lo + 1) for i in range(n)]


def _batch(case):
    """[(new tokens, cached tokens)] of an attention case."""
    seqs = []
    for part in case["batch"].split(","):
        what, span = part.split("@")
        new, count = (int(v) for v in what.split("x"))
        lo, hi = (int(v) for v in span.split("-"))
        seqs += [(new, c) for c in _spread(count, lo, hi)]
    return seqs


def _padded(case):
    """Bytes of the largest temporary of an attention case's plain form."""
    most = 0
    for one in (True, False):
        group = [(n, c) for n, c in _batch(case) if (n == 1) == one]
        if group:
            keys, new = max(n + c for n, c in group), max(n for n, _ in group)
            most = max(most, 4 * len(group) * keys * max(case["kv_heads"] * case["dim"], case["q_heads"] * new))
    return most / 2


def _lengths(case):
    return _spread(case["requests"], case["lo"], case["hi"])


def _pages_of(tokens, page):
    return -(-tokens // page)


def _page_bytes(case):
    return case["layers"] * 2 * case["kv_heads"] * case["page"] * case["dim"] * 2


def _pool_pages(case):
    pages = [_pages_of(n, case["page"]) for n in _lengths(case)]
    if case["op"] == "fork":
        return sum(pages) + len(pages) * case["samples"] + 7
    if case["op"] == "turnover":
        return sum(pages) + sum(sorted(_pages_of(n, case["page"]) for n in _lengths(case))) // 4 + 9
    return int(sum(pages) / case["live"]) + 1


def work(case):
    """What a pass cannot do without: every input read once, every output written once."""
    if case["op"] == "attention":
        rows, keys, pairs = 0, 0, 0
        for n, c in _batch(case):
            rows, keys, pairs = rows + n, keys + n + c, pairs + n * c + n * (n + 1) // 2
        return {"bytes": 4 * case["dim"] * (keys * case["kv_heads"] + rows * case["q_heads"]),
                "flops": 4 * case["dim"] * case["q_heads"] * pairs}
    if case["op"] == "rope":
        heads, one = case["q_heads"] + case["kv_heads"], 2 * case["rows"] * case["dim"]
        each = {"plain": 2 * heads, "append": 2 * heads + 2 * case["kv_heads"],
                "train": (2 + (3 if case["norm"] else 2)) * heads}[case["mode"]]
        return {"bytes": one * each + case["rows"] * (4 * case["rot"] + 4), "flops": 8 * case["rows"] * heads * case["dim"]}
    if case["op"] == "fork":
        filled = sum(n % case["page"] for n in _lengths(case)) * case["samples"]
        kept = sum(_pages_of(n, case["page"]) for n in _lengths(case)) * case["samples"]
        return {"bytes": 2 * filled * _page_bytes(case) / case["page"] + 16 * kept + 4 * _pool_pages(case), "flops": 0}
    if case["op"] == "turnover":
        new = sum(_lengths(case)[::case["every"]])
        return {"bytes": 12 * new + 16 * new / case["page"] + 4 * _pool_pages(case) + 24 * case["requests"], "flops": 0}
    pages = sum(_pages_of(n, case["page"]) for n in _lengths(case))
    moved = pages * (1 - pages / _pool_pages(case))
    return {"bytes": 2 * moved * _page_bytes(case) + 8 * pages + 8 * _pool_pages(case), "flops": 0}


# ---- inputs ------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _tables(lengths, page, pool, r, spare_rows=0, width=None):
    """Page tables [requests + spare rows, widest] of requests whose pages lie anywhere in the pool, and the pages' uses."""
    ids = r.sample(range(pool), sum(_pages_of(n, page) for n in lengths))
    width = width or max([_pages_of(n, page) for n in lengths] + [1])
    rows, refs, at = [], [0] * pool, 0
    for n in lengths:
        k = _pages_of(n, page)
        rows.append(ids[at:at + k] + [-1] * (width - k))
        at += k
    for i in ids:
        refs[i] = 1
    rows += [[-1] * width] * spare_rows
    return (torch.tensor(rows, dtype=torch.int32).cuda(), torch.tensor(refs, dtype=torch.int32).cuda())


def prepare(case, seed):
    g, r, dt = _gen(seed), random.Random(int(seed)), DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "attention":
        seqs = _batch(case)
        ones = [c for n, c in seqs if n == 1]
        k = r.randrange(len(ones)) if ones else 0  # who has which context is the seed's
        ones = ones[k:] + ones[:k]
        seqs = [(n, c) for n, c in seqs if n > 1] + [(1, c) for c in ones]
        lens, D, Hq, Hkv, P = [n + c for n, c in seqs], case["dim"], case["q_heads"], case["kv_heads"], case["page"]
        pool = sum(_pages_of(n, P) for n in lens) + 3
        s["table"], _ = _tables(lens, P, pool, r)
        shape = (pool, P, Hkv, D) if case["nhd"] else (pool, Hkv, P, D)
        # keys lie some way off the origin, as a model's do; sizes as behind a norm
        kc, vc = _randn(g, *shape, dtype=dt) + 0.5 * _randn(g, D, dtype=dt), _randn(g, *shape, dtype=dt)
        s["k_cache"], s["v_cache"] = (kc.transpose(1, 2), vc.transpose(1, 2)) if case["nhd"] else (kc, vc)
        s["new"], s["lens"], s["rows"] = [n for n, _ in seqs], lens, sum(n for n, _ in seqs)
        s["q"] = _randn(g, s["rows"], Hq, D, dtype=dt)
        s["q_indptr"] = torch.tensor([0] + [n for n, _ in seqs], dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        s["kv_len"] = torch.tensor(lens, dtype=torch.int32).cuda()
    elif case["op"] == "rope":
        T, Hq, Hkv, D, rot, P = (case[k] for k in ("rows", "q_heads", "kv_heads", "dim", "rot", "page"))
        qkv = _randn(g, T, (Hq + 2 * Hkv) * D, dtype=dt)  # one projection's output, the three side by side
        s["q"], s["k"], s["v"] = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
        far = 16384
        angle = torch.arange(far, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
        first = r.randrange(far - T) if case["mode"] != "append" else 0
        s["positions"] = (torch.arange(T, dtype=torch.int32, device="cuda") + first if case["mode"] != "append" else
                          torch.randint(0, far, (T,), generator=g, device="cuda", dtype=torch.int32))
        weight = lambda: (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dt) if case["norm"] else None
        s["q_weight"], s["k_weight"] = weight(), weight()
        if case["mode"] == "append":
            pool = _pages_of(T, P) * 2 + 1
            s["k_cache"], s["v_cache"] = (torch.zeros(pool, Hkv, P, D, dtype=dt, device="cuda") for _ in range(2))
            s["slots"] = torch.randperm(pool * P, generator=g, device="cuda")[:T].contiguous()
        if case["mode"] == "train":
            s["q"], s["k"] = (t.contiguous().requires_grad_(True) for t in (s["q"], s["k"]))
            if case["norm"]:
                s["q_weight"].requires_grad_(True), s["k_weight"].requires_grad_(True)
            s["gq"], s["gk"] = _randn(g, T, Hq, D, dtype=dt), _randn(g, T, Hkv, D, dtype=dt)
    else:
        lens, P, pool = _lengths(case), case["page"], _pool_pages(case)
        k = r.randrange(len(lens)) if case["op"] != "turnover" else 0
        children = len(lens) * case.get("samples", 0)
        s["table0"], s["refs0"] = _tables(lens[k:] + lens[:k], P, pool, r, children,
                                          _pages_of(case["hi"], P) if case["op"] == "turnover" else None)
        s["length0"] = torch.tensor(lens[k:] + lens[:k] + [0] * children, dtype=torch.int32).cuda()
        s["table"], s["refs"], s["length"] = s["table0"].clone(), s["refs0"].clone(), s["length0"].clone()
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        if case["op"] != "turnover":
            s["pool"] = _randn(g, pool, case["layers"], 2, case["kv_heads"], P, case["dim"], dtype=dt)
        if case["op"] == "fork":
            s["parents"] = torch.arange(len(lens), dtype=torch.int32).repeat_interleave(case["samples"]).cuda()
            s["children"] = torch.arange(len(lens), len(lens) + children, dtype=torch.int32).cuda()
        if case["op"] == "turnover":
            done = list(range(len(lens)))[::case["every"]]
            new = [lens[i] for i in done]
            s["done"] = torch.tensor(done, dtype=torch.int32).cuda()
            s["requests"] = torch.arange(len(lens), dtype=torch.int32).cuda()
            counts = torch.zeros(len(lens), dtype=torch.int32)
            counts[torch.tensor(done)] = torch.tensor(new, dtype=torch.int32)
            s["counts"], s["rows"] = counts.cuda(), sum(new)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------

def _attend(q, first, new, lens, table, k_cache, v_cache):
    """Attention of a group of requests padded to their longest: [rows of the group in order, Hq, D] in float."""
    S, n, L, dev = len(lens), max(new), max(lens), q.device
    Hq, D = q.shape[1:]
    Hkv, P = k_cache.shape[1:3]
    new_, lens_, first_ = (torch.tensor(v, device=dev) for v in (new, lens, first))
    j = torch.arange(n, device=dev)
    rows = (first_[:, None] + j).clamp(max=q.shape[0] - 1)                       # [S, n]
    pages = table[:, :_pages_of(L, P)].long().clamp(min=0)
    k, v = (c[pages].float().transpose(1, 2).reshape(S, Hkv, -1, D) for c in (k_cache, v_cache))
    qg = q[rows].float().reshape(S, n, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, -1, D)
    score = (qg @ k.transpose(2, 3)).mul_(D ** -0.5).reshape(S, Hq, n, -1)
    at = torch.arange(score.shape[-1], device=dev)
    score.masked_fill_(at > ((lens_ - new_)[:, None] + j)[:, None, :, None], -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    score = score.div_(score.sum(-1, keepdim=True))
    v = v * (at < lens_[:, None])[:, None, :, None]
    out = (score.reshape(S, Hkv, -1, score.shape[-1]) @ v).reshape(S, Hq, n, D).transpose(1, 2)
    return out[j < new_[:, None]]


def _attention_plain(s):
    chunks = sum(n > 1 for n in s["new"])
    first = s["q_indptr"].tolist()
    args = lambda a, b: (s["q"], first[a:b], s["new"][a:b], s["lens"][a:b], s["table"][a:b], s["k_cache"], s["v_cache"])
    parts = [_attend(*args(0, chunks))] if chunks else []
    parts += [_attend(*args(chunks, len(s["new"])))] if chunks < len(s["new"]) else []
    return torch.cat(parts).to(s["q"].dtype)


def _normed(x, w):
    x = x.float()
    if w is None:
        return x, None
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return x * r * w.float(), r


def _turned(y, cos, sin):
    h = cos.shape[-1]
    a, b = y[..., :h], y[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * h:]], -1)


def _rope_grad(g, x, w, r, cos, sin):
    g = _turned(g.float(), cos, -sin)
    if w is None:
        return g.to(x.dtype), None
    gw, x_ = g * w.float(), x.float()
    dx = r * (gw - x_ * r.square() * (gw * x_).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * x_ * r).sum((0, 1)).to(w.dtype)


def _rope_plain(s):
    q, k, dt = s["q"].detach(), s["k"].detach(), s["q"].dtype
    cos, sin = s["table"][s["positions"].long()][:, None].chunk(2, -1)
    (qn, qr), (kn, kr) = _normed(q, s["q_weight"]), _normed(k, s["k_weight"])
    qo, ko = _turned(qn, cos, sin).to(dt), _turned(kn, cos, sin).to(dt)
    if s["case"]["mode"] == "plain":
        return qo, ko
    if s["case"]["mode"] == "append":
        page, at = s["slots"] // s["case"]["page"], s["slots"] % s["case"]["page"]
        s["k_cache"][page, :, at] = ko
        s["v_cache"][page, :, at] = s["v"]
        return qo, s["k_cache"], s["v_cache"]
    dq, dqw = _rope_grad(s["gq"], q, s["q_weight"], qr, cos, sin)
    dk, dkw = _rope_grad(s["gk"], k, s["k_weight"], kr, cos, sin)
    return [qo, ko, dq, dk] + ([dqw, dkw] if dqw is not None else [])


def _free_plain(table, length, refs, requests):
    ids = table[requests.long()]
    refs.index_add_(0, ids[ids >= 0].long(), -torch.ones_like(ids[ids >= 0]))
    table[requests.long()] = -1
    length[requests.long()] = 0


def _fork_plain(s):
    pool, table, length, refs, P = s["pool"], s["table"], s["length"], s["refs"], s["case"]["page"]
    parents, children = s["parents"].long(), s["children"].long()
    n = length[parents].long()
    full, rest = n // P, n % P
    free = (refs == 0).nonzero()[:, 0]
    fresh = free[(rest > 0).cumsum(0) - 1]
    col = torch.arange(table.shape[1], device=table.device)
    ids = torch.where(col < full[:, None], table[parents], -1)
    shared = ids[ids >= 0].long()
    last = table[parents].gather(1, full.clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    cut = rest > 0
    ids[cut] = ids[cut].scatter(1, full[cut][:, None], fresh[cut][:, None].int())
    table[children] = ids
    length[children] = n.int()
    refs.index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    refs[fresh[cut]] = 1
    flat = pool.view(pool.shape[0], -1, *pool.shape[-2:])
    take = (torch.arange(P, device=pool.device) < rest[cut][:, None])[:, None, :, None]
    flat[fresh[cut]] = torch.where(take, flat[last[cut].long()], flat[fresh[cut]])


def _extend_plain(s):
    table, length, refs, P = s["table"], s["length"], s["refs"], s["case"]["page"]
    req, old = s["requests"].long(), length[s["requests"].long()].long()
    new = old + s["counts"]
    had, has = (old + P - 1) // P, (new + P - 1) // P
    start = (has - had).cumsum(0) - (has - had)
    free = (refs == 0).nonzero()[:, 0]
    col = torch.arange(table.shape[1], device=table.device)
    take = (col >= had[:, None]) & (col < has[:, None])
    got = free[(start[:, None] + col - had[:, None]).clamp(0, free.shape[0] - 1)]
    table[req] = torch.where(take, got.int(), table[req])
    refs[got[take]] = 1
    length[req] = new.int()
    indptr = torch.cat([new.new_zeros(1), s["counts"].long().cumsum(0)])
    rows = torch.arange(s["rows"], device=table.device)
    seq = torch.searchsorted(indptr, rows, right=True) - 1
    pos = old[seq] + rows - indptr[seq]
    slots = table[req[seq], pos // P].long() * P + pos % P
    return indptr.int(), new.int(), pos.int(), slots


def _compact_plain(s):
    pool, table, refs = s["pool"], s["table"], s["refs"]
    live = refs > 0
    n = live.sum()
    at = torch.arange(refs.shape[0], device=refs.device)
    to, frm = (~live & (at < n)).nonzero()[:, 0], (live & (at >= n)).nonzero()[:, 0]
    pool[to] = pool[frm]
    moved = at.clone()
    moved[frm] = to
    table.copy_(torch.where(table >= 0, moved[table.long().clamp(min=0)].int(), -1))
    refs[to] = refs[frm]
    refs[frm] = 0


def _pages_pass(s):
    """Fork: the children's tables and pages as the fork leaves them.  Turnover: the step's tables.  Compact: all of it."""
    case = s["case"]
    if own:
        from loquetier_amd.ops import _kernels as K
    if case["op"] == "fork":
        if own:
            K.kv_fork(s["pool"], s["table"], s["length"], s["refs"], s["parents"], s["children"], s["status"])
        else:
            _fork_plain(s)
        forked = s["table"].clone(), s["length"].clone(), s["refs"].clone()
        if own:
            K.kv_free(s["table"], s["length"], s["refs"], s["children"], case["page"], s["status"])
        else:
            _free_plain(s["table"], s["length"], s["refs"], s["children"])
        return forked, s["table"], s["length"], s["refs"], s["pool"]
    if case["op"] == "turnover":
        if own:
            K.kv_free(s["table"], s["length"], s["refs"], s["done"], case["page"], s["status"])
            step = K.kv_extend(s["table"], s["length"], s["refs"], s["requests"], s["counts"], s["rows"], case["page"], s["status"])
        else:
            _free_plain(s["table"], s["length"], s["refs"], s["done"])
            step = _extend_plain(s)
        return tuple(step), s["table"], s["length"], s["refs"]
    s["table"].copy_(s["table0"])  # the pages that move keep their contents, so the same pool can be packed again
    s["refs"].copy_(s["refs0"])
    if own:
        K.kv_compact(s["pool"], s["table"], s["refs"])
    else:
        _compact_plain(s)
    return s["table"], s["refs"], s["pool"]


def run(s):
    case = s["case"]
    if case["op"] not in ("attention", "rope"):
        return _pages_pass(s)
    if not own:
        return _attention_plain(s) if case["op"] == "attention" else _rope_plain(s)
    from loquetier_amd.kernel_utils import qk_norm_rope
    from loquetier_amd.ops import _kernels as K
    if case["op"] == "attention":
        plan = K.AttentionPlan(s["q_indptr"], s["kv_len"], s["table"], s["rows"], case["q_heads"], case["kv_heads"], case["page"])
        out = torch.empty_like(s["q"])
        K.paged_attention(out, s["q"], s["k_cache"], s["v_cache"], plan)
        return out
    if case["mode"] == "train":
        outs = qk_norm_rope.apply(s["q"], s["k"], s["q_weight"], s["k_weight"], s["table"], s["positions"], EPS)
        leaves = [s["q"], s["k"]] + ([s["q_weight"], s["k_weight"]] if case["norm"] else [])
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, (s["gq"], s["gk"])))
    q_out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    if case["mode"] == "append":
        K.qk_norm_rope(q_out, None, s["q"], s["k"], s["table"], s["positions"], s["q_weight"], s["k_weight"], EPS,
                       v=s["v"], k_cache=s["k_cache"], v_cache=s["v_cache"], slots=s["slots"])
        return q_out, s["k_cache"], s["v_cache"]
    k_out = torch.empty(s["k"].shape, dtype=s["k"].dtype, device=s["k"].device)
    K.qk_norm_rope(q_out, k_out, s["q"], s["k"], s["table"], s["positions"], s["q_weight"], s["k_weight"], EPS)
    return q_out, k_out


# ---- the definitions in 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] not in ("attention", "rope"):
        return None  # whole numbers and copies
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _attention_exact(case, s)
    cos, sin = s["table"][s["positions"].long()].double().chunk(2, -1)
    turn = torch.complex(cos, sin)[:, None]
    h = turn.shape[-1]

    def of(x, w):  # one complex number for each pair of dimensions, turned by the angle
        y = x if w is None else x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w
        z = torch.complex(y[..., :h], y[..., h:2 * h]) * turn
        return torch.cat([z.real, z.imag, y[..., 2 * h:]], -1)

    grad = case["mode"] == "train"
    leaf = lambda t: None if t is None else t.detach().double().requires_grad_(grad)
    q, k, qw, kw = (leaf(s[n]) for n in ("q", "k", "q_weight", "k_weight"))
    qo, ko = of(q, qw), of(k, kw)
    if case["mode"] == "plain":
        return qo, ko
    if case["mode"] == "append":
        flat = [torch.zeros(s["k_cache"].shape, dtype=torch.float64, device="cuda").transpose(1, 2).contiguous() for _ in range(2)]
        for f, x in zip(flat, (ko, s["v"].double())):
            f.flatten(0, 1)[s["slots"]] = x
        return qo, flat[0].transpose(1, 2), flat[1].transpose(1, 2)
    leaves = [q, k] + ([qw, kw] if case["norm"] else [])
    return [qo.detach(), ko.detach()] + list(torch.autograd.grad((qo, ko), leaves, (s["gq"].double(), s["gk"].double())))


def _attention_exact(case, s):
    Hq, Hkv, D, P = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    if work(case)["flops"] > 2e12 or len(s["lens"]) * Hkv > 10000:
        return None
    out, row, group = torch.zeros(s["rows"], Hq, D, dtype=torch.float64, device="cuda"), 0, Hq // Hkv
    for i, (new, length) in enumerate(zip(s["new"], s["lens"])):
        token = torch.arange(length, device="cuda")
        page, at = s["table"][i].long()[token // P], token % P
        for head in range(Hkv):
            k, v = s["k_cache"][page, head, at].double(), s["v_cache"][page, head, at].double()
            q = s["q"][row:row + new, head * group:(head + 1) * group].double()
            for a in range(0, new, 512):
                score = torch.matmul(q[a:a + 512].flatten(0, 1), k.t().contiguous()) / math.sqrt(D)
                last = length - new + torch.arange(a, min(new, a + 512), device="cuda").repeat_interleave(group)
                score = torch.where(token <= last[:, None], score, -math.inf)
                out[row + a:row + min(new, a + 512), head * group:(head + 1) * group] = \
                    torch.matmul(torch.softmax(score, 1), v).unflatten(0, (-1, group))
        row += new
    return out
