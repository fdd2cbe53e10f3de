"""What the operators around a fine-tuning step of adapters are measured on: the residual's addition with the norm behind it, the
loss over the vocabulary with its gradient, and the update of many tensors.

`listed()` names the cases, `draw(rng)` makes further ones of the same ranges.  A case is a dict of plain values:

  op        "loss"   linear_cross_entropy; grad "none": row by row, without gradients; "x": means by partition and the gradient of the
                     rows; "xw": that of the vocabulary's matrix too
            "norm"   add_rms_norm; mode "train": forward and backward through autograd; "serve": the sum, the norm, and the norm in 8
                     bits with a scale for each row (group 0) or each `group` columns
            "adamw"  adamw_step of `adapters` adapters of `layers` layers
  dtype     "fp16" or "bf16"
  rows, hidden, vocab, parts, labelled   loss: rows, their width, vocabulary, partitions, share of rows that have a label
  rows, cols                             norm
  rank, shapes, bits, master             adamw: "OUTxIN,..." of a layer's projections, states of 8 or 32 bits, with or without float weights
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
BLOCK = 256    # weights that share a scale of the 8-bit states; tensors begin at a multiple of it in the flat states
MOST8 = 448.0  # the largest e4m3


def _loss(dtype, rows, hidden, vocab, grad, parts=1, labelled=1.0):
    return dict(op="loss", dtype=dtype, rows=rows, hidden=hidden, vocab=vocab, grad=grad, parts=parts, labelled=labelled)


def _norm(dtype, mode, rows, cols, group=0):
    return dict(op="norm", dtype=dtype, mode=mode, rows=rows, cols=cols, group=group)


def _adamw(dtype, adapters, layers, rank, shapes, bits, master):
    return dict(op="adamw", dtype=dtype, adapters=adapters, layers=layers, rank=rank, shapes=shapes, bits=bits, master=master)


QKVO = "4096x4096,4096x4096,4096x4096,4096x4096"
ALL7 = QKVO + ",11008x4096,11008x4096,4096x11008"


def listed():
    cases = {
        # a few rows of a small model's evaluation: launches are all there is
        "loss_small": _loss("fp16", 33, 512, 2000, "none"),
        # the last rows of evaluation requests against a large vocabulary: its matrix is read once
        "loss_eval": _loss("bf16", 200, 4096, 128256, "none"),
        # four adapters' training partitions of 1024 rows, prompts without labels, frozen head
        "loss_adapters": _loss("bf16", 4096, 4096, 32000, "x", 4, 0.6),
        # the head is trained too
        "loss_head": _loss("fp16", 2048, 4096, 32000, "xw", 2),
        # long sequences over a large vocabulary, every row labelled, odd sizes
        "loss_long": _loss("bf16", 4099, 4096, 128256, "x", 3),
        # a decode batch: the residual, the norm and its 8-bit form for base matrices held in 8 bits
        "norm_decode": _norm("fp16", "serve", 256, 4096),
        # a prefill batch, scales by 128 columns
        "norm_prefill": _norm("bf16", "serve", 2112, 4096, 128),
        # four training sequences of 1024 rows
        "norm_train": _norm("bf16", "train", 4096, 4096),
        # a small model's odd batch
        "norm_train_odd": _norm("fp16", "train", 1021, 1048),
        # one adapter on q/k/v/o of eight layers, states in float
        "adamw_adapter": _adamw("fp16", 1, 8, 16, QKVO, 32, True),
        # four adapters on all projections of eight layers, float weights beside the 16-bit ones
        "adamw_adapters": _adamw("bf16", 4, 8, 32, ALL7, 32, True),
        # the same with states in 8 bits
        "adamw_8bit": _adamw("bf16", 4, 8, 32, ALL7, 8, True),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 5e14)


def draw(rng: random.Random):
    """A case of the ranges the listed ones stand for: 1 to 8192 rows of 64 to 8192 columns against 100 to 160000 words in 1 to 16
    partitions; norms of 1 to 16384 rows of 64 to 16384 columns; 1 to 8 adapters of ranks 8 to 64 on 1 to 32 layers of any sizes."""
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("loss", "norm", "adamw")}
    while True:
        dtype, op = rng.choice(["fp16", "bf16"]), rng.choice(["loss", "loss", "norm", "adamw"])
        if op == "loss":
            case = _loss(dtype, log(1, 8192), 8 * log(8, 1024), log(100, 160000), rng.choice(["none", "x", "x", "xw"]), log(1, 16),
                         rng.choice([1.0, round(rng.uniform(0.1, 1.0), 2)]))
        elif op == "norm":
            cols = 8 * log(8, 2048)
            case = _norm(dtype, rng.choice(["train", "serve"]), log(1, 16384), cols)
            if case["mode"] == "serve" and rng.random() < 0.5:
                case["cols"] = max(128, cols // 128 * 128)
                case["group"] = 128
        else:
            sizes = [8 * log(32, 1376) for _ in range(4)]
            shapes = ",".join(f"{rng.choice(sizes)}x{rng.choice(sizes)}" for _ in range(rng.randint(1, 7)))
            case = _adamw(dtype, log(1, 8), log(1, 32), rng.choice([8, 16, 16, 32, 64]), shapes, rng.choice([8, 32]),
                          rng.random() < 0.6)
            if len(_sizes(case)) > 1200:
                continue
        if _cost(case) <= most[op]:
            return case


# ---- sizes of a case ---------------------------------------------------------------------------------------

def _has_label(case):
    """Which rows have a label, the same for every seed."""
    n = case["rows"]
    return [(i * 2654435761 + 12345) % 4294967296 < case["labelled"] * 4294967296 for i in range(n)]


def _sizes(case):
    """Weights' sizes of an adamw case, adapter by adapter: A [rank, in] and B [out, rank] of each projection."""
    one = []
    for shape in case["shapes"].split(","):
        out, in_ = (int(v) for v in shape.split("x"))
        one += [(case["rank"], in_), (out, case["rank"])]
    return one * (case["layers"] * case["adapters"])


def work(case):
    """What a pass cannot do without: every input read once, every output written once, the products of the labelled rows."""
    if case["op"] == "loss":
        T, H, V, n = case["rows"], case["hidden"], case["vocab"], sum(_has_label(case))
        products = {"none": 1, "x": 2, "xw": 3}[case["grad"]]
        return {"bytes": 2 * V * H * (2 if case["grad"] == "xw" else 1) + 2 * T * H * (1 if case["grad"] == "none" else 2) + 12 * T,
                "flops": 2 * products * n * V * H}
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        if case["mode"] == "train":
            return {"bytes": 2 * n * (4 + 4) + 4 * case["cols"], "flops": 16 * n}
        scales = case["rows"] * (case["cols"] // case["group"] if case["group"] else 1)
        return {"bytes": 9 * n + 4 * scales + 2 * case["cols"], "flops": 8 * n}
    n = sum(a * b for a, b in _sizes(case))
    return {"bytes": n * (6 + (8 if case["master"] else 0) + (16 if case["bits"] == 32 else 4)), "flops": 14 * n}


# ---- inputs ------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rounded8(x):
    """Blocks [n, BLOCK] of floats in e4m3 and their scales."""
    scale = x.abs().amax(1) / MOST8
    return (x / torch.where(scale > 0, scale, 1)[:, None]).to(torch.float8_e4m3fn), scale


def _root8(v):
    """Blocks of second averages: their roots in e4m3, none of which becomes zero, and their scales."""
    code, scale = _rounded8(v.sqrt())
    least = torch.full((), 2.0 ** -9, device=v.device).to(torch.float8_e4m3fn)
    return torch.where((v > 0) & (code.float() == 0), least, code), scale


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    s = dict(case=case)
    if case["op"] == "loss":
        T, H, V = case["rows"], case["hidden"], case["vocab"]
        # logits of a trained model: spread 2.5, the label's some way above, by an amount that differs from row to row
        s["w"] = (torch.randn(V, H, generator=g, device="cuda", dtype=dt) * (2.5 / math.sqrt(H))).requires_grad_(case["grad"] == "xw")
        labels = torch.randint(0, V, (T,), generator=g, device="cuda")
        x = randn(T, H) + torch.rand(T, 1, generator=g, device="cuda") * 1.6 * s["w"].detach()[labels].float()
        s["x"] = x.to(dt).requires_grad_(case["grad"] != "none")
        s["labels"] = torch.where(torch.tensor(_has_label(case)).cuda(), labels, -100)
        if case["grad"] != "none":
            P = case["parts"]
            s["partition"] = torch.tensor([T * p // P for p in range(P + 1)], dtype=torch.int32).cuda()
            s["g"] = 0.5 + torch.rand(P, generator=g, device="cuda")
    elif case["op"] == "norm":
        T, H = case["rows"], case["cols"]
        s["x"], s["residual"] = (0.3 * randn(T, H)).to(dt), (2 * randn(T, H) * (0.5 + randn(H).abs())).to(dt)
        s["w"] = (1 + 0.1 * randn(H)).to(dt)
        if case["mode"] == "train":
            for n in ("x", "residual", "w"):
                s[n].requires_grad_(True)
            s["g"], s["gh"] = randn(T, H).to(dt), (0.5 * randn(T, H)).to(dt)
    else:
        sizes = _sizes(case)
        # the weights' tensors lie in one buffer, and so do their gradients
        s["weights"], gradients = ((randn(sum(a * b for a, b in sizes)) * by).to(dt) for by in (0.02, 1e-3))
        s["params"], s["grads"] = ([t.view(n) for t, n in zip(flat.split([a * b for a, b in sizes]), sizes)]
                                   for flat in (s["weights"], gradients))
        blocks = [-(-a * b // BLOCK) for a, b in sizes]
        n = sum(blocks)
        s["blocks"], s["block_tensor"] = blocks, torch.arange(len(sizes)).repeat_interleave(torch.tensor(blocks)).cuda()
        there = _flat([torch.ones_like(t) for t in s["params"]], s)  # the rest of a tensor's last block is zeros
        m, v = randn(n, BLOCK) * 1e-3 * there, ((randn(n, BLOCK) * 1e-3).square() + 1e-8) * there
        if case["bits"] == 8:
            (s["m"], s["m_scale"]), (s["v"], s["v_scale"]) = _rounded8(m), _root8(v)
        else:
            s["m"], s["v"], s["m_scale"], s["v_scale"] = m, v, None, None
        s["m"], s["v"] = s["m"].flatten(), s["v"].flatten()
        s["master"] = None
        if case["master"]:  # what the 16-bit weights are the rounding of
            s["master"] = _flat(s["params"], s) * (1 + 0.0005 * torch.rand(n, BLOCK, generator=g, device="cuda"))
            s["master"] = torch.where(s["master"].to(dt).float() == _flat(s["params"], s), s["master"], _flat(s["params"], s)).flatten()
        A = case["adapters"]
        s["group"] = torch.arange(A, dtype=torch.int32).repeat_interleave(len(sizes) // A).cuda()
        s["hyper"] = torch.tensor([[1e-4 * (1 + a), 0.9, 0.999, 1e-8, 0.01] for a in range(A)], dtype=torch.float32).cuda()
        s["step"] = torch.randint(50, 500, (A,), generator=g, device="cuda", dtype=torch.int32)[s["group"].long()].contiguous()
    return s


def _padded(t, dtype):
    """A tensor's values in whole blocks, the last filled up with zeros."""
    t = t.detach().flatten().to(dtype)
    return torch.nn.functional.pad(t, (0, -t.numel() % BLOCK))


def _flat(tensors, s, dtype=torch.float32):
    return torch.cat([_padded(t, dtype) for t in tensors]).view(-1, BLOCK)


def _unflat(flat, tensors, s):
    parts = flat.flatten().split([b * BLOCK for b in s["blocks"]])
    return [p[:t.numel()].view(t.shape) for p, t in zip(parts, tensors)]


# ---- the plain forms ---------------------------------------------------------------------------------------

def _row_weight(labels, partition, g):
    """What each row's loss counts in the sum of g's products with the partitions' means, and the rows' partitions."""
    T, P = labels.shape[0], partition.shape[0] - 1
    part = torch.searchsorted(partition, torch.arange(T, device=labels.device, dtype=torch.int32), right=True) - 1
    counted = labels >= 0
    count = torch.zeros(P, device=labels.device).index_add_(0, part, counted.float())
    return part, count, torch.where(counted, g[part] / count[part].clamp(min=1), 0)


def _loss_plain(s):
    grad, labels = s["case"]["grad"], s["labels"]
    x, w = s["x"].detach(), s["w"].detach().float()
    rows = (labels >= 0).nonzero()[:, 0]
    xr, label = x[rows].float(), labels[rows]
    z = xr @ w.t()
    top = z.amax(1, keepdim=True)
    at_label = z.gather(1, label[:, None])[:, 0]
    e = z.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    row_loss = total[:, 0].log() + top[:, 0] - at_label
    loss = torch.zeros(labels.shape[0], device=x.device)
    loss[rows] = row_loss
    if grad == "none":
        return loss
    part, count, weight = _row_weight(labels, s["partition"], s["g"])
    means = torch.zeros_like(count).index_add_(0, part, loss) / count.clamp(min=1)
    p = e.mul_(weight[rows][:, None] / total)
    p[torch.arange(rows.shape[0], device=x.device), label] -= weight[rows]
    dx = torch.zeros_like(x)
    dx[rows] = (p @ w).to(x.dtype)
    return [means, dx] + ([(p.t() @ xr).to(x.dtype)] if grad == "xw" else [])


def _norm_plain(s):
    case, dt = s["case"], s["x"].dtype
    w = s["w"].detach().float()
    h = (s["x"].detach().float() + s["residual"].detach().float()).to(dt)
    hf = h.float()
    r = (hf.square().mean(-1, keepdim=True) + EPS).rsqrt()
    y = hf * r * w
    if case["mode"] == "serve":
        g = y.unflatten(1, (-1, case["group"] or case["cols"]))
        scale = g.abs().amax(-1) / MOST8
        out8 = (g / torch.where(scale > 0, scale, 1)[..., None]).to(torch.float8_e4m3fn).flatten(1)
        return h, y.to(dt), out8, scale
    gf = s["g"].float()
    gw = gf * w
    dh = s["gh"].float() + r * (gw - hf * r.square() * (gw * hf).mean(-1, keepdim=True))
    dh = dh.to(dt)
    return [y.to(dt), h, dh, dh, (gf * hf * r).sum(0).to(dt)]


def _adamw_plain(s):
    dt, of = s["params"][0].dtype, s["block_tensor"]
    s["step"] += 1
    lr, b1, b2, eps, wd = s["hyper"][s["group"].long()].double().unbind(1)
    size, root = lr / (1 - b1 ** s["step"]), (1 - b2 ** s["step"]).sqrt()
    lr, b1, b2, eps, wd, size, root, nb1, nb2 = (c.float()[of][:, None] for c in (lr, b1, b2, eps, wd, size, root, 1 - b1, 1 - b2))
    g, p = _flat(s["grads"], s), _flat(s["params"], s)
    if s["master"] is not None:
        full = s["master"].view(-1, BLOCK)
        p = torch.where(full.to(dt).float() == p, full, p)
    m, v = s["m"].view(-1, BLOCK).float(), s["v"].view(-1, BLOCK).float()
    if s["m_scale"] is not None:
        m, v = m * s["m_scale"][:, None], (v * s["v_scale"][:, None]).square()
    m = b1 * m + nb1 * g
    v = b2 * v + nb2 * g * g
    p = p - lr * wd * p
    p = p - size * m / (v.sqrt() / root + eps)
    if s["m_scale"] is not None:
        (m, ms), (v, vs) = _rounded8(m), _root8(v)
        s["m_scale"].copy_(ms)
        s["v_scale"].copy_(vs)
    s["m"].copy_(m.flatten())
    s["v"].copy_(v.flatten())
    if s["master"] is not None:
        s["master"].copy_(p.flatten())
    torch._foreach_copy_(s["params"], _unflat(p.to(dt), s["params"], s))


def _adamw_out(s):
    return [s["weights"], s["m"], s["v"]] + [s[n] for n in ("m_scale", "v_scale", "master") if s[n] is not None] + [s["step"]]


def run(s):
    op = s["case"]["op"]
    if not own:
        if op == "adamw":
            _adamw_plain(s)
            return _adamw_out(s)
        return _loss_plain(s) if op == "loss" else _norm_plain(s)
    from loquetier_amd.kernel_utils import add_rms_norm, linear_cross_entropy
    from loquetier_amd.ops import _kernels as K
    if op == "loss":
        if s["case"]["grad"] == "none":
            return linear_cross_entropy.apply(s["x"], s["w"], s["labels"])
        loss = linear_cross_entropy.apply(s["x"], s["w"], s["labels"], s["partition"])
        leaves = [s["x"]] + ([s["w"]] if s["case"]["grad"] == "xw" else [])
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves, s["g"]))
    if op == "norm":
        x, residual, w = s["x"], s["residual"], s["w"]
        if s["case"]["mode"] == "train":
            out, h = add_rms_norm.apply(x, residual, w, EPS)
            return [out.detach(), h.detach()] + list(torch.autograd.grad((out, h), (x, residual, w), (s["g"], s["gh"])))
        T, H = x.shape
        h, out, out8 = torch.empty_like(x), torch.empty_like(x), torch.empty(T, H, dtype=torch.float8_e4m3fn, device=x.device)
        scale = torch.empty(T, H // s["case"]["group"] if s["case"]["group"] else 1, device=x.device)
        K.add_rms_norm(out, None, h, x, residual, w, EPS, out8, scale)
        return h, out, out8, scale
    K.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], s["hyper"], s["group"], s["m_scale"], s["v_scale"], s["master"])
    return _adamw_out(s)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"loss": _loss_exact, "norm": _norm_exact, "adamw": _adamw_exact}[case["op"]](case, s)


def _loss_exact(case, s):
    T, H, V = case["rows"], case["hidden"], case["vocab"]
    x, w = s["x"].detach().double(), s["w"].detach().double()
    loss, dx = torch.zeros(T, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    dw = torch.zeros(V, H, dtype=torch.float64, device="cuda") if case["grad"] == "xw" else None
    valid = s["labels"] >= 0
    weight, means = valid.double(), None
    if case["grad"] != "none":
        edges = s["partition"].tolist()
        for p, (a, b) in enumerate(zip(edges, edges[1:])):
            weight[a:b] *= s["g"][p].double() / max(1, int(valid[a:b].sum()))
    for a in range(0, T, 1024):
        rows = a + valid[a:a + 1024].nonzero()[:, 0]
        z = torch.matmul(x[rows], w.t())
        lse = torch.logsumexp(z, 1)
        loss[rows] = lse - z[torch.arange(len(rows)), s["labels"][rows]]
        if case["grad"] == "none":
            continue
        z = torch.exp(z - lse[:, None])
        z[torch.arange(len(rows)), s["labels"][rows]] -= 1
        z *= weight[rows][:, None]
        dx[rows] = torch.matmul(z, w)
        if dw is not None:
            dw += torch.matmul(z.t(), x[rows])
    if case["grad"] == "none":
        return loss
    means = torch.stack([loss[a:b].sum() / max(1, int(valid[a:b].sum())) for a, b in zip(edges, edges[1:])])
    return [means, dx] + ([dw] if dw is not None else [])


def _norm_exact(case, s):
    dt = s["x"].dtype
    x, residual, w = (s[n].detach().double() for n in ("x", "residual", "w"))
    total = x + residual
    h = total.to(dt).double()
    if case["mode"] == "serve":
        y = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * w
        groups = y.reshape(y.shape[0], -1, case["group"] or case["cols"])
        scale = groups.abs().amax(2) / MOST8
        return total, y, (groups / scale[:, :, None].clamp(min=1e-300)).reshape(y.shape), scale
    leaf, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = leaf / torch.sqrt((leaf * leaf).mean(1, keepdim=True) + EPS) * wl
    dh, dw = torch.autograd.grad((y, leaf * 1.0), (leaf, wl), (s["g"].double(), s["gh"].double()))
    return [y.detach(), total, dh, dh, dw]


def _adamw_exact(case, s):
    step = (s["step"] + 1).tolist()
    hyper, group = s["hyper"].double().tolist(), s["group"].tolist()
    blocks = lambda name: s[name].view(-1, BLOCK).double()
    m, v = blocks("m"), blocks("v")
    if case["bits"] == 8:
        m, v = m * s["m_scale"].double()[:, None], (v * s["v_scale"].double()[:, None]) ** 2
    full = None if s["master"] is None else blocks("master").clone()
    params, at = [], 0
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        lr, b1, b2, eps, wd = hyper[group[i]]
        n, span = p.numel(), slice(at, at + s["blocks"][i])
        at += s["blocks"][i]
        one_m, one_v, g = m[span].view(-1)[:n], v[span].view(-1)[:n], g.double().flatten()
        w = p.double().flatten()
        if full is not None:
            kept = full[span].view(-1)[:n]
            w = torch.where(kept.to(p.dtype).double() == w, kept, w)
        one_m.mul_(b1).add_(g, alpha=1 - b1)
        one_v.mul_(b2).add_(g * g, alpha=1 - b2)
        w = w * (1 - lr * wd) - lr * (one_m / (1 - b1 ** step[i])) / ((one_v / (1 - b2 ** step[i])).sqrt() + eps)
        params.append(w)
        if full is not None:
            full[span].view(-1)[:n] = w
    out = [torch.cat(params)]
    if case["bits"] == 8:
        r = v.sqrt()
        ms, vs = m.abs().amax(1) / MOST8, r.amax(1) / MOST8
        out += [(m / ms[:, None].clamp(min=1e-300)).flatten(), (r / vs[:, None].clamp(min=1e-300)).flatten(), ms, vs]
    else:
        out += [m.flatten(), v.flatten()]
    return out + ([] if full is None else [full.flatten()]) + [torch.tensor(step, dtype=torch.int32).cuda()]
