"""Norms of queries and keys by head with their rotation, forward, backward and into a cache's pages, against the formulas in 64
bits.

Bounds: every output is computed in float from 16-bit inputs and rounded once, so it is off by half a step of its own size
(eps / 2, relative) and by the float arithmetic: a sum of at most 512 squares in some order, a square root, a division and a few
products, 64 float half-steps of the larger operand with room, relative to the sizes that are added (which may cancel).  A
weight's gradient sums n = rows x heads such terms in float: n half-steps of the sum of the terms' sizes at the most.  fp16 results under
2^-14 are off by at most half a step of 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TDT = {"fp16": torch.float16, "bf16": torch.bfloat16}
F32 = 2.0 ** -24


@pytest.fixture(scope="module")
def K(gpu_device):
    from loquetier_amd import _lib
    from loquetier_amd.ops import _kernels
    _lib.load()
    return _kernels


def turn(y, cos, sin):
    h = cos.shape[-1]
    a, b = y[..., :h], y[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * h:]], -1)


def sizes(y, cos, sin):
    """|a c| + |b s|: what the rotation adds."""
    h = cos.shape[-1]
    a, b = y[..., :h].abs(), y[..., h:2 * h].abs()
    return torch.cat([a * cos.abs() + b * sin.abs(), b * cos.abs() + a * sin.abs(), y[..., 2 * h:].abs()], -1)


def forward(x, w, cos, sin, eps):
    y = x if w is None else x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
    return turn(y, cos, sin), sizes(y, cos, sin)


def near(got, want, size, n=64):
    u = torch.finfo(got.dtype).eps / 2
    bound = u * want.abs() + n * F32 * size * (1 + u) + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"{float((err / bound).max())} times the bound"


def case(dt, T, Hq, Hkv, D, rot, norm, seed=0, dev="cuda", n_pos=4000):
    from loquetier_amd.ops import _kernels as K
    g = torch.Generator(device="cpu").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(dev).to(TDT[dt])
    qkv = mk(T, (Hq + 2 * Hkv) * D)
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
    table = K.rope_table(n_pos, rot, 500000.0, dev)
    pos = torch.randint(0, n_pos, (T,), generator=g, dtype=torch.int32).to(dev)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(dev).to(TDT[dt]) if n else None for n in norm)
    return q, k, v, table, pos, wq, wk


def angles(table, pos):
    cos, sin = table[pos.long().clamp(0, table.shape[0] - 1)].double()[:, None].chunk(2, -1)
    return cos, sin


SHAPES = [  # rows, q heads, kv heads, head size, rotated
    (1, 1, 1, 16, 16), (3, 5, 1, 64, 64), (17, 32, 8, 128, 128), (5, 7, 7, 96, 48), (2, 3, 2, 80, 16), (129, 4, 2, 256, 64),
    (33, 2, 1, 512, 512), (700, 32, 8, 128, 128), (1500, 12, 4, 64, 32), (2, 64, 64, 128, 128)]


def test_rope_table_far_positions(K):
    t = K.rope_table(100001, 32, 10000.0, "cuda")
    assert t.shape == (100001, 32) and t.dtype == torch.float32
    import math
    for p in (0, 1, 99999, 100000):
        for j in (0, 3, 15):
            a = p * 10000.0 ** (-2 * j / 32)
            # (the angle, at most 1e5, is off by 2^-53 of it a few times over)
            assert abs(float(t[p, j]) - math.cos(a)) <= F32 + 1e-10 and abs(float(t[p, 16 + j]) - math.sin(a)) <= F32 + 1e-10
    scaled = K.rope_table(9, 32, device="cuda", inv_freq=torch.full((16,), 0.25))
    assert abs(float(scaled[8, 5]) - math.cos(2.0)) <= F32


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("norm", [(True, True), (False, False), (True, False)], ids=["norms", "plain", "qnorm"])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", SHAPES)
def test_forward(K, dt, norm, T, Hq, Hkv, D, rot):
    q, k, _, table, pos, wq, wk = case(dt, T, Hq, Hkv, D, rot, norm)
    qo, ko = torch.empty(T, Hq, D, dtype=q.dtype, device="cuda"), torch.empty(T, Hkv, D, dtype=q.dtype, device="cuda")
    K.qk_norm_rope(qo, ko, q, k, table, pos, wq, wk, 1e-5)
    cos, sin = angles(table, pos)
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        near(got, *forward(x.double(), None if w is None else w.double(), cos, sin, 1e-5))
    # in place
    q2, k2 = q.contiguous(), k.contiguous()
    K.qk_norm_rope(q2, k2, q2, k2, table, pos, wq, wk, 1e-5)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("norm", [(True, True), (False, False), (False, True)], ids=["norms", "plain", "knorm"])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", SHAPES)
def test_backward(K, dt, norm, T, Hq, Hkv, D, rot):
    from loquetier_amd.kernel_utils import qk_norm_rope
    q, k, _, table, pos, wq, wk = case(dt, T, Hq, Hkv, D, rot, norm, seed=1)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k)]
    ws = [None if w is None else w.clone().requires_grad_(True) for w in (wq, wk)]
    qo, ko = qk_norm_rope.apply(*leaves, *ws, table, pos, 1e-5)
    g = torch.Generator(device="cpu").manual_seed(2)
    gq, gk = (torch.randn(*o.shape, generator=g).cuda().to(o.dtype) for o in (qo, ko))
    torch.autograd.backward((qo, ko), (gq, gk))
    cos, sin = angles(table, pos)
    for x, w, go in ((leaves[0], ws[0], gq), (leaves[1], ws[1], gk)):
        gy, size = turn(go.double(), cos, -sin), sizes(go.double(), cos, -sin)
        if w is None:
            near(x.grad, gy, size)
            continue
        xd, wd = x.detach().double(), w.detach().double()
        r = (xd.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
        dx = r * (gy * wd - xd * r.pow(2) * (gy * wd * xd).mean(-1, keepdim=True))
        dsize = r * (size * wd.abs() + xd.abs() * r.pow(2) * (size * wd.abs() * xd.abs()).mean(-1, keepdim=True))
        near(x.grad, dx, dsize, 64 + D)
        # and against differences, taken by autograd of the formula in 64 bits
        xv, wv = xd.clone().requires_grad_(True), wd.clone().requires_grad_(True)
        dx2, dw2 = torch.autograd.grad(forward(xv, wv, cos, sin, 1e-5)[0], (xv, wv), go.double())
        assert torch.allclose(dx, dx2, rtol=1e-9, atol=1e-12)
        terms = size * xd.abs() * r
        near(w.grad, dw2, terms.sum((0, 1)), 64 + T * x.shape[1])


def test_gradient_against_differences():
    """The formula the kernel is held to, by differences of the forward in 64 bits (on the CPU)."""
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(3, 2, 32, generator=g, dtype=torch.float64), torch.rand(32, generator=g, dtype=torch.float64) + 0.5
    a = torch.rand(3, 1, 8, generator=g, dtype=torch.float64) * 6
    x.requires_grad_(True), w.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda x, w: forward(x, w, a.cos(), a.sin(), 1e-5)[0], (x, w))


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,P,nhd", [(1, 4, 4, 128, 128, 16, False), (37, 32, 8, 128, 128, 16, False),
                                                  (300, 6, 2, 64, 32, 20, True), (1, 2, 1, 96, 96, 1, False)])
@pytest.mark.parametrize("norm", [True, False])
def test_append(K, dt, T, Hq, Hkv, D, rot, P, nhd, norm):
    q, k, v, table, pos, wq, wk = case(dt, T, Hq, Hkv, D, rot, (norm, norm), seed=3)
    pages = 2 * T // P + 3
    shape = (pages, P, Hkv, D) if nhd else (pages, Hkv, P, D)
    kc, vc = (torch.full(shape, 7.0, dtype=q.dtype, device="cuda") for _ in range(2))
    if nhd:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    g = torch.Generator().manual_seed(4)
    slots = torch.randperm(pages * P, generator=g)[:T].cuda()
    if T > 5:  # rows that are not cached
        slots[1], slots[3] = -1, pages * P
    qo, ko = torch.empty_like(q.contiguous()), torch.empty_like(k.contiguous())
    K.qk_norm_rope(qo, ko, q, k, table, pos, wq, wk, 1e-5)
    q2 = torch.empty_like(qo)
    K.qk_norm_rope(q2, None, q, k, table, pos, wq, wk, 1e-5, v=v, k_cache=kc, v_cache=vc, slots=slots)
    assert torch.equal(q2, qo)
    want_k, want_v = (torch.full((pages, P, Hkv, D), 7.0, dtype=q.dtype, device="cuda") for _ in range(2))
    ok = (slots >= 0) & (slots < pages * P)
    want_k.flatten(0, 1)[slots[ok]] = ko[ok]
    want_v.flatten(0, 1)[slots[ok]] = v[ok]
    assert torch.equal(kc.transpose(1, 2), want_k) and torch.equal(vc.transpose(1, 2), want_v)


def test_padding_and_positions_past_the_table(K):
    q, k, v, table, pos, wq, wk = case("bf16", 9, 4, 2, 128, 128, (True, True), n_pos=50)
    q, k = q.clone(), k.clone()
    pos[2], pos[5] = -1, 50
    q[2, 1, 3] = float("nan")  # whatever a padded row holds stays with it
    qo, ko = torch.empty(9, 4, 128, dtype=q.dtype, device="cuda"), torch.empty(9, 2, 128, dtype=q.dtype, device="cuda")
    K.qk_norm_rope(qo, ko, q, k, table, pos, wq, wk)
    assert not bool(qo[2].any()) and not bool(ko[2].any())
    assert bool(qo[5].isnan().all()) and bool(ko[5].isnan().all())
    rest = [0, 1, 3, 4, 6, 7, 8]
    assert bool(qo[rest].isfinite().all()) and bool(ko[rest].isfinite().all())
    # the padded row has no gradient and adds nothing to the weights'
    pos[5] = 3
    grads = []
    for keep in ([0, 1, 2, 3, 4, 5, 6, 7, 8], [0, 1, 3, 4, 5, 6, 7, 8]):
        qq, kk, pp = q[keep].contiguous(), k[keep].contiguous(), pos[keep].contiguous()
        gq, gk = torch.ones_like(qq), torch.ones_like(kk)
        dq, dk, dwq, dwk = torch.empty_like(qq), torch.empty_like(kk), torch.empty_like(wq), torch.empty_like(wk)
        K.qk_norm_rope_backward(dq, dk, dwq, dwk, gq, gk, qq, kk, table, pp, wq, wk)
        grads.append((dq, dk, dwq, dwk))
    (dq, dk, dwq, dwk), (eq, ek, ewq, ewk) = grads
    assert not bool(dq[2].any()) and not bool(dk[2].any())
    keep = [0, 1, 3, 4, 5, 6, 7, 8]
    assert torch.equal(dq[keep], eq) and torch.equal(dk[keep], ek)
    # (the rows lie with other waves, so the weights' sums are taken in another order)
    assert torch.allclose(dwq.float(), ewq.float(), rtol=2 ** -7, atol=1e-3) and bool(dwk.isfinite().all())


def test_padding_is_not_cached(K):
    q, k, v, table, pos, _, _ = case("fp16", 6, 4, 2, 64, 64, (False, False), n_pos=50)
    kc, vc = (torch.full((3, 2, 16, 64), 7.0, dtype=q.dtype, device="cuda") for _ in range(2))
    pos[1] = pos[4] = -1
    slots = torch.arange(6, device="cuda") * 5
    K.qk_norm_rope(torch.empty_like(q.contiguous()), None, q, k, table, pos, v=v, k_cache=kc, v_cache=vc, slots=slots)
    for c, x in ((kc, None), (vc, v)):
        flat = c.transpose(1, 2).flatten(0, 1)
        assert bool((flat[slots[[1, 4]]] == 7).all()) and not bool((flat[slots[[0, 2, 3, 5]]] == 7).any())
        if x is not None:
            assert torch.equal(flat[slots[[0, 2, 3, 5]]], x[[0, 2, 3, 5]])


def test_training_step_in_a_graph(K):
    """Forward and backward captured, replayed with new inputs between the program's own work, against eager passes."""
    from loquetier_amd.kernel_utils import qk_norm_rope
    q, k, _, table, pos, wq, wk = case("bf16", 60, 8, 2, 128, 128, (True, True), seed=12)
    g = torch.Generator(device="cuda").manual_seed(1)
    inputs = [[torch.randn(t.shape, generator=g, device="cuda").to(t.dtype) for t in (q, k, q, k)] for _ in range(5)]

    def step(q, k, gq, gk):
        a, b = qk_norm_rope.apply(q, k, wq, wk, table, pos, 1e-6)
        return [a.detach(), b.detach(), *torch.autograd.grad((a, b), (q, k, wq, wk), (gq, gk))]

    wq.requires_grad_(True), wk.requires_grad_(True)
    want = [[t.clone() for t in step(x[0].clone().requires_grad_(True), x[1].clone().requires_grad_(True), *x[2:])] for x in inputs]
    static = [t.clone() for t in inputs[0]]
    static[0].requires_grad_(True), static[1].requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(*static)
    for x, w in zip(inputs, want):
        with torch.no_grad():
            for s, t in zip(static, x):
                s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        torch.ones(3000, device="cuda").sum().item()
        assert all(torch.equal(a, b) for a, b in zip(out, w))


def test_infinities_stay_in_their_pairs(K):
    """A dimension that is not rotated passes through beside an infinity."""
    q, k, _, table, pos, _, _ = case("bf16", 4, 2, 1, 64, 32, (False, False))
    q = q.clone()
    q[1, 0, 40], q[2, 1, 3] = float("inf"), float("-inf")
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    K.qk_norm_rope(qo, ko, q, k, table, pos)
    want = turn(q.double(), *angles(table, pos))
    assert torch.equal(qo[..., 32:], q[..., 32:])
    bad = ~want.isfinite()
    assert torch.equal(~qo.isfinite(), bad) and int(bad.sum()) <= 3


def test_strided_expanded_and_repeated(K):
    """Views with strides, gradients that are expanded, and the same call twice (the weights' sums have a fixed order)."""
    from loquetier_amd.kernel_utils import qk_norm_rope
    q, k, _, table, pos, wq, wk = case("fp16", 50, 8, 2, 64, 64, (True, True), seed=9)
    big = torch.zeros(100, 16, 72, dtype=q.dtype, device="cuda")
    qs = big[::2, ::2, :64]
    qs.copy_(q)
    qo, ko, q1, k1 = (torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (q, k, q, k))
    K.qk_norm_rope(qo, ko, qs, k, table, pos, wq, wk)
    K.qk_norm_rope(q1, k1, q, k, table, pos, wq, wk)
    assert torch.equal(qo, q1) and torch.equal(ko, k1)
    outs = []
    for _ in range(2):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
        a, b = qk_norm_rope.apply(*leaves, table, pos, 1e-6)
        (a.sum() + 2 * b.sum()).backward()
        outs.append([t.grad for t in leaves])
    assert all(torch.equal(x, y) for x, y in zip(*outs))
    # one weight for both: autograd adds the two
    w = wq.clone().requires_grad_(True)
    a, b = qk_norm_rope.apply(q, k, w, w, table, pos, 1e-6)
    torch.autograd.backward((a, b), (torch.ones_like(a), torch.ones_like(b)))
    u, t = (wq.clone().requires_grad_(True) for _ in range(2))
    a, b = qk_norm_rope.apply(q, k, u, t, table, pos, 1e-6)
    torch.autograd.backward((a, b), (torch.ones_like(a), torch.ones_like(b)))
    assert torch.equal(w.grad, u.grad + t.grad)


def test_no_rows(K):
    q, k, v, table, pos, wq, wk = case("bf16", 0, 4, 2, 64, 64, (True, True))
    from loquetier_amd.kernel_utils import qk_norm_rope
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
    a, b = qk_norm_rope.apply(*leaves, table, pos, 1e-6)
    (a.sum() + b.sum()).backward()
    assert a.shape == (0, 4, 64) and not bool(leaves[2].grad.any()) and not bool(leaves[3].grad.any())


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch, K):
    from loquetier_amd import _lib
    if request.param == "python":
        monkeypatch.setattr(K, "_host", lambda: _lib._NoHost)


@pytest.mark.parametrize("norm", [(True, True), (True, False), (False, False)], ids=["norms", "qnorm", "plain"])
def test_gradients_are_not_differentiated(K, path, norm):
    """A graph of the gradients raises where it is differentiated, by every way to what they hang on; without one nothing changes."""
    from loquetier_amd.kernel_utils import qk_norm_rope
    q, k, _, table, pos, wq, wk = case("bf16", 6, 4, 2, 64, 64, norm, seed=14)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk) if t is not None]
    args = lambda: (leaves[0], leaves[1], leaves[2] if norm[0] else None, leaves[-1] if norm[1] else None, table, pos, 1e-6)
    gq, gk = torch.ones_like(leaves[0]), torch.ones_like(leaves[1])
    want = torch.autograd.grad(qk_norm_rope.apply(*args()), leaves, (gq, gk))
    got = torch.autograd.grad(qk_norm_rope.apply(*args()), leaves, (gq, gk), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    again = "cannot be differentiated"
    if any(norm):  # the gradients hang on q, which other terms lead to as well
        for x, g in zip(leaves, got):
            with pytest.raises(RuntimeError, match=again):
                torch.autograd.grad(g.float().square().sum() + leaves[0].float().square().sum(), leaves[0], retain_graph=True)
        with pytest.raises(RuntimeError, match=again):
            (sum(g.float().square().sum() for g in got) + leaves[0].float().sum()).backward()
    else:  # a rotation by itself: the gradients hang on the outputs' alone
        assert not any(g.requires_grad for g in got)
    gq.requires_grad_(True)
    got = torch.autograd.grad(qk_norm_rope.apply(*args()), leaves, (gq, gk), create_graph=True)
    with pytest.raises(RuntimeError, match=again):
        torch.autograd.grad(got[0].float().sum(), gq)
    assert leaves[0].grad is None
