"""Norms and rotation of large batches: forward batches whose waves take two runs of heads, shared evenly over a row's waves or not, and backward
batches whose waves walk several rows, on both sides of the sizes from which they do; and the norm weights' gradients, to the rounding that
their sums can have.

Bounds of outputs and of the gradients of queries and keys as in test_gpu_qk_norm_rope.  A weight's gradient: each of its terms is off by 64 float
half-steps of its size at most, as an output is, and is then added up in a tree: a lane's rows and steps of heads one after the other, the wave's groups of
lanes, the four waves, up to every 64th workgroup's sum one after the other, and six levels.  Each addition rounds what has been added so far,
which is no more than the sum of the terms' sizes, so the sum is off by as many half-steps of that as the tree is deep; then the result's own
rounding."""
import pytest
import torch

from test_gpu_qk_norm_rope import F32, K, angles, case, forward, near, sizes, turn  # noqa: F401

pytestmark = pytest.mark.gpu

# rows, q heads, kv heads, head size, rotated.  Two runs a wave from rows x ceil(runs / 2) = 4096 on; several rows a wave from 2049 rows on.
SHAPES = [
    (1365, 32, 8, 128, 128),   # five runs of heads a row: the last batch with a run a wave
    (1366, 32, 8, 128, 128),   # the first with two, the third wave of a row takes one
    (2048, 9, 3, 128, 64),     # two runs; one row a wave in the backward
    (2049, 9, 3, 128, 64),     # its first workgroup takes a second row
    (4095, 9, 5, 64, 32), (4096, 9, 5, 64, 32),  # one run, on both sides
    (4099, 17, 3, 96, 96),     # three runs, head sizes that leave lanes idle
    (5001, 3, 1, 512, 256),    # two runs of two heads
    (6200, 5, 2, 80, 16),
]


def depth(T, H, D):
    """Additions that a term of a weight's gradient goes through, at most."""
    lanes = 1
    while lanes * 16 < D:
        lanes *= 2
    per = 64 // lanes
    blocks = min(-(-T // 4), 512)
    return -(-T // (4 * blocks)) * -(-H // per) + per.bit_length() + 2 + -(-blocks // 64) + 6


def padded(pos):
    pos[::97] = -1
    pos[-1] = 5
    return pos


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("norm", [(True, True), (False, False), (False, True)], ids=["norms", "plain", "knorm"])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", SHAPES)
def test_forward_and_backward(K, dt, norm, T, Hq, Hkv, D, rot):
    from loquetier_amd.kernel_utils import qk_norm_rope
    q, k, _, table, pos, wq, wk = case(dt, T, Hq, Hkv, D, rot, norm, seed=T)
    live = (padded(pos) >= 0)[:, None, None]
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k)]
    ws = [None if w is None else w.clone().requires_grad_(True) for w in (wq, wk)]
    out = qk_norm_rope.apply(*leaves, *ws, table, pos, 1e-5)
    g = torch.Generator(device="cuda").manual_seed(T)
    grads = [torch.randn(o.shape, generator=g, device="cuda").to(o.dtype) for o in out]
    torch.autograd.backward(out, grads)
    cos, sin = angles(table, pos)
    for o, x, w, go in zip(out, leaves, ws, grads):
        xd = x.detach().double()
        want, size = forward(xd, None if w is None else w.detach().double(), cos, sin, 1e-5)
        near(o.detach(), want * live, size * live)
        gy, size = turn(go.double(), cos, -sin) * live, sizes(go.double(), cos, -sin) * live
        if w is None:
            near(x.grad, gy, size)
            continue
        wd = w.detach().double()
        r = (xd.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
        dx = r * (gy * wd - xd * r.pow(2) * (gy * wd * xd).mean(-1, keepdim=True))
        near(x.grad, dx, r * (size * wd.abs() + xd.abs() * r.pow(2) * (size * wd.abs() * xd.abs()).mean(-1, keepdim=True)), 64 + D)
        near(w.grad, (gy * xd * r).sum((0, 1)), (size * xd.abs() * r).sum((0, 1)), 64 + depth(T, x.shape[1], D))


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,P", [(2112, 32, 32, 128, 128, 16), (1500, 17, 9, 128, 64, 20), (4100, 9, 3, 64, 64, 7),
                                              (1025, 32, 8, 256, 256, 16)])
def test_append(K, dt, norm, T, Hq, Hkv, D, rot, P):
    q, k, v, table, pos, wq, wk = case(dt, T, Hq, Hkv, D, rot, (norm, norm), seed=T)
    padded(pos)
    pages = 2 * T // P + 3
    kc, vc = (torch.full((pages, Hkv, P, D), 7.0, dtype=q.dtype, device="cuda") for _ in range(2))
    slots = torch.randperm(pages * P, generator=torch.Generator().manual_seed(4))[:T].cuda()
    slots[1], slots[3] = -1, pages * P
    qo, ko, q2 = (torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (q, k, q))
    K.qk_norm_rope(qo, ko, q, k, table, pos, wq, wk, 1e-5)
    cos, sin = angles(table, pos)
    live = (pos >= 0)[:, None, None]
    want, size = forward(q.double(), None if wq is None else wq.double(), cos, sin, 1e-5)
    near(qo, want * live, size * live)
    K.qk_norm_rope(q2, None, q, k, table, pos, wq, wk, 1e-5, v=v, k_cache=kc, v_cache=vc, slots=slots)
    assert torch.equal(q2, qo)
    ok = (slots >= 0) & (slots < pages * P) & (pos >= 0)
    for cache, x in ((kc, ko), (vc, v)):
        flat = torch.full((pages * P, Hkv, D), 7.0, dtype=q.dtype, device="cuda")
        flat[slots[ok]] = x[ok]
        assert torch.equal(cache.transpose(1, 2).flatten(0, 1), flat)


@pytest.mark.parametrize("T", [1, 4, 5, 129, 2048, 2049, 2053, 4097])
@pytest.mark.parametrize("H,D,rot", [(1, 128, 128), (9, 128, 64), (32, 128, 128), (5, 80, 80), (3, 512, 512), (33, 64, 16)])
def test_one_gradient(K, T, H, D, rot):
    """A gradient of one row and head alone, first, last and between: the weights' gradient is its term, the sums of all others are zero."""
    q, k, _, table, pos, wq, wk = case("bf16", T, H, H, D, rot, (True, True), seed=T + H)
    cos, sin = angles(table, pos)
    for row, head in {(0, 0), (T - 1, H - 1), (T - 1, 0), (0, H - 1), (T // 2, H // 2)}:
        gq, gk = torch.zeros_like(q), torch.zeros_like(k)
        gq[row, head] = torch.randn(D, device="cuda").to(q.dtype)
        gk[T - 1 - row, head] = torch.randn(D, device="cuda").to(q.dtype)
        dq, dk, dwq, dwk = (torch.full(t.shape, 5.0, dtype=t.dtype, device="cuda") for t in (q, k, wq, wk))
        K.qk_norm_rope_backward(dq, dk, dwq, dwk, gq, gk, q, k, table, pos, wq, wk, 1e-5)
        for g, x, dx, dw, at in ((gq, q, dq, dwq, row), (gk, k, dk, dwk, T - 1 - row)):
            gd, xd, c, s = g[at:at + 1].double(), x[at:at + 1].double(), cos[at:at + 1], sin[at:at + 1]
            r = (xd.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
            # (one term is not zero, so no addition rounds)
            near(dw, (turn(gd, c, -s) * xd * r).sum((0, 1)), (sizes(gd, c, -s) * xd.abs() * r).sum((0, 1)))
            assert bool(dx[at, head].any()) and int((dx != 0).any(-1).sum()) == 1
