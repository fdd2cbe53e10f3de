"""linear_cross_entropy against its definition in 64 bits: rows and vocabularies around the tiles' edges, rows without labels,
partitions, gradients of both inputs.

Tolerances.  Logits are sums of H exact products in float, in an order that the matrix cores choose: off by at most H 2^-24 sum |x w|,
here far less (errors of random sign); 2e-6 of the largest |x||w| covers them, and losses, differences of two such numbers, are taken
to 1e-5 of it.  An entry G = c (p - [label]) has p = exp(z - lse): off by p times the logits' error, and by some steps of a float
of the exponential and the logarithm (v_exp_f32 and v_log_f32, 2^-23 each; 1e-6 in all) - of p, not of G, which is near 0 where a label is
nearly certain.  It is then rounded to 16 bits, at most eps / 2 of |G|, multiplied in float, and the result is rounded once more:
|error| <= sum |G w| eps / 2 + sum |c p w| (2e-6 |x||w| + 1e-6) + |dx| eps / 2, and a float's rounding of the sums, 1e-7 of their largest.
With partitions the rows are rounded once more for dw, times what c is of a power of two: sum |G x| eps / 2 again."""
import math

import pytest
import torch

from loquetier_amd.kernel_utils import linear_cross_entropy
from loquetier_amd.ops import _kernels as K

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16


def make(T, H, V, dt, seed=0, labelled=1.0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, H, generator=g) * (spread / math.sqrt(H))).to(dt)
    labels = torch.randint(0, V, (T,), generator=g)
    x = (torch.randn(T, H, generator=g) + torch.rand(T, 1, generator=g) * w[labels].float()).to(dt)
    labels[torch.rand(T, generator=g) >= labelled] = -100
    return x.cuda(), w.cuda(), labels.cuda()


def want(x, w, labels, c):
    """losses, dx, dw and the sums of absolute values that bound their errors, in 64 bits; c: each row's weight."""
    x, w = x.double().cpu(), w.double().cpu()
    labels, c = labels.cpu(), c.double().cpu()
    V = w.shape[0]
    ok = (labels >= 0) & (labels < V)
    z = x @ w.t()
    lse = torch.logsumexp(z, 1)
    safe = labels.clamp(0, V - 1)
    loss = torch.where(ok, lse - z.gather(1, safe[:, None])[:, 0], 0)
    P = torch.exp(z - lse[:, None]) * torch.where(ok, c, 0)[:, None]
    G = P.clone()
    G[torch.arange(len(labels)), safe] -= torch.where(ok, c, 0)
    bx, bw = [M.abs() @ w.abs() for M in (G, P)], [M.abs().t() @ x.abs() for M in (G, P)]
    return loss, torch.where(ok, lse, 0), G @ w, G.t() @ x, bx, bw


def close(got, exact, bounds, eps, top, roundings=1):
    off, (bound, soft) = (got.double().cpu() - exact).abs(), bounds
    limit = roundings * bound * eps / 2 + soft * (2e-6 * top + 1e-6) + exact.abs() * eps / 2 + 1e-7 * bound.max()
    limit += torch.finfo(got.dtype).smallest_normal * eps  # (a step of the subnormal numbers)
    assert torch.isfinite(got).all()
    assert (off <= limit).all(), (off / limit).max()


def check(x, w, labels, partition=None, want_w=True, grad=None):
    T = x.shape[0]
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(want_w)
    out = linear_cross_entropy.apply(x, w, labels, partition)
    g = torch.rand(out.shape, generator=torch.Generator().manual_seed(3)).cuda() + 0.5 if grad is None else grad
    grads = torch.autograd.grad(out, [x, w] if want_w else [x], g)
    ok = (labels >= 0) & (labels < w.shape[0])
    if partition is None:
        c = g
    else:
        c = torch.zeros(T, device="cuda")
        for p, (a, b) in enumerate(zip(partition.tolist(), partition.tolist()[1:])):
            c[a:b] = g[p] / max(1, int(ok[a:b].sum()))
    loss, lse, dx, dw, bx, bw = want(x.detach(), w.detach(), labels, c)
    top = (x.detach().double().norm(dim=1).max() * w.detach().double().norm(dim=1).max()).item()
    if partition is None:
        assert out.dtype == torch.float32 and (out.double().cpu() - loss).abs().max() <= 1e-5 * max(1, top)
    else:
        edges = partition.tolist()
        means = torch.stack([loss[a:b].sum() / max(1, int(ok[a:b].sum())) for a, b in zip(edges, edges[1:])])
        assert (out.double().cpu() - means).abs().max() <= 1e-5 * max(1, top)
    eps = torch.finfo(x.dtype).eps
    close(grads[0], dx, bx, eps, top)
    if want_w:
        close(grads[1], dw, bw, eps, top, 1 if partition is None else 2)
    return out, grads


@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("T,H,V", [(1, 64, 100), (1, 8, 1), (3, 72, 257), (33, 512, 2000), (64, 128, 300), (65, 128, 300), (130, 200, 1023),
                                   (256, 64, 256), (257, 264, 513), (300, 1032, 777), (600, 256, 4097),
                                   # (tiles of 256 rows: enough of them)
                                   (513, 200, 20000), (1300, 136, 6000), (257, 8, 33001)])
def test_rows_and_gradients(T, H, V, dt):
    x, w, labels = make(T, H, V, dt, T + V)
    check(x, w, labels)
    check(x, w, labels, want_w=False)  # (a frozen vocabulary: another route)


@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("T,H,V,labelled", [(40, 136, 500, 0.5), (512, 256, 1500, 0.6), (700, 520, 900, 0.1)])
def test_rows_without_labels(T, H, V, labelled, dt):
    x, w, labels = make(T, H, V, dt, T, labelled)
    x[labels < 0] = float("nan")  # (nothing of them is used)
    xz = torch.where(labels[:, None] < 0, torch.zeros_like(x), x)
    edges = torch.tensor([0, T // 3, T // 3, T // 2, T], dtype=torch.int32, device="cuda")  # (one has no rows)
    a = x.detach().requires_grad_(True)
    out = linear_cross_entropy.apply(a, w, labels, edges)
    got = torch.autograd.grad(out, a, torch.ones_like(out))[0]
    ref_out, ref = check(xz, w, labels, edges, want_w=False, grad=torch.ones_like(out))
    assert torch.equal(out, ref_out) and torch.equal(got, ref[0])
    assert out[1] == 0 and not got[labels < 0].any()


def test_no_row_has_a_label():
    x, w, labels = make(100, 64, 300, BF16)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    for bad in (-100, 300, 1 << 40, -(1 << 40)):
        labels.fill_(bad)
        out = linear_cross_entropy.apply(x, w, labels)
        dx, dw = torch.autograd.grad(out.sum(), (x, w))
        assert not out.any() and not dx.any() and not dw.any()
    part = torch.tensor([0, 50, 100], dtype=torch.int32, device="cuda")
    out = linear_cross_entropy.apply(x, w, labels, part)
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    assert not out.any() and not dx.any() and not dw.any()


def test_rows_outside_the_partitions():
    x, w, labels = make(90, 64, 300, FP16)
    part = torch.tensor([20, 50, 70], dtype=torch.int32, device="cuda")
    check(x, w, labels, part)
    x = x.requires_grad_(True)
    out = linear_cross_entropy.apply(x, w, labels, part)
    dx = torch.autograd.grad(out.sum(), x)[0]
    assert not dx[:20].any() and not dx[70:].any() and dx[20:70].any()


def test_one_partitions_loss_alone():
    x, w, labels = make(600, 128, 700, BF16)
    part = torch.tensor([0, 200, 600], dtype=torch.int32, device="cuda")
    check(x, w, labels, part, grad=torch.tensor([0.0, 2.0], device="cuda"))
    x = x.requires_grad_(True)
    dx = torch.autograd.grad(linear_cross_entropy.apply(x, w, labels, part)[1], x)[0]
    assert not dx[:200].any() and dx[200:].any()


def test_frozen_rows_and_kept_sums():
    x, w, labels = make(100, 64, 300, BF16)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    both = torch.autograd.grad(linear_cross_entropy.apply(a, b, labels).sum(), (a, b))
    assert torch.equal(torch.autograd.grad(linear_cross_entropy.apply(x, b, labels).sum(), b)[0], both[1])
    # the calls behind it: what the forward keeps serves several backwards, of any gradients
    f = lambda n: torch.empty(n, device="cuda")
    kept = torch.empty(K.linear_cross_entropy_kept_size(100, 64, 300), dtype=torch.uint8, device="cuda")
    loss, lse, one, three, other = f(100), f(100), torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    K.linear_cross_entropy(loss, lse, x, w, labels, kept=kept)
    g = torch.ones(100, device="cuda")
    K.linear_cross_entropy_backward(one, None, g, loss, lse, x, w, labels, kept=kept)
    K.linear_cross_entropy_backward(three, None, 4 * g, loss, lse, x, w, labels, kept=kept)
    K.linear_cross_entropy_backward(other, None, g, loss, lse, x, w, labels)
    assert torch.equal(three.float(), 4 * one.float()) and torch.equal(other, both[0])
    # two routes, each within eps / 2 of sum |G w| <= 2 max |w| and eps / 2 of its own rounding
    assert (other.float() - one.float()).abs().max() <= 4 * 2.0 ** -8 * 2 * w.float().abs().max()


@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("T", [600, 2400])
def test_references_move_from_piece_to_piece(T, dt):
    """Logits that grow along the vocabulary by far more than 16-bit exponents hold, so that every tile, and every piece (512 MiB of
    exponentials: one, three), takes the rows' reference along, in some rows; in others the first holds the largest."""
    H, V = 64, 250000
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(T, H, generator=g), 0.3 * torch.randn(V, H, generator=g)
    x[:, 0], x[:, 1] = 1.0, 0.0
    x[::3, 1] = 1.0
    x[1::3, 1] = -0.25
    w[:, 1] = torch.arange(V) * (300.0 / V)
    labels = torch.randint(0, V, (T,), generator=g)
    labels[::2] = torch.randint(V - 2000, V, (T // 2,), generator=g)
    x, w, labels = x.to(dt).cuda().requires_grad_(True), w.to(dt).cuda(), labels.cuda()
    out = linear_cross_entropy.apply(x, w, labels)
    dx, = torch.autograd.grad(out.sum(), x)
    z = x.detach().double() @ w.double().t().contiguous()
    lse = torch.logsumexp(z, 1)
    at = torch.arange(T, device="cuda")
    # (of the row's largest logits too: sums of 64 terms in float, some of 300)
    assert ((out.double() - (lse - z[at, labels])).abs() <= 2e-5 + 1e-6 * (z[at, labels].abs() + lse.abs())).all()
    P = torch.exp(z - lse[:, None])
    exact = P @ w.double() - w.double()[labels]
    eps = torch.finfo(dt).eps
    # entries below 2^-28 of a row's largest (fp16) lose bits of a 2^-39th of it: V 2^-39 |w| at most
    limit = (P @ w.double().abs()) * (eps / 2 + 1e-5) + exact.abs() * eps / 2 + V * 2.0 ** -39 * w.double().abs().amax(0) + 1e-6
    assert ((dx.double() - exact).abs() <= limit).all()


@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("T,V", [(700, 100001), (2200, 300001)])
def test_pieces_of_the_vocabulary(T, V, dt):
    """G of one piece and of three (512 MiB of it at a time)."""
    x, w, labels = make(T, 64, V, dt, 5)
    x = x.requires_grad_(True)
    w = w.requires_grad_(True)
    out = linear_cross_entropy.apply(x, w, labels)
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    z = x.detach().double() @ w.detach().double().t().contiguous()
    lse = torch.logsumexp(z, 1)
    at = torch.arange(T, device="cuda")
    assert (out.double() - (lse - z[at, labels])).abs().max() < 2e-5
    G = torch.exp(z - lse[:, None])
    G[at, labels] -= 1
    eps = torch.finfo(dt).eps
    for got, a, b in ((dx, G, w.detach().double()), (dw, G.t().contiguous(), x.detach().double())):
        exact, bound = a @ b, a.abs() @ b.abs()
        assert ((got.double() - exact).abs() <= bound * (eps / 2 + 1e-5) + exact.abs() * eps / 2 + 1e-7).all()


@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("T,H,V,labelled", [(1, 64, 100, 1.0), (7, 1304, 805, 1.0), (32, 264, 1000, 1.0), (32, 264, 1000, 0.6), (9, 104, 156, 0.5)])
def test_few_rows_keep_what_rounding_takes(T, H, V, labelled, dt):
    """The vocabulary's gradient of up to 32 rows: entries of G are held in two numbers, off by (eps / 2)^2, so that the result's own
    rounding is what is left (and the logits' error, of p)."""
    x, w, labels = make(T, H, V, dt, T + H, labelled)
    part = torch.tensor([0, T // 3, T - T // 4, T], dtype=torch.int32, device="cuda")
    grad = torch.tensor([1.3, 0.7, 1.1], device="cuda")
    w = w.requires_grad_(True)
    out = linear_cross_entropy.apply(x, w, labels, part)
    dw, = torch.autograd.grad(out, w, grad)
    c = torch.zeros(T, dtype=torch.float64)
    for p, (a, b) in enumerate(zip(part.tolist(), part.tolist()[1:])):
        c[a:b] = grad.double().cpu()[p] / max(1, int((labels[a:b] >= 0).sum()))
    _, _, _, exact, _, (bound, soft) = want(x, w.detach(), labels, c)
    eps = torch.finfo(dt).eps
    top = float(x.float().norm(dim=1).max() * w.detach().float().norm(dim=1).max())
    limit = exact.abs() * eps / 2 + bound * (eps * eps / 4 + 4 * 2.0 ** -24) + soft * (2e-6 * top + 1e-6) + 1e-7 * bound.max()
    limit += torch.finfo(dt).smallest_normal * eps
    assert ((dw.double().cpu() - exact).abs() <= limit).all()


@pytest.mark.parametrize("dt", [FP16, BF16])
def test_a_partitions_rows_do_not_share_an_error(dt):
    """c of the second partition lies half a step above a 16-bit number, and so would G, nearly -c, at all its labels: an error of eps / 2 of
    almost all of the gradient.  As it is, the rows times c's part of a power of two are rounded, and the result: each uniform in half a
    step, (eps / 2)^2 / 3 at most in the mean square; the other entries of G (a 100th of the squares here) add theirs."""
    T, V, eps = 300, 20000, torch.finfo(dt).eps
    x, w, labels = make(T, 256, V, dt, 9, spread=0.5)
    w = w.requires_grad_(True)
    part = torch.tensor([0, 20, 300], dtype=torch.int32, device="cuda")
    out = linear_cross_entropy.apply(x, w, labels, part)
    dw, = torch.autograd.grad(out, w, torch.tensor([40.0, 280 * (1 + eps / 2)], device="cuda"))
    c = torch.full((T,), 1 + eps / 2, dtype=torch.float64)
    c[:20] = 2.0
    exact = want(x, w.detach(), labels, c)[3]
    assert (dw.double().cpu() - exact).norm() <= 1.1 * math.sqrt(2 / 3) * eps / 2 * exact.norm()


def test_few_rows_of_infinite_gradients():
    x, w, labels = make(3, 64, 100, BF16)
    w = w.requires_grad_(True)
    out = linear_cross_entropy.apply(x, w, labels)
    dw, = torch.autograd.grad(out, w, torch.tensor([1.0, float("inf"), 1.0], device="cuda"))
    at = labels[1]
    assert torch.equal(dw[at], torch.where(x[1] > 0, -float("inf"), float("inf")).to(BF16))


def test_no_partition_at_all():
    """An edge alone: no row lies in a partition."""
    x, w, labels = make(70, 64, 300, BF16)
    part = torch.tensor([0], dtype=torch.int32, device="cuda")
    loss, lse = torch.full((70,), 7.0, device="cuda"), torch.full((70,), 7.0, device="cuda")
    K.linear_cross_entropy(loss, lse, x, w, labels, part)
    assert not loss.any() and not lse.any()
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    out = linear_cross_entropy.apply(x, w, labels, part)
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    assert out.shape == (0,) and not dx.any() and not dw.any()


def test_offsets_past_32_bits():
    """A vocabulary's matrix of more than 4 GiB in one piece, and rows of more than 4 GiB, against products of chunks in float32."""
    for T, H, V in ((300, 8192, 290000), (290000, 8192, 300)):
        g = torch.Generator(device="cuda").manual_seed(T)
        x = (torch.randn(T, H, generator=g, device="cuda", dtype=BF16)).requires_grad_(True)
        w = (torch.randn(V, H, generator=g, device="cuda", dtype=BF16) * (1.0 / 64)).requires_grad_(True)
        labels = torch.randint(0, V, (T,), generator=g, device="cuda")
        out = linear_cross_entropy.apply(x, w, labels)
        dx, dw = torch.autograd.grad(out.sum(), (x, w))
        frozen, = torch.autograd.grad(linear_cross_entropy.apply(x, w.detach(), labels).sum(), x)
        xd, wd = x.detach(), w.detach()
        for rows in (slice(0, 40), slice(T - 40, T)):  # (whole rows of the gradient of x)
            xr = xd[rows].float()
            z = torch.cat([xr @ wd[i:i + 20000].float().t() for i in range(0, V, 20000)], 1)
            lse = torch.logsumexp(z, 1)
            at = torch.arange(40, device="cuda")
            # (logits of size 1.4 sqrt(2): sums of 8192 products, 8192 2^-24 of |x||w| at most and both sides' error far less)
            assert (out[rows] - (lse - z[at, labels[rows]])).abs().max() < 1e-3
            G = torch.exp(z - lse[:, None])
            G[at, labels[rows]] -= 1
            exact = sum(G[:, i:i + 20000] @ wd[i:i + 20000].float() for i in range(0, V, 20000))
            # |error| <= sum |G w| eps / 2 and its own rounding, and of exp(z - lse) 1e-3 of sum |p w|
            bound = sum(G[:, i:i + 20000].abs() @ wd[i:i + 20000].float().abs() for i in range(0, V, 20000))
            for got in (dx, frozen):
                assert ((got[rows].float() - exact).abs() <= bound * (2.0 ** -8 + 1e-3) + exact.abs() * 2.0 ** -8 + 1e-6).all()
        lse = torch.empty(T, device="cuda")
        K.linear_cross_entropy(torch.empty_like(lse), lse, xd, wd, labels)
        for cols in (slice(0, 40), slice(V - 40, V)):  # (whole rows of the gradient of w)
            at = torch.arange(cols.start, cols.stop, device="cuda")
            exact = bound = 0.0
            for i in range(0, T, 20000):
                xr = xd[i:i + 20000].float()
                G = torch.exp(xr @ wd[cols].float().t() - lse[i:i + 20000, None]) - (labels[i:i + 20000, None] == at).float()
                exact, bound = exact + G.t().contiguous() @ xr, bound + G.abs().t().contiguous() @ xr.abs()
            assert ((dw[cols].float() - exact).abs() <= bound * (2.0 ** -8 + 1e-3) + exact.abs() * 2.0 ** -8 + 1e-6).all()


def test_old_bytes_of_the_workspace():
    """Nothing is read of a workspace, or of what is kept, before it is written."""
    for T, H, V, labelled in ((70, 136, 300, 0.5), (700, 264, 1000, 0.7), (513, 200, 20000, 0.9)):
        x, w, labels = make(T, H, V, BF16, 4, labelled)
        got = []
        for byte in (0, 255):
            f = lambda *s: torch.empty(*s, device="cuda")
            mem = lambda what: torch.full((K._lib.size_query("smlm_vocab_loss_workspace_size", T, H, V, what),), byte, dtype=torch.uint8, device="cuda")
            L, st = K._lib.load(), torch.cuda.current_stream().cuda_stream
            loss, lse, alone, lone_lse, g = f(T), f(T), f(T), f(T), torch.ones(T, device="cuda")
            dx, dw, dx_alone, dx_kept = (torch.empty_like(t) for t in (x, w, x, x))
            kept, ws = mem(5), mem(4)
            p = lambda t: t.data_ptr()
            rc = L.smlm_vocab_loss_fwd(p(loss), p(lse), None, None, p(kept), kept.numel(), p(x), p(w), p(labels), None, 0, p(ws), ws.numel(),
                                       T, H, V, 1, st)
            rc |= L.smlm_vocab_loss_bwd_kept(p(dx_kept), p(g), p(kept), kept.numel(), p(w), None, None, 0, T, H, V, 1, st)
            w0, w3, w1 = mem(0), mem(3), mem(1)
            rc |= L.smlm_vocab_loss_fwd(p(alone), p(lone_lse), None, None, None, 0, p(x), p(w), p(labels), None, 0, p(w0), w0.numel(),
                                        T, H, V, 1, st)
            rc |= L.smlm_vocab_loss_bwd(p(dx), p(dw), p(g), p(loss), p(lse), p(x), p(w), p(labels), None, None, 0, p(w3), w3.numel(),
                                        T, H, V, 1, st)
            rc |= L.smlm_vocab_loss_bwd(p(dx_alone), None, p(g), p(loss), p(lse), p(x), p(w), p(labels), None, None, 0, p(w1), w1.numel(),
                                        T, H, V, 1, st)
            assert rc == 0
            got.append([loss, lse, alone, lone_lse, dx, dw, dx_alone, dx_kept])
        for a, b in zip(*got):
            assert torch.isfinite(a).all() and torch.equal(a, b)


def test_small_gradients_in_fp16():
    """Gradients far below one, and rows whose weights differ by 2^20: G is held relative to the largest."""
    x, w, labels = make(80, 128, 5000, FP16, 1)
    x = x.requires_grad_(True)
    g = torch.full((80,), 2.0 ** -6, device="cuda")
    g[40:] = 2.0 ** -26
    dx, = torch.autograd.grad(linear_cross_entropy.apply(x, w, labels), x, g * 2.0 ** 20)
    loss, _, want_x, _, bound, _ = want(x.detach(), w, labels, g * 2.0 ** 20)
    off = (dx.double().cpu() - want_x).abs()
    limit = bound[0] * 2.0 ** -11 + bound[1] * 1e-4 + want_x.abs() * 2.0 ** -11 + 2.0 ** -25
    assert (off <= limit).all(), (off / limit).max()


def test_infinities_and_nan_stay_in_their_rows():
    x, w, labels = make(70, 64, 300, BF16, 2)
    x[3], x[5, 0] = float("nan"), float("inf")
    x = x.requires_grad_(True)
    out = linear_cross_entropy.apply(x, w, labels)
    dx, = torch.autograd.grad(out.sum(), x)
    bad = torch.zeros(70, dtype=torch.bool, device="cuda")
    bad[3] = bad[5] = True
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()
    assert torch.isnan(dx[bad]).any(1).all() and torch.isfinite(dx[~bad]).all()


def test_large_logits():
    """Logits of some thousands: the maximum is taken off before the exponentials."""
    x, w, labels = make(50, 128, 700, BF16, 4, spread=400.0)
    x = x.requires_grad_(True)
    out = linear_cross_entropy.apply(x, w, labels)
    loss, *_ = want(x.detach(), w, labels, torch.ones(50))
    assert ((out.double().cpu() - loss).abs() <= 1e-5 * (1 + loss.abs()) + 5e-3).all()
    assert torch.isfinite(torch.autograd.grad(out.sum(), x)[0]).all()


@pytest.mark.parametrize("dt", [FP16, BF16])
def test_labels_that_are_nearly_certain(dt):
    """Rows whose label has all but 2^-5 to 2^-40 of the probability: losses and gradients are exact relative to their size (the logits' own
    error aside: 2e-6 of the largest |x||w|, which moves others / e by as much), and where others vanish they are 0."""
    T, H, V = 72, 128, 400
    x, w, labels = make(T, H, V, dt, 11, spread=1.0)
    boost = torch.linspace(1, 40, T)[:, None].cuda()
    x = (0.1 * x.float() + boost * w[labels].float()).to(dt)
    for frozen in (True, False):
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(not frozen)
        out = linear_cross_entropy.apply(a, b, labels)
        dx, = torch.autograd.grad(out.sum(), a)
        z = x.double() @ w.double().t().contiguous()
        at = torch.arange(T, device="cuda")
        own = z[at, labels]
        z[at, labels] = -float("inf")
        others = torch.exp(z - own[:, None])
        loss = torch.log1p(others.sum(1))
        top = (x.double().norm(dim=1).max() * w.double().norm(dim=1).max()).item()
        soft = 4e-6 * top + 4e-6
        keep = loss > 1e-30
        assert ((out.double() - loss).abs() <= loss * soft)[keep].all()
        P = others / (1 + others.sum(1, keepdim=True))
        exact = P @ w.double() - P.sum(1, keepdim=True) * w.double()[labels]
        size = P @ w.double().abs() + P.sum(1, keepdim=True) * w.double()[labels].abs()
        eps, f = torch.finfo(dt).eps, torch.finfo(dt)
        limit = size * (eps / 2 + 2 * soft) + exact.abs() * eps / 2 + f.smallest_normal * f.eps
        assert ((dx.double() - exact).abs() <= limit).all()


def test_differences():
    """The gradient against central differences of the loss: x moves along a direction by powers of two that bf16 holds."""
    x, w, labels = make(8, 64, 200, BF16, 6)
    x = (x.float() * 16).round().clamp(-64, 64).div(16).to(BF16)  # (multiples of 2^-4 up to 4: sums with 2^-5 are exact)
    a = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(linear_cross_entropy.apply(a, w, labels).sum(), a)
    d = (torch.rand(8, 64, generator=torch.Generator().manual_seed(1)) < 0.5).to(BF16).cuda() * 2 - 1
    step = 2.0 ** -5
    up, down = (linear_cross_entropy.apply(x + s * d, w, labels) for s in (step, -step))
    slope = (up - down) / (2 * step)
    along = (dx.float() * d.float()).sum(1)
    # third derivative of a logsumexp along d: at most 2 max |w . d|^3, the difference quotient off by step^2 / 6 of it
    far = (w.double() @ d.double().t()).abs().amax(0).cpu()
    limit = step ** 2 / 3 * far ** 3 + 2e-5 / step + 2.0 ** -8 * 2 * (dx.float().abs() * 2).sum(1).cpu() + 64 * 2.0 ** -9 * w.abs().max().item()
    assert ((slope - along).abs().cpu() <= limit).all()


def test_captured_and_replayed():
    x, w, labels = make(300, 128, 1000, BF16, 7, 0.7)
    part = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    ws = K.Workspace(x.device)
    f = lambda n: torch.empty(n, device="cuda")
    loss, lse, means, weight, dx, dw = f(300), f(300), f(2), f(2), torch.empty_like(x), torch.empty_like(w)
    g, dk = torch.ones(2, device="cuda"), torch.empty_like(x)
    kept = torch.empty(K.linear_cross_entropy_kept_size(300, 128, 1000), dtype=torch.uint8, device="cuda")

    def step():
        K.linear_cross_entropy(loss, lse, x, w, labels, part, means, weight, ws)
        K.linear_cross_entropy_backward(dx, dw, g, loss, lse, x, w, labels, part, weight, ws)
        K.linear_cross_entropy(loss, lse, x, w, labels, part, means, weight, ws, kept)
        K.linear_cross_entropy_backward(dk, None, g, loss, lse, x, w, labels, part, weight, ws, kept)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
    torch.cuda.current_stream().wait_stream(s)
    for seed in (8, 9, 10):
        x2, w2, l2 = make(300, 128, 1000, BF16, seed, 0.4 + 0.1 * (seed - 8))
        x.copy_(x2), w.copy_(w2), labels.copy_(l2)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (means, dx, dw, dk)]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (means, dx, dw, dk)))
        check(x, w, labels, part)


def test_another_stream_and_the_same_bits():
    x, w, labels = make(500, 256, 3000, FP16, 8)
    x = x.requires_grad_(True)
    run = lambda: (lambda o: (o.detach(), torch.autograd.grad(o.sum(), x)[0]))(linear_cross_entropy.apply(x, w, labels))
    first = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_second_derivatives_are_refused():
    x, w, labels = make(8, 64, 100, BF16)
    x = x.requires_grad_(True)
    dx, = torch.autograd.grad(linear_cross_entropy.apply(x, w, labels).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        torch.autograd.grad(dx.float().sum(), x)


@pytest.mark.parametrize("T", [0, 4])
def test_empty(T):
    x = torch.randn(T, 64, device="cuda").to(BF16).requires_grad_(True)
    w = torch.randn(10, 64, device="cuda").to(BF16).requires_grad_(True)
    labels = torch.zeros(T, dtype=torch.int64, device="cuda")
    out = linear_cross_entropy.apply(x, w, labels, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert out.shape == (0,)
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    assert not dx.any() and not dw.any() and dx.shape == x.shape
    if T == 0:
        out = linear_cross_entropy.apply(x, w, labels)
        assert out.shape == (0,) and not torch.autograd.grad(out.sum(), w)[0].any()


def test_refusals():
    x, w, labels = make(8, 64, 100, BF16)
    ok = lambda **k: linear_cross_entropy.apply(*{**dict(x=x, w=w, labels=labels, partition=None), **k}.values())
    part = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    for bad, text in ((dict(x=x.float(), w=w.float()), "No suitable kernel"), (dict(x=x.half()), "dtype"),
                      (dict(x=x[:, :60].contiguous(), w=w[:, :60].contiguous()), "No suitable kernel"),
                      (dict(x=x[:, :32]), "contiguous"), (dict(w=w[:, :32].contiguous()), "columns"),
                      (dict(labels=labels.int()), "int64"), (dict(labels=labels[:4]), "one entry per row"),
                      (dict(x=x.cpu()), "CUDA"), (dict(partition=part.long()), "int32"), (dict(x=x[0]), "2D"),
                      (dict(partition=part[:0]), "partition"), (dict(w=w[:0]), "No suitable kernel")):
        with pytest.raises(RuntimeError, match=text):
            ok(**bad)


def at_the_label(x, w, labels, row, value, rest=0.0):
    """Makes value the row's logit at its label, and rest (0: finite ones) all its others; other rows keep theirs."""
    x[:, 0], w[:, 0] = 0, math.copysign(1.0, rest) if rest else 0
    big = 1e30 if x.dtype == BF16 and not rest else float("inf")  # (1e30 1e30 is an infinity; fp16's largest numbers make none)
    x[row, 0], w[labels[row], 0] = big, math.copysign(1e30 if big < math.inf else 1.0, value)


@pytest.mark.parametrize("frozen", [True, False])
@pytest.mark.parametrize("T,V", [(70, 300), (20, 300), (600, 20000)])
@pytest.mark.parametrize("dt,rest", [(BF16, 0.0), (BF16, -math.inf), (FP16, -math.inf)])
def test_a_label_of_infinite_probability(T, V, frozen, dt, rest):
    """The label's logit is +infinity, the others are finite or -infinity: a softmax divides infinity by infinity, and the row's loss and
    gradient are NaN as its."""
    x, w, labels = make(T, 64, V, dt, 12)
    at_the_label(x, w, labels, 5, math.inf, rest)
    others = torch.arange(T, device="cuda") != 5
    x, w = x.requires_grad_(True), w.requires_grad_(not frozen)
    out = linear_cross_entropy.apply(x, w, labels)
    assert torch.isnan(out[5]) and torch.isfinite(out[others]).all()
    assert torch.isnan(linear_cross_entropy.apply(x.detach(), w.detach(), labels)[5])
    dx, = torch.autograd.grad(out.sum(), x)
    assert torch.isnan(dx[5]).any() and torch.isfinite(dx[others]).all()


def test_one_entry_that_is_no_number():
    """A vocabulary of one entry: no other logit says that the label's is NaN or an infinity."""
    x, w, labels = make(6, 64, 1, BF16, 2)
    x[1], x[2, 0], w[0, 0] = float("nan"), float("inf"), 1.0
    x[3, 0] = -float("inf")
    out = linear_cross_entropy.apply(x, w, labels)
    assert torch.isnan(out[1:4]).all() and not out[0].any() and not out[4:].any()


@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("T,V", [(70, 300), (20, 300), (600, 20000)])
def test_a_label_far_below_the_others(T, V, dt):
    """The label's logit is near -2^20: the logsumexp is of the others and as exact as theirs (2e-6 of |x||w| without the label's column; exponentials,
    sum and logarithm 2e-6 and 2^-22 of it), where loss + z would be off by a float's step of 2^20; so are the gradients of both routes."""
    x, w, labels = make(T, 64, V, dt, 13)
    x[:, 0], w[:, 0] = 0, 0
    top = (x.double().norm(dim=1).max() * w.double().norm(dim=1).max()).item()
    x[5, 0], w[labels[5], 0] = 1024, -1024
    z = x.double() @ w.double().t().contiguous()
    exact = torch.logsumexp(z, 1)
    for kept in (None, torch.empty(K.linear_cross_entropy_kept_size(T, 64, V), dtype=torch.uint8, device="cuda")):
        loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
        K.linear_cross_entropy(loss, lse, x, w, labels, kept=kept)
        assert (lse.double() - exact)[5].abs() <= 2e-6 * top + 2e-6 + 2.0 ** -22 * exact[5].abs()
        # (the logit itself: 64 products summed in float, 64 2^-24 2^20 at most; and z log2 e - ref, its difference with the sum's logarithm and its
        # product with ln 2, half a float's step of 2^-3 each, with 2^20 2e-8 for log2 e as a float: 0.25 in all)
        assert (loss.double() - (exact - z[torch.arange(T), labels]))[5].abs() <= 4.25
    check(x, w, labels)
    check(x, w, labels, want_w=False)


@pytest.mark.parametrize("T,V", [(70, 300), (20, 300), (600, 20000)])
def test_a_label_of_no_probability(T, V):
    """The label's logit is -infinity: the loss is infinite, the logsumexp that of the others, and the gradient finite: it pulls with all its
    weight.  Both routes."""
    x, w, labels = make(T, 64, V, BF16, 14)
    at_the_label(x, w, labels, 5, -math.inf)
    z = x.double() @ w.double().t().contiguous()
    z[5, labels[5]] = -math.inf
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    K.linear_cross_entropy(loss, lse, x, w, labels)
    assert loss[5] == math.inf and (lse.double() - torch.logsumexp(z, 1)).abs().max() <= 1e-4
    P = torch.softmax(z, 1)
    exact = (P @ w.double() - w.double()[labels])[5]
    for frozen in (True, False):
        a = x.clone().requires_grad_(True)
        out = linear_cross_entropy.apply(a, w.clone().requires_grad_(not frozen), labels)
        dx, = torch.autograd.grad(out, a, torch.ones_like(out))
        # |error| <= sum |G w| eps / 2 and its own rounding; 1e-4 of p by the logits
        limit = (P[5] @ w.double().abs() + w.double()[labels[5]].abs()) * 2.0 ** -8 * 1.02 + exact.abs() * 2.0 ** -8
        assert ((dx[5].double() - exact).abs() <= limit).all()


@pytest.mark.parametrize("T", [4, 40])
def test_few_rows_of_a_vocabulary_past_32_bits(T):
    """G of few rows is held in 64, each of 2^27 bytes if it were one piece: past 2^32 bytes the second half would be the first's again."""
    V = (1 << 26) + 5
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, 8, generator=g, device="cuda", dtype=BF16).requires_grad_(True)
    w = torch.randn(V, 8, generator=g, device="cuda", dtype=BF16).requires_grad_(True)
    labels = torch.randint(0, V, (T,), generator=g, device="cuda")
    labels[0], labels[1] = V - 1, 0
    out = linear_cross_entropy.apply(x, w, labels)
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    step, xd, wd = 1 << 22, x.detach().float(), w.detach()
    lse = torch.logsumexp(torch.stack([torch.logsumexp(xd @ wd[i:i + step].float().t().contiguous(), 1) for i in range(0, V, step)]), 0)
    at = (xd * wd[labels].float()).sum(1)
    assert (out.detach() - (lse - at)).abs().max() < 1e-4
    exact_dx = bound_dx = 0.0
    eps = 2.0 ** -7
    for i in range(0, V, step):
        wi = wd[i:i + step].float()
        G = torch.exp(xd @ wi.t().contiguous() - lse[:, None])
        here = ((labels >= i) & (labels < i + wi.shape[0])).nonzero()[:, 0]
        G[here, labels[here] - i] -= 1
        exact_dx, bound_dx = exact_dx + G.double() @ wi.double(), bound_dx + G.abs().double() @ wi.abs().double()
        exact, bound = G.t().contiguous() @ xd, G.abs().t().contiguous() @ xd.abs()
        # |error| <= sum |G x| eps / 2 and eps / 2 of the result, and 1e-4 of p by the logits
        assert ((dw[i:i + step].float() - exact).abs() <= bound * (eps / 2 + 2e-4) + exact.abs() * eps / 2 + 1e-12).all(), i
    assert ((dx.double() - exact_dx).abs() <= bound_dx * (eps / 2 + 2e-4) + exact_dx.abs() * eps / 2 + 1e-6).all()


def test_more_tiles_than_a_launch_takes():
    """The losses alone of 2^20 rows against 2^20 entries, 2^24 tiles: more threads than HIP launches at once."""
    T = V = 1 << 20
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w = (torch.randn(n, 8, generator=g, device="cuda", dtype=BF16) for n in (T, V))
    labels = torch.randint(0, V, (T,), generator=g, device="cuda")
    out = linear_cross_entropy.apply(x, w, labels)
    for rows in (slice(0, 300), slice(T // 2, T // 2 + 300), slice(T - 300, T)):
        z = x[rows].float() @ w.float().t().contiguous()
        exact = torch.logsumexp(z, 1) - z[torch.arange(300), labels[rows]]
        assert (out[rows] - exact).abs().max() < 1e-4  # (logits of size 8: 2e-6 of |x||w| and as much of a logsumexp in float)


def test_more_rows_than_a_launch_takes():
    """2^26 rows, four a workgroup of those that move rows and fold their gradients; every 2^12th has a label."""
    T, V = (1 << 26) + 7, 40
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, 8, generator=g, device="cuda", dtype=BF16).requires_grad_(True)
    w = torch.randn(V, 8, generator=g, device="cuda", dtype=BF16).requires_grad_(True)
    labels = torch.full((T,), -100, device="cuda")
    at = torch.arange(0, T, 1 << 12, device="cuda")
    at[-1] = T - 1
    labels[at] = torch.randint(0, V, at.shape, generator=g, device="cuda")
    z = x.detach()[at].float() @ w.detach().float().t().contiguous()
    G = torch.softmax(z, 1)
    loss = torch.logsumexp(z, 1) - z[torch.arange(len(at)), labels[at]]
    G[torch.arange(len(at)), labels[at]] -= 1
    exact, bound = G @ w.detach().float(), G.abs() @ w.detach().float().abs()
    for frozen in (True, False):
        out = linear_cross_entropy.apply(x, w.detach() if frozen else w, labels)
        dx = torch.autograd.grad(out.sum(), [x] if frozen else [x, w])[0]
        assert (out.detach()[at] - loss).abs().max() < 1e-4 and int(out.count_nonzero()) == len(at)
        assert ((dx[at].float() - exact).abs() <= bound * (2.0 ** -8 + 2e-4) + exact.abs() * 2.0 ** -8 + 1e-6).all()
        assert int(dx.any(1).count_nonzero()) == len(at)


def test_more_partitions_than_a_launch_takes():
    """2^22 partitions of a row or none, a workgroup of 1024 each."""
    T, P = 1 << 20, (1 << 22) + 9
    x, w, labels = make(64, 8, 50, BF16, 3)
    x, labels = x.repeat(T // 64, 1), labels.repeat(T // 64)
    part = (torch.arange(P + 1, device="cuda") // 4).clamp(max=T).int()
    rows = linear_cross_entropy.apply(x, w, labels)
    means = linear_cross_entropy.apply(x, w, labels, part)
    first = torch.arange(P, device="cuda") % 4 == 3
    first &= torch.arange(P, device="cuda") // 4 < T
    assert torch.equal(means[first], rows) and not means[~first].any()


@pytest.mark.parametrize("T", [20, 80, 300])
@pytest.mark.parametrize("parted", [True, False])
@pytest.mark.parametrize("apart", [13, 20, 26])
@pytest.mark.parametrize("want_w", [True, False])
def test_small_weights_beside_large_ones_in_fp16(T, parted, apart, want_w):
    """Half of the rows weigh 2^-13 to 2^-26 of the others, with the vocabulary's gradient beside the rows', so G is made: entries are off by eps / 2
    or 2^-28 of their own row's weight, and rows' gradients by sum |w| of that; in the vocabulary's gradient the rows are rounded once
    more where they take the rest of the weight, by eps / 2 or 2^-36 of the largest weight's |x|."""
    H, V, eps = 128, 5000, 2.0 ** -10
    x, w, labels = make(T, H, V, FP16, T)
    g = torch.full((T,), 2.0 ** 10, device="cuda")
    half = T // 2
    g[half:] *= 2.0 ** -apart
    part = torch.tensor([0, half, T], dtype=torch.int32, device="cuda")
    grad = torch.stack([g[0] * half, g[-1] * (T - half)]) if parted else g
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(want_w)
    if want_w:
        out = linear_cross_entropy.apply(a, b, labels, part if parted else None)
        dx, dw = torch.autograd.grad(out, (a, b), grad)
    else:  # (the same G, without what the forward keeps)
        loss, lse, dx, means, weight = *(torch.empty(T, device="cuda") for _ in range(2)), torch.empty_like(x), *(torch.empty(2, device="cuda") for _ in range(2))
        K.linear_cross_entropy(loss, lse, x, w, labels, *((part, means, weight) if parted else ()))
        K.linear_cross_entropy_backward(dx, None, grad, loss, lse, x, w, labels, *((part, weight) if parted else ()))
    _, _, want_x, want_dw, bx, bw = want(x, w, labels, g)
    top = (x.double().norm(dim=1).max() * w.double().norm(dim=1).max()).item()
    c, X, W = g.double().cpu(), x.double().cpu().abs(), w.double().cpu().abs()
    off = (dx.double().cpu() - want_x).abs()
    limit = bx[0] * eps / 2 + bx[1] * (2e-6 * top + 2e-6) + want_x.abs() * eps / 2 + c[:, None] * 2.0 ** -28 * W.sum(0) + 2.0 ** -25
    assert (off <= limit).all(), (off / limit).max()
    if want_w:
        off = (dw.double().cpu() - want_dw).abs()
        limit = bw[0] * eps + bw[1] * (2e-6 * top + 2e-6) + want_dw.abs() * eps / 2 + c @ X * 2.0 ** -28 + 2.0 ** 10 * T * 2.0 ** -36 + 2.0 ** -25
        assert (off <= limit).all(), (off / limit).max()
