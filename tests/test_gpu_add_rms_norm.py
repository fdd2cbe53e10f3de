"""add_rms_norm against its definition in 64 bits: widths at the edges of each kernel route, 8-bit outputs by row and by 128 columns, the
backward with and without a gradient of the sum.

Tolerances.  The sum is the float sum of two 16-bit values rounded once: torch's own, bit for bit.  The norm: squares and their sum in
float (relative error of the mean well under 1e-6: terms of one sign, summed in 64 or 256 lanes), a square root, a division and two
products, 2^-24 each: 2e-6 relative; then half a step of 16 bits (eps / 2), or of the subnormal numbers.  8 bits: y / scale is at most 448 and rounded to half a step,
2^-4 of the value or 2^-10 below the normal ones (in units of the scale); the scale itself is off by 2e-6 relative.
Backward: dh = gh + r (gw - h r^2 mean(gw h)): a sum of three terms, each to 4e-6 of its size, rounded once; dw: a sum over rows in
float, 2e-6 of the sum of absolute values, rounded once."""
import pytest
import torch

from loquetier_amd.kernel_utils import add_rms_norm
from loquetier_amd.ops import _kernels as K

pytestmark = pytest.mark.gpu
FP16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
EPS = 1e-5


def make(rows, cols, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *n: torch.randn(*n, generator=g)
    return [t.to(dt).cuda() for t in (0.3 * r(rows, cols), 2 * r(rows, cols) * (0.2 + r(cols).abs()), 1 + 0.2 * r(cols))]


def total(x, residual):
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def norm64(h, w):
    h = h.double()
    r = 1 / (h.square().mean(1, keepdim=True) + EPS).sqrt()
    return h * r * w.double(), r


def near(got, exact, dt, rel=2e-6, size=None):
    f = torch.finfo(dt)
    limit = exact.abs() * f.eps / 2 + (exact.abs() if size is None else size) * rel + f.smallest_normal * f.eps
    off = (got.double() - exact).abs()
    assert (off <= limit).all(), (off / limit).max()


def near8(out8, scale, y, cols):
    group = cols // scale.shape[1]
    y = y.unflatten(1, (-1, group))
    most = y.abs().amax(2)
    assert ((scale.double() - most / 448).abs() <= 3e-6 * most / 448).all()
    got = out8.float().double().unflatten(1, (-1, group)) * scale.double()[..., None]
    limit = y.abs() * (2.0 ** -4 + 1e-5) + scale.double()[..., None] * 2.0 ** -10 * 1.001
    assert ((got - y).abs() <= limit).all()
    assert (out8.float().unflatten(1, (-1, group)).abs().amax(2)[most > 0] == 448).all()


SHAPES = [(1, 8), (3, 64), (5, 512), (4, 520), (7, 1024), (9, 1048), (6, 2048), (1, 4096), (1030, 4096), (1025, 2056), (5, 4104), (3, 8192),
          (2, 8200), (3, 16384), (2, 16392), (3, 20480)]


@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("with_residual", [True, False])
def test_forward(rows, cols, with_residual, dt):
    x, residual, w = make(rows, cols, dt, rows + cols)
    residual = residual if with_residual else None
    h = torch.empty_like(x) if with_residual else None
    out, rms = torch.empty_like(x), torch.empty(rows, 1, device="cuda")
    out8, scale = torch.empty(rows, cols, dtype=F8, device="cuda"), torch.empty(rows, 1, device="cuda")
    K.add_rms_norm(out, rms, h, x, residual, w, EPS, out8, scale)
    want = total(x, residual)
    y, r = norm64(want, w)
    if h is not None:
        assert torch.equal(h, want)
    assert ((rms.double() - r).abs() <= 2e-6 * r).all()
    near(out, y, dt)
    near8(out8, scale, y, cols)
    alone = torch.empty_like(x)
    K.add_rms_norm(alone, None, None, x, residual, w, EPS)
    assert torch.equal(alone, out)
    only8, scale2 = torch.empty_like(out8), torch.empty_like(scale)
    K.add_rms_norm(None, None, None, x, residual, w, EPS, only8, scale2)
    assert torch.equal(only8.view(torch.uint8), out8.view(torch.uint8)) and torch.equal(scale, scale2)
    if cols % 128 == 0:
        scale = torch.empty(rows, cols // 128, device="cuda")
        K.add_rms_norm(out, None, h, x, residual, w, EPS, out8, scale)
        near8(out8, scale, y, cols)
        assert torch.equal(out, alone)


@pytest.mark.parametrize("cols", [1048, 4096, 8192, 20480])
def test_in_place(cols):
    x, residual, w = make(37, cols, BF16, cols)
    out, h = torch.empty_like(x), torch.empty_like(x)
    K.add_rms_norm(out, None, h, x, residual, w, EPS)
    for which in range(3):
        a, b = x.clone(), residual.clone()
        o, s = [(torch.empty_like(x), b), (a, b), (b, a)][which]
        K.add_rms_norm(o, None, s, a, b, w, EPS)
        assert torch.equal(o, out) and torch.equal(s, h)
    a = x.clone()
    K.add_rms_norm(a, None, None, a, None, w, EPS)
    alone = torch.empty_like(x)
    K.rms_norm(alone, torch.empty(37, 1, device="cuda"), x, w, EPS)
    assert torch.equal(a, alone)


def test_rows_of_zeros_and_no_numbers():
    x, residual, w = make(6, 256, BF16, 1)
    x[0], residual[0] = 0, 0
    x[1, 3], x[2, 200], x[3] = float("inf"), float("nan"), float("nan")
    x[4], residual[4] = 1, -1
    for shape in ((6, 1), (6, 2)):
        out, h = torch.empty_like(x), torch.empty_like(x)
        out8, scale = torch.empty(6, 256, dtype=F8, device="cuda"), torch.empty(*shape, device="cuda")
        K.add_rms_norm(out, None, h, x, residual, w, EPS, out8, scale)
        for row in (0, 4):
            assert not out[row].any() and not out8[row].float().any() and not scale[row].any()
        assert torch.isnan(out[1, 3]) and not out[1, torch.arange(256) != 3].any()
        assert torch.isnan(scale[1, 0]) and torch.isnan(out[2]).all() and torch.isnan(scale[2]).all() and torch.isnan(scale[3]).all()
        y, _ = norm64(h[5:], w)
        near(out[5:], y, BF16)
        near8(out8[5:], scale[5:], y, 256)


@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 64), (130, 520), (1021, 1048), (300, 4096), (77, 8200), (9, 16384), (5, 20480)])
@pytest.mark.parametrize("with_sum", [True, False])
def test_gradients(rows, cols, with_sum, dt):
    x, residual, w = (t.requires_grad_(True) for t in make(rows, cols, dt, rows))
    g, gh, _ = make(rows, cols, dt, rows + 1)
    gh = gh if with_sum else None
    out, h = add_rms_norm.apply(x, residual, w, EPS)
    dx, dr, dw = torch.autograd.grad((out, h) if with_sum else out, (x, residual, w), (g, gh) if with_sum else g)
    assert torch.equal(dx, dr) and torch.equal(h, total(x.detach(), residual.detach()))
    h64, w64, g64 = h.detach().double(), w.detach().double(), g.double()
    y, r = norm64(h.detach(), w.detach())
    near(out.detach(), y, dt)
    gw = g64 * w64
    back = h64 * r * r * (gw * h64).mean(1, keepdim=True)
    size = r * (gw.abs() + h64.abs() * r * r * (gw * h64).abs().mean(1, keepdim=True)) + (gh.double().abs() if with_sum else 0)
    near(dx, r * (gw - back) + (gh.double() if with_sum else 0), dt, 4e-6, size)
    near(dw, (g64 * h64 * r).sum(0), dt, 4e-6, (g64 * h64 * r).abs().sum(0))


def test_gradients_without_the_norm_and_the_old_norms():
    x, residual, w = (t.requires_grad_(True) for t in make(64, 1024, BF16))
    g = make(64, 1024, BF16, 5)[0]
    out, h = add_rms_norm.apply(x, residual, w, EPS)
    dx, dr, dw = torch.autograd.grad(h, (x, residual, w), g, allow_unused=True)
    assert torch.equal(dx, g) and torch.equal(dr, g) and dw is None
    # without a sum's gradient: bit for bit the norm's backward of the stored sum, given the same root mean squares (which each
    # forward sums in an order of its own)
    out, h = add_rms_norm.apply(x, residual, w, EPS)
    dx, dw = torch.autograd.grad(out, (x, w), g)
    rms, alone = torch.empty(64, 1, device="cuda"), torch.empty_like(out)
    K.add_rms_norm(alone, rms, None, x.detach(), residual.detach(), w.detach(), EPS)
    ds, dv = torch.empty_like(dx), torch.empty_like(dw)
    K.rms_norm_backward(ds, dv, g, h.detach(), w.detach(), rms)
    assert torch.equal(alone, out) and torch.equal(ds, dx) and torch.equal(dv, dw)


def test_differences():
    """The gradient of x against central differences; sums in 64 bits of outputs rounded to fp16 (half a step of 2^-10 of each)."""
    x, residual, w = make(4, 64, FP16, 3)
    x = (x.float() * 64).round().div(64).half()
    residual = (residual.float() * 64).round().div(64).half()
    a = x.clone().requires_grad_(True)
    out, _ = add_rms_norm.apply(a, residual, w, EPS)
    c = make(4, 64, FP16, 4)[0]
    dx, = torch.autograd.grad(out, a, c)
    d = ((torch.rand(4, 64, generator=torch.Generator().manual_seed(1)) < 0.5).half() * 2 - 1).cuda()
    step = 2.0 ** -4
    f = lambda s: (add_rms_norm.apply(x + s * d, residual, w, EPS)[0].double() * c.double()).sum(1)
    slope, along = (f(step) - f(-step)) / (2 * step), (dx.double() * d.double()).sum(1)
    h = total(x, residual).double()
    r = 1 / (h.square().mean(1) + EPS).sqrt()
    # outputs: rounded, 2^-11 of each; dx likewise; the third derivative along d (|d| has a mean square of one): at most 15 r^3 sum |c w| max(1, |h r|)
    size = (c.double().abs() * w.double().abs() * (1 + (h * r[:, None]).abs())).sum(1)
    limit = 2.0 ** -11 * (out.double().abs() * c.double().abs()).sum(1) / step + 2.0 ** -11 * dx.double().abs().sum(1) + \
        step ** 2 / 6 * 15 * r ** 3 * size + 1e-3
    assert ((slope - along).abs() <= limit).all()


def test_captured_and_another_stream():
    x, residual, w = make(64, 1024, BF16)
    out, h, out8, scale = torch.empty_like(x), torch.empty_like(x), torch.empty(64, 1024, dtype=F8, device="cuda"), torch.empty(64, 8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        K.add_rms_norm(out, None, h, x, residual, w, EPS, out8, scale)
        with torch.cuda.graph(graph, stream=s):
            K.add_rms_norm(out, None, h, x, residual, w, EPS, out8, scale)
    torch.cuda.current_stream().wait_stream(s)
    for seed in range(3):
        for t, n in zip((x, residual, w), make(64, 1024, BF16, seed + 10)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        y, _ = norm64(total(x, residual), w)
        near(out, y, BF16)
        near8(out8, scale, y, 1024)


def test_second_derivatives_are_refused_and_no_rows():
    x, residual, w = (t.requires_grad_(True) for t in make(4, 64, BF16))
    out, h = add_rms_norm.apply(x, residual, w, EPS)
    dx, = torch.autograd.grad(out.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        torch.autograd.grad(dx.float().sum(), x)
    x, residual = x[:0].detach().requires_grad_(True), residual[:0].detach()
    out, h = add_rms_norm.apply(x, residual, w, EPS)
    dx, dw = torch.autograd.grad((out, h), (x, w), (torch.empty_like(out), torch.empty_like(h)))
    assert out.shape == (0, 64) and dx.shape == (0, 64) and not dw.any()


def test_refusals():
    x, residual, w = make(8, 256, BF16)
    e = lambda *n, dt=BF16: torch.empty(*n, dtype=dt, device="cuda")
    ok = dict(output=e(8, 256), rms_output=None, residual_output=None, input=x, residual=residual, weight=w, epsilon=EPS)
    for bad, text in ((dict(input=x.float()), "No suitable kernel"), (dict(weight=w[:8]), "one entry per column"),
                      (dict(residual=residual.half()), "bfloat16"), (dict(residual=residual[:4]), "same shape"),
                      (dict(residual=None, residual_output=e(8, 256)), "sum with a residual"), (dict(output=None), "output is needed"),
                      (dict(output8=e(8, 256, dt=F8)), "come together"), (dict(scale=e(8, 1, dt=torch.float32)), "come together"),
                      (dict(output8=e(8, 256, dt=torch.uint8), scale=e(8, 1, dt=torch.float32)), "float8"),
                      (dict(output8=e(8, 256, dt=F8), scale=e(8, 3, dt=torch.float32)), "scale must be"),
                      (dict(output8=e(8, 256, dt=F8), scale=e(8, 1)), "float32"), (dict(rms_output=e(8, dt=torch.float32)), "2D"),
                      (dict(input=x[:, ::2]), "contiguous"), (dict(input=x.cpu()), "CUDA"), (dict(output=e(8, 128)), "same shape")):
        with pytest.raises(RuntimeError, match=text):
            K.add_rms_norm(**{**ok, **bad})
    y = x[:, :136].contiguous()
    with pytest.raises(RuntimeError, match="scale must be"):
        K.add_rms_norm(e(8, 136), None, None, y, None, w[:136], EPS, e(8, 136, dt=F8), e(8, 2, dt=torch.float32))


@pytest.mark.parametrize("rows,cols,group", [(2112, 4096, 128), (2112, 4096, 4096), (16000, 512, 128), (300, 20480, 128), (300, 20480, 20480)])
@pytest.mark.parametrize("dt", [FP16, BF16])
def test_codes_are_those_of_the_quotients(rows, cols, group, dt):
    """The 8-bit values are the rounding of the correctly rounded y / scale (a product with 1 / scale is off by more, and between two codes takes
    the other one), so the norm in tensor expressions gives the same codes: of the kernel's own h, rms and scales, bit for bit."""
    x, residual, w = make(rows, cols, dt, rows + group)
    h, rms, scale = torch.empty_like(x), torch.empty(rows, 1, device="cuda"), torch.empty(rows, cols // group, device="cuda")
    out8 = torch.empty(rows, cols, dtype=F8, device="cuda")
    K.add_rms_norm(None, rms, h, x, residual, w, EPS, out8, scale)
    y = (h.float() * rms * w.float()).unflatten(1, (-1, group))
    assert torch.equal((y / scale[..., None]).flatten(1).to(F8).float(), out8.float())


def test_an_infinite_norm_leaves_its_groups_other_codes():
    x = torch.ones(2, 256, dtype=BF16, device="cuda")
    w = torch.ones(256, dtype=BF16, device="cuda")
    x[0, :128] = 0
    x[0, 3], w[3] = 8.0, 3e38  # (y overflows there)
    out8, scale = torch.empty(2, 256, dtype=F8, device="cuda"), torch.empty(2, 2, device="cuda")
    K.add_rms_norm(None, None, None, x, None, w, EPS, out8, scale)
    codes = out8.float()
    assert scale[0, 0] == float("inf") and torch.isnan(codes[0, 3]) and not codes[0, :128][torch.arange(128) != 3].any()
    assert torch.isfinite(scale[:, 1]).all() and torch.isfinite(codes[:, 128:]).all()


def test_more_rows_than_a_launch_takes():
    """2^24 workgroups of 256 are more threads than HIP launches at once.  Rows repeat, so that a few tell of all."""
    rows, cols = (1 << 26) + 5, 8
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < rows * cols * 8 + (1 << 33):
        pytest.skip("needs the memory")
    few = 1 << 12
    x, residual, w = make(few, cols, BF16, 3)
    want = [torch.empty_like(x), torch.empty(few, 1, device="cuda"), torch.empty_like(x)]
    K.add_rms_norm(*want, x, residual, w, EPS)
    x = x.repeat(-(-rows // few), 1)[:rows]
    x[-1] = 1.0  # (the last row is its own)
    residual = residual.repeat(-(-rows // few), 1)[:rows]
    out, rms, h = torch.empty_like(x), torch.empty(rows, 1, device="cuda"), torch.empty_like(x)
    K.add_rms_norm(out, rms, h, x, residual, w, EPS)
    whole = rows // few * few
    for got, one in zip((out, rms, h), want):
        got = got[:whole].view(-1, *one.shape)
        assert all(torch.allclose(got[i:i + 64].float(), one.float(), rtol=2e-2, atol=1e-6) for i in range(0, len(got), 64))
    y, _ = norm64(total(x[-1:], residual[-1:]), w)
    near(out[-1:], y, BF16)
