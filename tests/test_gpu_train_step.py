"""A fine-tuning step of the operators around the projections together, as a model runs them: the residual's norms, a projection with
its adapters, the loss by train partition, the adapters' update; and the native host path against the Python functions it stands in for."""
import pytest
import torch

from loquetier_amd import _lib
from loquetier_amd.kernel_utils import BatchLenInfo, add_rms_norm, linear_cross_entropy
from loquetier_amd.mixed_lora import MixedLoraContext, MixedLoraLinear, NamedLoraLayer
from loquetier_amd.ops import _kernels as K
from loquetier_amd.optim import AdamW

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16
H, V, R, EPS = 256, 1000, 16, 1e-5
BOUNDS, ADAPTERS, TRAIN = [0, 40, 97, 104, 105, 106], [1, 2, 0, 2, 1], [1, 2]  # two train sequences, a prompt, two single tokens
SCALING = [0.5, 1.0, 2.0]


class Model:
    def __init__(self, dt, bits=32):
        g = torch.Generator().manual_seed(7)
        mk = lambda *s, by=1.0: (torch.randn(*s, generator=g) * by).to(dt).cuda()
        base = torch.nn.Linear(H, H, bias=False, device="cuda", dtype=dt)
        base.weight.data.copy_(mk(H, H, by=H ** -0.5))
        base.weight.requires_grad_(False)
        self.base, self.named = base, [NamedLoraLayer(f"a{i}", mk(R, H, by=H ** -0.5), mk(H, R, by=0.25), torch.nn.Identity(), SCALING[i]) for i in range(3)]
        self.ctx = MixedLoraContext()
        self.layer = MixedLoraLinear(self.ctx, base, self.named, R, dt, is_scaled=False, fused=True)
        self.layer.set_trainable(TRAIN)
        self.norms = [(1 + 0.1 * torch.randn(H, generator=g)).to(dt).cuda().requires_grad_(True) for _ in range(2)]
        self.head = mk(V, H, by=2 * H ** -0.5)
        self.x, self.residual = (mk(BOUNDS[-1], H).requires_grad_(True) for _ in range(2))
        labels = torch.randint(0, V, (BOUNDS[-1],), generator=g)
        labels[::7] = -100
        labels[97:] = -100
        self.labels = labels.cuda()
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        self.partition = i32([0, 40, 97])
        self.blen = BatchLenInfo([(1, 40), (1, 57)], [7], 2, [], torch.device("cuda"))
        self.segment, self.lens = i32(BOUNDS), i32([b - a for a, b in zip(BOUNDS, BOUNDS[1:])])
        self.adapters = [[self.layer.get_parameter(f"lora-{i}-{m}") for m in "AB"] for i in TRAIN]
        self.opt = AdamW([dict(params=p, lr=1e-3 * (i + 1)) for i, p in enumerate(self.adapters)], state_bits=bits)
        self.leaves = [self.x, self.residual, *self.norms, *sum(self.adapters, [])]

    def losses(self):
        self.ctx.update(blen=self.blen, lora_ids=ADAPTERS, lora_len=self.lens, segment=self.segment, train_idx=TRAIN)
        y, h = add_rms_norm.apply(self.x, self.residual, self.norms[0], EPS)
        y, h = add_rms_norm.apply(self.layer(y), h, self.norms[1], EPS)
        return linear_cross_entropy.apply(y, self.head, self.labels, self.partition)

    def step(self):
        for t in self.leaves:
            t.grad = None
        losses = self.losses()
        losses.sum().backward()
        self.opt.step()
        return losses.detach()

    def exact(self):
        """The losses and gradients of the formulas in 64 bits."""
        d = {id(t): t.detach().double().cpu().requires_grad_(True) for t in self.leaves}
        norm = lambda h, w: h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * w
        x, r, n0, n1 = (d[id(t)] for t in (self.x, self.residual, *self.norms))
        h = x + r
        y = norm(h, n0)
        out = y @ self.base.weight.detach().double().cpu().t()
        rows = []
        for (a, b), i in zip(zip(BOUNDS, BOUNDS[1:]), ADAPTERS):
            wa, wb = [d[id(p)] for p in self.adapters[TRAIN.index(i)]] if i in TRAIN else (
                self.named[i].wa.double().cpu(), self.named[i].wb.double().cpu())
            rows.append(SCALING[i] * (y[a:b] @ wa.t() @ wb.t()))
        h = h + out + torch.cat(rows)
        z, labels = norm(h, n1) @ self.head.double().cpu().t(), self.labels.cpu()
        ends = self.partition.tolist()
        losses = torch.stack([torch.nn.functional.cross_entropy(z[a:b], labels[a:b], ignore_index=-100) for a, b in zip(ends, ends[1:])])
        losses.sum().backward()
        return losses.detach(), [d[id(t)].grad for t in self.leaves]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", [FP16, BF16])
def test_a_step(dt, bits):
    """On the way from a leaf to its gradient a value is rounded at most 12 times (the sums, norms, the adapters' middle, the projection, the
    exponentials, and the gradients of each), each time by eps / 2 of itself; what follows multiplies such an error of random sign by no
    more than about 2 (a norm divides by a length near one, logits have a size near 2).  24 eps / 2 of a gradient's length covers them."""
    m = Model(dt, bits)
    for step in range(2):
        before = [p.detach().clone() for p in sum(m.adapters, [])]
        want, grads = m.exact()
        kept = [m.opt.state_of(p)["master"].double() if step else p.detach().double() for p in sum(m.adapters, [])]
        old = [m.opt.state_of(p) for p in sum(m.adapters, [])]
        losses = m.step()
        eps = torch.finfo(dt).eps
        assert ((losses.double().cpu() - want).abs() <= 24 * eps / 2 * want).all()
        for t, g in zip(m.leaves, grads):
            assert t.grad is not None and torch.isfinite(t.grad).all()
            assert (t.grad.double().cpu() - g).norm() <= 24 * eps / 2 * g.norm()
        assert m.x.grad.data_ptr() != m.residual.grad.data_ptr() and not m.x.grad[97:].any()  # (rows without a loss)
        for i, (p, was, w, o) in enumerate(zip(sum(m.adapters, []), before, kept, old)):
            g, lr = p.grad.double(), 1e-3 * (i // 2 + 1)
            b1, b2 = torch.tensor([0.9, 0.999]).tolist()  # (the rates' floats: the averages' sums and their ages go by the same)
            a = b1 * o["exp_avg"].double() + (1 - b1) * g
            v = b2 * o["exp_avg_sq"].double() + (1 - b2) * g * g
            w = w - lr * 0.01 * w - lr / (1 - b1 ** (step + 1)) * a / ((v / (1 - b2 ** (step + 1))).sqrt() + 1e-8)
            got = m.opt.state_of(p)["master"]
            # some float roundings of the weight and of the step (2^-24 each; v_rcp_f32 and v_sqrt_f32 2^-23)
            assert ((got.double() - w).abs() <= 4 * 2.0 ** -24 * w.abs() + 16 * 2.0 ** -24 * 4 * lr).all()
            assert torch.equal(p.detach(), got.to(dt)) and not torch.equal(p.detach(), was)


def everything(monkeypatch=None):
    m = Model(BF16, 8)
    out = [m.step() for _ in range(2)] + [t.grad for t in m.leaves] + [p.detach() for p in sum(m.adapters, [])]
    out += [t.view(torch.uint8) for t in m.opt._sets[0].tensors.values()]
    w = m.head.clone().requires_grad_(True)
    losses = linear_cross_entropy.apply(m.x, w, m.labels)
    out += [losses.detach(), *torch.autograd.grad(losses.sum(), (m.x, w))]
    x, e8, sc = m.x.detach(), torch.empty(106, H, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(106, 2, device="cuda")
    y, h = torch.empty_like(x), torch.empty_like(x)
    K.add_rms_norm(y, None, h, x, m.residual.detach(), m.norms[0].detach(), EPS, e8, sc)
    return out + [y, h, e8.view(torch.uint8), sc]


def test_native_and_python_have_the_same_bits(monkeypatch):
    assert K._host() is not _lib._NoHost, "the native host path is not built"
    native = everything()
    monkeypatch.setattr(K, "_host", lambda: _lib._NoHost)
    python = everything()
    assert len(native) == len(python) and all(torch.equal(a, b) for a, b in zip(native, python))


def test_taken_and_handed_back():
    """Plain calls are taken; others are handed back with nothing written."""
    h = K._host()
    x, w, v = torch.randn(6, 64, device="cuda").half(), torch.ones(64, device="cuda").half(), torch.randn(50, 64, device="cuda").half()
    y = torch.arange(6, device="cuda")
    assert h.add_rms_norm(x, x, w, EPS) is not None and h.linear_cross_entropy(x, v, y) is not None
    assert h.add_rms_norm(x, x[:5], w, EPS) is None and h.add_rms_norm(x.float(), x.float(), w, EPS) is None
    assert h.add_rms_norm(x, x, w[:56], EPS) is None and h.add_rms_norm(x.t(), x.t(), w, EPS) is None and h.add_rms_norm(x, x, w.cpu(), EPS) is None
    assert h.linear_cross_entropy(x, v[:, :56], y) is None and h.linear_cross_entropy(x, v, y.int()) is None
    assert h.linear_cross_entropy(x, v, y[:5]) is None and h.linear_cross_entropy(x, v.bfloat16(), y) is None
    assert h.linear_cross_entropy(x, v, y, y) is None and h.linear_cross_entropy(x[:0], v, y[:0]) is None
    out = torch.zeros_like(x)
    call = lambda *a: h.add_rms(*a, None, None)
    assert call(out, None, None, x, None, w, EPS) is True and bool(out.any())
    kept = out.clone()
    assert call(out, None, out, x, None, w, EPS) is False and call(None, None, None, x, x, w, EPS) is False
    assert call(out, y, None, x, None, w, EPS) is False and call(out[:5], None, None, x, None, w, EPS) is False
    assert torch.equal(out, kept)
    p, f, i = [torch.ones(10, device="cuda").half()], torch.zeros(256, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    rates = torch.zeros(1, 5, device="cuda")
    step = lambda p=p, g=p, m=f, s=i, r=rates: h.adamw_step(p, g, m, f.clone(), s, r, i.clone(), None, None, None, None)
    assert step() is True and i.item() == 1
    assert step(g=[]) is False and step(m=f[:100]) is False and step(s=i.long()) is False and step(r=rates[:, :4]) is False
    assert step(p=p * 2, g=p * 2) is False and step(g=[p[0].float()]) is False and step(p=[p[0].cpu()]) is False
    assert i.item() == 1


def test_groups_that_join_behind_a_captured_step():
    """A captured step goes on with its own table of rates, which stays and follows the groups; so does one whose states were set back."""
    w = [torch.randn(500).to(BF16).cuda().requires_grad_(True) for _ in range(3)]
    for p in w:
        p.grad = torch.ones_like(p)
    opt = AdamW(w[:2], lr=0.0, weight_decay=0.0)
    fresh = opt.state_dict()
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        opt.step()
        with torch.cuda.graph(graph, stream=s):
            opt.step()
    torch.cuda.current_stream().wait_stream(s)
    opt.add_param_group(dict(params=[w[2]], lr=0.5))
    opt.param_groups[0]["lr"] = 0.25
    opt.update_rates()
    junk = [torch.full((n,), float("nan"), device="cuda") for n in (5, 10, 15, 128)]  # (into what might have been freed)
    was = [p.detach().clone() for p in w]
    graph.replay()
    torch.cuda.synchronize()
    assert all(((a.float() - p.detach().float() - 0.25).abs() <= 0.25 * 2.0 ** -8 + 2.0 ** -8 * a.float().abs()).all() for a, p in zip(was[:2], w))
    assert torch.equal(was[2], w[2].detach()) and len(junk) == 4
    opt = AdamW(w[:2], lr=0.5)
    opt.step()
    opt.load_state_dict({**fresh, "state": dict(bits=32, sets=[])})
    assert opt.state_of(w[0])["step"] == 0 and not opt.state_of(w[0])["exp_avg"].any()
