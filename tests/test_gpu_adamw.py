"""adamw_step and optim.AdamW against the formulas in 64 bits.

Tolerances.  Averages: two products and a sum in float, 3 x 2^-24 of the summands' sizes (2e-7 is taken of each).  The update lr m / (...): a
root, two products, a reciprocal (v_rcp_f32 and v_sqrt_f32: 2^-23 each), a sum: 1e-6 of the update, and 2^-23 of the weight for the two subtractions;
16-bit weights are rounded once more, eps / 2.  8 bits: values relative to the block's scale, rounded to 2^-4 of the value or 2^-10 of the
scale below the normal numbers."""
import copy
import math
import pickle

import pytest
import torch

from loquetier_amd.ops import _kernels as K
from loquetier_amd.optim import AdamW

pytestmark = pytest.mark.gpu
FP16, BF16, F32, F8 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn
B = K.ADAMW_BLOCK


class Problem:
    def __init__(self, sizes, dt, bits, master, seed=0, groups=2, odd=()):
        g = torch.Generator().manual_seed(seed)
        r = lambda *n: torch.randn(*n, generator=g)

        def tensor(i, n, by):  # (some start off the alignment of four elements)
            flat = (r(n + 1) * by).to(dt).cuda()
            return flat[1:] if i in odd else flat[:n].clone()
        self.params = [tensor(i, n, 0.05) for i, n in enumerate(sizes)]
        self.grads = [tensor(i, n, 1e-2) for i, n in enumerate(sizes)]
        self.blocks = [-(-n // B) for n in sizes]
        n = sum(self.blocks)
        there = torch.cat([torch.nn.functional.pad(torch.ones(s), (0, -s % B)) for s in sizes]).view(n, B) if n else torch.zeros(0, B)
        m, v = r(n, B) * 1e-3 * there, (r(n, B) * 1e-2).square() * there
        self.bits = bits
        if bits == 8:
            self.ms, self.vs = m.abs().amax(1) / 448, v.sqrt().amax(1) / 448
            code = lambda a, s: (a / torch.where(s > 0, s, 1)[:, None]).to(F8).flatten().cuda()
            self.m, self.v = code(m, self.ms), code(v.sqrt(), self.vs)
            self.ms, self.vs = self.ms.cuda(), self.vs.cuda()
        else:
            self.m, self.v, self.ms, self.vs = m.flatten().cuda(), v.flatten().cuda(), None, None
        self.master = None
        if master:
            self.master = torch.zeros(n * B).cuda()
            for i, (at, k) in enumerate(self.spans()):
                self.master[at:at + k] = self.params[i].float() * (1 + 1e-4 * r(k).cuda())
        self.hyper = torch.tensor([[1e-2 / (1 + j), 0.9 - 0.1 * j, 0.999 - 0.01 * j, 1e-8 * 10 ** j, 0.01 * j] for j in range(groups)]).cuda()
        self.group = (torch.arange(len(sizes), dtype=torch.int32) % groups).cuda()
        self.step = (torch.arange(len(sizes), dtype=torch.int32) * 7 % 50).cuda()

    def spans(self):
        at = 0
        for p, b in zip(self.params, self.blocks):
            yield at, p.numel()
            at += b * B

    def averages(self):
        m, v = self.m.float().double().view(-1, B), self.v.float().double().view(-1, B)
        if self.bits == 8:
            m, v = m * self.ms.double()[:, None], (v * self.vs.double()[:, None]).square()
        return m.flatten(), v.flatten()

    def run(self, grads=None):
        K.adamw_step(self.params, self.grads if grads is None else grads, self.m, self.v, self.step, self.hyper, self.group, self.ms,
                     self.vs, self.master)

    def check(self, grads=None):
        """One step, against the formulas in 64 bits."""
        grads = self.grads if grads is None else grads
        m0, v0 = self.averages()
        before = [p.clone() for p in self.params]
        full = None if self.master is None else self.master.clone()
        raw = self.m.clone(), self.v.clone(), None if self.ms is None else (self.ms.clone(), self.vs.clone())
        steps = self.step.clone()
        self.run(grads)
        m1, v1 = self.averages()
        dt = before[0].dtype
        eps = torch.finfo(dt).eps
        for i, (at, n) in enumerate(self.spans()):
            blocks = slice(at // B, at // B + self.blocks[i])
            if grads[i] is None or n == 0:
                assert torch.equal(self.params[i], before[i]) and (n == 0 and grads[i] is not None or self.step[i] == steps[i])
                if n:
                    assert torch.equal(self.m[at:at + n].view(torch.uint8), raw[0][at:at + n].view(torch.uint8))
                    assert full is None or torch.equal(self.master[at:at + n], full[at:at + n])
                continue
            assert self.step[i] == steps[i] + 1
            lr, b1, b2, e, wd = self.hyper[self.group[i]].double().tolist()
            t = int(self.step[i])
            g, w = grads[i].double().flatten(), before[i].double().flatten()
            if full is not None:
                kept = full[at:at + n]
                w = torch.where(kept.to(dt).double() == w, kept.double(), w)
            m, v = b1 * m0[at:at + n] + (1 - b1) * g, b2 * v0[at:at + n] + (1 - b2) * g * g
            den = (v / (1 - b2 ** t)).sqrt() + e
            update = lr / (1 - b1 ** t) * m / den
            new = w * (1 - lr * wd) - update
            size_m = b1 * m0[at:at + n].abs() + (1 - b1) * g.abs()
            size = new.abs() * 2.0 ** -23 + w.abs() * 2.0 ** -23 + update.abs() * 1e-6 + lr / (1 - b1 ** t) * size_m / den * 4e-7
            off = (self.params[i].double().flatten() - new).abs()
            tiny = torch.finfo(dt).smallest_normal * eps if dt != F32 else 1e-38
            limit = size + (0 if dt == F32 else new.abs() * eps / 2 * (1 + 1e-3) + tiny)
            assert (off <= limit).all(), (i, (off / limit).max())
            if full is not None:
                assert ((self.master[at:at + n].double() - new).abs() <= size + 1e-38).all()
                assert torch.equal(self.master[at:at + n].to(dt), self.params[i].flatten())
            for got, exact, scale, sizes in ((m1[at:at + n], m, self.ms, size_m), (v1[at:at + n], v, self.vs, v)):
                if scale is None:
                    assert ((got - exact).abs() <= sizes * 4e-7 + 1e-38).all()
                    continue
                root = exact is v
                a, b = (got.sqrt(), exact.sqrt()) if root else (got, exact)
                s = scale[blocks].double().repeat_interleave(B)[:n]
                top = torch.nn.functional.pad(b.abs(), (0, -n % B)).view(-1, B).amax(1)
                assert ((scale[blocks].double() - top / 448).abs() <= 2e-6 * top / 448).all()
                limit = b.abs() * (2.0 ** -4 + 1e-5) + s * 2.0 ** (-9 if root else -10) * 1.001 + sizes.sqrt() * 0 + 1e-38
                assert ((a - b).abs() <= limit).all(), ((a - b).abs() / limit).max()
                if root:
                    assert (got[exact > 0] > 0).all()
        rest = torch.ones(self.m.numel(), dtype=torch.bool, device="cuda")
        for at, n in self.spans():
            rest[at:at + n] = False
        assert not self.m.float()[rest].any() and not self.v.float()[rest].any()


SIZES = [[1], [256], [3, 1, 255, 257, 4], [4096, 0, 1000, 65536, 0, 511], [5] * 40 + [70000] + [0] * 3 + [1024] * 130 + [2]]


@pytest.mark.parametrize("sizes", SIZES, ids=len)
@pytest.mark.parametrize("dt,master", [(FP16, True), (BF16, True), (BF16, False), (FP16, False), (F32, False)])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps(sizes, dt, master, bits):
    p = Problem(sizes, dt, bits, master, len(sizes))
    p.check()
    p.check()
    p.check([g if i % 3 else None for i, g in enumerate(p.grads)])


@pytest.mark.parametrize("dt,master", [(BF16, True), (FP16, False), (F32, False)])
@pytest.mark.parametrize("bits", [32, 8])
def test_addresses_off_the_alignment(dt, master, bits):
    p = Problem([300, 1000, 5, 4096, 777], dt, bits, master, 3, odd=(0, 2, 3))
    assert p.params[0].data_ptr() % 8 if dt != F32 else p.params[0].data_ptr() % 16
    guards = [t._base.clone() for t in (p.params[0], p.params[2], p.params[3])]
    p.check()
    for t, g in zip((p.params[0], p.params[2], p.params[3]), guards):
        assert t._base[0] == g[0]
    p.check()


def test_a_weight_that_was_set_takes_its_masters_place():
    p = Problem([1000], BF16, 32, True)
    p.run()
    p.params[0][:500] = torch.randn(500, device="cuda").to(BF16)
    p.check()
    assert (p.master[:500].double() - p.params[0][:500].double()).abs().max() < 1e-1


def test_no_gradient_at_all_and_a_group_that_is_none():
    p = Problem([300, 400], BF16, 32, True)
    p.check([None, None])
    before = [t.clone() for t in p.params]
    p.group[1] = 5
    steps = p.step.clone()
    p.run()
    assert torch.equal(p.params[1], before[1]) and p.step[1] == steps[1] and not torch.equal(p.params[0], before[0])


def test_infinities_stay_in_their_block():
    for bits in (32, 8):
        p = Problem([1024, 256], F32, bits, False)
        p.grads[0][300] = float("inf")
        p.run()
        bad = torch.zeros(1024, dtype=torch.bool, device="cuda")
        bad[300] = True
        assert torch.isnan(p.params[0][bad]).all() and torch.isfinite(p.params[0][~bad]).all() and torch.isfinite(p.params[1]).all()
        p.grads[0][300] = 0
        p.run()
        if bits == 8:
            bad[256:512] = True  # (a block's values share a scale)
        assert torch.isfinite(p.params[0][~bad]).all() and torch.isfinite(p.params[1]).all()


def test_many_steps_follow_torch():
    """A hundred steps in float beside torch's in 64 bits: errors of a step, 1e-6 of the update and 2^-23 of the weight, add up."""
    g = torch.Generator().manual_seed(0)
    w = [torch.randn(40, 30, generator=g).cuda(), torch.randn(500, generator=g).cuda()]
    mine, theirs = [t.clone().requires_grad_(True) for t in w], [t.double().requires_grad_(True) for t in w]
    a = AdamW([dict(params=mine[:1], lr=1e-2), dict(params=mine[1:], weight_decay=0.1)], lr=1e-3, eps=1e-6)
    b = torch.optim.AdamW([dict(params=theirs[:1], lr=1e-2), dict(params=theirs[1:], weight_decay=0.1)], lr=1e-3, eps=1e-6)
    for s in range(100):
        for p, q in zip(mine, theirs):
            p.grad = torch.randn(p.shape, generator=g).cuda()
            q.grad = p.grad.double()
        if s == 50:
            for o in (a, b):
                o.param_groups[0]["lr"] = 5e-3
        a.step(), b.step()
    for p, q, lr in zip(mine, theirs, (1e-2, 1e-3)):
        assert (p.double() - q).abs().max() < 100 * (2.0 ** -23 * q.abs().max().item() + 2e-6 * lr * 10)
    state = a.state_of(mine[1])
    assert state["step"] == 100 and (state["exp_avg"].double() - b.state[theirs[1]]["exp_avg"]).abs().max() < 1e-5


def test_adapters_take_steps_by_turns():
    w = [torch.randn(64, 32).to(BF16).cuda().requires_grad_(True) for _ in range(2)]
    opt = AdamW([dict(params=[w[0]]), dict(params=[w[1]])], lr=1e-2, state_bits=8)
    start = w[1].detach().clone()
    for _ in range(3):
        w[0].grad, w[1].grad = torch.randn_like(w[0]), None
        opt.step()
    assert torch.equal(w[1], start) and opt.state_of(w[1])["step"] == 0 and opt.state_of(w[0])["step"] == 3
    w[1].grad = torch.ones_like(w[1])
    opt.step()
    # the first step moves each weight by lr (1 of 1e-8, and the decay), rounded
    assert ((start.double() * (1 - 1e-4) - w[1].detach().double() - 1e-2).abs() <= start.double().abs() * 2.0 ** -8 + 1e-4).all()


def test_small_updates_add_up_in_the_masters():
    w = torch.ones(512, dtype=BF16, device="cuda").requires_grad_(True)
    opt = AdamW([w], lr=1e-4, weight_decay=0.0)
    for _ in range(100):
        w.grad = torch.ones_like(w)
        opt.step()
    assert (opt.state_of(w)["master"].double() - (1 - 100 * 1e-4)).abs().max() < 1e-5
    assert torch.equal(w.detach(), opt.state_of(w)["master"].to(BF16)) and (w != 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_and_loaded(bits):
    make = lambda: [torch.randn(100, 20, generator=torch.Generator().manual_seed(i)).to(BF16).cuda().requires_grad_(True) for i in range(3)]
    a, b = make(), make()
    x, y = AdamW(a, lr=1e-2, state_bits=bits), AdamW(b, lr=1e-3, state_bits=bits)
    grads = lambda s: [torch.randn(100, 20, generator=torch.Generator().manual_seed(10 * s + i)).to(BF16).cuda() for i in range(3)]

    def step(o, ps, s):
        for p, g in zip(ps, grads(s)):
            p.grad = g
        o.step()
    for s in range(3):
        step(x, a, s)
    saved = x.state_dict()
    y.load_state_dict(saved)
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    for s in range(3, 6):
        step(x, a, s), step(y, b, s)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and y.param_groups[0]["lr"] == 1e-2
    with pytest.raises(ValueError, match="other tensors"):
        AdamW(make()[:2], state_bits=bits).load_state_dict({**saved, "param_groups": AdamW(make()[:2]).state_dict()["param_groups"]})
    with pytest.raises(ValueError, match="bits"):
        AdamW(make(), state_bits=40 - bits).load_state_dict(saved)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed(bits):
    sizes = [1000] * 20
    w = [torch.randn(n).to(BF16).cuda().requires_grad_(True) for n in sizes]
    v = [t.detach().clone().requires_grad_(True) for t in w]
    for p, q in zip(w, v):
        p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
    a, b = AdamW(w, lr=1e-2, state_bits=bits), AdamW(v, lr=1e-2, state_bits=bits)
    draw = lambda: [p.grad.copy_(torch.randn_like(p)) for p in w] and [q.grad.copy_(p.grad) for p, q in zip(w, v)]
    draw()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        a.step()
        with torch.cuda.graph(graph, stream=s):
            a.step()
    torch.cuda.current_stream().wait_stream(s)
    b.step()
    for i in range(4):
        draw()
        if i == 2:
            for o in (a, b):
                o.param_groups[0]["lr"] = 1e-3
            a.update_rates()
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(w, v)), i
    assert a.state_of(w[0])["step"] == 5


def test_states_are_not_made_while_a_graph_is_captured():
    w = torch.randn(100).cuda().requires_grad_(True)
    w.grad = torch.randn_like(w)
    opt = AdamW([w])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        with pytest.raises(RuntimeError, match="eager step"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
                opt.step()


def test_refusals():
    p = Problem([300, 400], BF16, 32, True)
    call = lambda **k: K.adamw_step(*{**dict(params=p.params, grads=p.grads, m=p.m, v=p.v, step=p.step, hyper=p.hyper, group=p.group, ms=p.ms,
                                             vs=p.vs, master=p.master), **k}.values())
    for bad, text in ((dict(grads=p.grads[:1]), "one entry per tensor"), (dict(params=[p.params[0], p.params[0]], grads=[p.grads[0]] * 2), "twice"),
                      (dict(params=[p.params[0], p.params[1].half()]), "one dtype"), (dict(grads=[p.grads[0], p.grads[1].float()]), "match"),
                      (dict(grads=[p.grads[0], p.grads[1][:3]]), "match"), (dict(m=p.m[:256]), "entries"), (dict(v=p.v.half()), "float32"),
                      (dict(ms=torch.empty(4, device="cuda")), "8 bits"), (dict(m=p.m.to(F8), v=p.v.to(F8)), "8 bits"), (dict(step=p.step[:1]), "one entry"),
                      (dict(hyper=p.hyper[:, :4].contiguous()), "five columns"), (dict(params=[t.cpu() for t in p.params]), "on cuda"),
                      (dict(params=[t.double() for t in p.params], grads=[t.double() for t in p.grads]), "No suitable kernel"),
                      (dict(params=[t.float() for t in p.params], grads=[t.float() for t in p.grads]), "No suitable kernel"),
                      (dict(master=p.master[:256]), "entries"), (dict(params=[p.params[0], torch.empty(800, dtype=BF16, device="cuda")[::2]]), "contiguous")):
        with pytest.raises(RuntimeError, match=text):
            call(**bad)
    with pytest.raises(ValueError):
        AdamW(p.params, lr=-1.0)
    with pytest.raises(ValueError):
        AdamW(p.params, state_bits=16)
    opt = AdamW([torch.randn(4).requires_grad_(True)])
    opt.param_groups[0]["params"][0].grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="No suitable kernel"):
        opt.step()


@pytest.mark.parametrize("dt,master", [(BF16, True), (FP16, False), (F32, False)])
def test_codes_are_those_of_the_tensor_expressions(dt, master):
    """8-bit states, bit for bit: each operation of the averages is rounded by itself, as tensor expressions round it, so no code is its
    neighbour.  Products, sums and quotients are the host's (IEEE), the root is that of tensors on the GPU (sqrtf, which may be a float's step off)."""
    p = Problem([70000, 300, 5, 1 << 20], dt, 8, master, 17)
    f = lambda t: t.float().cpu().view(-1, B)
    m, v = f(p.m) * p.ms.cpu()[:, None], (f(p.v) * p.vs.cpu()[:, None]).square()
    flat = torch.cat([torch.nn.functional.pad(g.float().cpu(), (0, -g.numel() % B)) for g in p.grads]).view(-1, B)
    of = torch.arange(4).repeat_interleave(torch.tensor(p.blocks)) % 2
    b1, b2 = p.hyper.cpu()[of, 1:3].unbind(1)
    n1, n2 = ((1 - b.double()).float()[:, None] for b in (b1, b2))
    m = b1[:, None] * m + n1 * flat
    r = (b2[:, None] * v + n2 * flat * flat).cuda().sqrt().cpu()
    p.run()
    for got, scale, exact, least in ((p.m, p.ms, m, 0.0), (p.v, p.vs, r, 2.0 ** -9)):
        s = exact.abs().amax(1) * torch.tensor(1 / 448)  # (a float's 1 / 448)
        assert torch.equal(scale.cpu(), s)
        q = exact / torch.where(s > 0, s, 1)[:, None]
        assert torch.equal(f(got), torch.where((exact > 0) & (q < least), least, q).to(F8).float())


def test_more_blocks_than_a_launch_takes():
    """2^34 weights, 2^26 blocks of a wave each: more threads than HIP launches at once.  (100 GB; mostly zeros, which stay.)"""
    torch.cuda.empty_cache()
    n = (1 << 34) + 300
    if torch.cuda.mem_get_info()[0] < n * 6.2 + (1 << 33):
        pytest.skip("needs 115 GB")
    blocks = -(-n // B)
    zeros = lambda k, dt: torch.zeros(k, dtype=torch.uint8 if dt == F8 else dt, device="cuda").view(dt)
    w, g, m, v = zeros(n, BF16), zeros(n, BF16), zeros(blocks * B, F8), zeros(blocks * B, F8)
    ms, vs = zeros(blocks, F32), zeros(blocks, F32)
    at = torch.tensor([0, 1 << 32, (1 << 33) - 1, (1 << 34) - 1, n - 1], device="cuda")
    w[at], g[at] = 1.0, torch.tensor([1.0, -1.0, 2.0, 1.0, -1.0], dtype=BF16, device="cuda")
    step, group = zeros(1, torch.int32), zeros(1, torch.int32)
    K.adamw_step([w], [g], m, v, step, torch.tensor([[0.125, 0.9, 0.999, 1e-8, 0.0]], device="cuda"), group, ms, vs)
    assert step.item() == 1
    # (a first step is lr, up to 1e-6 of it: 1 -+ 0.125 to half a step of bf16)
    want = torch.tensor([0.875, 1.125, 0.875, 0.875, 1.125], device="cuda")
    assert ((w[at].float() - want).abs() <= 2.0 ** -8 * want).all()
    assert sum(int(w[i:i + (1 << 30)].count_nonzero()) for i in range(0, n, 1 << 30)) == 5
    assert ((ms[at // B] * 448 - 0.1 * g[at].abs().float()).abs() < 1e-6).all() and int(ms.count_nonzero()) == 5


def tensors(*sizes, dt=BF16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, generator=g).to(dt).cuda().requires_grad_(True) for n in sizes]


def take_step(opt, params, seed):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (torch.randn(p.shape, generator=g) * 1e-2).to(p.dtype).cuda()
    opt.step()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [True, False])
def test_saved_after_a_group_joined(bits, master):
    """An adapter that joins while others train: the states go to and from an optimizer that has had all groups from the start, and one
    whose groups joined as they did, and go on there bit for bit."""
    a, c = tensors(300, 5, 1000), tensors(64, 700, dt=F32, seed=1)
    new = lambda: AdamW([dict(params=a[:1] + c[:1], lr=1e-2)], lr=1e-3, state_bits=bits, master=master)
    x = new()
    take_step(x, a[:1] + c[:1], 1)
    x.add_param_group(dict(params=a[1:2]))
    take_step(x, a[:2] + c[:1], 2)
    x.add_param_group(dict(params=[c[1], a[2]]))
    take_step(x, a + c, 3)
    saved = x.state_dict()
    copies = []
    for joins in (False, True):
        b, d = ([t.detach().clone().requires_grad_(True) for t in ts] for ts in (a, c))
        if joins:
            y = AdamW([dict(params=b[:1] + d[:1], lr=1e-2)], lr=1e-3, state_bits=bits, master=master)
            take_step(y, b[:1] + d[:1], 4)
            y.add_param_group(dict(params=b[1:2]))
            take_step(y, b[:1], 5)
            y.add_param_group(dict(params=[d[1], b[2]]))
            with torch.no_grad():
                for p, q in zip(a + c, b + d):
                    q.copy_(p)
        else:
            y = AdamW([dict(params=b[:1] + d[:1]), dict(params=b[1:2]), dict(params=[d[1], b[2]])], state_bits=bits, master=master)
        y.load_state_dict(saved)
        again = y.state_dict()
        assert again["param_groups"] == saved["param_groups"]
        for s, t in zip(saved["state"]["sets"], again["state"]["sets"]):
            assert all(u is None and t[n] is None or torch.equal(u.view(torch.uint8), t[n].view(torch.uint8)) for n, u in s.items())
        copies.append((y, b + d))
    for i in range(4, 7):
        take_step(x, a + c, i)
        for y, ps in copies:
            take_step(y, ps, i)
    for y, ps in copies:
        assert all(torch.equal(p, q) for p, q in zip(a + c, ps))
        assert all(torch.equal(x.state_of(p)[n], y.state_of(q)[n]) for p, q in zip(a + c, ps) for n in x.state_of(p))


def test_saved_before_a_joined_groups_first_step():
    a = tensors(300, 500)
    x = AdamW([dict(params=a[:1])])
    take_step(x, a[:1], 1)
    x.add_param_group(dict(params=a[1:]))
    b = [t.detach().clone().requires_grad_(True) for t in a]
    y = AdamW([dict(params=b[:1]), dict(params=b[1:])])
    y.load_state_dict(x.state_dict())
    take_step(x, a, 2), take_step(y, b, 2)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and [int(y.state_of(q)["step"]) for q in b] == [2, 1]


def test_a_refused_load_changes_nothing():
    a = tensors(300, 500)
    x = AdamW([dict(params=a[:1]), dict(params=a[1:], weight_decay=0.5)], lr=1e-2)
    take_step(x, a, 1)
    def other(sizes, groups, **kw):
        b = tensors(*sizes)
        y = AdamW([dict(params=[b[i] for i in g]) for g in groups], lr=0.5, **kw)
        take_step(y, b, 2)
        return y.state_dict()
    b = tensors(300, 500)
    theirs = torch.optim.AdamW([dict(params=b[:1]), dict(params=b[1:])], lr=0.5)
    take_step(theirs, b, 3)
    before = x.state_dict()
    for bad in (other([300, 5000], [[0], [1]]), other([300, 500], [[0], [1]], state_bits=8), other([300, 500], [[0], [1]], master=False),
                other([300, 500], [[0, 1]]), other([300], [[0]]), theirs.state_dict()):
        with pytest.raises(ValueError):
            x.load_state_dict(bad)
        after = x.state_dict()
        assert after["param_groups"] == before["param_groups"]
        assert all(torch.equal(t, after["state"]["sets"][0][n]) for n, t in before["state"]["sets"][0].items() if t is not None)


def test_states_of_tensors_of_other_shapes(tmp_path):
    """Tensors that fill as many blocks in all as the saved ones are others all the same; what is saved goes through a file and the host."""
    a = tensors(300, 200)
    x = AdamW(a, state_bits=8)
    take_step(x, a, 1)
    for sizes in ((200, 300), (301, 200), ((30, 10), 200)):
        with pytest.raises(ValueError, match="other tensors"):
            AdamW([torch.zeros(n, dtype=BF16, device="cuda").requires_grad_(True) for n in sizes], state_bits=8).load_state_dict(x.state_dict())
    torch.save(x.state_dict(), tmp_path / "state")
    saved = torch.load(tmp_path / "state", map_location="cpu", weights_only=True)
    b = [t.detach().clone().requires_grad_(True) for t in a]
    y = AdamW(b, state_bits=8)
    y.load_state_dict(saved)
    take_step(x, a, 2), take_step(y, b, 2)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    del saved["state"]["shapes"]  # (as they were saved without)
    AdamW(b, state_bits=8).load_state_dict(saved)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("again", [copy.deepcopy, lambda pair: pickle.loads(pickle.dumps(pair))], ids=["copied", "pickled"])
def test_copies_go_on_alone(bits, again):
    a = tensors(300, 500)
    x = AdamW([dict(params=a[:1], lr=1e-2)], state_bits=bits)
    take_step(x, a[:1], 1)
    x.add_param_group(dict(params=a[1:]))
    take_step(x, a, 2)
    y, b = again((x, a))
    assert all(p is q for p, q in zip(b, [p for g in y.param_groups for p in g["params"]]))
    before = x.state_dict()["state"]["sets"][0]
    take_step(y, b, 3)
    assert all(torch.equal(t.view(torch.uint8), before[n].view(torch.uint8))
               for n, t in x.state_dict()["state"]["sets"][0].items() if t is not None)
    take_step(x, a, 3)
    x.param_groups[0]["lr"] = y.param_groups[0]["lr"] = 1e-3
    take_step(x, a, 4), take_step(y, b, 4)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert all(torch.equal(x.state_of(p)[n], y.state_of(q)[n]) for p, q in zip(a, b) for n in x.state_of(p))


def test_groups_that_leave_and_join():
    """An adapter's group is taken out and another's joins, in one step or two: the one that left stays as it is, gradient or not, the others keep their
    rates, the new one learns, and one that comes back goes on."""
    a = tensors(300, 500, 700)
    new = lambda ps: AdamW([dict(params=[p], lr=r) for p, r in zip(ps, (1e-2, 2e-2))])
    x = new(a)
    take_step(x, a[:2], 1)
    left = x.param_groups.pop(0)
    x.add_param_group(dict(params=[a[2]], lr=4e-2))
    before = [t.detach().clone() for t in a]
    take_step(x, a, 2)
    assert torch.equal(a[0], before[0]) and x.state_of(a[0])["step"] == 1
    for p, b, lr in ((a[1], before[1], 2e-2), (a[2], before[2], 4e-2)):
        b = b.clone().requires_grad_(True)
        y = AdamW([b], lr=lr)
        if p is a[1]:
            g = torch.Generator().manual_seed(1)
            torch.randn(300, generator=g)
            c = tensors(300, 500, 700)[1]
            y = AdamW([c], lr=lr)
            c.grad = (torch.randn(500, generator=g) * 1e-2).to(BF16).cuda()
            y.step()
            b = c
        b.grad = p.grad.clone()
        y.step()
        assert torch.equal(p, b)
    del x.param_groups[0]
    x.step()
    x.param_groups.insert(0, left)
    take_step(x, a[:1], 3)
    assert [int(x.state_of(p)["step"]) for p in a] == [2, 2, 3]
    del x.param_groups[:]
    before = [t.detach().clone() for t in a]
    x.step()
    assert all(torch.equal(p, b) for p, b in zip(a, before))


def test_tensors_that_overlap_are_refused():
    """Two waves would update the same weight, one after the other or not.  Tensors side by side, and one without a gradient, are none of that."""
    flat, g = torch.randn(600, device="cuda").to(BF16), torch.randn(600, device="cuda").to(BF16)
    p = Problem([300, 300], BF16, 32, True)
    for a, b, ok in ((flat[:300], flat[300:], True), (flat[:300], flat[296:596], False), (flat[200:500], flat[:300], False)):
        p.params, p.grads = [a, b], [g[:300], g[300:]]
        if ok:
            p.run()
            continue
        before = flat.clone()
        with pytest.raises(RuntimeError, match="overlap"):
            p.run()
        assert torch.equal(flat, before)
        p.run([g[:300], None])
        assert not torch.equal(flat, before)


def test_groups_that_join_one_after_another_beside_a_captured_step():
    a = tensors(300, 500, 64)
    for t in a:
        t.grad = torch.ones_like(t)
    x = AdamW(a[:1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        x.step()
        with torch.cuda.graph(graph, stream=s):
            x.step()
    torch.cuda.current_stream().wait_stream(s)
    for i in (1, 2):
        x.add_param_group(dict(params=a[i:i + 1], lr=1e-2))
        x.step()
        graph.replay()
        torch.cuda.synchronize()
    assert [int(x.state_of(p)["step"]) for p in a] == [5, 2, 1]


def test_groups_that_leave_and_join_beside_a_captured_step():
    a, b = tensors(300, 500), tensors(300, 500)
    x, y = (AdamW([dict(params=t[:1], lr=1e-2), dict(params=t[1:], lr=2e-2)]) for t in (a, b))
    for t in a + b:
        t.grad = torch.ones_like(t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        x.step()
        with torch.cuda.graph(graph, stream=s):
            x.step()
    torch.cuda.current_stream().wait_stream(s)
    y.step()
    same = lambda: all(torch.equal(p, q) for p, q in zip(a, b))

    def replay():
        x.update_rates()
        graph.replay()
        torch.cuda.synchronize()
        y.step()
    replay()
    assert same()
    left = [o.param_groups.pop(0) for o in (x, y)]  # (the other's group moves up)
    before = a[0].detach().clone()
    replay()
    assert same() and torch.equal(a[0], before)
    for o, g in zip((x, y), left):
        o.param_groups.append(g)
    replay()
    assert same() and not torch.equal(a[0], before)
    more = tensors(64)
    x.add_param_group(dict(params=more))
    x.update_rates()  # (a larger table; the captured step's is kept up)
    replay()
    assert same()
    x.param_groups.insert(0, x.param_groups.pop())
    with pytest.raises(RuntimeError, match="append"):
        x.update_rates()
    x.param_groups.append(x.param_groups.pop(0))
    replay()
    assert same()
