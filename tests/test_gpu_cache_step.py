"""The operators between the projections as a server runs them: prompts and decoding requests in one batch, answers forked from a
prompt, requests that end, a packed pool, a captured decode step, two caches on two streams."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HQ, HKV, D, P, L = 8, 2, 64, 16, 2


@pytest.fixture(scope="module")
def K(gpu_device):
    from loquetier_amd import _lib
    from loquetier_amd.ops import _kernels
    _lib.load()
    return _kernels


class Server:
    """A cache, and beside it every request's keys and values by layer as they were handed over."""

    def __init__(self, K, dtype=torch.bfloat16, pages=200, seed=0):
        from loquetier_amd.kvcache import PagedKvCache
        self.cache = PagedKvCache(pages, L, HKV, D, max_requests=24, max_tokens=600, page_size=P, dtype=dtype)
        self.table = K.rope_table(600, D, device="cuda")
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype, self.K = dtype, K
        self.kept = {}
        self.wq, self.wk = ((1 + 0.1 * torch.randn(D, generator=self.g, device="cuda")).to(dtype) for _ in range(2))

    def step(self, requests, counts, extra=0):
        T = sum(counts) + extra
        s = self.cache.extend(requests, counts, T)
        plan = self.cache.plan(s, HQ)
        outs = []
        for layer in range(L):
            qkv = torch.randn(T, (HQ + 2 * HKV) * D, generator=self.g, device="cuda").to(self.dtype)
            q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([HQ * D, HKV * D, HKV * D], 1))
            outs.append((q, self.cache.attend(layer, q, k, v, s, plan, self.table, self.wq, self.wk)))
            row = 0
            for r, n in zip(requests, counts):
                if r >= 0:
                    self.kept.setdefault(r, [[] for _ in range(L)])[layer].append((k[row:row + n].double(), v[row:row + n].double()))
                row += n
        self.cache.check()
        for layer, (q, out) in enumerate(outs):
            row = 0
            for r, n in zip(requests, counts):
                if r >= 0 and n:
                    self.compare(r, layer, q[row:row + n], out[row:row + n])
                row += n
            assert not bool(out[row:].any())

    def turn(self, x, w, pos):
        cos, sin = self.table[pos].double()[:, None].chunk(2, -1)
        y = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        a, b = y.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    def compare(self, r, layer, q, out):
        k, v = (torch.cat(t) for t in zip(*self.kept[r][layer]))
        n, length = q.shape[0], k.shape[0]
        k = self.turn(k, self.wk, torch.arange(length, device="cuda")).repeat_interleave(HQ // HKV, 1)
        q = self.turn(q.double(), self.wq, torch.arange(length - n, length, device="cuda"))
        s = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * D ** -0.5
        s = s.masked_fill(torch.arange(length, device="cuda") > torch.arange(length - n, length, device="cuda")[:, None], float("-inf"))
        p, vv = torch.softmax(s, -1), v.repeat_interleave(HQ // HKV, 1).transpose(0, 1)
        want, size = torch.matmul(p, vv).transpose(0, 1), torch.matmul(p, vv.abs()).transpose(0, 1)
        # queries and keys are rounded between the two operators (u each, of normed heads of 1.1^2 D at most in square, so a score
        # moves by 2 u 1.1^4 sqrt(D) or so at the very most, and a weight by that share, twice with their sum), the weights once, and
        # the result once
        u = torch.finfo(self.dtype).eps / 2
        bound = u * want.abs() + (u + 4 * u * 1.5 * D ** 0.5) * size
        assert bool(((out.double() - want).abs() <= bound + 1e-9).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_serving(K, dtype):
    s = Server(K, dtype)
    s.step([0, 1, 2], [37, 130, 1])
    s.step([0, 1, 2, 3], [1, 1, 1, 64])            # a prompt joins decoding requests
    s.step([3, 0, -1, 2], [50, 1, 0, 1], extra=3)  # its second chunk; a place left open; rows of padding
    s.cache.fork([1, 1, 3], [4, 5, 6])             # answers to one prompt
    for p, c in ((1, 4), (1, 5), (3, 6)):
        s.kept[c] = [list(l) for l in s.kept[p]]
    s.step([1, 4, 5, 6, 3, 0], [1, 1, 1, 1, 1, 1])
    s.cache.free([1, 2])
    s.kept.pop(1), s.kept.pop(2)
    s.step([4, 5, 1, 2], [1, 2, 20, 200])          # their numbers come again
    s.cache.free([0, 5])
    s.kept.pop(0), s.kept.pop(5)
    s.cache.compact()
    live = int((s.cache.refs > 0).sum())
    assert bool((s.cache.refs[:live] > 0).all())
    s.step([1, 2, 3, 4, 6], [1, 1, 1, 17, 1])
    for r in list(s.kept):
        assert int(s.cache.length[r]) == sum(k.shape[0] for k, _ in s.kept[r][0])
    s.cache.free(list(s.kept))
    assert not bool(s.cache.refs.any()) and bool((s.cache.table == -1).all())


def test_a_refused_step_leaves_the_cache_whole(K):
    s = Server(K, pages=12)
    s.step([0, 1], [100, 50])
    before = [t.clone() for t in (s.cache.pool, s.cache.table, s.cache.length, s.cache.refs)]
    bad = s.cache.extend([2], [60])
    plan = s.cache.plan(bad, HQ)
    q = torch.ones(60, HQ, D, dtype=torch.bfloat16, device="cuda")
    out = s.cache.attend(0, q, q[:, :HKV], q[:, :HKV], bad, plan, s.table)
    assert not bool(out.any())
    assert all(torch.equal(a, b) for a, b in zip(before, (s.cache.pool, s.cache.table, s.cache.length, s.cache.refs)))
    with pytest.raises(RuntimeError, match="no free pages"):
        s.cache.check()
    s.cache.check()
    s.step([0, 1], [1, 1])


def test_decode_step_in_a_graph(K):
    """One decode step, captured, replayed step after step with the program's own work in between, against eager steps of another cache."""
    from loquetier_amd.kvcache import PagedKvCache
    R = 5

    def make():
        c = PagedKvCache(120, 1, HKV, D, R, 400, P)
        g = torch.Generator(device="cuda").manual_seed(3)
        n = [3, 40, 15, 16, 260]
        st = c.extend(list(range(R)), n)
        k, v = c.layer(0)
        x = torch.randn(sum(n), HQ + 2 * HKV, D, generator=g, device="cuda").to(torch.bfloat16)
        q = torch.empty_like(x[:, :HQ])
        K.qk_norm_rope(q, None, x[:, :HQ], x[:, HQ:HQ + HKV], table, st.positions, v=x[:, HQ + HKV:], k_cache=k, v_cache=v, slots=st.slots)
        return c

    table = K.rope_table(400, D, device="cuda")
    requests = torch.arange(R, dtype=torch.int32, device="cuda")
    ones = torch.ones(R, dtype=torch.int32, device="cuda")
    x = torch.zeros(R, HQ + 2 * HKV, D, dtype=torch.bfloat16, device="cuda")

    def step(c):
        s = c.extend(requests, ones, R)
        return c.attend(0, x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:], s, c.plan(s, HQ), table)

    eager, graphed = make(), make()
    g = torch.Generator(device="cuda").manual_seed(4)
    inputs = [torch.randn(x.shape, generator=g, device="cuda").to(torch.bfloat16) for _ in range(40)]
    want = []
    for i in inputs:
        x.copy_(i)
        want.append(step(eager))
    eager.check()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x.copy_(inputs[0])
        assert torch.equal(step(graphed), want[0])  # (the eager pass that sizes the workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(graphed)
    for i, w in zip(inputs[1:], want[1:]):
        x.copy_(i)
        graph.replay()
        torch.cuda.synchronize()
        torch.ones(1000, device="cuda").sum().item()
        assert torch.equal(out, w)
    graphed.check()
    assert torch.equal(graphed.pool, eager.pool) and torch.equal(graphed.length, eager.length)


def test_two_caches_on_two_streams(K):
    """Each with its own workspace: the same results as one after the other."""
    def work(s):
        s.step([0, 1, 2], [300, 1, 17])
        for _ in range(3):
            s.step([0, 1, 2], [1, 1, 1])

    servers = [Server(K, seed=i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in servers]
    for s, st in zip(servers, streams):
        with torch.cuda.stream(st):
            s.step([3], [200])
    for s, st in zip(servers, streams):
        with torch.cuda.stream(st):
            work(s)
    torch.cuda.synchronize()


def test_training_rows_beside_serving_rows(K):
    """[train | decode] in one batch: the training rows' slots are -1 and their gradient flows through the rotation."""
    from loquetier_amd.kernel_utils import qk_norm_rope
    from loquetier_amd.kvcache import PagedKvCache
    c = PagedKvCache(20, 1, HKV, D, 4, 100, P)
    table = K.rope_table(200, D, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    mk = lambda n, h: torch.randn(n, h, D, generator=g, device="cuda").to(torch.bfloat16)
    q, k = mk(48, HQ).requires_grad_(True), mk(48, HKV).requires_grad_(True)
    pos = torch.arange(48, dtype=torch.int32, device="cuda")
    qo, ko = qk_norm_rope.apply(q, k, None, None, table, pos, 1e-6)
    (qo.float().square().sum() + ko.float().square().sum()).backward()
    # a rotation keeps lengths: the gradient of the squares is twice the input, to the roundings of output, gradient and result
    for t in (q, k):
        pair = t.detach().float().abs()
        pair = pair + pair.roll(D // 2, -1)
        assert bool(((t.grad.float() - 2 * t.detach().float()).abs() <= 2 * 4 * 2 ** -8 * pair).all())
    s = c.extend([0, 1], [30, 2])
    x = mk(32, HQ)
    out = c.attend(0, x, mk(32, HKV), mk(32, HKV), s, c.plan(s, HQ), table)
    assert bool(out.isfinite().all()) and int(c.refs.sum()) == 3


def test_python_refusals(K):
    x = torch.zeros(4, HQ, D, dtype=torch.bfloat16, device="cuda")
    k = x[:, :HKV]
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, pos = K.rope_table(9, D, device="cuda"), i32(0, 1, 2, 3)
    cache = torch.zeros(3, HKV, P, D, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    rope = lambda **kw: K.qk_norm_rope(**{**dict(q_out=x.clone(), k_out=k.clone(), q=x, k=k, table=table, positions=pos), **kw})
    for kw, what in ((dict(q=x.float(), k=k.float()), "No suitable kernel"), (dict(k=k[:3]), "same rows"), (dict(positions=pos[:3]), "one entry per row"),
                     (dict(positions=pos.long()), "positions must be"), (dict(table=table.double()), "table must be"),
                     (dict(table=table[:, :24].contiguous()), "rot_dim"), (dict(q_weight=torch.ones(3, dtype=x.dtype, device="cuda")), "entries"),
                     (dict(q_out=k.clone()), "same shape"), (dict(k_out=None), "left out"), (dict(slots=slots), "come together"),
                     (dict(q=x.transpose(1, 2).contiguous().transpose(1, 2)), "next to each other"),
                     (dict(v=k, k_cache=cache, v_cache=cache.clone().transpose(1, 2).contiguous().transpose(1, 2), slots=slots), "same shape and strides"),
                     (dict(q_out=x[:1].expand(4, HQ, D)), "expanded"), (dict(v=k, k_cache=cache[:1].expand(3, HKV, P, D),
                      v_cache=cache[:1].expand(3, HKV, P, D), slots=slots), "expanded"),
                     (dict(v=k, k_cache=cache[..., :32], v_cache=cache[..., :32], slots=slots), "must be"),
                     (dict(v=k, k_cache=cache, v_cache=cache, slots=slots[:2]), "one entry per row"),
                     (dict(k_out=None, v=k, k_cache=cache[:0], v_cache=cache[:0], slots=slots), "no pages")):
        with pytest.raises(RuntimeError, match=what):
            rope(**kw)
    pt = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="multiple of kv_heads"):
        K.AttentionPlan(i32(0, 1, 2), i32(1, 1), pt, 2, 5, 2, P)
    with pytest.raises(RuntimeError, match="one entry more"):
        K.AttentionPlan(i32(0, 1, 2), i32(1), pt, 2, 4, 2, P)
    with pytest.raises(RuntimeError, match="a row for each"):
        K.AttentionPlan(i32(0, 1, 2), i32(1, 1), pt[:1], 2, 4, 2, P)
    plan = K.AttentionPlan(i32(0, 2, 4), i32(2, 2), pt, 4, HQ, HKV, P)
    for args, what in (((x[:3], x[:3], cache, cache), "plan is for"), ((x, x, cache[:, :1], cache[:, :1]), "must be"),
                       ((x, x, cache[:, :, :8], cache[:, :, :8]), "pages of"), ((x, x.half(), cache, cache), "dtype"),
                       ((x, x, cache, cache.half()), "dtype"), ((x[:1].expand(4, HQ, D), x, cache, cache), "expanded")):
        with pytest.raises(RuntimeError, match=what):
            K.paged_attention(*args, plan)
    with pytest.raises(RuntimeError, match="scale"):
        K.paged_attention(x, x, cache, cache, plan, scale=-1.0)
    with pytest.raises(RuntimeError, match="one page per entry"):
        K.kv_compact(cache, pt, i32(0, 0))
    with pytest.raises(RuntimeError, match="one entry per"):
        K.kv_extend(pt, i32(0, 0), i32(0, 0, 0), i32(0), i32(0, 0), 1, P)
