"""The native host path of the operators between the projections against the Python functions it stands in for: the same bits, and
the calls it does not know handed back (its other tests run through it as everybody's calls do)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from loquetier_amd import _lib
    from loquetier_amd.ops import _kernels
    _lib.load()
    assert _kernels._host() is not _lib._NoHost, "the native host path is not built"
    return _kernels


def everything(K):
    from loquetier_amd.kernel_utils import qk_norm_rope
    from loquetier_amd.kvcache import PagedKvCache
    g = torch.Generator(device="cuda").manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
    c = PagedKvCache(60, 1, 2, 64, 8, 300, 16)
    table = K.rope_table(300, 64, device="cuda")
    out = []
    for req, n in (([0, 1], [37, 100]), ([1, 0, 2], [1, 1, 5])):
        s = c.extend(req, n)
        x = mk(sum(n), 12, 64)
        out += [*s, c.attend(0, x[:, :8], x[:, 8:10], x[:, 10:], s, c.plan(s, 8), table)]
    c.fork([0, 1, 1], [3, 4, 5])
    out += [c.table.clone(), c.refs.clone()]
    c.free([0, 4])
    out += [c.table, c.refs, c.length, c.pool, c.status]
    q, k = mk(50, 8, 64).requires_grad_(True), mk(50, 2, 64).requires_grad_(True)
    wq = mk(64).requires_grad_(True)
    o = qk_norm_rope.apply(q, k, wq, None, table, torch.arange(50, dtype=torch.int32, device="cuda"), 1e-5)
    torch.autograd.backward(o, (mk(50, 8, 64), mk(50, 1, 64).expand(50, 2, 64)))
    return out + [t.detach() for t in o] + [q.grad, k.grad, wq.grad]


def test_same_bits(K, monkeypatch):
    from loquetier_amd import _lib
    native = everything(K)
    monkeypatch.setattr(K, "_host", lambda: _lib._NoHost)
    python = everything(K)
    assert len(native) == len(python) and all(torch.equal(a, b) for a, b in zip(native, python))


def test_taken_and_handed_back(K):
    """Plain calls are taken; others are handed back with nothing written."""
    h = K._host()
    x = torch.randn(4, 8, 64, device="cuda").half()
    table, pos = K.rope_table(9, 64, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(x)
    rope = lambda *a: h.rope(*a, None, None, 1e-6, None, None, None, None)
    assert rope(out, out[:, :2].clone(), x, x[:, :2], table, pos) is True and bool(out.any())
    kept = out.clone()
    assert rope(out, None, x, x[:, :2], table, pos) is False
    assert rope(out, out[:, :3], x, x[:, :2], table, pos) is False
    assert rope(out, out[:, :2], x.float(), x[:, :2], table, pos) is False
    assert rope(out, out[:, :2], x, x[:, :2], table[:, :24], pos) is False
    assert rope(out, out[:, :2], x, x[:, :2], table, pos.long()) is False
    assert rope(out, out[:, :2], x, x[:, :2].cpu(), table, pos) is False
    assert torch.equal(out, kept)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    assert h.attention_plan(i32(0, 4), i32(4), i32(0).view(1, 1), 4, 8, 3, 16, None) is None
    assert h.attention_plan(i32(0, 4), i32(4, 4), i32(0).view(1, 1), 4, 8, 2, 16, None) is None
    assert h.kv_extend(i32(0).view(1, 1), i32(0), i32(0), i32(0), i32(0, 1), 1, 16, None, None) is None
    assert h.kv_free(i32(0).view(1, 1), i32(0), i32(0), i32(0), 0, None) is False
    assert h.kv_fork(x, i32(0).view(1, 1), i32(0), i32(0), i32(0), i32(0), None, None) is False


def test_saved_tensors_that_come_back_otherwise(K):
    from loquetier_amd.kernel_utils import qk_norm_rope
    q, k = (torch.randn(6, n, 64, device="cuda").half().requires_grad_(True) for n in (4, 2))
    w = torch.ones(64, dtype=torch.float16, device="cuda", requires_grad=True)
    table, pos = K.rope_table(9, 64, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda")
    for unpack in (lambda t: t.float() if t.dtype == torch.float16 else t, lambda t: t[:3] if t.dim() == 3 else t, lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            a, b = qk_norm_rope.apply(q, k, w, w, table, pos, 1e-6)
        with pytest.raises(RuntimeError):
            (a.sum() + b.sum()).backward()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):  # as offloading does
        a, b = qk_norm_rope.apply(q, k, w, w, table, pos, 1e-6)
    (a.sum() + b.sum()).backward()
    assert bool(q.grad.isfinite().all())


def test_one_output_used(K):
    from loquetier_amd.kernel_utils import qk_norm_rope
    q, k = (torch.randn(6, n, 64, device="cuda").half().requires_grad_(True) for n in (4, 2))
    table, pos = K.rope_table(9, 64, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda")
    a, _ = qk_norm_rope.apply(q, k, None, None, table, pos, 1e-6)
    a.sum().backward()
    assert bool(q.grad.any()) and (k.grad is None or not bool(k.grad.any()))
