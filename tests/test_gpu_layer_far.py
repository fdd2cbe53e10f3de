"""Offsets past 2^31 elements: the rotation's rows and places, pages that do not hold whole loads of attention, and copies of pages.  Each call
against the same one on small tensors, bit for bit."""
import pytest
import torch

from test_gpu_paged_attention import batch, run
from test_gpu_qk_norm_rope import case

pytestmark = pytest.mark.gpu

FAR = 2 ** 29  # elements from row to row: five rows reach past 2^31


@pytest.fixture(scope="module")
def K(gpu_device):
    from loquetier_amd import _lib
    from loquetier_amd.ops import _kernels
    _lib.load()
    return _kernels


def far_rows(like, fill=None):
    """[rows, heads, D] with rows FAR apart, holding `like`."""
    T, H, D = like.shape
    t = torch.empty((T - 1) * FAR + H * D, dtype=like.dtype, device="cuda").as_strided((T, H, D), (FAR, D, 1))
    t.copy_(like) if fill is None else t.fill_(fill)
    return t


@pytest.mark.parametrize("norm", [True, False])
def test_rotation_of_rows_far_apart(K, norm):
    T, Hq, Hkv, D = 6, 9, 2, 128
    q, k, _, table, pos, wq, wk = case("bf16", T, Hq, Hkv, D, 64, (norm, norm), seed=2)
    near = [torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (q, k)]
    K.qk_norm_rope(*near, q, k, table, pos, wq, wk)
    far = [far_rows(t, 7.0) for t in (q, k)]
    K.qk_norm_rope(*far, far_rows(q), far_rows(k), table, pos, wq, wk)
    assert all(torch.equal(a, b) for a, b in zip(near, far))
    gq, gk = (torch.randn(t.shape, device="cuda").to(t.dtype) for t in (q, k))
    dw = lambda: [torch.empty_like(w) if norm else None for w in (wq, wk)]
    dw0, dw1 = dw(), dw()
    K.qk_norm_rope_backward(*near, *dw0, gq, gk, q, k, table, pos, wq, wk)
    K.qk_norm_rope_backward(*far, *dw1, far_rows(gq), far_rows(gk), far_rows(q), far_rows(k), table, pos, wq, wk)
    assert all(torch.equal(a, b) for a, b in zip(near, far))
    assert not norm or all(torch.equal(a, b) for a, b in zip(dw0, dw1))


@pytest.mark.parametrize("P", [16, 20])
def test_places_far_apart(K, P):
    T, Hq, Hkv, D = 40, 4, 8, 128
    q, k, v, table, pos, _, _ = case("fp16", T, Hq, Hkv, D, 128, (False, False), seed=3)
    few = 2 * T // P + 1
    pages = 2 ** 31 // (P * Hkv * D) + few + 5
    slots = torch.randperm(few * P, generator=torch.Generator().manual_seed(1))[:T].cuda()
    small, large = ([torch.full((n, Hkv, P, D), 7.0, dtype=q.dtype, device="cuda") for _ in range(2)] for n in (few, pages))
    out = [torch.empty(q.shape, dtype=q.dtype, device="cuda") for _ in range(2)]
    K.qk_norm_rope(out[0], None, q, k, table, pos, v=v, k_cache=small[0], v_cache=small[1], slots=slots)
    K.qk_norm_rope(out[1], None, q, k, table, pos, v=v, k_cache=large[0], v_cache=large[1], slots=slots + (pages - few) * P)
    assert torch.equal(*out)
    for a, b in zip(small, large):
        assert torch.equal(a, b[-few:]) and bool((b[:few] == 7).all())


@pytest.mark.parametrize("P,D", [(20, 128), (7, 128), (8, 64), (5, 64)])
def test_odd_pages_far_apart(K, P, D):
    """Pages of four keys' multiples, of eight's with heads of 64, and of no load's: few rows, a chunk, a long one that is cut."""
    Hkv = 8
    small = batch("bf16", [(1, 300), (70, 100), (9, 3000)], 16, Hkv, D, P, seed=8)
    n = small["kc"].shape[0]
    pages = 2 ** 31 // (P * Hkv * D) + n + 5
    kc, vc = (torch.empty(pages, Hkv, P, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kc[-n:], vc[-n:] = small["kc"], small["vc"]
    table = torch.where(small["table"] >= 0, small["table"] + (pages - n), -1).contiguous()
    assert torch.equal(run(K, dict(small, kc=kc, vc=vc, table=table)), run(K, small))


def test_rows_of_attention_far_apart(K):
    b = batch("bf16", [(1, 900), (5, 30)], 8, 8, 128, 16, seed=9)  # few rows
    want = run(K, b)
    out = far_rows(b["q"], 7.0)
    assert torch.equal(run(K, dict(b, q=far_rows(b["q"])), out=out), want)
    b = batch("bf16", [(5, 900)], 32, 8, 128, 16, seed=9)  # tiles of many
    want = run(K, b)
    out = far_rows(b["q"], 7.0)
    assert torch.equal(run(K, dict(b, q=far_rows(b["q"])), out=out), want)


def test_pages_copied_far(K):
    """A pool of 45 pages of 2^26 elements: copies, a fork's last page, pages that move."""
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    N, P = 45, 8
    pool = torch.zeros(N, 2 ** 12, P, 2 ** 11, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    page = lambda: torch.randn(*pool.shape[1:], generator=g, device="cuda").to(pool.dtype)
    a, b = page(), page()
    pool[0], pool[44] = a, b
    K.kv_copy_pages(pool, ints([0, 44]), ints([43, 42]))
    assert torch.equal(pool[43], a) and torch.equal(pool[42], b) and torch.equal(pool[0], a) and torch.equal(pool[44], b)
    pool[42:44].zero_()
    # request 0 has pages 44 and 41, the last with three places filled; the lowest free page is 40
    pool[41] = a
    table, length, status = ints([[44, 41], [-1, -1]]), ints([P + 3, 0]), ints([0])
    refs = ints([1] * 40 + [0, 1, 0, 0, 1])
    K.kv_fork(pool, table, length, refs, ints([0]), ints([1]), status)
    assert table.tolist() == [[44, 41], [44, 40]] and length.tolist() == [P + 3, P + 3] and status.item() == 0
    assert torch.equal(pool[40, :, :3], a[:, :3]) and not bool(pool[40, :, 3:].any())
    # in use from here: 40, 41 and 44, which become 0, 1 and 2
    refs[:40] = 0
    K.kv_compact(pool, table, refs)
    moved = {40: 0, 41: 1, 44: 2}
    assert table.tolist() == [[moved[44], moved[41]], [moved[44], moved[40]]]
    assert refs.tolist() == [1, 1, 2] + [0] * 42
    assert torch.equal(pool[2], b) and torch.equal(pool[1], a) and torch.equal(pool[0, :, :3], a[:, :3])
