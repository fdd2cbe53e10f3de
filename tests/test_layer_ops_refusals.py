"""What the operators between the projections refuse, through the C ABI, before any launch (no GPU needed: made-up addresses
are never read), and from Python for tensors that are not on a GPU."""
import ctypes as C

import pytest
import torch

from loquetier_amd import _lib as lib

ARG, DTYPE, ALIGN, WORKSPACE, LIMIT = -1, -2, -3, -4, -6
A = 1 << 20  # an aligned address


@pytest.fixture(scope="module")
def L():
    return lib.load()


def rope(**kw):
    heads = lambda **h: lib.Heads(**{**dict(data=A, row_stride=512, head_stride=128), **h})
    a = lib.QkRope(q=heads(), k=heads(), v=heads(), q_out=heads(), k_out=heads(), table=A, positions=A, rows=4, q_heads=4, kv_heads=4,
                   head_dim=128, rot_dim=128, table_rows=10, dtype=0, eps=1e-6, page_size=16, n_pages=4)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), ARG), (dict(q_heads=0), ARG), (dict(kv_heads=0), ARG), (dict(head_dim=0), ARG), (dict(rot_dim=144), ARG),
    (dict(head_dim=120, rot_dim=64), ALIGN), (dict(rot_dim=24), ALIGN), (dict(head_dim=528), LIMIT), (dict(dtype=7), DTYPE),
    (dict(table=0), ARG), (dict(positions=0), ARG), (dict(table=A + 4), ALIGN), (dict(q_weight=A + 2), ALIGN),
    (dict(q=lib.Heads()), ARG), (dict(k_out=lib.Heads()), ARG), (dict(q=lib.Heads(A + 2, 512, 128)), ALIGN),
    (dict(k=lib.Heads(A, 510, 128)), ALIGN), (dict(q_out=lib.Heads(A, 512, 130)), ALIGN), (dict(k_cache=A), ARG),
    (dict(k_cache=A, v_cache=A), ARG), (dict(k_cache=A, v_cache=A, slots=A, page_size=0), ARG),
    (dict(k_cache=A, v_cache=A, slots=A, v=lib.Heads()), ARG), (dict(k_cache=A, v_cache=A, slots=A, slot_stride=4), ALIGN),
    (dict(k_cache=A, v_cache=A, slots=A, n_pages=1 << 28), LIMIT)])
def test_rope(L, change, code):
    assert L.smlm_qk_norm_rope_fwd(C.byref(rope(**change)), None) == code


def test_rope_backward(L):
    h = C.byref(lib.Heads(A, 512, 128))
    assert L.smlm_qk_norm_rope_fwd(None, None) == ARG
    assert L.smlm_qk_norm_rope_bwd(C.byref(rope()), h, None, h, h, None, None, None, 0, None) == ARG
    assert L.smlm_qk_norm_rope_bwd(C.byref(rope(q_weight=A)), h, h, h, h, A, None, None, 0, None) == ARG      # no workspace
    assert L.smlm_qk_norm_rope_bwd(C.byref(rope(q_weight=A)), h, h, h, h, A, None, A, 8, None) == WORKSPACE
    assert L.smlm_qk_norm_rope_bwd(C.byref(rope(q_weight=A)), h, h, h, h, None, None, A, 1 << 20, None) == ARG  # no gradient
    assert L.smlm_qk_norm_rope_bwd(C.byref(rope(q_weight=A, rows=0)), h, h, h, h, A, None, A, 1 << 20, None) == ARG
    odd = C.byref(lib.Heads(A, 512, 4))
    assert L.smlm_qk_norm_rope_bwd(C.byref(rope()), h, h, odd, h, None, None, None, 0, None) == ALIGN
    n = C.c_size_t()
    assert L.smlm_qk_norm_rope_bwd_workspace_size(4, 4, 4, 1024, C.byref(n)) == LIMIT
    assert L.smlm_qk_norm_rope_bwd_workspace_size(-1, 4, 4, 128, C.byref(n)) == ARG


def test_pages(L):
    n = C.c_size_t()
    assert L.smlm_kv_workspace_size(4, -1, 3, C.byref(n)) == ARG
    assert L.smlm_kv_workspace_size(4, 10, 3, C.byref(n)) == 0
    ext = lambda ws=A, size=n.value, R=4, M=4, N=10, S=3, rows=5, P=16, req=A: L.smlm_kv_extend(
        A, A, A, req, A, A, A, A, A, ws, size, R, M, N, S, rows, P, None, None)
    assert ext(P=0) == ARG and ext(rows=-1) == ARG and ext(req=None) == ARG and ext(ws=None) == ARG
    assert ext(size=16) == WORKSPACE and ext(ws=A + 8) == ALIGN
    assert ext(N=1 << 28) == LIMIT and ext(M=1 << 21) == LIMIT and ext(rows=(1 << 20) + 1) == LIMIT
    assert L.smlm_kv_free(A, A, A, None, 4, 4, 10, 3, 16, None, None) == ARG
    assert L.smlm_kv_free(A, A, A, A, 4, 4, 10, 3, 0, None, None) == ARG
    fork = lambda pool=A, blocks=2, place=256, ws=A, size=n.value, par=A: L.smlm_kv_fork(
        pool, A, A, A, par, A, ws, size, 4, 4, 10, 3, blocks, 16, place, None, None)
    assert fork(pool=A + 8) == ALIGN and fork(place=24) == ALIGN and fork(blocks=0) == ARG and fork(par=None) == ARG
    assert fork(size=16) == WORKSPACE and fork(pool=None) == ARG and fork(place=1 << 27) == LIMIT
    assert L.smlm_kv_compact(A, A, A, A, 16, 4, 4, 10, 2, 16, 256, None) == WORKSPACE
    assert L.smlm_kv_compact(A, None, A, A, n.value, 4, 4, 10, 2, 16, 256, None) == ARG
    assert L.smlm_kv_copy_pages(A, A, None, 3, 10, 2, 16, 256, None) == ARG
    assert L.smlm_kv_copy_pages(A, A, A, -3, 10, 2, 16, 256, None) == ARG


def test_attention(L):
    n, w = C.c_size_t(), C.c_size_t()
    assert L.smlm_attn_plan_size(10, 3, 8, 3, C.byref(n)) == ARG       # heads that do not divide
    assert L.smlm_attn_plan_size(1 << 28, 3, 8, 2, C.byref(n)) == LIMIT
    assert L.smlm_attn_plan_size(10, 3, 8, 2, C.byref(n)) == 0
    assert L.smlm_paged_attn_workspace_size(10, 3, 100, 16, 8, 2, 128, C.byref(w)) == 0 and w.value > 0
    build = lambda plan=A, size=n.value, indptr=A, S=3, P=16, M=100: L.smlm_attn_plan_build(plan, size, indptr, A, None, 10, S, 3, M, P, 8, 2, None)
    assert build(plan=None) == ARG and build(size=8) == WORKSPACE and build(indptr=None) == ARG and build(plan=A + 4) == ALIGN
    assert build(P=0) == ARG and build(M=1 << 19, P=1 << 13) == LIMIT
    h = lib.Heads(A, 1024, 128)

    def attn(out=h, q=h, k=A, page=8192, plan=A, plan_size=n.value, ws=A, size=w.value, pages=9, P=16, hd=128, dtype=0, scale=0.1, T=10):
        return L.smlm_paged_attn(C.byref(out), C.byref(q), k, A, page, 4096, 128, A, plan, plan_size, ws, size, T, 3, 3, 100, pages, P, 8, 2,
                                 hd, dtype, scale, None)
    assert attn(hd=96) == LIMIT and attn(dtype=3) == DTYPE and attn(scale=0.0) == ARG and attn(scale=-1.0) == ARG
    assert attn(scale=float("nan")) == ARG and attn(scale=float("inf")) == ARG and attn(pages=-1) == ARG and attn(P=0) == ARG
    assert attn(plan=None) == ARG and attn(plan_size=8) == WORKSPACE and attn(ws=None) == ARG and attn(size=8) == WORKSPACE
    assert attn(out=lib.Heads()) == ARG and attn(q=lib.Heads(A, 1024, 4)) == ALIGN and attn(page=4) == ALIGN and attn(k=A + 8) == ALIGN
    assert attn(T=0) == 0  # nothing to do


def test_python_surface_wants_gpu_tensors():
    from loquetier_amd.kernel_utils import qk_norm_rope
    from loquetier_amd.ops import _kernels as K
    x, i = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    table = K.rope_table(5, 64)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        K.qk_norm_rope(x, x, x, x, table, i)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        qk_norm_rope.apply(x, x, None, None, table, i)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        K.AttentionPlan(i, i[:1], torch.zeros(1, 1, dtype=torch.int32), 2, 4, 4, 16)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        K.kv_free(torch.zeros(1, 1, dtype=torch.int32), i[:1], i, i, 16)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        K.kv_copy_pages(torch.zeros(2, 2, 16, 64), i, i)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        K.rope_table(5, 24)
    with pytest.raises(RuntimeError, match="entries"):
        K.rope_table(5, 64, inv_freq=torch.ones(3))


def test_division_by_the_page_size():
    """The constants that the kernel divides by: exact for every page size and any token a table can hold."""
    import random
    r = random.Random(0)
    for P in list(range(1, 300)) + [2 ** 20 - 1, 2 ** 20, 2 ** 20 + 1, 2 ** 31 - 1]:
        s = (P - 1).bit_length()
        m = ((1 << 32) * ((1 << s) - P)) // P + 1
        assert m < 1 << 32
        for x in [0, 1, P - 1, P, P + 1, 2 * P - 1, 2 ** 31 - 1] + [r.randrange(2 ** 31) for _ in range(20)]:
            assert (((x * m) >> 32) + x) >> s == x // P


def test_extend_with_a_limit(L):
    n = C.c_size_t()
    assert L.smlm_kv_workspace_size(4, 10, 3, C.byref(n)) == 0
    ext = lambda most=9, ws=A, size=n.value, P=16: L.smlm_kv_extend_upto(
        A, A, A, A, A, A, A, A, A, ws, size, 4, 4, 10, 3, 5, P, most, None, None)
    assert ext(most=-1) == ARG and ext(P=0) == ARG and ext(ws=None) == ARG and ext(size=16) == WORKSPACE


@pytest.mark.parametrize("dim,dtype", [(96, torch.bfloat16), (256, torch.float16), (0, torch.bfloat16), (128, torch.float32), (64, torch.int8)])
def test_a_cache_that_attention_cannot_read(dim, dtype):
    """Refused when it is made, not when its pages have been written."""
    from loquetier_amd.kvcache import PagedKvCache
    with pytest.raises(RuntimeError, match="No suitable kernel"):
        PagedKvCache(2, 1, 1, dim, 1, 16, dtype=dtype, device="cpu")


def test_a_cache_that_it_can_read():
    from loquetier_amd.kvcache import PagedKvCache
    for dim, dtype in ((64, torch.float16), (128, torch.bfloat16)):
        assert PagedKvCache(2, 1, 1, dim, 1, 16, dtype=dtype, device="cpu").pool.shape == (2, 1, 2, 1, 16, dim)
