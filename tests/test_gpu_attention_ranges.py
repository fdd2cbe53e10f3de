"""Row ranges that break the contract of the attention's plan: a q_indptr that decreases, with so many sequences that their tiles come to more
than the plan has room for.  The plan holds nothing then, and a call with it writes nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from loquetier_amd import _lib
    from loquetier_amd.ops import _kernels
    _lib.load()
    return _kernels


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def attend(K, indptr, lens, T, Hkv, most):
    q = torch.randn(T, Hkv, 64, device="cuda").bfloat16()
    k, v = (torch.randn(4, Hkv, 16, 64, device="cuda").bfloat16() for _ in range(2))
    table = torch.zeros(len(lens), most // 16, dtype=torch.int32, device="cuda")
    plan = K.AttentionPlan(ints(indptr), ints(lens), table, T, Hkv, Hkv, 16)
    out = torch.full_like(q, 9.0)
    K.paged_attention(out, q, k, v, plan)
    return out, plan.buf[:8].view(torch.int32).tolist()


@pytest.mark.parametrize("S", [200, 1500])
@pytest.mark.parametrize("long", [64, 100000])
def test_ranges_that_go_back_and_forth(K, S, long):
    T = 4096
    indptr = [0 if i % 2 == 0 else T for i in range(S)] + [0, T]
    out, head = attend(K, indptr, [64] * S + [long], T, 8, 100000)
    assert head == [0, 0]  # no items, no joins: nothing left to read that was not written
    assert bool((out == 9).all())


@pytest.mark.parametrize("indptr", [[0, 190, 10, 204], [0, 204, 0, 204], [-5, 300, 9, 400], [204, 1, 204, 0], [0, 1, 0, 0]])
def test_one_step_back(K, indptr):
    out, head = attend(K, indptr, [400, 2500, 3], 204, 2, 2560)
    assert head == [0, 0] and bool((out == 9).all())


def test_ranges_past_the_batch(K):
    """Ranges that only grow past the rows are cut at the last one."""
    out, head = attend(K, [-3, 2, 150, 300, 500], [5, 900, 900, 7], 204, 2, 1024)
    assert head[0] > 0 and bool(out.isfinite().all()) and not bool((out == 9).all(-1).any())
