"""What a cache does not take: requests past `max_tokens`, which need not fill a last page."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from loquetier_amd import _lib
    from loquetier_amd.ops import _kernels
    _lib.load()
    return _kernels


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch, K):
    from loquetier_amd import _lib
    if request.param == "python":
        monkeypatch.setattr(K, "_host", lambda: _lib._NoHost)


def state(c):
    return [t.clone() for t in (c.pool, c.table, c.length, c.refs)]


def test_one_token_past_max_tokens(K, path):
    """20 tokens in pages of 16: the 21st has a place in the second page, and a rotation table of 20 positions no angle for it."""
    from loquetier_amd.kvcache import PagedKvCache
    c = PagedKvCache(9, 1, 2, 64, 4, 20, 16)
    table = K.rope_table(20, 64, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)

    def step(requests, counts):
        s = c.extend(requests, counts)
        x = torch.randn(sum(counts), 8, 64, generator=g, device="cuda").to(torch.bfloat16)
        return c.attend(0, x[:, :4], x[:, 4:6], x[:, 6:], s, c.plan(s, 4), table)

    assert bool(step([0, 1], [19, 20]).isfinite().all())
    assert bool(step([0], [1]).isfinite().all())
    c.check()
    before = state(c)
    for requests, counts in (([0], [1]), ([2, 1], [3, 1]), ([3], [21])):
        out = step(requests, counts)
        assert not bool(out.any()) and all(torch.equal(a, b) for a, b in zip(before, state(c)))
        with pytest.raises(RuntimeError, match="longer than max_tokens"):
            c.check()
    c.fork([0], [2])  # a fork is as long as what it is forked from
    c.check()
    step([2], [1])
    with pytest.raises(RuntimeError, match="longer than max_tokens"):
        c.check()
    assert bool(c.pool.isfinite().all()) and c.length.tolist() == [20, 20, 20, 0]


@pytest.mark.parametrize("S,rows", [(3, 40), (900, 6000), (1100, 1200)])
def test_limit_by_size_of_the_step(K, path, S, rows):
    """Steps of few rows, of few sequences, of more: the last token that fits and the one past it; without a limit, the table's width."""
    from loquetier_amd import _lib
    P, M, most = 4, 3, 10
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, length, refs = torch.full((S, M), -1, dtype=torch.int32, device="cuda"), ints([0] * S), ints([0] * (3 * S))
    status = ints([0])
    req = ints(list(range(S)))
    step = lambda counts, **kw: K.kv_extend(table, length, refs, req, ints(counts), rows, P, status, **kw)
    full = [most if i in (1, S - 1) else 0 for i in range(S)]
    assert step(full, max_tokens=most)[1].tolist() == full and status.item() == 0
    before = [t.clone() for t in (table, length, refs)]
    for i in (1, S - 1):
        got = step([int(j == i) for j in range(S)], max_tokens=most)
        assert not any(bool(t.any()) for t in got[:2]) and bool((got[3] == -1).all())
        assert status.item() == _lib.SMLM_KV_TOO_LONG
        status.zero_()
    assert all(torch.equal(a, b) for a, b in zip(before, (table, length, refs)))
    one = [int(j == 1) for j in range(S)]
    for _ in range(2):  # the table has places for two more
        step(one)
    step(one, max_tokens=10 ** 12)
    assert status.item() == _lib.SMLM_KV_TOO_LONG and length[1].item() == P * M
    with pytest.raises(RuntimeError, match="max_tokens"):
        step(one, max_tokens=-1)
