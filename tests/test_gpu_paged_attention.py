"""Attention over a paged cache against softmax in 64 bits.

Bound, elementwise, with u = eps / 2 of the element type: the result's own rounding, u |o|; the probabilities' rounding, at most u
each (of a 16-bit number, whose smallest step in fp16 is 2^-24: 2^-25 |v| a key more), so u sum p |v|; the scores' float
error: a dot product of D terms is off by D 2^-24 sum |q k|, which moves every p, and their sum, by that share of itself: twice that times
sum p |v|, with 2^-16 more for the exponential, the running rescaling and the sums over the keys (L 2^-24 at L up to 2^8 steps of a tile)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TDT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def K(gpu_device):
    from loquetier_amd import _lib
    from loquetier_amd.ops import _kernels
    _lib.load()
    return _kernels


def batch(dt, seqs, Hq, Hkv, D, P, nhd=False, seed=0, spare=3, before=0, after=0):
    """seqs: [(new, cached)]; `before` and `after`: rows of no sequence."""
    g = torch.Generator().manual_seed(seed)
    lens = [n + c for n, c in seqs]
    need = [-(-l // P) for l in lens]
    pool = sum(need) + spare
    perm = torch.randperm(pool, generator=g).tolist()
    M = max(need + [1])
    table, at = [], 0
    for n in need:
        table.append(perm[at:at + n] + [-1] * (M - n))
        at += n
    gd = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=gd, device="cuda").to(TDT[dt])
    shape = (pool, P, Hkv, D) if nhd else (pool, Hkv, P, D)
    kc, vc = mk(*shape), mk(*shape)
    if nhd:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    T = before + sum(n for n, _ in seqs) + after
    indptr = torch.tensor([before] + [n for n, _ in seqs]).cumsum(0).to(torch.int32).cuda()
    return dict(q=mk(T, Hq, D), kc=kc, vc=vc, table=torch.tensor(table, dtype=torch.int32).reshape(len(seqs), M).cuda(), indptr=indptr,
                lens=torch.tensor(lens, dtype=torch.int32).cuda(), T=T, P=P, Hq=Hq, Hkv=Hkv, D=D, seqs=seqs, before=before)


def run(K, b, fill=0.0, scale=None, requests=None, out=None):
    plan = K.AttentionPlan(b["indptr"], b["lens"], b["table"], b["T"], b["Hq"], b["Hkv"], b["P"], requests)
    out = torch.full_like(b["q"], fill) if out is None else out
    K.paged_attention(out, b["q"], b["kc"], b["vc"], plan, scale)
    return out


def expected(b, scale=None, rows=None):
    """(result, bound) in 64 bits by sequence."""
    Hq, Hkv, D, P = b["Hq"], b["Hkv"], b["D"], b["P"]
    g, scale = Hq // Hkv, scale or D ** -0.5
    dt = b["q"].dtype
    u = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    out, bound = (torch.zeros(b["T"], Hq, D, dtype=torch.float64, device="cuda") for _ in range(2))
    row, N = b["before"], b["kc"].shape[0]
    for i, (new, cached) in enumerate(b["seqs"]):
        L = int(b["lens"][i])
        if L > 0 and new > 0:
            tok = torch.arange(L, device="cuda")
            page = b["table"][i].long()[tok // P]
            bad = (page < 0) | (page >= N)
            page = page.clamp(0, N - 1)
            k, v = (c.transpose(1, 2)[page, tok % P].double().repeat_interleave(g, 1) for c in (b["kc"], b["vc"]))   # [L, Hq, D]
            last = L - new + torch.arange(new, device="cuda")
            off = (tok > last[:, None]) | bad
            for a in range(0, new, 256):
                q = b["q"][row + a:row + min(new, a + 256)].double()
                kt, o = k.permute(1, 2, 0).contiguous(), off[a:a + 256]
                s = (torch.matmul(q.transpose(0, 1), kt) * scale).masked_fill(o, -math.inf)
                size = (torch.matmul(q.abs().transpose(0, 1), kt.abs()) * scale).masked_fill(o, 0).amax(-1, keepdim=True)
                p = torch.softmax(s, -1).nan_to_num(0.0) if not bool(s.isnan().any()) else torch.softmax(s, -1)
                vt = v.transpose(0, 1)
                # a value that a row does not see has no part in it, whatever it is
                r = torch.matmul(p, vt.nan_to_num(0.0, 0.0, 0.0))
                pv = torch.matmul(p, vt.abs().nan_to_num(0.0, 0.0, 0.0))
                sees = (~o).double()
                odd = torch.matmul(sees, (~vt.isfinite()).double().contiguous()) > 0
                r = r.masked_fill(odd, math.nan)
                some = torch.matmul(sees, vt.abs().nan_to_num(0.0, 0.0, 0.0))
                e = u * r.abs() + (u + 2 * D * 2.0 ** -24 * size + 2.0 ** -16) * pv + tiny * (some + 1)
                out[row + a:row + min(new, a + 256)] = r.transpose(0, 1)
                bound[row + a:row + min(new, a + 256)] = e.transpose(0, 1)
        row += new
    return out, bound


def near(got, want, bound):
    bad = want.isnan()
    assert bool((~got[bad].isfinite()).all()) and bool(got[~bad].isfinite().all())
    err = (got.double() - want).abs()[~bad]
    assert bool((err <= bound[~bad] + 1e-12).all()), f"{float((err / bound[~bad].clamp(min=1e-12)).max())} times the bound"


BATCHES = {
    "one token": [(1, 0)],
    "decode": [(1, c) for c in (0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 500, 1033)],
    "long decode": [(1, 20000), (1, 3)],
    "short chunks": [(2, 0), (3, 50), (4, 129), (5, 0), (7, 200), (16, 16), (17, 1000)],
    "chunk": [(130, 0), (200, 77)],
    "long chunk": [(333, 2000)],
    "many splits of a chunk": [(40, 9000)],
    "mixed": [(64, 0), (1, 40), (129, 300), (1, 0), (0, 25), (2, 700), (1, 256)],
}


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D,P,nhd", [(8, 8, 128, 16, False), (8, 2, 128, 16, True), (8, 1, 64, 16, False), (6, 2, 64, 20, True),
                                            (5, 1, 128, 7, False), (32, 8, 128, 64, False), (2, 1, 128, 1, False), (3, 3, 64, 128, False), (64, 1, 64, 1000, True), (40, 1, 128, 8, False)])
@pytest.mark.parametrize("name", BATCHES)
def test_batches(K, dt, Hq, Hkv, D, P, nhd, name):
    b = batch(dt, BATCHES[name], Hq, Hkv, D, P, nhd)
    near(run(K, b), *expected(b))


@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (8, 1)])
def test_rows_of_no_sequence_are_left_alone(K, Hq, Hkv):
    b = batch("bf16", [(1, 30), (0, 4), (50, 9)], Hq, Hkv, 128, 16, before=3, after=5)
    out = run(K, b, fill=7.0)
    want, bound = expected(b)
    near(out[3:-5], want[3:-5], bound[3:-5])
    assert bool((out[:3] == 7).all()) and bool((out[-5:] == 7).all())


@pytest.mark.parametrize("new", [1, 3, 200])
def test_rows_that_see_no_token(K, new):
    """A length below the rows' number: the first rows see nothing and are zero; a length of zero: all of them."""
    b = batch("fp16", [(new, 4), (new, 10), (1, 0)], 8, 2, 64, 16)
    b["lens"][0] = 0
    b["lens"][1] = new - 1
    b["seqs"] = [(new, -new), (new, -1), (1, 0)]
    out = run(K, b, fill=3.0)
    near(out, *expected(b))
    assert not bool(out[:new].any()) and not bool(out[new].any())


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("seqs", [[(1, 37), (1, 200)], [(5, 44), (3, 0)], [(200, 100)], [(150, 0), (1, 77)]])
def test_odd_values_where_nothing_looks(K, dt, seqs):
    """NaN and infinities in free pages, in places past a sequence's end, and in tokens that only later rows see."""
    for value in (math.nan, math.inf, -math.inf):
        b = batch(dt, seqs, 4, 2, 128, 16, seed=3)
        want, bound = expected(b)
        used = torch.zeros(b["kc"].shape[0], 16, dtype=torch.bool, device="cuda")
        for i, (n, c) in enumerate(seqs):
            tok = torch.arange(n + c, device="cuda")
            used[b["table"][i].long()[tok // 16], tok % 16] = True
        for cache in (b["kc"], b["vc"]):
            cache.transpose(1, 2)[~used] = value
        near(run(K, b), want, bound)
        # the value of a token in the middle of the new ones: only rows from it on see it
        n, c = max(seqs)
        if n > 1:
            i = seqs.index((n, c))
            t = c + n // 2
            page = int(b["table"][i][t // 16])
            b["vc"][page, 1, t % 16, 5] = value
            want, bound = expected(b)
            out = run(K, b)
            row = sum(m for m, _ in seqs[:i])
            assert bool(want[row + n // 2, 2, 5].isnan()) and not bool(want[row:row + n // 2].isnan().any())
            near(out, want, bound)
            b["kc"][page, 1, t % 16, 5] = math.nan  # and its key: those rows are lost, the ones before are not
            out = run(K, b)
            near(out[row:row + n // 2], want[row:row + n // 2], bound[row:row + n // 2])
            assert bool(out[row + n // 2:row + n, 2:].isnan().all())


@pytest.mark.parametrize("new", [1, 6, 140])
def test_pages_the_pool_does_not_hold(K, new):
    b = batch("bf16", [(new, 300), (new, 90)], 4, 1, 64, 16)
    b["table"][0, 3], b["table"][0, 7], b["table"][1, 0] = -1, b["kc"].shape[0], 2 ** 30
    near(run(K, b), *expected(b))


def test_lengths_past_the_table(K):
    b = batch("fp16", [(1, 31), (4, 60)], 4, 4, 64, 16)
    b["lens"][1] = 10 ** 9  # only what the table holds counts
    b2 = dict(b, lens=torch.tensor([32, 64], dtype=torch.int32).cuda())
    assert torch.equal(run(K, b), run(K, b2))


def test_requests_name_rows_of_the_table(K):
    b = batch("bf16", [(1, 100), (30, 40), (2, 2)], 8, 2, 128, 16)
    want = run(K, b)
    order = torch.tensor([4, 0, 2], dtype=torch.int32).cuda()
    table = torch.full((5, b["table"].shape[1]), -1, dtype=torch.int32, device="cuda")
    table[order.long()] = b["table"]
    assert torch.equal(run(K, dict(b, table=table), requests=order), want)
    # a request that the table does not hold sees nothing
    order = order.clone()
    order[1] = 5
    out = run(K, dict(b, table=table), requests=order)
    assert not bool(out[1:31].any()) and torch.equal(out[0], want[0]) and torch.equal(out[31:], want[31:])


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_large_scores_and_scale(K, dt):
    """Scores of hundreds, rising and falling over the keys, and another scale."""
    b = batch(dt, [(1, 700), (100, 400), (3, 1500)], 8, 2, 128, 16, seed=5)
    b["kc"].mul_(6.0)
    near(run(K, b), *expected(b))
    near(run(K, b, scale=0.01), *expected(b, 0.01))


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("new", [1, 9, 150])
def test_many_small_weights(K, dt, new):
    """One token of great weight and thousands whose weights, 2^-15 of it each, come to as much together: they count, and so does
    their sum."""
    b = batch(dt, [(new, 50000)], 4, 1, 64, 16, seed=6)
    b["q"].zero_()
    b["q"][..., 0] = 8.0
    b["kc"].zero_()
    b["vc"].copy_(torch.where(b["vc"] > 0, 1.0, 0.5))
    page, at = int(b["table"][0, 700]), 5
    b["kc"][page, 0, at, 0] = 8.0
    b["vc"][page, 0, at] = 4.0
    scale = 15 * math.log(2) / 64
    want, bound = expected(b, scale)
    assert 1.5 < float(want[0, 0, 0]) < 3.5  # (neither the one nor the others alone)
    near(run(K, b, scale=scale), want, bound)


def test_strided_tensors(K):
    b = batch("bf16", [(1, 70), (60, 30)], 4, 2, 64, 16)
    want = run(K, b)
    wide = torch.zeros(b["T"], 8, 72, dtype=torch.bfloat16, device="cuda")
    wide[:, ::2, :64] = b["q"]
    out = torch.zeros(b["T"], 6, 64, dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros(b["kc"].shape[0], 3, 2, 2, 16, 64, dtype=torch.bfloat16, device="cuda")  # a layer of several
    pool[:, 1, 0], pool[:, 1, 1] = b["kc"], b["vc"]
    c = dict(b, q=wide[:, ::2, :64], kc=pool[:, 1, 0], vc=pool[:, 1, 1])
    assert torch.equal(run(K, c, out=out[:, 1:5]), want) and not bool(out[:, 0].any()) and not bool(out[:, 5].any())


def test_far_offsets(K):
    """Pages past 2^31 elements of the pool."""
    P, Hkv, D = 64, 8, 128
    pages = 2 ** 31 // (P * Hkv * D) + 40
    kc, vc = (torch.empty(pages, Hkv, P, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    small = batch("bf16", [(1, 300), (70, 100)], 16, Hkv, D, P, seed=8)
    n = small["kc"].shape[0]
    kc[-n:], vc[-n:] = small["kc"], small["vc"]
    table = torch.where(small["table"] >= 0, small["table"] + (pages - n), -1).contiguous()
    assert torch.equal(run(K, dict(small, kc=kc, vc=vc, table=table)), run(K, small))


def test_same_bits_again(K):
    b = batch("fp16", [(1, 5000)] * 3 + [(300, 4000)], 8, 2, 128, 16)
    first = run(K, b)
    for _ in range(3):
        assert torch.equal(run(K, b), first)


def test_in_place(K):
    for seqs in ([(1, 9000)] * 2, [(1, 50), (300, 2000), (20, 7), (3, 0)]):
        b = batch("bf16", seqs, 8, 2, 128, 16, seed=11)
        want = run(K, b)
        q = b["q"].clone()
        assert torch.equal(run(K, dict(b, q=q), out=q), want)


@pytest.mark.parametrize("g", [1, 4])
def test_more_sequences_than_the_plan_keeps_in_lds(K, g):
    import random
    r = random.Random(g)
    seqs = [(r.choice([0, 1, 1, 1, 2, 5, 40]), r.choice([0, 1, 30, 200, 900])) for _ in range(1500)]
    b = batch("fp16", seqs, g, 1, 64, 16, seed=12)
    near(run(K, b), *expected(b))


@pytest.mark.parametrize("count,Hkv", [(300, 2), (1300, 1)])
def test_more_chunks_than_the_card_takes_at_a_time(K, count, Hkv):
    """The plan then sorts them by length, in LDS and past it: lengths of nothing and of one key among them, some single tokens."""
    import random
    r = random.Random(count)
    seqs = [(r.choice([9, 20, 33, 70]), r.choice([0, 0, 1, 40, 300, 900])) for _ in range(count)] + [(1, 5), (1, 400)] * 10
    r.shuffle(seqs)
    b = batch("bf16", seqs, 4 * Hkv, Hkv, 64, 16, seed=24)
    for i in range(0, len(seqs), 50):
        b["lens"][i] = i // 50 % 3  # shorter than its rows
    near(run(K, b), *expected(b))


def test_a_plan_for_another_table_does_nothing(K):
    b = batch("bf16", [(1, 400), (200, 500)], 4, 2, 64, 16)
    plan = K.AttentionPlan(b["indptr"], b["lens"], b["table"], b["T"], 4, 2, 16)
    plan.page_table = b["table"][:, :3].contiguous()
    out = torch.full_like(b["q"], 5.0)
    K.paged_attention(out, b["q"], b["kc"], b["vc"], plan)
    assert bool((out == 5).all())


@pytest.mark.parametrize("T,S,heads", [(120, 2, (4, 2)), (201, 1, (4, 2)), (201, 2, (4, 1)), (201, 2, (2, 1))])
def test_a_plan_for_other_sizes_does_nothing(K, T, S, heads):
    b = batch("bf16", [(1, 400), (200, 500)], 4, 2, 64, 16)
    plan = K.AttentionPlan(b["indptr"], b["lens"], b["table"], b["T"], 4, 2, 16)
    plan.T, plan.S, (plan.q_heads, plan.kv_heads) = T, S, heads
    q, (kc, vc) = b["q"][:T, :heads[0]], (c[:, :heads[1]] for c in (b["kc"], b["vc"]))
    out = torch.full_like(b["q"], 5.0)
    if heads[1] == 1:  # (one kv head's tiles are cut into more items than two's: the host knows that the plan is too small)
        with pytest.raises(RuntimeError):
            K.paged_attention(out[:T, :heads[0]], q, kc, vc, plan)
    else:
        K.paged_attention(out[:T, :heads[0]], q, kc, vc, plan)
    assert bool((out == 5).all())


def test_sequences_that_overlap_stay_in_bounds(K):
    """Row ranges that decrease, overlap or leave the batch break the contract; what is written stays within the batch's rows."""
    b = batch("bf16", [(1, 400), (200, 2500), (1, 3)], 4, 2, 64, 16, after=3)
    for indptr in ([0, 190, 10, 204], [0, 204, 0, 204], [-5, 300, 9, 400], [204, 1, 204, 0]):
        out = torch.full((b["T"] + 2, 4, 64), 9.0, dtype=torch.bfloat16, device="cuda")
        c = dict(b, indptr=torch.tensor(indptr, dtype=torch.int32).cuda())
        run(K, c, out=out[1:-1])
        assert bool((out[0] == 9).all()) and bool((out[-1] == 9).all())


@pytest.mark.parametrize("P,D", [(16, 128), (48, 64), (20, 128), (8, 64), (7, 128)])
def test_ends_of_tiles_and_pages(K, P, D):
    """Lengths around tiles of 64 keys and pairs of them, for chunks of some rows and many, no number in any other place of the pool."""
    seqs = [(n, length - n) for length in (40, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 320) for n in (9, 40)]
    b = batch("bf16", seqs, 4, 2, D, P, seed=21)
    want, bound = expected(b)
    used = torch.zeros(b["kc"].shape[0], P, dtype=torch.bool, device="cuda")
    for i, (n, c) in enumerate(seqs):
        tok = torch.arange(n + c, device="cuda")
        used[b["table"][i].long()[tok // P], tok % P] = True
    for cache in (b["kc"], b["vc"]):
        cache.transpose(1, 2)[~used] = math.nan
    near(run(K, b), want, bound)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (8, 2), (6, 2)])
def test_tile_rows_around_the_paths(K, dt, Hq, Hkv):
    """Rows of a kv head up to 16 and past it, up to 128 and past it, over lengths that are cut into few parts and many."""
    g = Hq // Hkv
    news = sorted({max(1, n // g + d) for n in (16, 32, 128) for d in (0, 1)})
    near(*((lambda b: (run(K, b), *expected(b)))(batch(dt, [(n, c) for n in news for c in (0, 70, 600)], Hq, Hkv, 64, 16, seed=22))))
    for n in news[:3]:
        b = batch(dt, [(n, 17000)], Hq, Hkv, 64, 16, seed=23)
        near(run(K, b), *expected(b))


def test_empty_batches(K):
    b = batch("bf16", [(0, 5), (0, 0)], 4, 2, 64, 16, after=4)
    assert bool((run(K, b, fill=2.0) == 2).all())
    b = batch("bf16", [(1, 4)], 4, 2, 64, 16)
    none = dict(b, kc=b["kc"][:0], vc=b["vc"][:0])
    assert not bool(run(K, none, fill=2.0).any())
    q0 = dict(b, q=b["q"][:0], T=0, indptr=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert run(K, q0).shape == (0, 4, 64)
