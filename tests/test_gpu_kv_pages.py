"""Pages of a cache on the device against the same rules in Python lists.  Whole numbers and copies: equal."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from loquetier_amd import _lib
    from loquetier_amd.ops import _kernels
    _lib.load()
    return _kernels


class Model:
    """The rules, one request at a time; the pool as a list of [blocks][place] values."""

    def __init__(self, n_pages, blocks, page_size, requests, width, fill):
        self.P, self.M = page_size, width
        self.table = [[-1] * width for _ in range(requests)]
        self.length, self.refs = [0] * requests, [0] * n_pages
        self.pool, self.blocks = [[[fill(n, b, p) for p in range(page_size)] for b in range(blocks)] for n in range(n_pages)], blocks
        self.status = 0

    def pages(self, n):
        return -(-n // self.P)

    def free_pages(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def extend(self, requests, counts, rows):
        err, seen = 0, set()
        need = 0
        for r, n in zip(requests, counts):
            if r < 0:
                continue
            if r >= len(self.table) or n < 0 or r in seen:
                err |= 1
                continue
            seen.add(r)
            if self.pages(self.length[r] + n) > self.M:
                err |= 2
            need += self.pages(self.length[r] + n) - self.pages(self.length[r])
        if sum(n for r, n in zip(requests, counts) if r >= 0) > rows:
            err |= 4
        if not err and need > len(self.free_pages()):
            err |= 8
        if err:
            self.status |= err
            return [0] * (len(requests) + 1), [0] * len(requests), [-1] * rows, [-1] * rows
        indptr, lens, pos, slots, free = [0], [], [], [], self.free_pages()
        for r, n in zip(requests, counts):
            if r < 0:
                indptr.append(indptr[-1]), lens.append(0)
                continue
            for t in range(self.length[r], self.length[r] + n):
                if t % self.P == 0:
                    self.table[r][t // self.P] = free.pop(0)
                    self.refs[self.table[r][t // self.P]] = 1
                pos.append(t), slots.append(self.table[r][t // self.P] * self.P + t % self.P)
            self.length[r] += n
            indptr.append(indptr[-1] + n), lens.append(self.length[r])
        return indptr, lens, pos + [-1] * (rows - len(pos)), slots + [-1] * (rows - len(slots))

    def fork(self, parents, children):
        err, seen, need = 0, set(), 0
        for p, c in zip(parents, children):
            if c < 0:
                continue
            if not 0 <= p < len(self.table) or c >= len(self.table) or c in seen or self.length[c]:
                err |= 1
                continue
            seen.add(c)
            need += self.length[p] % self.P != 0
        if not err and need > len(self.free_pages()):
            err |= 8
        self.status |= err
        if err:
            return
        free, length = self.free_pages(), list(self.length)  # (a parent counts as it was before the call, an empty child too)
        for p, c in zip(parents, children):
            if c < 0:
                continue
            n = length[p]
            for i in range(n // self.P):
                self.table[c][i] = self.table[p][i]
                self.refs[self.table[p][i]] += 1
            if n % self.P:
                new, old = free.pop(0), self.table[p][n // self.P]
                self.table[c][n // self.P], self.refs[new] = new, 1
                for b in range(self.blocks):
                    self.pool[new][b][:n % self.P] = self.pool[old][b][:n % self.P]
            self.length[c] = n

    def free(self, requests):
        for r in requests:
            if r >= len(self.table):
                self.status |= 1
            elif r >= 0:
                for i in range(self.pages(self.length[r])):
                    self.refs[self.table[r][i]] -= 1
                    self.table[r][i] = -1
                self.length[r] = 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [i for i in range(live) if self.refs[i] == 0]
        moved = {}
        for i in range(live, len(self.refs)):
            if self.refs[i] > 0:
                to = holes.pop(0)
                moved[i] = to
                self.pool[to] = [list(b) for b in self.pool[i]]
                self.refs[to], self.refs[i] = self.refs[i], 0
        self.table = [[moved.get(i, i) for i in row] for row in self.table]


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


class Device:
    """The tensors of the same state; a place is 8 values of fp16, all the model's."""

    def __init__(self, m, K):
        self.K, self.P = K, m.P
        self.pool = torch.tensor(m.pool, dtype=torch.float16).cuda()[..., None].expand(-1, -1, -1, 8).contiguous()
        self.table, self.length, self.refs, self.status = ints(m.table), ints(m.length), ints(m.refs), ints([0])

    def same(self, m):
        assert self.table.tolist() == m.table and self.length.tolist() == m.length and self.refs.tolist() == m.refs
        assert self.status.item() == m.status
        assert torch.equal(self.pool, torch.tensor(m.pool, dtype=torch.float16).cuda()[..., None].expand(-1, -1, -1, 8))


def both(K, n_pages=40, blocks=3, P=4, requests=12, width=9):
    m = Model(n_pages, blocks, P, requests, width, lambda n, b, p: (n * 131 + b * 17 + p) % 2000)
    return m, Device(m, K)


def do_extend(m, d, req, counts, rows):
    want = m.extend(req, counts, rows)
    got = d.K.kv_extend(d.table, d.length, d.refs, ints(req), ints(counts), rows, d.P, d.status)
    assert [t.tolist() for t in got] == [list(w) for w in want]
    d.same(m)


@pytest.mark.parametrize("P,seed", [(4, 0), (1, 1), (7, 2), (16, 3), (4, 4), (5, 5)])
def test_lives_of_pages(K, P, seed):
    r = random.Random(seed)
    m, d = both(K, n_pages=r.choice([17, 40, 90]), P=P, requests=r.choice([3, 12, 30]), width=9)
    R = len(m.table)
    for _ in range(25):
        op = r.choice(["extend", "extend", "extend", "fork", "fork", "free", "free", "compact"])
        some = r.sample(range(R), r.randint(1, R)) + [-1] * r.randint(0, 2)
        r.shuffle(some)
        if op == "extend":
            counts = [r.choice([0, 1, 1, r.randint(0, 3 * P)]) for _ in some]
            do_extend(m, d, some, counts, max(0, sum(c for q, c in zip(some, counts) if q >= 0) + r.choice([0, 0, 5, -1])))
            continue
        if op == "fork":
            empty = [i for i in range(R) if m.length[i] == 0] or [0]
            children = r.sample(empty, r.randint(1, len(empty)))
            parents = [r.randrange(R) for _ in children]
            m.fork(parents, children)
            K.kv_fork(d.pool, d.table, d.length, d.refs, ints(parents), ints(children), d.status)
        elif op == "free":
            names = some[:3] + some[:1] + ([R + 4] if r.random() < 0.2 else [])  # one named twice, one unknown
            m.free(names)
            K.kv_free(d.table, d.length, d.refs, ints(names), d.P, d.status)
        else:
            m.compact()
            K.kv_compact(d.pool, d.table, d.refs)
        d.same(m)


def test_refused_whole(K):
    """What cannot be done in full changes nothing: tables, pages and lengths stay, the status says why."""
    m, d = both(K, n_pages=8, P=4, requests=6, width=4)
    do_extend(m, d, [0, 1], [9, 5], 14)
    for req, counts, rows in (([2, 3], [4, 16], 20),    # no pages
                              ([2, 2], [1, 1], 2),      # named twice
                              ([2, 6], [1, 1], 2),      # unknown
                              ([2, 1], [1, -1], 2),     # a count below zero
                              ([0], [8], 8),            # longer than a row of the table
                              ([2, 3], [2, 2], 3)):     # more tokens than rows
        m.status = 0
        d.status.zero_()
        do_extend(m, d, req, counts, rows)
        assert m.status
    for parents, children in (([0, 0], [2, 2]), ([0], [1]), ([7], [2]), ([-1], [2]), ([0], [6])):
        m.status = 0
        d.status.zero_()
        m.fork(parents, children)
        K.kv_fork(d.pool, d.table, d.length, d.refs, ints(parents), ints(children), d.status)
        assert m.status == 1
        d.same(m)
    do_extend(m, d, [2, 3], [4, 4], 8)
    m.status = 0
    d.status.zero_()
    m.fork([0, 0], [4, 5])  # two part-filled pages to copy, one page free
    K.kv_fork(d.pool, d.table, d.length, d.refs, ints([0, 0]), ints([4, 5]), d.status)
    assert m.status == 8
    d.same(m)


def test_many_pages_and_rows(K):
    """More pages than one pass of the search takes, more sequences than threads, prompts long and short, fork from a shared prompt."""
    r = random.Random(7)
    m, d = both(K, n_pages=40003, blocks=1, P=2, requests=1500, width=30)
    req = r.sample(range(1500), 1300)
    counts = [r.randint(0, 40) for _ in req]
    do_extend(m, d, req, counts, sum(counts))
    gone = req[::3]
    m.free(gone)
    K.kv_free(d.table, d.length, d.refs, ints(gone), 2, d.status)
    d.same(m)
    children = [i for i in range(1500) if m.length[i] == 0][:400]
    parents = [req[1]] * 200 + [r.choice(req[1::3]) for _ in range(len(children) - 200)]
    m.fork(parents, children)
    K.kv_fork(d.pool, d.table, d.length, d.refs, ints(parents), ints(children), d.status)
    d.same(m)
    m.compact()
    K.kv_compact(d.pool, d.table, d.refs)
    d.same(m)
    do_extend(m, d, req, [1] * len(req), len(req) + 100)


@pytest.mark.parametrize("S,rows,R", [(1024, 4096, 1100), (1025, 4096, 1100), (300, 4097, 400), (1, 4096, 3), (5, 40, 9000), (1030, 1500, 9000)])
def test_steps_of_few_rows_and_others(K, S, rows, R):
    """Around the sizes up to which a step takes one launch: steps that use all rows and fewer, and refusals."""
    r = random.Random(S)
    m, d = both(K, n_pages=6000, blocks=1, P=5, requests=R, width=900)
    req = r.sample(range(R), S)
    for used in (rows, rows // 2):
        cuts = sorted(r.randint(0, used) for _ in range(S - 1))
        do_extend(m, d, req, [b - a for a, b in zip([0] + cuts, cuts + [used])], rows)
        r.shuffle(req)
    ones = [1] * S
    for names, counts, bits in ((req[:-1] + [R], ones, 1), (req[:-1] + [req[0]], ones, 1) if S > 1 else ([-3, R], [1, 1], 1),
                                (req, [rows + 1] + ones[1:], 4), (req, [0] * (S - 1) + [-1], 1)):
        m.status = 0
        d.status.zero_()
        do_extend(m, d, names, counts, rows)
        assert m.status & bits
    free = sum(x == 0 for x in m.refs)
    m.refs[:] = [x or 1 for x in m.refs[:-2]] + m.refs[-2:]  # all but two pages held
    d.refs.copy_(ints(m.refs))
    m.status = 0
    d.status.zero_()
    do_extend(m, d, req, [min(11 * 5, rows)] + [0] * (S - 1), rows)
    assert free > 2 and m.status & 8
    m.status = 0
    d.status.zero_()
    do_extend(m, d, req, [min(2, rows)] + [0] * (S - 1), rows)
    assert m.status == 0


def test_empty_calls(K):
    m, d = both(K)
    do_extend(m, d, [], [], 0)
    do_extend(m, d, [3], [0], 4)
    do_extend(m, d, [-1], [5], 2)
    for f in (lambda: K.kv_fork(d.pool, d.table, d.length, d.refs, ints([]), ints([]), d.status),
              lambda: K.kv_free(d.table, d.length, d.refs, ints([]), d.P, d.status),
              lambda: K.kv_compact(d.pool, d.table, d.refs),
              lambda: K.kv_copy_pages(d.pool, ints([]), ints([])),
              lambda: K.kv_fork(d.pool, d.table, d.length, d.refs, ints([3, 3]), ints([4, 5]), d.status)):
        f()
        d.same(m)


@pytest.mark.parametrize("shape", [(9, 2, 2, 8, 16, 128), (5, 1, 1, 3, 1, 8), (7, 3, 5, 64), (4, 1, 2, 1, 300, 256)])
def test_copy_pages(K, shape):
    dt = torch.bfloat16
    pool = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(dt).cuda()
    want = pool.clone()
    want[[0, 3]] = pool[[2, 1]]
    K.kv_copy_pages(pool, ints([2, 1, 0, 99, -1]), ints([0, 3, 77, 2, 2]))  # three of them with a page that is not there
    assert torch.equal(pool, want)


def test_free_takes_each_request_by_itself(K):
    """A list that names an unknown request, one twice and one that is skipped: the rest is freed, the unknown one reported."""
    m, d = both(K, n_pages=30, P=4, requests=6, width=5)
    do_extend(m, d, [0, 1, 2, 3], [9, 17, 4, 1], 31)
    m.fork([1], [4])
    K.kv_fork(d.pool, d.table, d.length, d.refs, ints([1]), ints([4]), d.status)
    K.kv_free(d.table, d.length, d.refs, ints([0, 6, 1, -2, 1, 2 ** 31 - 1]), d.P, d.status)
    assert d.status.item() == 1 and d.length.tolist() == [0, 0, 4, 1, 17, 0]
    assert d.table.tolist()[0] == d.table.tolist()[1] == [-1] * 5
    assert [n for n, r in enumerate(d.refs.tolist()) if r] == sorted({i for row in d.table.tolist() for i in row if i >= 0})
    assert set(d.refs.tolist()) == {0, 1}  # (what the fork shares has one holder left)
    m.free([0, 6, 1, -2, 1, 2 ** 31 - 1])
    d.same(m)
