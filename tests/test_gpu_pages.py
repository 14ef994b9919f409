"""The pages of a cache on the GPU: given out, shared, copied, moved together and taken back, against the same done one entry after
the other (oracle/pages.py)."""
import random

import pytest
import torch

import linear_moe_amd as L
from oracle import pages as oracle

pytestmark = pytest.mark.gpu


class State:
    """A random consistent cache on both sides: rows that share beginnings, holes, some pages with a hold of the program."""

    def __init__(self, dev, seed, N, M, P, S, shapes=((2, 16),), dtypes=(torch.bfloat16,), full=0.7):
        r = random.Random(seed)
        self.N, self.M, self.P, self.S, self.dev = N, M, P, S, dev
        self.table, self.lens, self.refs = [[-1] * M for _ in range(N)], [0] * N, [0] * P
        free = list(range(P))
        r.shuffle(free)
        for n in range(N):
            m = 0
            if n and r.random() < 0.4:
                other = r.randrange(n)
                m = r.randrange(0, M + 1)
                for j in range(m):
                    x = self.table[other][j]
                    if 0 <= x < P:
                        self.table[n][j] = x
                        self.refs[x] += 1
                m = next((j for j in range(M) if self.table[n][j] < 0), M)
                for j in range(m, M):
                    x = self.table[n][j]
                    if x >= 0:
                        self.refs[x] -= 1
                        self.table[n][j] = -1
            more = r.randrange(0, M - m + 1) if r.random() < full else 0
            for j in range(m, m + more):
                if free:
                    self.table[n][j] = free.pop()
                    self.refs[self.table[n][j]] += 1
            held = next((j for j in range(M) if self.table[n][j] < 0), M)
            self.lens[n] = max(0, held * S - r.randrange(0, 2 * S)) if held else 0
            for j in range(held, M):
                self.table[n][j] = r.choice((-1, -1, -9, P, 2 ** 31 - 1))
        for _ in range(min(2, len(free))):
            self.refs[free.pop()] += 1                      # held by the program alone
        g = torch.Generator().manual_seed(seed)
        self.pages = [(torch.randint(0, 255, (P, S, *s), generator=g).to(d)) for s, d in zip(shapes, dtypes)]
        i32 = dict(dtype=torch.int32, device=dev)
        self.d_table = torch.tensor(self.table, **i32).view(N, M)
        self.d_lens, self.d_refs = torch.tensor(self.lens, **i32), torch.tensor(self.refs, **i32)
        self.d_pages = [p.to(dev) for p in self.pages]

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def copied(self, copies):
        for p in self.pages:
            old = p.clone()
            for a, b in copies:
                p[b] = old[a]

    def check(self):
        assert self.d_table.cpu().tolist() == self.table
        assert self.d_lens.cpu().tolist() == self.lens and self.d_refs.cpu().tolist() == self.refs
        for a, b in zip(self.d_pages, self.pages):
            assert torch.equal(a.cpu(), b)

    def free(self, rows):
        L.paged_free(self.d_table, self.d_lens, self.d_refs, self.ints(rows))
        oracle.free(self.table, self.lens, self.refs, rows)
        self.check()

    def fork(self, src, dst):
        L.paged_fork(self.d_table, self.d_lens, self.d_refs, self.ints(src), self.ints(dst))
        oracle.fork(self.table, self.lens, self.refs, src, dst)
        self.check()

    def reserve(self, tokens):
        each = isinstance(tokens, int)
        fits = L.paged_reserve(self.d_pages, self.d_table, self.d_lens, self.d_refs, tokens if each else self.ints(tokens))
        want, copies = oracle.reserve(self.table, self.lens, self.refs, [tokens] * self.N if each else tokens, self.S)
        self.copied(copies)
        assert fits.dtype == torch.bool and fits.cpu().tolist() == want
        self.check()
        return want

    def compact(self):
        live, moved = L.paged_compact(self.d_pages, self.d_table, self.d_refs)
        want, where, copies = oracle.compact(self.table, self.refs)
        self.copied(copies)
        assert live.cpu().tolist() == [want] and moved.cpu().tolist() == where
        self.check()

    def consistent(self, holds=2):
        names = [x for row in self.table for x in row if 0 <= x < self.P]
        assert all(self.refs[p] >= names.count(p) for p in range(self.P)) and sum(self.refs) <= len(names) + holds


SIZES = [(1, 1, 1, 1), (4, 5, 20, 3), (7, 12, 90, 16), (3, 200, 500, 4), (40, 9, 150, 8), (70, 30, 900, 2)]


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("N,M,P,S", SIZES)
def test_each_alone(cuda, seed, N, M, P, S):
    r = random.Random(seed + 100 * N)
    new = lambda i=0: State(cuda, 10 * seed + i, N, M, P, S)
    rows = lambda k, lo=0, hi=N: [r.randrange(lo, hi) for _ in range(k)]
    new().free(rows(N // 2 + 1))
    new().free(rows(2 * N, -2, N + 2))                          # twice, and none
    new().fork(rows(N), rows(N))                                # given and taken, several for one
    new().fork(rows(2 * N, -1, N + 1), rows(2 * N, -1, N + 1))
    order = list(range(N))
    r.shuffle(order)
    new().fork(order, list(range(N)))
    for i, tokens in enumerate((0, 1, S, 3 * S + 1, M * S + 1, [r.randrange(-2, 2 * S + 2) for _ in range(N)], [r.choice((0, 1, 2 ** 31 - 1)) for _ in range(N)])):
        new(i).reserve(tokens)
    new().compact()


@pytest.mark.parametrize("seed", range(6))
def test_a_life_of_a_cache(cuda, seed):
    """Steps in any order; every page stays counted."""
    r = random.Random(seed)
    N, M, P, S = r.choice(SIZES[1:])
    st = State(cuda, seed, N, M, P, S, shapes=((2, 16), (2, 1), (3,)), dtypes=(torch.bfloat16, torch.uint8, torch.float32))
    for _ in range(12):
        what = r.randrange(4)
        if what == 0:
            st.free([r.randrange(N) for _ in range(r.randrange(1, 4))])
        elif what == 1:
            k = r.randrange(1, N + 1)
            st.fork([r.randrange(N) for _ in range(k)], r.sample(range(N), k))
        elif what == 2:
            tokens = [r.randrange(0, 2 * S) for _ in range(N)]
            fits = st.reserve(tokens)
            st.lens = [n + t if ok else n for n, t, ok in zip(st.lens, tokens, fits)]
            st.d_lens.copy_(torch.tensor(st.lens, dtype=torch.int32))
        else:
            st.compact()
        st.consistent()


def test_when_the_pages_end(cuda):
    """Rows are served in their order: the first that lacks a page and all behind that need one get none, and what those would have
    copied stays shared -- its last holder gets no page to itself."""
    st = State(cuda, 1, 6, 4, 8, 4, full=0.0)
    st.table = [[0, -1, -1, -1], [0, -1, -1, -1], [1, -1, -1, -1], [1, -1, -1, -1], [2, -1, -1, -1], [3, -1, -1, -1]]
    st.lens, st.refs = [3, 3, 2, 2, 4, 1], [2, 2, 1, 1, 1, 1, 0, 1]          # one free page
    st.d_table.copy_(st.ints(st.table)), st.d_lens.copy_(st.ints(st.lens)), st.d_refs.copy_(st.ints(st.refs))
    want = st.reserve(1)
    assert want == [True, True, False, False, False, True]                     # row 1 keeps page 0, row 3 does not get to write on page 1
    assert st.table[0][0] == 6 and st.table[1][0] == 0 and st.table[2][0] == st.table[3][0] == 1


def test_many(cuda):
    """More rows and pages than the deciding work-group has threads."""
    for seed, (N, M, P, S) in enumerate(((1500, 6, 9000, 4), (30, 1200, 40000, 2), (2000, 3, 1000, 1))):
        st = State(cuda, seed, N, M, P, S, shapes=((4,),), dtypes=(torch.int32,))
        r = random.Random(seed)
        st.free([r.randrange(N) for _ in range(N // 4)])
        st.fork([r.randrange(N) for _ in range(N // 2)], r.sample(range(N), N // 2))
        st.reserve([r.randrange(0, 3 * S) for _ in range(N)])
        st.compact()
        st.reserve(1)


def test_shared_pages_whose_numbers_are_alike(cuda):
    """Rows of one token that share pages 512, 1024, 2048 and 4096 apart, and neighbours."""
    for step in (1, 512, 1024, 2048, 4096):
        n, r = 15, random.Random(step)
        st = State(cuda, 2, 4 * n, 3, 15 * 4096 + 1, 4, full=0.0, shapes=((1,),), dtypes=(torch.uint8,))
        pages = [step * i for i in range(n)] * 4
        r.shuffle(pages)
        st.table = [[p, -1, -1] for p in pages]
        st.lens, st.refs = [r.randrange(1, 4) for _ in pages], [0] * st.P
        for i in range(n):
            st.refs[step * i] = 4 + (i % 5 == 0)                               # (some held by the program as well)
        st.d_table.copy_(st.ints(st.table)), st.d_lens.copy_(st.ints(st.lens)), st.d_refs.copy_(st.ints(st.refs))
        st.reserve([r.choice((0, 1, 1, 1)) for _ in pages])
        st.reserve(2)


@pytest.mark.parametrize("N,M,F", [(300, 2, 256), (300, 2, 257), (40, 1024, 8), (40, 1025, 8), (260, 32, 256), (260, 33, 256), (5, 3000, 4), (200, 1, 200), (3, 1, 40)])
def test_forks_of_many_rows(cuda, N, M, F):
    """Chains and rings of rows, rows twice, rows that are none."""
    r = random.Random(N * M + F)
    st = State(cuda, 60, N, M, 3 * N + M, 2)
    for _ in range(3):
        st.fork([r.randrange(-1, N + 1) for _ in range(F)], [r.randrange(-1, N + 1) for _ in range(F)])
    ring = [i % N for i in range(min(F, N))]
    st.fork(ring, ring[1:] + ring[:1])


def test_layouts_of_pages(cuda):
    """Tensors of pages in other orders and as parts of others; what lies between stays."""
    N, M, P, S = 5, 6, 40, 8
    make = [
        lambda: torch.randn(P, S, 2, 16, device=cuda),
        lambda: torch.randn(P, 2, S, 16, device=cuda).transpose(1, 2),
        lambda: torch.randn(2 * P, S, 3, 16, device=cuda)[::2, :, 1:],
        lambda: torch.randint(0, 255, (P, 2, S, 3), device=cuda, dtype=torch.uint8).transpose(1, 2),
        lambda: torch.randint(0, 255, (P, S, 2, 7), device=cuda, dtype=torch.uint8)[..., 1:4],
        lambda: torch.randn(S, P, 20, device=cuda).transpose(0, 1),
        lambda: torch.randn(P, S, device=cuda),
        lambda: torch.randn(P, S, 4, 5, 6, device=cuda)[:, :, 1:, :, 2:4],
        lambda: torch.randn(P, S, 5, 2, 16, device=cuda)[:, :, :, 1],
        lambda: torch.randn(P, S, 2, 2, device=cuda)[..., 0],
        lambda: torch.randn(P, 4, S, 2, device=cuda)[:, 0, :, 1],
    ]
    for k, f in enumerate(make):
        st = State(cuda, 50 + k, N, M, P, S)
        x = f()
        base = x._base if x._base is not None else x
        untouched = base.clone()
        st.pages, st.d_pages = [x.cpu().clone()], [x]
        st.reserve(S + 1)
        st.free([0, 3])
        st.compact()
        mark = torch.zeros_like(base, dtype=torch.bool)
        view = torch.as_strided(mark, x.shape, x.stride(), x.storage_offset())
        view.fill_(True)
        assert torch.equal(base[~mark], untouched[~mark])
    # many tensors in one call, of different sizes
    st = State(cuda, 70, N, M, P, S, shapes=tuple((1 + i % 5, 8) for i in range(70)), dtypes=tuple((torch.bfloat16, torch.uint8, torch.float32)[i % 3] for i in range(70)))
    st.reserve(2 * S)
    st.free([1])
    st.compact()


def test_graph(cuda):
    """One captured step, replayed on a state that has moved on."""
    N, M, P, S = 6, 8, 60, 4
    st = State(cuda, 3, N, M, P, S)
    src, dst, rows, tokens = st.ints([0, 1]), st.ints([2, 3]), st.ints([4]), st.ints([1] * N)

    def step(d):
        L.paged_free(d[0], d[1], d[2], rows)
        L.paged_fork(d[0], d[1], d[2], src, dst)
        fits = L.paged_reserve(d[3], d[0], d[1], d[2], tokens)
        live, moved = L.paged_compact(d[3], d[0], d[2])
        return fits, live, moved
    mine = (st.d_table, st.d_lens, st.d_refs, st.d_pages)
    spare = tuple(x.clone() for x in mine[:3]) + ([p.clone() for p in st.d_pages],)
    twin = tuple(x.clone() for x in mine[:3]) + ([p.clone() for p in st.d_pages],)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(spare)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(mine)
    r = random.Random(4)
    for _ in range(6):
        g.replay()
        want = step(twin)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(mine[:3], twin[:3])) and torch.equal(mine[3][0], twin[3][0])
        for x, hi in ((src, N), (dst, N), (rows, N + 2), (tokens, 2 * S)):
            x.copy_(torch.tensor([r.randrange(hi) for _ in range(x.numel())], dtype=torch.int32))
        more = torch.where(out[0], tokens, 0).to(torch.int32) * 0 + 1
        for d in (mine, twin):
            d[1].add_(more).clamp_(max=M * S - 1)


def test_two_at_once(cuda):
    """Two caches on two streams at the same time: each as by itself."""
    N, M, P, S = 40, 12, 700, 8
    states = [State(cuda, 90 + i, N, M, P, S) for i in range(2)]
    twins = [tuple(x.clone() for x in (st.d_table, st.d_lens, st.d_refs)) + ([p.clone() for p in st.d_pages],) for st in states]
    rows, src, dst = states[0].ints([1, 5, 39]), states[0].ints([0, 2, 2]), states[0].ints([1, 5, 7])

    def life(d):
        out = []
        for j in range(3):
            L.paged_free(d[0], d[1], d[2], rows)
            L.paged_fork(d[0], d[1], d[2], src, dst)
            out.append(L.paged_reserve(d[3], d[0], d[1], d[2], j + 1))
            out += L.paged_compact(d[3], d[0], d[2])
        return out + [x.clone() for x in (*d[:3], *d[3])]
    want = [life(d) for d in twins]
    torch.cuda.synchronize()
    got = []
    for st in states:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(life((st.d_table, st.d_lens, st.d_refs, st.d_pages)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(want, got) for a, b in zip(x, y))


def test_the_path_in_python_does_the_same(cuda):
    """Calls that need a conversion (numbers of 64 bits, a generator of tensors)."""
    for native in (True, False):
        st = State(cuda, 80, 6, 8, 60, 4, shapes=((2, 16), (3,)), dtypes=(torch.bfloat16, torch.uint8))
        conv = (lambda x: x) if native else (lambda x: x.long())
        pages = lambda: tuple(st.d_pages) if native else (p for p in st.d_pages)
        L.paged_free(st.d_table, st.d_lens, st.d_refs, conv(st.ints([1, 1, 9])))
        L.paged_fork(st.d_table, st.d_lens, st.d_refs, conv(st.ints([0, 2])), conv(st.ints([1, 4])))
        fits = L.paged_reserve(pages(), st.d_table, st.d_lens, st.d_refs, conv(st.ints([1, 2, 3, 4, 5, 6])))
        live, moved = L.paged_compact(pages(), st.d_table, st.d_refs)
        got = [st.d_table, st.d_lens, st.d_refs, fits, live, moved, *st.d_pages]
        if native:
            first = got
    assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_nothing(cuda):
    i32 = dict(dtype=torch.int32, device=cuda)
    none = torch.zeros(0, **i32)
    for N, M, P in ((0, 3, 5), (3, 0, 5), (3, 3, 0), (0, 0, 0)):
        table, lens, refs = torch.full((N, M), -1, **i32), torch.zeros(N, **i32), torch.zeros(P, **i32)
        pages = torch.zeros(P, 4, 2, device=cuda)
        L.paged_free(table, lens, refs, none)
        L.paged_free(table, lens, refs, torch.zeros(2, **i32))
        L.paged_fork(table, lens, refs, none, none)
        assert L.paged_reserve(pages, table, lens, refs, 0).tolist() == [True] * N
        fits = L.paged_reserve(pages, table, lens, refs, 1).tolist()
        assert fits == [M > 0 and P > 0] * N
        live, moved = L.paged_compact((), table, refs)
        assert live.tolist() == [N if M and P else 0] and moved.tolist() == list(range(P))


def test_refusals(cuda):
    i32 = dict(dtype=torch.int32, device=cuda)
    table, lens, refs, pages, rows = torch.full((3, 4), -1, **i32), torch.zeros(3, **i32), torch.zeros(6, **i32), torch.zeros(6, 4, 2, device=cuda), torch.zeros(2, **i32)
    state = dict(page_table=table, lens=lens, refs=refs)
    for change in (dict(page_table=table.long()), dict(page_table=table[0]), dict(page_table=table.t().contiguous().t()), dict(page_table=table[:1].expand(3, 4)),
                   dict(lens=lens.long()), dict(lens=lens[:2]), dict(lens=lens.cpu()), dict(refs=refs.long()), dict(refs=torch.zeros(12, **i32)[::2]), dict(refs=refs[:, None])):
        for f, more in ((L.paged_free, dict(rows=rows)), (L.paged_fork, dict(src=rows, dst=rows)), (L.paged_reserve, dict(pages=pages, tokens=1))):
            with pytest.raises(ValueError):
                f(**{**state, **more, **change})
    for change in (dict(pages=pages[:5]), dict(pages=pages.cpu()), dict(pages=(pages, torch.zeros(6, 5, 2, device=cuda))), dict(pages=pages[:, 0, 0]),
                   dict(pages=torch.zeros(1, 4, 2, device=cuda).expand(6, 4, 2)), dict(pages=torch.zeros(6, 4, 1, device=cuda).expand(6, 4, 2)),
                   dict(pages=torch.zeros(6, 5, 3, 4, 9, device=cuda)[:, :4, :2, :3, :8]),
                   dict(tokens=-1), dict(tokens=2 ** 31), dict(tokens=torch.zeros(2, **i32)), dict(tokens=torch.zeros(3, device=cuda))):
        with pytest.raises(ValueError):
            L.paged_reserve(**{**state, **dict(pages=pages, tokens=1), **change})
    for change in (dict(src=rows[:1]), dict(src=rows.float()), dict(dst=rows[None]), dict(dst=rows.cpu())):
        with pytest.raises(ValueError):
            L.paged_fork(**{**state, **dict(src=rows, dst=rows), **change})
    with pytest.raises(ValueError):
        L.paged_reserve((), **state, tokens=1)
    with pytest.raises(ValueError):
        L.paged_free(**state, rows=rows[None])
    with pytest.raises(RuntimeError):
        L.paged_free(table.cpu(), lens.cpu(), refs.cpu(), rows.cpu())
    with pytest.raises(RuntimeError):
        L.paged_reserve(pages.clone().requires_grad_(True), table, lens, refs, 1)
