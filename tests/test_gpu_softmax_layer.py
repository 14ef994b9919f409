"""A softmax layer of a hybrid model as it is served, all of it together: pages given out, queries and keys normed and turned, a prompt
written and attended to as the cache holds it, tokens generated, sequences forked, ended, the cache moved together -- against float64 on
what an ordinary dictionary says every sequence holds; and its training step through norm, rotation and attention."""
import pytest
import torch

import linear_moe_amd as L
from oracle import kv4, rope, softmax
from tests.util import gen

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


class Layer:
    def __init__(self, dev, N, P, S, HQ, HKV, D, bits4, heads_first, dtype=BF16):
        self.dev, self.N, self.S, self.HQ, self.HKV, self.D, self.bits4, self.dtype = dev, N, S, HQ, HKV, D, bits4, dtype
        self.table = torch.full((N, 12), -1, dtype=torch.int32, device=dev)
        self.lens, self.refs = torch.zeros(N, dtype=torch.int32, device=dev), torch.zeros(P, dtype=torch.int32, device=dev)
        make = lambda d, t: torch.zeros(P, HKV, S, d, dtype=t, device=dev).transpose(1, 2) if heads_first else torch.zeros(P, S, HKV, d, dtype=t, device=dev)
        if bits4:
            self.k, self.v = make(D // 2, torch.uint8), make(D // 2, torch.uint8)
            self.scales = dict(k_scales=make(D // 32, torch.uint8), v_scales=make(D // 32, torch.uint8))
        else:
            self.k, self.v, self.scales = make(D, dtype), make(D, dtype), {}
        self.pages = (self.k, self.v, *self.scales.values())
        self.cos, self.sin = L.rope_table(400, D, device=dev)
        self.w = [(1 + 0.2 * gen(5 + i, D, dtype=dtype)).to(dev) for i in range(2)]
        self.held = [[] for _ in range(N)]                   # (k, v) of every token, as the cache holds them

    def kept(self, x):
        return kv4.values(*kv4.pack(x)) if self.bits4 else x.double()

    def qk(self, q, k, **where):
        z = L.qk_norm_rope(q, k, *self.w, self.cos, self.sin, head_first=False, **where)
        return z

    def prompts(self, seed, lens):
        """Prompts for the sequences with a length, packed."""
        T = sum(lens)
        q, k, v = (gen(seed + i, 1, T, h, self.D, dtype=self.dtype).to(self.dev) for i, h in enumerate((self.HQ, self.HKV, self.HKV)))
        cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=self.dev)
        assert L.paged_reserve(self.pages, self.table, self.lens, self.refs, torch.tensor(lens, dtype=torch.int32, device=self.dev)).all()
        q, k = self.qk(q, k, cu_seqlens=cu)
        L.paged_kv_append(self.k, self.v, k, v, self.table, self.lens, cu_seqlens=cu, head_first=False, **self.scales)
        kk, vv = L.paged_kv_read(self.k, self.v, self.table, self.lens, T, cu_seqlens=cu, head_first=False, dtype=self.dtype, **self.scales)
        assert torch.equal(kk.double(), self.kept(k)) and torch.equal(vv.double(), self.kept(v))
        o = L.softmax_attn(q, kk, vv, cu_seqlens=cu, head_first=False)
        at = 0
        for n, m in enumerate(lens):
            rows = slice(at, at + m)
            self.held[n] += list(zip(self.kept(k[0, rows]), self.kept(v[0, rows])))
            if m:
                self.check(n, q[0, rows], o[0, rows])
            at += m
        self.lens += torch.tensor(lens, dtype=torch.int32, device=self.dev)

    def step(self, seed):
        """A token of every sequence."""
        q, k, v = (gen(seed + i, self.N, 1, h, self.D, dtype=self.dtype).to(self.dev) for i, h in enumerate((self.HQ, self.HKV, self.HKV)))
        assert L.paged_reserve(self.pages, self.table, self.lens, self.refs, 1).all()
        q, k = self.qk(q, k, offsets=self.lens)
        o = L.paged_attn_decode(q, self.k, self.v, self.table, self.lens, k=k, v=v, head_first=False, **self.scales)
        self.lens += 1
        for n in range(self.N):
            self.held[n].append((self.kept(k[n, 0]), self.kept(v[n, 0])))
            self.check(n, q[n], o[n])

    def check(self, n, q, o):
        k, v = (torch.stack(x) for x in zip(*self.held[n]))
        for h in range(self.HQ):
            ref, tol = softmax.head(q[:, h], k[:, h // (self.HQ // self.HKV)], v[:, h // (self.HQ // self.HKV)], self.D ** -0.5, dtype=self.dtype)
            assert ((o[:, h].double() - ref).abs() <= tol).all(), (n, h)

    def ints(self, *x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def fork(self, src, dst):
        L.paged_fork(self.table, self.lens, self.refs, self.ints(*src), self.ints(*dst))
        old = [list(x) for x in self.held]
        for s, d in zip(src, dst):
            self.held[d] = list(old[s])

    def free(self, *rows):
        L.paged_free(self.table, self.lens, self.refs, self.ints(*rows))
        for r in rows:
            self.held[r] = []

    def counted(self):
        """Every page is counted as often as it is named, and lens are those of the dictionary."""
        names = self.table[self.table >= 0].flatten()
        assert torch.equal(torch.bincount(names, minlength=self.refs.numel()).int(), self.refs)
        assert self.lens.tolist() == [len(x) for x in self.held]


@pytest.mark.parametrize("bits4,heads_first,S,D,dtype", [(True, True, 16, 64, BF16), (True, False, 24, 128, BF16), (True, True, 32, 96, F32), (False, False, 16, 64, BF16), (False, True, 5, 32, F32)])
def test_served(cuda, bits4, heads_first, S, D, dtype):
    m = Layer(cuda, 5, 60, S, 4, 2, D, bits4, heads_first, dtype)
    m.prompts(100, [37, 1, 16, 0, 3])
    for i in range(3):
        m.step(200 + 10 * i)
    m.counted()
    m.fork([0, 0, 2], [1, 3, 4])                             # three go on from others' beginnings, each on its own
    m.counted()
    for i in range(2):
        m.step(300 + 10 * i)
    m.fork([4, 3], [3, 4])                                   # two change places
    m.free(0, 2)
    m.counted()
    live, moved = L.paged_compact(m.pages, m.table, m.refs)
    assert int(live) == int((m.refs > 0).sum()) and bool((m.refs[:int(live)] > 0).all())
    m.counted()
    for i in range(2):
        m.step(400 + 10 * i)                                 # (sequences 0 and 2 begin anew)
    m.free(3)
    m.counted()


def test_a_captured_step(cuda):
    """Reserve, norm and rotation, attention and the length, captured once and replayed: the steps of the same calls made one by one."""
    a, b, spare = (Layer(cuda, 4, 40, 16, 4, 2, 64, True, True) for _ in range(3))
    for m in (a, b, spare):
        m.prompts(600, [14, 30, 1, 5])
        m.fork([1], [3])
    q, k, v = (torch.empty(4, 1, h, 64, dtype=BF16, device=cuda) for h in (4, 2, 2))

    def step(m):
        fits = L.paged_reserve(m.pages, m.table, m.lens, m.refs, 1)
        zq, zk = m.qk(q, k, offsets=m.lens)
        o = L.paged_attn_decode(zq, m.k, m.v, m.table, m.lens, k=zk, v=v, head_first=False, **m.scales)
        m.lens.add_(1)
        return fits, o
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(spare)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(a)
    for i in range(20):
        for j, x in enumerate((q, k, v)):
            x.copy_(gen(700 + 3 * i + j, *x.shape, dtype=BF16))
        g.replay()
        want = step(b)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)) and bool(out[0].all())
        assert all(torch.equal(x, y) for x, y in zip((a.table, a.lens, a.refs, *a.pages), (b.table, b.lens, b.refs, *b.pages)))


def test_training_step(cuda):
    """Norm, rotation and attention in float32, gradients of q, k, v and the weights against float64."""
    lens, HQ, HKV, D = [40, 1, 23], 4, 2, 64
    T = sum(lens)
    x = [gen(800 + i, 1, T, h, D) for i, h in enumerate((HQ, HKV, HKV))]
    w = [1 + 0.2 * gen(810 + i, D) for i in range(2)]
    do = gen(820, 1, T, HQ, D)
    cos, sin = L.rope_table(64, D)
    cu = torch.tensor([0, 40, 41, 64], dtype=torch.int32)
    leaves = [y.to(cuda).requires_grad_(True) for y in (*x, *w)]
    q, k = L.qk_norm_rope(leaves[0], leaves[1], *leaves[3:], cos.to(cuda), sin.to(cuda), cu_seqlens=cu.to(cuda), head_first=False)
    o = L.softmax_attn(q, k, leaves[2], cu_seqlens=cu.to(cuda), head_first=False)
    got = torch.autograd.grad(o, leaves, do.to(cuda))
    ref = [y.double().requires_grad_(True) for y in (*x, *w)]
    pos = torch.cat([torch.arange(n) for n in lens])
    c, s = (y.double()[pos][None, :, None] for y in (cos, sin))
    rq, rk = rope.forward(ref[0], ref[3], c, s, D, False, 1e-6), rope.forward(ref[1], ref[4], c, s, D, False, 1e-6)
    outs, at = [], 0
    for n in lens:
        rows = slice(at, at + n)
        hidden = torch.ones(n, n, dtype=torch.bool).triu(1)
        for h in range(HQ):
            p = torch.softmax((rq[0, rows, h] @ rk[0, rows, h // 2].T * D ** -0.5).masked_fill(hidden, float("-inf")), 1)
            outs.append((p @ ref[2][0, rows, h // 2] * do[0, rows, h].double()).sum())
        at += n
    want = torch.autograd.grad(sum(outs), ref)
    for a, b in zip(got, want):
        # float32 throughout: some hundred roundings of 2^-24, of sums whose terms are at most a few times the result's size
        assert (a.cpu().double() - b).abs().max() <= 1e-4 * b.abs().max()
