"""The paged cache on the GPU: attention of one token over it against float64 within derived bounds (oracle/softmax.py), what
is written into it bit for bit, and a run of prompt, cache and generated tokens together."""
import pytest
import torch

import linear_moe_amd as L
from oracle import softmax
from tests.util import gen

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


class Cache:
    """Pages of sequences in shuffled order; what no token owns holds `fill`."""

    def __init__(self, seed, lens, S, HKV, K, V, dtype, spare=1, fill=float("nan"), heads_first=False):
        g = torch.Generator().manual_seed(seed)
        self.S, self.lens = S, list(lens)
        cols = max((n + spare + S - 1) // S for n in lens) + 1
        need = [(n + spare + S - 1) // S for n in lens]
        P = sum(need) + 2
        ids = torch.randperm(P, generator=g).tolist()
        self.table = torch.full((len(lens), cols), -7, dtype=torch.int32)
        at = 0
        for n, m in enumerate(need):
            self.table[n, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
            at += m
        shape = (P, HKV, S) if heads_first else (P, S, HKV)
        self.k, self.v = (torch.full((*shape, D), fill, dtype=dtype) for D in (K, V))
        if heads_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.rows = [(gen(seed + 2 * n + 1, m, HKV, K, dtype=dtype), gen(seed + 2 * n + 2, m, HKV, V, dtype=dtype)) for n, m in enumerate(lens)]
        for n, (kk, vv) in enumerate(self.rows):
            for j in range(self.lens[n]):
                self.put(n, j, kk[j], vv[j])

    def put(self, n, j, kk, vv):
        page = int(self.table[n, j // self.S])
        self.k[page, j % self.S], self.v[page, j % self.S] = kk, vv

    def to(self, dev):
        # (strides kept)
        out = []
        for x in (self.k, self.v):
            y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=dev)
            out.append(y.copy_(x))
        return (*out, self.table.to(dev), torch.tensor(self.lens, dtype=torch.int32, device=dev))


def same(a, b):
    """The same bits, NaN included."""
    view = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.cpu().contiguous().view(view), b.cpu().contiguous().view(view))


def alibi(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)])


def decode_and_check(cuda, c, HQ, K, V, dtype, append=False, softcap=0.0, slopes=None, head_first=False, seed=900):
    HKV, N = c.k.shape[2], len(c.lens)
    G = HQ // HKV
    q, kn, vn = gen(seed, N, 1, HQ, K, dtype=dtype), gen(seed + 1, N, 1, HKV, K, dtype=dtype), gen(seed + 2, N, 1, HKV, V, dtype=dtype)
    kp, vp, table, lens = c.to(cuda)
    lay = (lambda x: x.transpose(1, 2)) if head_first else (lambda x: x)
    new = dict(k=lay(kn.to(cuda)), v=lay(vn.to(cuda))) if append else {}
    o = lay(L.paged_attn_decode(lay(q.to(cuda)), kp, vp, table, lens, softcap=softcap, slopes=None if slopes is None else slopes.to(cuda),
                                head_first=head_first, **new))
    assert o.shape == (N, 1, HQ, V) and o.dtype == dtype
    if append:
        for n, m in enumerate(c.lens):
            c.put(n, m, kn[n, 0], vn[n, 0])
    assert same(kp, c.k) and same(vp, c.v)                   # the new token where it belongs, nothing else touched
    for n in range(N):
        kk, vv = c.rows[n]
        if append:
            kk, vv = torch.cat([kk, kn[n]]), torch.cat([vv, vn[n]])
        if kk.shape[0] == 0:
            assert (o[n] == 0).all()
            continue
        for h in range(HQ):
            ref = softmax.head(q[n, :, h], kk[:, h // G], vv[:, h // G], K ** -0.5, cap=softcap, slope=0.0 if slopes is None else float(slopes[h]),
                               dtype=dtype)
            softmax.check(o[n, :, h], ref, (n, h))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("S", [1, 7, 16, 24, 32, 64, 100])
@pytest.mark.parametrize("append", [False, True])
def test_pages_of_any_size(cuda, dtype, S, append):
    c = Cache(S, [0, 1, S - 1, S, S + 1, 31, 32, 33, 127, 128, 129, 200], S, 2, 64, 64, dtype)
    decode_and_check(cuda, c, 4, 64, 64, dtype, append)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("HQ,HKV", [(1, 1), (3, 3), (4, 1), (5, 1), (16, 1), (17, 1), (40, 2)])
@pytest.mark.parametrize("K,V", [(128, 128), (64, 128), (96, 40), (8, 8)])
def test_heads(cuda, dtype, HQ, HKV, K, V):
    c = Cache(3, [5, 70, 300], 16, HKV, K, V, dtype)
    decode_and_check(cuda, c, HQ, K, V, dtype, append=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap,bias", [(3.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("append", [False, True])
def test_scores(cuda, dtype, cap, bias, append):
    c = Cache(5, [1, 90, 1000], 32, 2, 64, 64, dtype)
    decode_and_check(cuda, c, 4, 64, 64, dtype, append, cap, alibi(4) if bias else None)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("head_first", [False, True])
@pytest.mark.parametrize("pages_heads_first", [False, True])
def test_layouts(cuda, dtype, head_first, pages_heads_first):
    c = Cache(9, [3, 77, 140], 16, 3, 64, 64, dtype, heads_first=pages_heads_first)
    decode_and_check(cuda, c, 6, 64, 64, dtype, True, head_first=head_first)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens", [[3000], [1, 9000], [2047, 2048, 2049, 0]])
@pytest.mark.parametrize("append", [False, True])
def test_long_caches_are_cut_and_joined(cuda, dtype, lens, append):
    c = Cache(11, lens, 64, 1, 64, 64, dtype)
    decode_and_check(cuda, c, 2, 64, 64, dtype, append, slopes=alibi(2))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pages_that_are_none(cuda, dtype):
    """Numbers outside 0 .. P - 1: their positions take no part, and nothing is written there."""
    c = Cache(13, [100, 100, 100, 64], 16, 1, 64, 64, dtype)
    kp, vp, table, lens = c.to(cuda)
    P = kp.shape[0]
    table[0, 2], table[1, :], table[2, 6], table[3, 4] = -1, 2 ** 31 - 1, P, -1
    keep = kp.clone(), vp.clone()
    q, kn, vn = (gen(90 + i, 4, 1, n, 64, dtype=dtype) for i, n in enumerate((2, 1, 1)))
    o = L.paged_attn_decode(q.to(cuda), kp, vp, table, lens, head_first=False)
    gone = [set(range(32, 48)), set(range(100)), set(range(96, 100)), set()]
    for n in range(4):
        live = [j for j in range(c.lens[n]) if j not in gone[n]]
        if not live:
            assert (o[n] == 0).all()
            continue
        kk, vv = c.rows[n][0][live], c.rows[n][1][live]
        for h in range(2):
            softmax.check(o[n, :, h], softmax.head(q[n, :, h], kk[:, 0], vv[:, 0], 0.125, dtype=dtype), (n, h))
    assert same(kp, keep[0]) and same(vp, keep[1])
    # the new token of sequence 2, 3 and 1 has no page: attended to, not kept; that of 0 has
    o = L.paged_attn_decode(q.to(cuda), kp, vp, table, lens, kn.to(cuda), vn.to(cuda), head_first=False)
    softmax.check(o[1], (vn[1].double().expand(1, 2, 64), vn[1].double().abs().expand(1, 2, 64) * torch.finfo(dtype).eps), "itself alone")
    c.put(0, 100, kn[0, 0], vn[0, 0])
    keep[0][int(c.table[0, 6]), 4], keep[1][int(c.table[0, 6]), 4] = kn[0, 0].to(cuda), vn[0, 0].to(cuda)
    assert same(kp, keep[0]) and same(vp, keep[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lengths_beyond_the_table(cuda, dtype):
    """lens below 0 count as 0, positions beyond the table do not exist; the new token is attended to all the same."""
    c = Cache(17, [32, 32, 32], 16, 1, 64, 64, dtype, spare=0)
    kp, vp, table, lens = c.to(cuda)
    table = table[:, :2]                      # (a view with its own row stride)
    lens.copy_(torch.tensor([-3, 1000, 32]))
    keep = kp.clone(), vp.clone()
    q, kn, vn = (gen(70 + i, 3, 1, 1, 64, dtype=dtype) for i in range(3))
    for new in (False, True):
        o = L.paged_attn_decode(q.to(cuda), kp, vp, table, lens, *((kn.to(cuda), vn.to(cuda)) if new else ()), head_first=False)
        for n, m in enumerate((0, 32, 32)):
            kk, vv = c.rows[n][0][:m, 0], c.rows[n][1][:m, 0]
            if new:
                kk, vv = torch.cat([kk, kn[n, 0]]), torch.cat([vv, vn[n, 0]])
            if kk.shape[0] == 0:
                assert (o[n] == 0).all()
            else:
                softmax.check(o[n, :, 0], softmax.head(q[n, :, 0], kk, vv, 0.125, dtype=dtype), (new, n))
        assert same(kp, keep[0]) and same(vp, keep[1])


def test_offsets_beyond_31_bits(cuda):
    """A cache of more than 2^31 elements: the pages used lie at its end."""
    P, S, HKV, D = 17000, 16, 64, 128
    kp, vp = (torch.empty(P, S, HKV, D, dtype=BF16, device=cuda) for _ in range(2))
    assert kp.numel() > 2 ** 31
    table = torch.tensor([[P - 1, 0, P - 2]], dtype=torch.int32, device=cuda)
    kk, vv, q = gen(1, 40, HKV, D, dtype=BF16), gen(2, 40, HKV, D, dtype=BF16), gen(3, 1, 1, HKV, D, dtype=BF16)
    lens = torch.tensor([0], dtype=torch.int32, device=cuda)
    L.paged_kv_append(kp, vp, kk[None].to(cuda), vv[None].to(cuda), table, lens, head_first=False)
    for j, page in enumerate((P - 1, 0, P - 2)):
        m = min(16, 40 - 16 * j)
        assert torch.equal(kp[page, :m].cpu(), kk[16 * j:16 * j + m]) and torch.equal(vp[page, :m].cpu(), vv[16 * j:16 * j + m])
    o = L.paged_attn_decode(q.to(cuda), kp, vp, table, lens + 40, head_first=False)
    for h in (0, 63):
        softmax.check(o[0, :, h], softmax.head(q[0, :, h], kk[:, h], vv[:, h], D ** -0.5, dtype=BF16), h)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("S", [1, 16, 24])
@pytest.mark.parametrize("packed,head_first", [(False, False), (False, True), (True, False)])
def test_append(cuda, dtype, S, packed, head_first):
    fresh = [5, 0, 40, 0, 0, 1, 33] if packed else [40] * 7
    start = [0, 3, 15, 16, 17, 31, 100]
    c = Cache(S, start, S, 3, 64, 40, dtype, spare=40)
    kp, vp, table, lens = c.to(cuda)
    T = sum(fresh) + 9 if packed else 40                       # (nine rows behind the last sequence)
    kn, vn = (gen(50 + i, 1 if packed else 7, T, 3, D, dtype=dtype) for i, D in enumerate((64, 40)))
    cu = [0]
    for f in fresh:
        cu.append(cu[-1] + f)
    lay = (lambda x: x.transpose(1, 2)) if head_first else (lambda x: x)
    got = L.paged_kv_append(kp, vp, lay(kn.to(cuda)), lay(vn.to(cuda)), table, lens, head_first=head_first,
                            cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=cuda) if packed else None)
    assert got is None
    for n in range(7):
        for t in range(fresh[n]):
            row = (0, cu[n] + t) if packed else (n, t)
            c.put(n, start[n] + t, kn[row], vn[row])
    assert same(kp, c.k) and same(vp, c.v)


def test_append_to_many_sequences(cuda):
    """More sequences than the search looks at in a round, many of them empty."""
    N = 700
    fresh = [(n * 7919) % 5 if n % 3 else 0 for n in range(N)]
    c = Cache(1, [n % 4 for n in range(N)], 4, 1, 8, 8, BF16, spare=5)
    kp, vp, table, lens = c.to(cuda)
    cu = [0]
    for f in fresh:
        cu.append(cu[-1] + f)
    kn, vn = gen(50, 1, cu[-1], 1, 8, dtype=BF16), gen(51, 1, cu[-1], 1, 8, dtype=BF16)
    for offs in (torch.tensor(cu, device=cuda), torch.tensor(cu)):
        L.paged_kv_append(kp, vp, kn.to(cuda), vn.to(cuda), table, lens, cu_seqlens=offs, head_first=False)
    for n in range(N):
        for t in range(fresh[n]):
            c.put(n, n % 4 + t, kn[0, cu[n] + t], vn[0, cu[n] + t])
    assert same(kp, c.k) and same(vp, c.v)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_leaves_out_what_has_no_page(cuda, dtype):
    c = Cache(2, [14, 14, 14], 16, 1, 64, 64, dtype, spare=30)
    kp, vp, table, lens = c.to(cuda)
    P = kp.shape[0]
    table[0, 1], table[1, 1], table[1, 2] = -1, P, 2 ** 31 - 1
    lens[2] = -1
    kn, vn = gen(5, 3, 100, 1, 64, dtype=dtype), gen(6, 3, 100, 1, 64, dtype=dtype)
    L.paged_kv_append(kp, vp, kn.to(cuda), vn.to(cuda), table, lens, head_first=False)
    for j in range(14, 16):
        for n in range(2):
            c.put(n, j, kn[n, j - 14], vn[n, j - 14])
    for j in range(32, 44 + 4):                                # sequence 0 goes on behind its missing page
        if int(c.table[0, j // 16]) >= 0:
            c.put(0, j, kn[0, j - 14], vn[0, j - 14])
    assert same(kp, c.k) and same(vp, c.v)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (8.0, True)])
def test_prompt_cache_and_generated_tokens_together(cuda, dtype, cap, bias):
    """Prompts through softmax_attn into the cache, then token by token: the same as one pass over the whole sequences."""
    HQ, HKV, D, S, more = 4, 2, 64, 16, 6
    prompts = [1, 30, 64, 100]
    total = [p + more for p in prompts]
    full = [tuple(gen(10 * n + i, total[n], h, D, dtype=dtype) for i, h in enumerate((HQ, HKV, HKV))) for n in range(4)]
    kw = dict(softcap=cap, slopes=alibi(HQ).to(cuda) if bias else None)
    pack = lambda i, cut: torch.cat([full[n][i][:cut[n]] for n in range(4)])[None].to(cuda)
    cu = torch.tensor([0] + torch.tensor(prompts).cumsum(0).tolist(), dtype=torch.int32, device=cuda)
    cols = max((t + S - 1) // S for t in total)
    table = torch.randperm(4 * cols, generator=torch.Generator().manual_seed(3)).view(4, cols).to(torch.int32).to(cuda)
    kp, vp = (torch.full((4 * cols, S, HKV, D), float("nan"), dtype=dtype, device=cuda) for _ in range(2))
    lens = torch.zeros(4, dtype=torch.int32, device=cuda)
    with torch.no_grad():
        q, k, v = (pack(i, prompts) for i in range(3))
        outs = [list(x) for x in L.softmax_attn(q, k, v, cu_seqlens=cu, head_first=False, **kw)[0].split(prompts)]
        L.paged_kv_append(kp, vp, k, v, table, lens, cu_seqlens=cu, head_first=False)
        lens += cu[1:] - cu[:-1]
        for step in range(more):
            q, k, v = (torch.stack([full[n][i][prompts[n] + step] for n in range(4)])[:, None].to(cuda) for i in range(3))
            if step % 2:
                L.paged_kv_append(kp, vp, k, v, table, lens, head_first=False)
                lens += 1
                o = L.paged_attn_decode(q, kp, vp, table, lens, head_first=False, **kw)
            else:
                o = L.paged_attn_decode(q, kp, vp, table, lens, k, v, head_first=False, **kw)
                lens += 1
            for n in range(4):
                outs[n].append(o[n, 0])
    for n in range(4):
        want = softmax.attn(*(x[None] for x in full[n]), softcap=cap, slopes=alibi(HQ) if bias else None)
        softmax.check(torch.stack(outs[n])[None], want["o"], n)


def test_a_captured_step_follows_lengths_and_pages(cuda):
    """Decoding steps in a graph: the token is written, the lengths advance, replay by replay; two graphs and an eager step take turns."""
    c = Cache(21, [3, 600, 30], 16, 2, 64, 64, BF16, spare=40, fill=0.0)
    kp, vp, table, lens = c.to(cuda)
    q, kn, vn = (gen(60 + i, 3, 1, h, 64, dtype=BF16).to(cuda) for i, h in enumerate((4, 2, 2)))
    twin = [x.clone() for x in (kp, vp, lens)]

    def step(kp, vp, lens):
        o = L.paged_attn_decode(q, kp, vp, table, lens, kn, vn, head_first=False)
        lens += 1
        return o

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kp.clone(), vp.clone(), lens.clone())
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step(kp, vp, lens)
        graphs.append((g, o))
    for i in range(8):
        for x, s in ((q, 1000), (kn, 2000), (vn, 3000)):
            x.copy_(gen(s + i, *x.shape, dtype=BF16))
        g, o = graphs[i % 2]
        g.replay()
        got = o.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step(*twin)), i
        assert torch.equal(kp, twin[0]) and torch.equal(vp, twin[1]) and torch.equal(lens, twin[2])


def test_sequences_that_share_pages(cuda):
    """Two sequences with the same pages in front (a shared prompt), each with its own last page."""
    c = Cache(23, [40, 0], 16, 1, 64, 64, BF16, spare=8)
    kp, vp, table, lens = c.to(cuda)
    table[1, :2] = table[0, :2]
    table[1, 2] = int(c.table[1, 0])
    kp[table[1, 2].long(), :8], vp[table[1, 2].long(), :8] = kp[table[0, 2].long(), :8].clone(), vp[table[0, 2].long(), :8].clone()
    lens.fill_(40)
    q = gen(1, 1, 1, 2, 64, dtype=BF16).to(cuda).expand(2, 1, 2, 64).contiguous()
    o = L.paged_attn_decode(q, kp, vp, table, lens, head_first=False)
    assert torch.equal(o[0], o[1])
    softmax.check(o[0, :, 0], softmax.head(q[0, :, 0].cpu(), c.rows[0][0][:, 0], c.rows[0][1][:, 0], 0.125, dtype=BF16))
