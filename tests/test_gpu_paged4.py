"""The cache in 4 bits on the GPU: what is written bit for bit (oracle/kv4.py), what is read back, and attention of one token over it
against float64 within the bounds of oracle/softmax.py, on the values that the cache holds."""
import pytest
import torch

import linear_moe_amd as L
from oracle import kv4, softmax
from tests.util import gen

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


class Cache4:
    """Pages of sequences in shuffled order; what no token owns is NaN (scale 255)."""

    def __init__(self, seed, lens, S, HKV, K, V, spare=1, heads_first=True, random_scales=False):
        g = torch.Generator().manual_seed(seed)
        self.S, self.lens = S, list(lens)
        need = [(n + spare + S - 1) // S for n in lens]
        P = sum(need) + 2
        ids = torch.randperm(P, generator=g).tolist()
        self.table = torch.full((len(lens), max(need) + 1), -7, dtype=torch.int32)
        at = 0
        for n, m in enumerate(need):
            self.table[n, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
            at += m
        shape = (P, HKV, S) if heads_first else (P, S, HKV)
        self.x = [torch.full((*shape, d), f, dtype=torch.uint8) for d, f in ((K // 2, 0x55), (K // 32, 255), (V // 2, 0x55), (V // 32, 255))]
        if heads_first:
            self.x = [y.transpose(1, 2) for y in self.x]
        self.rows = []
        for n, m in enumerate(lens):
            parts = []
            for i, D in enumerate((K, V)):
                codes, scales = kv4.pack(gen(seed + 2 * n + i + 1, m, HKV, D))
                if random_scales:
                    scales = torch.randint(120, 132, scales.shape, generator=g, dtype=torch.uint8)
                parts += [codes, scales]
            self.rows.append(parts)
            for j in range(m):
                self.put(n, j, [p[j] for p in parts])

    def put(self, n, j, parts):
        page = int(self.table[n, j // self.S])
        for y, p in zip(self.x, parts):
            y[page, j % self.S] = p

    def to(self, dev):
        out = [torch.empty_strided(y.shape, y.stride(), dtype=y.dtype, device=dev).copy_(y) for y in self.x]
        return out, self.table.to(dev), torch.tensor(self.lens, dtype=torch.int32, device=dev)

    def same(self, out):
        return all(torch.equal(a.cpu(), b) for a, b in zip(out, self.x))


def alibi(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)])


def decode_and_check(cuda, c, HQ, K, V, dtype, append=False, softcap=0.0, slopes=None, head_first=False, seed=900):
    HKV, N = c.x[0].shape[2], len(c.lens)
    G = HQ // HKV
    q, kn, vn = gen(seed, N, 1, HQ, K, dtype=dtype), gen(seed + 1, N, 1, HKV, K, dtype=dtype), gen(seed + 2, N, 1, HKV, V, dtype=dtype)
    (kp, ks, vp, vs), table, lens = c.to(cuda)
    lay = (lambda x: x.transpose(1, 2)) if head_first else (lambda x: x)
    new = dict(k=lay(kn.to(cuda)), v=lay(vn.to(cuda))) if append else {}
    o = lay(L.paged_attn_decode(lay(q.to(cuda)), kp, vp, table, lens, softcap=softcap, slopes=None if slopes is None else slopes.to(cuda),
                                head_first=head_first, k_scales=ks, v_scales=vs, **new))
    assert o.shape == (N, 1, HQ, V) and o.dtype == dtype
    fresh = [(*kv4.pack(kn[n, 0]), *kv4.pack(vn[n, 0])) for n in range(N)]
    if append:
        for n, m in enumerate(c.lens):
            if m // c.S < c.table.shape[1]:
                c.put(n, m, fresh[n])
    assert c.same((kp, ks, vp, vs))                       # the new token where it belongs, nothing else touched
    for n in range(N):
        rows = [torch.cat([a, b[None]]) for a, b in zip(c.rows[n], fresh[n])] if append else c.rows[n]
        kk, vv = kv4.values(*rows[:2]), kv4.values(*rows[2:])
        if kk.shape[0] == 0:
            assert (o[n] == 0).all()
            continue
        for h in range(HQ):
            slope = 0.0 if slopes is None else float(slopes[h])
            ref, tol = softmax.head(q[n, :, h], kk[:, h // G], vv[:, h // G], K ** -0.5, True, softcap, slope, dtype=dtype)
            off = (o[n, :, h].cpu().double() - ref).abs()
            assert (off <= tol).all(), (n, h, (off / tol).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("K,V", [(128, 128), (64, 64), (32, 32), (96, 96), (128, 32), (32, 128), (64, 96), (96, 64)])
def test_dims(cuda, dtype, append, K, V):
    decode_and_check(cuda, Cache4(3, [70, 1, 33, 0], 16, 2, K, V), 8, K, V, dtype, append)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("S", [1, 3, 16, 24, 32, 64, 100])
@pytest.mark.parametrize("heads_first", [True, False])
def test_pages(cuda, dtype, S, heads_first):
    lens = [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200]
    decode_and_check(cuda, Cache4(17, lens, S, 1, 64, 64, heads_first=heads_first), 2, 64, 64, dtype, append=True, head_first=S % 2 == 0)
    decode_and_check(cuda, Cache4(18, lens[::-1], S, 1, 128, 128, heads_first=heads_first), 1, 128, 128, dtype)


@pytest.mark.parametrize("HQ,HKV", [(1, 1), (16, 1), (17, 1), (40, 2), (15, 3), (33, 1)])
def test_heads(cuda, HQ, HKV):
    decode_and_check(cuda, Cache4(5, [45, 2], 16, HKV, 64, 64), HQ, 64, 64, BF16, append=True)


@pytest.mark.parametrize("softcap,bias", [(0.0, True), (20.0, False), (5.0, True)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_options(cuda, softcap, bias, dtype):
    for K in (64, 128):
        decode_and_check(cuda, Cache4(6, [90, 1, 0, 700], 32, 2, K, K), 6, K, K, dtype, True, softcap, alibi(6) if bias else None)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("append", [False, True])
def test_long(cuda, dtype, append):
    """Several stretches, joined; ends inside tiles, of a stretch and behind one."""
    decode_and_check(cuda, Cache4(8, [3001, 512, 511, 513, 1024, 0, 1025, 2047], 64, 1, 64, 64, random_scales=True), 4, 64, 64, dtype, append)
    decode_and_check(cuda, Cache4(9, [1700, 5], 100, 2, 128, 128), 4, 128, 128, dtype, append)


def test_pages_that_are_none(cuda):
    """Positions whose page is no page take no part; a new token without one is attended to, not kept; nothing at all gives zeros."""
    c = Cache4(10, [100, 40, 20], 16, 2, 64, 64)
    c.table[0, 1], c.table[0, 3] = -1, 2 ** 31 - 1
    c.table[1, :] = -5
    c.table[2, 1] = c.x[0].shape[0]
    keep = [[j for j in range(m) if 0 <= int(c.table[n, j // 16]) < c.x[0].shape[0]] for n, m in enumerate(c.lens)]
    q = gen(90, 3, 1, 4, 64, dtype=BF16)
    (kp, ks, vp, vs), table, lens = c.to(cuda)
    o = L.paged_attn_decode(q.to(cuda), kp, vp, table, lens, head_first=False, k_scales=ks, v_scales=vs)
    for n in range(3):
        kk, vv = kv4.values(*[p[keep[n]] for p in c.rows[n][:2]]), kv4.values(*[p[keep[n]] for p in c.rows[n][2:]])
        if not keep[n]:
            assert (o[n] == 0).all()
            continue
        for h in range(4):
            ref, tol = softmax.head(q[n, :, h], kk[:, h // 2], vv[:, h // 2], 0.125, False, dtype=BF16)
            assert ((o[n, :, h].cpu().double() - ref).abs() <= tol).all()
    k, v = gen(91, 3, 1, 2, 64, dtype=BF16).to(cuda), gen(92, 3, 1, 2, 64, dtype=BF16).to(cuda)
    full = torch.tensor([16 * c.table.shape[1]] * 3, dtype=torch.int32, device=cuda)
    table.fill_(-1)
    o = L.paged_attn_decode(q.to(cuda), kp, vp, table, full, k=k, v=v, head_first=False, k_scales=ks, v_scales=vs)
    assert c.same((kp, ks, vp, vs))
    held = kv4.values(*kv4.pack(v.cpu()))
    for h in range(4):
        assert torch.equal(o[:, 0, h].cpu().double(), held[:, 0, h // 2])
    lens.fill_(-3)                                             # as an empty cache, and a token that has no position
    o = L.paged_attn_decode(q.to(cuda), kp, vp, table, lens, head_first=False, k_scales=ks, v_scales=vs)
    assert (o == 0).all()


def test_many_sequences_and_heads_next_to_each_other(cuda):
    """Both orders of the work-groups, with stretches of their own for every head."""
    lens = [(37 * i) % 70 for i in range(50)]
    for heads_first in (True, False):
        decode_and_check(cuda, Cache4(14, lens, 16, 3, 64, 64, heads_first=heads_first), 6, 64, 64, BF16, append=True)
        decode_and_check(cuda, Cache4(15, [2500, 1, 1100, 40, 2048, 1024, 0, 7, 1025], 16, 2, 64, 64, heads_first=heads_first), 2, 64, 64, BF16)


@pytest.mark.parametrize("heads_first", [True, False])
@pytest.mark.parametrize("cols", [129, 257, 1100, 12800])
def test_tables_wider_than_their_sequences(cuda, cols, heads_first):
    """2 to 64 stretches that the table has room for, of which the sequences have none to four."""
    c = Cache4(19, [2500, 1, 0, 1024, 1025, 4000], 16, 2, 64, 64, heads_first=heads_first)
    if cols < c.table.shape[1]:
        c = Cache4(20, [2000, 1, 0, 1024, 1025], 16, 2, 64, 64, heads_first=heads_first)
    c.table = torch.cat([c.table, torch.full((len(c.lens), max(cols - c.table.shape[1], 0)), -1, dtype=torch.int32)], 1)
    decode_and_check(cuda, c, 4, 64, 64, BF16, append=True)


def test_fewer_stretches_than_a_long_sequence_would_have(cuda):
    """So many sequences and heads that a stretch is longer than it is for a few."""
    decode_and_check(cuda, Cache4(21, [9000] + [i % 4 for i in range(1499)], 16, 2, 32, 32), 2, 32, 32, BF16)
    N, HKV, D, S = 256, 64, 32, 16                                       # one stretch each, whatever its length
    lens = [1500] + [(5 * i) % 40 for i in range(1, N - 1)] + [1300]
    need = [(n + S - 1) // S for n in lens]
    table = torch.full((N, max(need)), -1, dtype=torch.int32)
    at = 0
    for n, m in enumerate(need):
        table[n, :m] = torch.arange(at, at + m)
        at += m
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)
    k, v, q = gen(300, 1, sum(lens), HKV, D, dtype=BF16), gen(301, 1, sum(lens), HKV, D, dtype=BF16), gen(302, N, 1, HKV, D, dtype=BF16)
    kp, ks, vp, vs = (torch.empty(at, HKV, S, d, dtype=torch.uint8, device=cuda).transpose(1, 2) for d in (D // 2, 1, D // 2, 1))
    sc = dict(k_scales=ks, v_scales=vs, head_first=False)
    L.paged_kv_append(kp, vp, k.to(cuda), v.to(cuda), table.to(cuda), torch.zeros(N, dtype=torch.int32, device=cuda), cu_seqlens=cu, **sc)
    o = L.paged_attn_decode(q.to(cuda), kp, vp, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), **sc).cpu().double()
    for n in (0, 1, 8, 100, N - 2, N - 1):
        if not lens[n]:
            assert (o[n] == 0).all()
            continue
        kk, vv = (kv4.values(*kv4.pack(x[0, cu[n]:cu[n + 1]])) for x in (k, v))
        for h in range(0, HKV, 9):
            ref, tol = softmax.head(q[n, :, h], kk[:, h], vv[:, h], D ** -0.5, dtype=BF16)
            assert ((o[n, :, h] - ref).abs() <= tol).all(), (n, h)


@pytest.mark.parametrize("heads_first", [True, False])
def test_one_stretch_for_many_work_groups(cuda, heads_first):
    """Tables of up to 5120 positions and two work-groups a CU; with the heads of a token next to each other, several stretches."""
    decode_and_check(cuda, Cache4(24, [5000, 2049, 0] + [i % 4 for i in range(300)], 16, 2, 32, 32, heads_first=heads_first), 2, 32, 32, BF16, append=True)
    decode_and_check(cuda, Cache4(25, [2000] + [i % 3 for i in range(40)], 24, 3, 64, 64, heads_first=heads_first), 3, 64, 64, F32)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tables_past_the_caches(cuda, dtype):
    """Tables of more than 256 MB of positions, most of them of no page: whole rows of 128 columns, and 96."""
    for D in (128, 96):
        c = Cache4(26, [300, 0, 1100, 33], 16, 2, D, D)
        c.table = torch.cat([c.table, torch.full((4, 16000), -1, dtype=torch.int32)], 1)
        decode_and_check(cuda, c, 4, D, D, dtype, append=True)
    c = Cache4(27, [4000, 1] + [i % 3 for i in range(300)], 16, 2, 128, 128)
    c.table = torch.cat([c.table, torch.full((302, 319 - c.table.shape[1]), -1, dtype=torch.int32)], 1)
    decode_and_check(cuda, c, 2, 128, 128, dtype, softcap=20.0, slopes=alibi(2))


def test_two_at_once(cuda):
    """Steps of two caches on two streams at the same time, and in inference mode: the bits of each by itself."""
    caches = [Cache4(22 + i, [4000, 70, 1500], 16, 2, 128, 128, spare=8) for i in range(2)]
    held = [c.to(cuda) for c in caches]
    q, k, v = (gen(310 + i, 3, 1, h, 128, dtype=BF16).to(cuda) for i, h in enumerate((8, 2, 2)))

    def steps(h, i):
        (kp, ks, vp, vs), table, lens = h
        out = []
        for j in range(4):
            out.append(L.paged_attn_decode(q * (i + 1), kp, vp, table, lens, k=k + j, v=v - j, head_first=False, k_scales=ks, v_scales=vs))
            lens += 1
        return out + list(L.paged_kv_read(kp, vp, table, lens - 20, 20, head_first=False, k_scales=ks, v_scales=vs))
    with torch.inference_mode():
        want = [steps(c.to(cuda), i) for i, c in enumerate(caches)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            got.append(steps(held[i], i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(want, got) for a, b in zip(x, y))


def test_a_score_that_grows(cuda):
    """Maxima that move late and by much, and ones that move by less than 2^8: the sums stay those of the definition."""
    for step, scale in ((0.02, 1.0), (0.3, 1.0), (3.0, 1.0), (-3.0, 1.0)):
        c = Cache4(16, [700], 16, 1, 64, 64)
        q = gen(80, 1, 1, 2, 64, dtype=BF16)
        # keys along q, longer and longer (in 4 bits: what the format keeps of them)
        grow = (1 + step * torch.arange(700).float() / 50) * scale
        kk = kv4.pack(q[0, 0, :1].float() * grow[:, None, None])
        c.rows[0][:2] = kk
        for j in range(700):
            c.put(0, j, [p[j] for p in c.rows[0]])
        (kp, ks, vp, vs), table, lens = c.to(cuda)
        o = L.paged_attn_decode(q.to(cuda), kp, vp, table, lens, head_first=False, k_scales=ks, v_scales=vs)
        for h in range(2):
            ref, tol = softmax.head(q[0, :, h], kv4.values(*c.rows[0][:2])[:, 0], kv4.values(*c.rows[0][2:])[:, 0], 0.125, dtype=BF16)
            assert ((o[0, :, h].cpu().double() - ref).abs() <= tol).all()


def test_nan_in_a_token_that_nobody_sees(cuda):
    """Slots behind a sequence hold NaN in all these tests; one that is seen makes its head NaN."""
    c = Cache4(11, [50], 16, 2, 64, 64)
    (kp, ks, vp, vs), table, lens = c.to(cuda)
    q = gen(93, 1, 1, 4, 64, dtype=BF16).to(cuda)
    ks[int(c.table[0, 1]), 3, 1, 0] = 255
    o = L.paged_attn_decode(q, kp, vp, table, lens, head_first=False, k_scales=ks, v_scales=vs)
    assert o[0, 0, :2].isfinite().all() and o[0, 0, 2:].isnan().all()


def edge_rows():
    """Every bfloat16 there is, and rows around the borders of the format."""
    every = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(BF16)
    rows = [every]                                             # (32 neighbours share a scale)
    g = torch.Generator().manual_seed(1)
    for e in (-126, -121, -120, -119, -118, -3, 0, 1, 120, 124, 125, 126, 127):
        y = torch.rand(64, generator=g) * 2 - 1
        y[0] = 1.0
        rows += [(y * m).double().mul(2.0 ** e).to(BF16) for m in (1.0, 1.5, 1.5078125, 1.9921875)]
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]).repeat(4) * torch.tensor([1.0, -1.0]).repeat_interleave(16)
    rows += [ties.to(BF16), torch.zeros(32, dtype=BF16), -torch.zeros(32, dtype=BF16)]
    return torch.cat(rows)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_is_written_and_read(cuda, dtype):
    x = edge_rows().to(dtype)
    if dtype == F32:                                           # and numbers between two bfloat16
        y = x.view(torch.int32).clone()
        x = torch.cat([x, (y + 1).view(F32), (y + 0x7fff).view(F32)])
    x = torch.cat([x, torch.zeros(-x.numel() % 128, dtype=dtype)]).view(1, -1, 1, 128)
    T, S = x.shape[1], 16
    P = (T + S - 1) // S
    for heads_first in (True, False):
        st = [torch.full((P, S, 1, d), 77, dtype=torch.uint8, device=cuda) for d in (64, 4, 64, 4)]
        table, lens = torch.arange(P, dtype=torch.int32, device=cuda)[None], torch.zeros(1, dtype=torch.int32, device=cuda)
        L.paged_kv_append(st[0], st[2], x.to(cuda), x.to(cuda), table, lens, head_first=False, k_scales=st[1], v_scales=st[3])
        codes, scales = kv4.pack(x[0])
        for i in (0, 2):
            got = [y.flatten(0, 1)[:T].cpu() for y in st[i:i + 2]]
            ok = (scales != 255).repeat_interleave(16, -1)
            assert torch.equal(got[1], scales) and torch.equal(got[0][ok], codes[ok])       # (codes under a NaN say nothing)
            assert (st[i].flatten(0, 1)[T:] == 77).all() and (st[i + 1].flatten(0, 1)[T:] == 77).all()
        want = kv4.values(codes, scales)
        for out in (BF16, F32):
            for y in L.paged_kv_read(st[0], st[2], table, lens, T, head_first=False, k_scales=st[1], v_scales=st[3], dtype=out):
                assert y.dtype == out and torch.equal(y[0].cpu().double().nan_to_num(nan=7e77), want.nan_to_num(nan=7e77))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bits4", [True, False])
@pytest.mark.parametrize("K,V,HKV,S", [(128, 128, 8, 16), (96, 32, 3, 24), (64, 64, 1, 5), (32, 64, 5, 100)])
def test_append_and_read(cuda, dtype, bits4, K, V, HKV, S):
    """Packed and padded prompts onto caches that hold something, read back; rows behind the last sequence and pages that are none."""
    starts, new = [0, 5, 16, 100, 7], [37, 0, 1, 64, 3]
    N, T = len(new), sum(new) + 4
    need = [(a + b + S - 1) // S for a, b in zip(starts, new)]
    P = sum(need) + 1
    ids = torch.randperm(P, generator=torch.Generator().manual_seed(2)).tolist()
    table, at = torch.full((N, max(need)), -1, dtype=torch.int32), 0
    for n, m in enumerate(need):
        table[n, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
        at += m
    table[3, (100 // S) + 1:] = P                                # the rest of sequence 3 has no pages
    k, v = gen(70, 1, T, HKV, K, dtype=dtype), gen(71, 1, T, HKV, V, dtype=dtype)
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=cuda)
    table_d, starts_d = table.to(cuda), torch.tensor(starts, dtype=torch.int64, device=cuda)
    if bits4:
        kp, ks, vp, vs = (torch.zeros(P, S, HKV, d, dtype=torch.uint8, device=cuda) for d in (K // 2, K // 32, V // 2, V // 32))
        sc = dict(k_scales=ks, v_scales=vs)
        held = [kv4.values(*kv4.pack(x)).to(dtype) for x in (k, v)]
    else:
        kp, vp = (torch.zeros(P, S, HKV, d, dtype=dtype, device=cuda) for d in (K, V))
        sc, held = {}, [k, v]
    L.paged_kv_append(kp, vp, k.to(cuda), v.to(cuda), table_d, starts_d, cu_seqlens=cu, head_first=False, **sc)
    got = L.paged_kv_read(kp, vp, table_d, starts_d, T, cu_seqlens=cu, head_first=False, dtype=dtype, **sc)
    last = (100 // S + 1) * S - 100                              # tokens of sequence 3 that have a page
    at = 0
    for n, m in enumerate(new):
        for y, want in zip(got, held):
            keep = min(m, last) if n == 3 else m
            assert torch.equal(y[0, at:at + keep].cpu(), want[0, at:at + keep]), n
            assert (y[0, at + keep:at + m] == 0).all()
        at += m
    assert all((y[0, at:] == 0).all() for y in got)
    # padded, heads first: the same rows by sequence
    most = max(new)
    for y, want in zip(L.paged_kv_read(kp, vp, table_d, starts_d, most, dtype=dtype, **sc), held):
        assert y.shape[:3] == (N, HKV, most)
        at = 0
        for n, m in enumerate(new):
            keep = min(m, last) if n == 3 else m
            assert torch.equal(y[n, :, :keep].cpu().transpose(0, 1), want[0, at:at + keep])
            at += m
    # written once more, from padded rows: the same bytes
    before = [x.clone() for x in (kp, vp, *sc.values())]
    kk, vv = L.paged_kv_read(kp, vp, table_d, starts_d, most, dtype=dtype, **sc)
    L.paged_kv_append(kp, vp, kk, vv, table_d, starts_d, **sc)
    if bits4:
        again = L.paged_kv_read(kp, vp, table_d, starts_d, most, dtype=dtype, **sc)
        assert torch.equal(again[0], kk) and torch.equal(again[1], vv)       # (what 4 bits hold stays what it is)
    else:
        assert all(torch.equal(a, b) for a, b in zip(before, (kp, vp)))


def test_large_results_are_read(cuda):
    """More than goes through the caches."""
    P, S, H, D = 80, 64, 16, 128
    for bits4 in (True, False):
        k, v = (gen(72 + i, 1, P * S, H, D, dtype=BF16).to(cuda) for i in range(2))
        table, zero = torch.arange(P, dtype=torch.int32, device=cuda)[None], torch.zeros(1, dtype=torch.int32, device=cuda)
        sc = dict(zip(("k_scales", "v_scales"), (torch.empty(P, S, H, D // 32, dtype=torch.uint8, device=cuda) for _ in range(2)))) if bits4 else {}
        kp, vp = (torch.empty(P, S, H, D // 2, dtype=torch.uint8, device=cuda) if bits4 else torch.empty(P, S, H, D, dtype=BF16, device=cuda) for _ in range(2))
        L.paged_kv_append(kp, vp, k, v, table, zero, head_first=False, **sc)
        for f32 in (False, True) if bits4 else (False,):
            got = L.paged_kv_read(kp, vp, table, zero, P * S, head_first=False, dtype=F32 if f32 else BF16, **sc)
            for x, y in zip(got, (k, v)):
                want = kv4.values(*kv4.pack(y)) if bits4 else y.double()
                assert torch.equal(x.double(), want)


def test_strides(cuda):
    """Pages as parts of larger tensors: keys and values of one buffer, every second page, heads in another order; scales with any strides."""
    c = Cache4(12, [70, 3], 16, 2, 64, 64)
    (kp, ks, vp, vs), table, lens = c.to(cuda)
    P, S, H, B = kp.shape
    q, kn, vn = (gen(94 + i, 2, 1, h, 64, dtype=BF16).to(cuda) for i, h in enumerate((4, 2, 2)))
    both = torch.zeros(2 * P, S, H + 1, 2, B, dtype=torch.uint8, device=cuda)
    k2, v2 = both[::2, :, 1:, 0], both[::2, :, 1:, 1]
    sc = torch.zeros(P, H, 3, S, 2, dtype=torch.uint8, device=cuda)
    ks2, vs2 = sc[:, :, 0].transpose(1, 2), sc[:, :, 2].transpose(1, 2)
    for a, b in ((k2, kp), (v2, vp), (ks2, ks), (vs2, vs)):
        a.copy_(b)
    a = L.paged_attn_decode(q, kp, vp, table, lens, k=kn, v=vn, head_first=False, k_scales=ks, v_scales=vs)
    b = L.paged_attn_decode(q, k2, v2, table, lens, k=kn, v=vn, head_first=False, k_scales=ks2, v_scales=vs2)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in ((k2, kp), (v2, vp), (ks2, ks), (vs2, vs)))
    assert (both[1::2] == 0).all() and (both[:, :, 0] == 0).all() and (sc[:, :, 1] == 0).all()
    wide = torch.full((2, 40), -1, dtype=torch.int64, device=cuda)
    wide[:, 1:1 + 2 * table.shape[1]:2] = table
    c2 = L.paged_attn_decode(q, kp, vp, wide[:, 1:1 + 2 * table.shape[1]:2], lens.long(), k=kn, v=vn, head_first=False, k_scales=ks, v_scales=vs)
    assert torch.equal(a, c2)


@pytest.mark.parametrize("S", [64, 60])
def test_far_pages(cuda, S):
    """Offsets beyond 2^32 bytes."""
    P, H, D = 40000, 16, 128                             # 2.6e9 bytes of codes
    k = torch.empty(P, H, S, D // 2, dtype=torch.uint8, device=cuda).transpose(1, 2)
    v = torch.empty(P, H, S, D // 2, dtype=torch.uint8, device=cuda).transpose(1, 2)
    ks, vs = (torch.empty(P, H, S, D // 32, dtype=torch.uint8, device=cuda).transpose(1, 2) for _ in range(2))
    both = torch.empty(2 * P, H, S, D // 2, dtype=torch.uint8, device=cuda)       # 5.2e9: every second page
    k = both[1::2].transpose(1, 2)
    far, near = torch.tensor([[P - 1, P - 2]], dtype=torch.int32, device=cuda), torch.tensor([[0, 1]], dtype=torch.int32, device=cuda)
    kn, vn = (gen(95 + i, 1, 100, H, D, dtype=BF16).to(cuda) for i in range(2))
    zero, q = torch.zeros(1, dtype=torch.int32, device=cuda), gen(97, 1, 1, H, D, dtype=BF16).to(cuda)
    out = []
    for table in (near, far):
        L.paged_kv_append(k, v, kn, vn, table, zero, head_first=False, k_scales=ks, v_scales=vs)
        out.append([L.paged_attn_decode(q, k, v, table, zero + 100, head_first=False, k_scales=ks, v_scales=vs),
                    *L.paged_kv_read(k, v, table, zero, 100, head_first=False, k_scales=ks, v_scales=vs)])
    assert all(torch.equal(a, b) for a, b in zip(*out)) and out[0][0].isfinite().all()
    assert torch.equal(out[1][1].cpu().double(), kv4.values(*kv4.pack(kn.cpu())))


def test_graph(cuda):
    """A step of writing and attending, captured and replayed while lens and the table move on."""
    c = Cache4(13, [30, 1, 500], 16, 2, 128, 128, spare=8)
    (kp, ks, vp, vs), table, lens = c.to(cuda)
    twin = [x.clone() for x in (kp, vp, ks, vs)]
    q, k, v = (torch.empty(3, 1, h, 128, dtype=BF16, device=cuda) for h in (8, 2, 2))
    step = lambda a, b, s, t: L.paged_attn_decode(q, a, b, table, lens, k=k, v=v, head_first=False, k_scales=s, v_scales=t)
    fill = lambda i: [x.copy_(gen(200 + 3 * i + j, *x.shape, dtype=BF16)) for j, x in enumerate((q, k, v))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    fill(0)
    with torch.cuda.stream(side):
        step(kp, vp, ks, vs)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = step(kp, vp, ks, vs)
    for i in range(1, 6):
        fill(i)
        g.replay()
        want = step(*twin)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and all(torch.equal(a, b) for a, b in zip((kp, vp, ks, vs), twin))
        lens += 1


def test_no_pages_and_no_sequences(cuda):
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=cuda)
    none, i32 = u8(0, 16, 2, 32), dict(dtype=torch.int32, device=cuda)
    q, k = gen(1, 2, 1, 4, 64, dtype=BF16).to(cuda), gen(2, 2, 1, 2, 64, dtype=BF16).to(cuda)
    sc = dict(k_scales=u8(0, 16, 2, 2), v_scales=u8(0, 16, 2, 2), head_first=False)
    for cols in (0, 3):
        table, lens = torch.zeros(2, cols, **i32), torch.tensor([5, 0], **i32)
        assert (L.paged_attn_decode(q, none, none, table, lens, **sc) == 0).all()
        o = L.paged_attn_decode(q, none, none, table, lens, k=k, v=k, **sc)
        assert torch.equal(o[:, :, ::2].cpu().double(), kv4.values(*kv4.pack(k.cpu())))
        L.paged_kv_append(none, none, k, k, table, lens, **sc)
        assert all((x == 0).all() for x in L.paged_kv_read(none, none, table, lens, 3, **sc))
    table, lens = torch.zeros(0, 3, **i32), torch.zeros(0, **i32)
    assert L.paged_attn_decode(q[:0], none, none, table, lens, **sc).shape == (0, 1, 4, 64)
    L.paged_kv_append(none, none, k[:0], k[:0], table, lens, **sc)
    assert [x.shape for x in L.paged_kv_read(none, none, table, lens, 3, **sc)] == [(0, 3, 2, 64)] * 2


def test_refusals(cuda):
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=cuda)
    kp, ks = u8(4, 16, 2, 32), u8(4, 16, 2, 2)
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    q, k = torch.zeros(2, 1, 4, 64, device=cuda), torch.zeros(2, 1, 2, 64, device=cuda)
    ok = dict(k_pages=kp, v_pages=kp, page_table=table, k_scales=ks, v_scales=ks, head_first=False)
    L.paged_attn_decode(q=q, lens=lens, **ok)
    bad = [dict(k_scales=None), dict(v_scales=None), dict(k_scales=ks.int()), dict(k_scales=ks[:3]), dict(k_scales=ks[..., :1]), dict(k_scales=ks.cpu()),
           dict(k_scales=u8(4, 16, 2, 4)[..., ::2]), dict(k_pages=kp.float(), v_pages=kp.float()), dict(v_pages=kp.int()), dict(k_pages=u8(4, 16, 2, 24)),
           dict(k_pages=u8(4, 16, 2, 80), v_pages=u8(4, 16, 2, 80), k_scales=u8(4, 16, 2, 5), v_scales=u8(4, 16, 2, 5)), dict(k_pages=u8(4, 16, 2, 33)[..., 1:]),
           dict(page_table=table.float()), dict(page_table=table[0])]
    for change in bad:
        with pytest.raises(ValueError):
            L.paged_attn_decode(**{**dict(q=q, lens=lens), **ok, **change})
        with pytest.raises(ValueError):
            L.paged_kv_append(**{**dict(k=k, v=k, lens=lens), **ok, **change})
        with pytest.raises(ValueError):
            L.paged_kv_read(**{**dict(starts=lens, T=2), **ok, **change})
    for change in (dict(q=q.half()), dict(q=q[:1]), dict(q=q[:, :, :3]), dict(k=k), dict(k=k.bfloat16(), v=k.bfloat16()), dict(lens=lens[:1]), dict(lens=lens.float()),
                   dict(softcap=-1.0)):
        with pytest.raises(ValueError):
            L.paged_attn_decode(**{**dict(q=q, lens=lens), **ok, **change})
    for change in (dict(k=k.half(), v=k.half()), dict(v=k.bfloat16()), dict(k=k[:1]), dict(cu_seqlens=torch.tensor([0, 1, 2], device=cuda), head_first=True)):
        with pytest.raises(ValueError):
            L.paged_kv_append(**{**dict(k=k, v=k, lens=lens), **ok, **change})
    for change in (dict(T=-1), dict(T=2 ** 31), dict(dtype=torch.float16), dict(cu_seqlens=torch.tensor([0, 1, 3])), dict(cu_seqlens=torch.tensor([0, 1], device=cuda))):
        with pytest.raises(ValueError):
            L.paged_kv_read(**{**dict(starts=lens, T=2), **ok, **change})
    with pytest.raises(ValueError):
        L.paged_kv_read(kp.bfloat16(), kp.bfloat16(), table, lens, 2, dtype=torch.float32)
    with pytest.raises(RuntimeError):
        L.paged_attn_decode(q=q.requires_grad_(True), lens=lens, **ok)
    with pytest.raises(RuntimeError):
        L.paged_kv_append(k=k.clone().requires_grad_(True), v=k, lens=lens, **ok)
