"""What stands around the softmax layers of a hybrid model: the norms and the rotation of queries and keys, a cache of keys and
values in 4 bits (written, read back, attended to), and the pages of a cache (given out, shared, copied on write, moved together, freed).

``listed()`` are fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds before the
call, ``run`` is one pass, ``work`` what that pass cannot do without and ``exact`` the same outputs in 64 bits.  With ``own``
false ``run`` computes the operators with elementary torch operations in 32 bits, rounded once at the end; with ``own``
true it makes the calls a user makes of the package."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GROUP = 32            # columns that share a scale in the 4-bit cache
EPS = 1e-6
BASE = 10000.0        # of the rotation's frequencies


def _rope(name, B, T, HQ, HKV, D, R=None, dtype="bf16", interleaved=False, weights=True, docs=0, start=0, grad=True):
    return dict(name=name, op="rope", B=B, T=T, HQ=HQ, HKV=HKV, D=D, R=D if R is None else R, dtype=dtype, interleaved=interleaved,
                weights=weights, docs=docs, start=start, grad=grad)


def _decode(name, N, L, HQ, HKV, D, page, dtype="bf16", softcap=0.0, slopes=False, append=False, heads_first=True):
    return dict(name=name, op="decode", N=N, L=L, HQ=HQ, HKV=HKV, D=D, page=page, dtype=dtype, softcap=softcap, slopes=slopes,
                append=append, heads_first=heads_first)


def _append(name, N, T, HKV, D, page, dtype="bf16", heads_first=True):
    return dict(name=name, op="append", N=N, T=T, HKV=HKV, D=D, page=page, dtype=dtype, heads_first=heads_first)


def _pages(name, N, L, HKV, D, page, ended, defrag=False, dtype="bf16"):
    return dict(name=name, op="pages", N=N, L=L, HKV=HKV, D=D, page=page, ended=ended, defrag=defrag, dtype=dtype)


def listed():
    return [
        # a generated token of one conversation: nothing but latency
        _rope("rope_token", 1, 1, 16, 4, 128, start=500, grad=False),
        # a long prompt, read in before generation: four query heads to a key head
        _rope("rope_prefill", 1, 8192, 32, 8, 128, grad=False),
        # training step on this package's headline shape (the largest case)
        _rope("rope_train", 4, 8192, 16, 4, 128),
        # training step on packed documents, half of the columns turned, neighbouring columns paired
        _rope("rope_train_packed", 1, 16381, 16, 8, 64, R=32, interleaved=True, docs=23),
        # a small layer in float32, without weights
        _rope("rope_train_f32", 2, 1000, 4, 2, 64, dtype="f32", weights=False),
        # one generated token of one conversation: latency
        _decode("decode4_1", 1, 500, 16, 4, 128, 16, append=True),
        # one generated token of a serving batch of unequal lengths
        _decode("decode4_64", 64, 4096, 32, 8, 128, 64),
        # one generated token over two very long documents
        _decode("decode4_long", 2, 131072, 16, 4, 128, 128),
        # the keys and values of seven prompts go into the cache, and come back as it holds them
        _append("append4_prompts", 7, 16384, 8, 128, 16),
        # those of one new token of each conversation, tokens of a page outside its heads
        _append("append4_tokens", 64, 64, 8, 128, 64, heads_first=False),
        # eight ways to go on from each of 32 conversations, of which half are dropped and taken again from others
        _pages("pages_fork", 256, 4096, 8, 128, 16, ended=128),
        # an eighth of the conversations ends, the cache is moved together, new prompts come
        _pages("pages_defrag", 64, 4096, 8, 128, 64, ended=8, defrag=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(("rope", "rope", "decode", "decode", "append", "pages"))
        dtype = "bf16" if rng.random() < 0.8 else "f32"
        G, HKV = rng.choice((1, 1, 2, 4, 5, 8)), rng.choice((1, 2, 3, 4, 8))
        page = rng.choice((16, 24, 32, 64, 100, 128))
        if op == "rope":
            D = rng.choice((64, 128, 128, 96, 80, 256, 36))
            T = _log_int(rng, 1, 16384)
            docs = min(T, _log_int(rng, 1, 40)) if rng.random() < 0.4 else 0
            B = 1 if docs else _log_int(rng, 1, 16)
            c = _rope(None, B, T, G * HKV, HKV, D, rng.choice((D, D, D // 4 * 2)), dtype, rng.random() < 0.4, rng.random() < 0.7, docs,
                      rng.choice((0, _log_int(rng, 1, 20000))), rng.random() < 0.6)
        elif op == "decode":
            c = _decode(None, _log_int(rng, 1, 128), _log_int(rng, 1, 65536), G * HKV, HKV, rng.choice((64, 128, 128, 96, 32)), page, dtype,
                        rng.choice((0.0, 0.0, 15.0, 50.0)), rng.random() < 0.3, rng.random() < 0.5, rng.random() < 0.7)
        elif op == "append":
            N = _log_int(rng, 1, 100)
            c = _append(None, N, max(N, _log_int(rng, 1, 16384)), HKV, rng.choice((64, 128, 128, 96, 32)), page, dtype, rng.random() < 0.7)
        else:
            N = _log_int(rng, 4, 300)
            defrag = rng.random() < 0.5
            c = _pages(None, N, _log_int(rng, 1, 8192), HKV, rng.choice((64, 128, 96)), page,
                       max(1, int(N * rng.uniform(0.05, 0.45 if defrag else 0.6))), defrag, dtype)
        # (the plain form of decoding spreads the cache out in 32 bits)
        if work(c)["bytes"] <= (2e8 if op == "decode" else most) and (op != "pages" or _pool(c) * page * HKV * c["D"] * 4 <= 2e9):
            del c["name"]
            return c


def _lengths(n, total):
    """n unequal lengths of one token at least (some of one), ``total`` together: the same for the same case."""
    rng = random.Random(n * 1000003 + total)
    w = [math.exp(rng.gauss(0.0, 1.2)) for _ in range(n)]
    free = total - n
    lens = [1 + int(free * x / sum(w)) for x in w]
    lens[0] += total - sum(lens)
    return lens


def _documents(case):
    return _lengths(case["docs"], case["T"]) if case["docs"] else [case["T"]] * case["B"]


def _cached(case):
    """Tokens per sequence of a case with a cache: from one to L."""
    N, L = case["N"], case["L"]
    return [max(1, round(L * (1.0 if N == 1 else 0.25 + 0.75 * i / (N - 1)))) for i in range(N)]


def _pool(case):
    """Pages of a case of pages: what all sequences hold, each of its own, with a page to grow, and some free ones."""
    S = case["page"]
    return sum(n // S + 2 for n in _cached(case)) + 8


def _defrag_groups(case):
    """Two groups of rows whose sequences end in turn, spread over the lengths."""
    N, E = case["N"], case["ended"]
    order = [i * N // (2 * E) for i in range(2 * E)]
    return order[::2], order[1::2]


def work(case):
    size, D, HKV = DTYPES[case["dtype"]].itemsize, case["D"], case["HKV"]
    row = D // 2 + D // GROUP                                       # a row of the 4-bit cache
    if case["op"] == "rope":
        tokens = case["B"] * case["T"]
        rows = tokens * (case["HQ"] + HKV)
        # q, k in and out, their gradients likewise; the table's rows that are met
        return {"bytes": rows * D * size * (4 if case["grad"] else 2) + max(_documents(case)) * case["R"] * 4,
                "flops": rows * D * (15 if case["grad"] else 6)}
    if case["op"] == "decode":
        tokens, new = sum(_cached(case)), case["N"] if case["append"] else 0
        moved = 2 * tokens * HKV * row + new * HKV * (2 * D * size + 2 * row + 2 * D * size) + 2 * case["N"] * case["HQ"] * D * size
        return {"bytes": moved, "flops": 4 * (tokens + new) * case["HQ"] * D}
    if case["op"] == "append":
        # in, the cache written, read, and out
        return {"bytes": case["T"] * HKV * (4 * D * size + 4 * row), "flops": 0}
    S = case["page"]
    held = [n // S + 1 for n in _cached(case)]
    block = 2 * S * HKV * D * size
    if case["defrag"]:
        moves = sum(held[i] for i in _defrag_groups(case)[0])
        M = max(held) + 1
        return {"bytes": 2 * moves * block + 8 * case["N"] * M + 12 * _pool(case), "flops": 0}
    E = case["ended"]
    entries = sum(held) * E / case["N"]
    return {"bytes": 2 * E * block + 12 * entries + 8 * _pool(case), "flops": 0}


def _slopes(H, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device=device)


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _table(positions, R, device):
    """cos and sin of position times frequency, angles in 64 bits."""
    freq = BASE ** (-torch.arange(0, R, 2, device=device, dtype=torch.float64) / R)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _cache(x, heads_first):
    """A random cache in 4 bits, [P, S, HKV, *] however it lies."""
    codes, scales = _to_4_bits(x)
    if heads_first:                                               # all tokens of a head next to each other inside a page
        codes, scales = (y.transpose(1, 2).contiguous().transpose(1, 2) for y in (codes, scales))
    return codes, scales


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    dt, D, HKV = DTYPES[case["dtype"]], case["D"], case["HKV"]
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev, dtype=dt)
    st = dict(case=case)
    if case["op"] == "rope":
        B, T, HQ = case["B"], case["T"], case["HQ"]
        lens = _documents(case)
        rng.shuffle(lens)
        qkv = randn(B, T, (HQ + 2 * HKV) * D)                    # one projection, of which q and k are views
        st.update(q=qkv[..., :HQ * D].view(B, T, HQ, D), k=qkv[..., HQ * D:(HQ + HKV) * D].view(B, T, HKV, D), lens=lens, cu=None, qw=None, kw=None,
                  offsets=None)
        start = [case["start"] - rng.randrange(case["start"] // 4 + 1) for _ in lens] if case["start"] else [0] * len(lens)
        st["start"] = start
        if case["start"]:
            st["offsets"] = torch.tensor(start, dtype=torch.int32, device=dev)
        st["cos"], st["sin"] = _table(max(lens) + case["start"], case["R"], dev)
        if case["docs"]:
            st["cu"] = torch.tensor(_offsets(lens), dtype=torch.int32, device=dev)
        if case["weights"]:
            st.update(qw=1 + 0.2 * randn(D), kw=1 + 0.2 * randn(D))
        if case["grad"]:
            st.update(dq=randn(B, T, HQ, D), dk=randn(B, T, HKV, D))
            st["leaves"] = [st[x].requires_grad_(True) for x in ("q", "k") + (("qw", "kw") if case["weights"] else ())]
        return st
    S, N = case["page"], case["N"]
    if case["op"] == "pages":
        return _prepare_pages(st, case, rng, randn, dev)
    # a cache: the pages of all sequences, shuffled, and a few that belong to none
    if case["op"] == "decode":
        start = _cached(case)
        rng.shuffle(start)
        fresh = [1 if case["append"] else 0] * N
        room = [(a + b + S - 1) // S for a, b in zip(start, fresh)]
    else:
        fresh = _lengths(N, case["T"])
        rng.shuffle(fresh)
        start = [rng.randrange(0, 2 * S) for _ in range(N)]
        room = [(2 * S - 1 + b + S - 1) // S for b in fresh]
    ids = list(range(sum(room) + 3))
    rng.shuffle(ids)
    table, at = torch.full((N, max(room)), -1, dtype=torch.int32), 0
    for n, m in enumerate(room):
        table[n, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
        at += m
    st["kp"], st["ks"] = _cache(randn(len(ids), S, HKV, D), case["heads_first"])
    st["vp"], st["vs"] = _cache(randn(len(ids), S, HKV, D), case["heads_first"])
    st.update(table=table.to(dev), start=start, fresh=fresh, lens=torch.tensor(start, dtype=torch.int32, device=dev),
              cu=torch.tensor(_offsets(fresh), dtype=torch.int32, device=dev), k=None, v=None)
    if case["op"] == "decode":
        st.update(q=randn(N, 1, case["HQ"], D), slopes=_slopes(case["HQ"], dev) if case["slopes"] else None)
        if case["append"]:
            st.update(k=randn(N, 1, HKV, D), v=randn(N, 1, HKV, D))
    else:
        st.update(k=randn(1, case["T"], HKV, D), v=randn(1, case["T"], HKV, D))
    return st


def _prepare_pages(st, case, rng, randn, dev):
    """Sequences with pages of their own (and one to grow into, where a length ends with its page), numbers shuffled."""
    S, N, E, P = case["page"], case["N"], case["ended"], _pool(case)
    lens = _cached(case)
    ids = list(range(sum(n // S + 1 for n in lens)))
    rng.shuffle(ids)
    table, refs, at = torch.full((N, max(lens) // S + 2), -1, dtype=torch.int32), torch.zeros(P, dtype=torch.int32), 0
    for n, a in enumerate(lens):
        m = a // S + 1
        table[n, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
        at += m
    refs[:at] = 1
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    st.update(pages=(randn(P, S, case["HKV"], case["D"]), randn(P, S, case["HKV"], case["D"])), table=table.to(dev), refs=refs.to(dev),
              lens=ints(lens), turn=0)
    if case["defrag"]:
        groups = _defrag_groups(case)
        st["ended"] = [ints(g) for g in groups]
        # (a new prompt as long as the one that ended there; a token for everybody else)
        st["tokens"] = [ints([lens[n] // S * S + 1 if n in set(g) else 1 for n in range(N)]) for g in groups]
    else:
        order = list(range(N))
        rng.shuffle(order)
        left = order[E:]
        st["ended"], st["src"] = ints(order[:E]), ints([rng.choice(left) for _ in range(E)])
        st["tokens"] = ints([1] * N)
    return st


def run(st):
    case = st["case"]
    return (_run_own if own else _run_plain)[case["op"]](st)


# ---- the package's calls ----
def _own_rope(st):
    import linear_moe_amd as L
    c = st["case"]
    q, k = L.qk_norm_rope(st["q"], st["k"], st["qw"], st["kw"], st["cos"], st["sin"], offsets=st["offsets"], cu_seqlens=st["cu"], eps=EPS,
                          interleaved=c["interleaved"], head_first=False)
    if not c["grad"]:
        return q, k
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), st["leaves"], (st["dq"], st["dk"]))


def _own_append(st):
    import linear_moe_amd as L
    L.paged_kv_append(st["kp"], st["vp"], st["k"], st["v"], st["table"], st["lens"], cu_seqlens=st["cu"], head_first=False, k_scales=st["ks"],
                      v_scales=st["vs"])
    return L.paged_kv_read(st["kp"], st["vp"], st["table"], st["lens"], st["case"]["T"], cu_seqlens=st["cu"], head_first=False,
                           k_scales=st["ks"], v_scales=st["vs"], dtype=st["k"].dtype)


def _own_decode(st):
    import linear_moe_amd as L
    c = st["case"]
    o = L.paged_attn_decode(st["q"], st["kp"], st["vp"], st["table"], st["lens"], k=st["k"], v=st["v"], softcap=c["softcap"],
                            slopes=st["slopes"], head_first=False, k_scales=st["ks"], v_scales=st["vs"])
    if not c["append"]:
        return o
    return (o,) + tuple(L.paged_kv_read(st["kp"], st["vp"], st["table"], st["lens"], 1, head_first=False, k_scales=st["ks"],
                                        v_scales=st["vs"], dtype=st["q"].dtype))


def _own_pages(st):
    import linear_moe_amd as L
    pages, table, lens, refs = st["pages"], st["table"], st["lens"], st["refs"]
    if st["case"]["defrag"]:
        turn = st["turn"]
        st["turn"] = 1 - turn
        L.paged_free(table, lens, refs, st["ended"][turn])
        live, moved = L.paged_compact(pages, table, refs)
        fits = L.paged_reserve(pages, table, lens, refs, st["tokens"][turn])
        return (table, lens, refs, fits, live, moved) + pages
    L.paged_free(table, lens, refs, st["ended"])
    L.paged_fork(table, lens, refs, st["src"], st["ended"])
    fits = L.paged_reserve(pages, table, lens, refs, st["tokens"])
    return (table, lens, refs, fits) + pages


# ---- the plain forms ----
def _positions(st):
    """Position of every token, in a row."""
    dev = st["q"].device
    lens, start = torch.tensor(st["lens"], device=dev), torch.tensor(st["start"], device=dev)
    seq = torch.repeat_interleave(torch.arange(len(st["lens"]), device=dev), lens)
    return torch.arange(seq.numel(), device=dev) - (lens.cumsum(0) - lens)[seq] + start[seq]


def _turn(x, c, s, R, interleaved):
    """The first R columns turned by the angles of c and s."""
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    ya, yb = a * c - b * s, b * c + a * s
    y = torch.stack((ya, yb), -1).flatten(-2) if interleaved else torch.cat((ya, yb), -1)
    return torch.cat((y, x[..., R:]), -1)


def _normed(x, w):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return r, x * r if w is None else x * r * w.float()


def _normed_back(x, r, w, g):
    """Gradients of x and w from that of x r w."""
    xhat = x * r
    gw = g if w is None else g * w.float()
    dx = r * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
    return dx, None if w is None else (g * xhat).sum((0, 1, 2))


def _plain_rope(st):
    case = st["case"]
    R, inter, B, T = case["R"], case["interleaved"], case["B"], case["T"]
    pos = _positions(st).view(B, T)
    c, s = st["cos"][pos][:, :, None], st["sin"][pos][:, :, None]
    q, k = st["q"].detach().float(), st["k"].detach().float()
    qw, kw = (None if w is None else w.detach() for w in (st["qw"], st["kw"]))
    (rq, nq), (rk, nk) = _normed(q, qw), _normed(k, kw)
    dt = st["q"].dtype
    out = _turn(nq, c, s, R, inter).to(dt), _turn(nk, c, s, R, inter).to(dt)
    if not case["grad"]:
        return out
    dq, dqw = _normed_back(q, rq, qw, _turn(st["dq"].float(), c, -s, R, inter))
    dk, dkw = _normed_back(k, rk, kw, _turn(st["dk"].float(), c, -s, R, inter))
    return out + (dq.to(dt), dk.to(dt)) + ((dqw.to(dt), dkw.to(dt)) if case["weights"] else ())


def _to_4_bits(x):
    """Codes, two in a byte (the even column in the low half: a sign, and which of 0 0.5 1 1.5 2 3 4 6), and per 32 columns the
    power of two that they are multiples of (plus 127): the least for which none is above 6."""
    g = x.float().unflatten(-1, (-1, GROUP))
    most = g.abs().amax(-1, keepdim=True)
    exponent = ((most.view(torch.int32) + 0x3FFFFF) >> 23) - 2            # 1.5 times a power of two is the last to fit
    exponent = exponent.clamp(7, 252)
    y = g * torch.exp2((127 - exponent).float())                          # (exact)
    size = y.abs().clamp(max=6.0)
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = torch.round(size / step) * step                                # (to even, as the codes count)
    code = torch.where(size < 2, size * 2, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(y).to(torch.uint8) << 3)).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), exponent[..., 0].to(torch.uint8)


def _from_4_bits(codes, scales):
    """The values, in 32 bits."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat((grid, -grid))
    x = torch.stack((grid[(codes & 15).int()], grid[(codes >> 4).int()]), -1).flatten(-2)
    return (x.unflatten(-1, (-1, GROUP)) * torch.exp2(scales.float() - 127)[..., None]).flatten(-2)


def _rows_of(table, pos, seq, S):
    """Page and slot that hold position pos of sequence seq."""
    return table[seq, pos // S].long(), pos % S


def _fresh(st):
    """Page and slot of every new token, in a row."""
    dev = st["table"].device
    fresh = torch.tensor(st["fresh"], device=dev)
    seq = torch.repeat_interleave(torch.arange(len(st["fresh"]), device=dev), fresh)
    pos = torch.arange(seq.numel(), device=dev) - st["cu"].long()[seq] + st["lens"].long()[seq]
    return _rows_of(st["table"], pos, seq, st["case"]["page"])


def _write(pages, scales, x, at):
    pages[at], scales[at] = _to_4_bits(x)
    return _from_4_bits(pages[at], scales[at]).to(x.dtype)


def _plain_append(st):
    at, shape = _fresh(st), st["k"].shape
    return tuple(_write(p, s, x.flatten(0, 1), at).view(shape) for p, s, x in ((st["kp"], st["ks"], st["k"]), (st["vp"], st["vs"], st["v"])))


def _plain_decode(st):
    c, dev = st["case"], st["q"].device
    S, N, HQ, HKV, D, cap = c["page"], c["N"], c["HQ"], c["HKV"], c["D"], c["softcap"]
    kept = _plain_append(st) if c["append"] else ()
    lens = st["lens"].long() + len(kept) // 2
    L = max(st["start"]) + len(kept) // 2
    pos = torch.arange(L, device=dev)
    seq = torch.arange(N, device=dev)[:, None]
    page, slot = _rows_of(st["table"], pos[None, :].expand(N, L), seq, S)
    live = pos[None, :] < lens[:, None]
    at = page.clamp(min=0), slot
    k, v = (_from_4_bits(p[at], s[at]).transpose(1, 2).contiguous() for p, s in ((st["kp"], st["ks"]), (st["vp"], st["vs"])))    # [N, HKV, L, D]
    q = st["q"].view(N, HKV, HQ // HKV, D).float()
    s = D ** -0.5 * (q @ k.transpose(2, 3).contiguous())                                          # [N, HKV, G, L]
    if cap:
        s = cap * torch.tanh(s / cap)
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, HKV, -1, 1) * (lens[:, None] - 1 - pos[None, :]).view(N, 1, 1, L)
    s = torch.where(live.view(N, 1, 1, L), s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = (p / p.sum(-1, keepdim=True)) @ v
    o = o.view(N, 1, HQ, D).to(st["q"].dtype)
    return (o,) + kept if kept else o


def _held(table, refs):
    """Which entries name a page, and their numbers (0 for the others)."""
    ok = (table >= 0) & (table < refs.numel())
    return ok, torch.where(ok, table, 0).long()


def _count(refs, ok, page, by):
    refs.index_add_(0, page.flatten(), torch.where(ok, by, 0).to(torch.int32).flatten())


def _free(table, lens, refs, rows):
    rows = rows.long()
    ok, page = _held(table[rows], refs)
    _count(refs, ok, page, -1)
    table[rows] = torch.where(ok, -1, table[rows])
    lens[rows] = 0


def _fork(table, lens, refs, src, dst):
    src, dst = src.long(), dst.long()
    new = table[src]
    _count(refs, *_held(table[dst], refs), -1)
    _count(refs, *_held(new, refs), 1)
    table[dst], lens[dst] = new, lens[src]


def _copy_pages(pages, src, dst):
    return tuple(x.index_copy_(0, dst, x[src]) for x in pages)


def _compact(pages, table, refs):
    P = refs.numel()
    used = refs > 0
    live = used.sum()
    front = torch.arange(P, device=refs.device) < live
    holes, movers = torch.nonzero(front & ~used)[:, 0], torch.nonzero(~front & used)[:, 0]
    moved = torch.arange(P, device=refs.device, dtype=torch.int32)
    moved[movers] = holes.int()
    _copy_pages(pages, movers, holes)
    refs[holes] = refs[movers]
    refs[movers] = 0
    ok, page = _held(table, refs)
    table.copy_(torch.where(ok, moved[page], table))
    return live.int().view(1), moved


def _reserve(pages, table, lens, refs, tokens, S):
    """In the order of the rows: every page that a row lacks, or shares with others, is given to it from the free ones in their order."""
    M, dev = table.shape[1], table.device
    col = torch.arange(M, device=dev)
    first, last = lens // S, (lens + tokens - 1) // S
    fits = (tokens <= 0) | (last < M)
    asked = (col >= first[:, None]) & (col <= last[:, None]) & (fits & (tokens > 0))[:, None]
    ok, page = _held(table, refs)
    item = torch.nonzero((asked & ok & (refs[page] > 1)).flatten())[:, 0]     # shared, in order
    shared = page.flatten()[item]
    by_page, order = torch.sort(shared, stable=True)
    place = torch.arange(item.numel(), device=dev)
    begin = torch.cummax(torch.where(torch.cat((by_page[:1] < 0, by_page[1:] == by_page[:-1])), 0, place), 0)[0]
    rank = torch.empty_like(place).index_copy_(0, order, place - begin)
    copied = item[refs[shared] - rank > 1]                                    # (the last to hold it keeps it)
    need = (asked & ~ok).flatten().index_fill_(0, copied, True).view_as(asked)
    free = torch.nonzero(refs <= 0)[:, 0]
    count = need.sum(1)
    fits = fits & ((count.cumsum(0) <= free.numel()) | (count == 0))
    need = need & fits[:, None]
    which = (need.flatten().cumsum(0) - 1).view_as(need)
    copies = torch.nonzero(need & ok)
    old = page[copies[:, 0], copies[:, 1]]
    new = free[which[copies[:, 0], copies[:, 1]]]
    _copy_pages(pages, old, new)
    refs.index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    refs[free[:need.sum()]] = 1
    table.copy_(torch.where(need, free[torch.where(need, which, 0)].int(), table))
    return fits


def _plain_pages(st):
    pages, table, lens, refs, S = st["pages"], st["table"], st["lens"], st["refs"], st["case"]["page"]
    if st["case"]["defrag"]:
        turn = st["turn"]
        st["turn"] = 1 - turn
        _free(table, lens, refs, st["ended"][turn])
        live, moved = _compact(pages, table, refs)
        fits = _reserve(pages, table, lens, refs, st["tokens"][turn], S)
        return (table, lens, refs, fits, live, moved) + pages
    _free(table, lens, refs, st["ended"])
    _fork(table, lens, refs, st["src"], st["ended"])
    fits = _reserve(pages, table, lens, refs, st["tokens"], S)
    return (table, lens, refs, fits) + pages


_run_own = {"rope": _own_rope, "decode": _own_decode, "append": _own_append, "pages": _own_pages}
_run_plain = {"rope": _plain_rope, "decode": _plain_decode, "append": _plain_append, "pages": _plain_pages}


# ---- 64 bits, from the definition ----
def _rope_64(x, w, c, s, R, interleaved):
    rms = torch.linalg.vector_norm(x, dim=-1, keepdim=True) / math.sqrt(x.shape[-1])
    y = x / torch.sqrt(rms * rms + EPS)
    if w is not None:
        y = y * w
    z = torch.complex(y[..., 0:R:2], y[..., 1:R:2]) if interleaved else torch.complex(y[..., :R // 2], y[..., R // 2:R])
    z = z * torch.complex(c, s)
    turned = torch.view_as_real(z).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)
    return torch.cat((turned, y[..., R:]), -1)


def _kept_64(x):
    """What 4 bits keep of x, in 64 bits: the nearest of 15 numbers, of two equally near that with an even code."""
    g = x.double().unflatten(-1, (-1, GROUP))
    most = g.abs().amax(-1, keepdim=True)
    e = torch.full_like(most, -120.0)
    for i in range(-120, 125):
        e = torch.where(6.0 * 2.0 ** i < most, float(i + 1), e)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    size = g.abs() / 2.0 ** e
    up = torch.bucketize(size, middle, right=False)               # how many middles lie below
    on = torch.bucketize(size, middle, right=True) > up           # on one: to the even code
    up = up + (on & (up % 2 == 1))
    return (grid[up] * torch.sign(g) * 2.0 ** e).flatten(-2)


def _values_64(codes, scales):
    b = codes.long()
    code = torch.stack((b % 16, b // 16), -1).flatten(-2)
    m, e = code % 2, code // 2 % 4
    size = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * 2.0 ** (e - 1).double())
    return torch.where(code >= 8, -size, size) * (2.0 ** (scales.double() - 127)).repeat_interleave(GROUP, -1)


def _attend(q, k, v, cap, slope):
    s = torch.einsum("id,jd->ij", q, k) / math.sqrt(q.shape[1])
    if cap:
        s = torch.tanh(s / cap) * cap
    if slope is not None:
        s = s - slope * torch.arange(k.shape[0] - 1, -1, -1, device=q.device).double()
    return torch.softmax(s, dim=1) @ v


def _exact_rope(case, st):
    R, B, T = case["R"], case["B"], case["T"]
    pos = [a + i for n, a in zip(st["lens"], st["start"]) for i in range(n)]
    pos = torch.tensor(pos, device=st["q"].device).view(B, T)
    c, s = (x.double()[pos][:, :, None] for x in (st["cos"], st["sin"]))
    names = ("q", "k") + (("qw", "kw") if case["weights"] else ())
    leaf = {n: st[n].detach().double().requires_grad_(case["grad"]) for n in names}
    out = tuple(_rope_64(leaf[x], leaf.get(x + "w"), c, s, R, case["interleaved"]) for x in "qk")
    if not case["grad"]:
        return out
    grads = torch.autograd.grad(out, [leaf[n] for n in names], (st["dq"].double(), st["dk"].double()))
    return tuple(x.detach() for x in out) + grads


def _exact_pages(case, st):
    """Page by page and row by row, on the host."""
    S, P = case["page"], st["refs"].numel()
    table, lens, refs = (st[x].tolist() for x in ("table", "lens", "refs"))
    origin = list(range(P))                          # whose contents at the start a page holds
    is_page = lambda x: 0 <= x < P
    turn = st["turn"]
    for r in (st["ended"][turn] if case["defrag"] else st["ended"]).tolist():
        for j, x in enumerate(table[r]):
            if is_page(x):
                refs[x] -= 1
                table[r][j] = -1
        lens[r] = 0
    extra = ()
    if case["defrag"]:
        live = sum(x > 0 for x in refs)
        holes, moved = [x for x in range(live) if refs[x] <= 0], list(range(P))
        for a, b in zip([x for x in range(live, P) if refs[x] > 0], holes):
            moved[a], origin[b], refs[b], refs[a] = b, origin[a], refs[a], 0
        table = [[moved[x] if is_page(x) else x for x in row] for row in table]
        extra = ([live], moved)
        tokens = st["tokens"][turn].tolist()
    else:
        before, lens0 = [list(row) for row in table], list(lens)
        for a, b in zip(st["src"].tolist(), st["ended"].tolist()):
            for x in before[a]:
                if is_page(x):
                    refs[x] += 1
            table[b], lens[b] = list(before[a]), lens0[a]
        tokens = st["tokens"].tolist()
    free, fits = [x for x in range(P) if refs[x] <= 0][::-1], []
    for row, n, t in zip(table, lens, tokens):
        cols = range(n // S, (n + t - 1) // S + 1) if t > 0 else range(0)
        want = [j for j in cols if not is_page(row[j]) or refs[row[j]] > 1]
        fits.append(len(want) <= len(free))
        for j in want if fits[-1] else ():
            p = free.pop()
            if is_page(row[j]):
                origin[p] = origin[row[j]]
                refs[row[j]] -= 1
            refs[p], row[j] = 1, p
    dev = st["refs"].device
    where = torch.tensor(origin, device=dev)
    ints = tuple(torch.tensor(x, dtype=torch.int32, device=dev) for x in (table, lens, refs))
    extra = tuple(torch.tensor(x, dtype=torch.int32, device=dev) for x in extra)
    return ints + (torch.tensor(fits, device=dev),) + extra + tuple(x[where].double() for x in st["pages"])


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, st)
    if case["op"] == "pages":
        return _exact_pages(case, st)
    if case["op"] == "append":
        return _kept_64(st["k"]), _kept_64(st["v"])
    kept = (_kept_64(st["k"]), _kept_64(st["v"])) if case["append"] else ()
    G, S = case["HQ"] // case["HKV"], case["page"]
    o = torch.empty(case["N"], 1, case["HQ"], case["D"], dtype=torch.float64, device=st["q"].device)
    for n, a in enumerate(st["start"]):
        mine = st["table"][n, :(a + S - 1) // S].long()
        k, v = (_values_64(p[mine], s[mine]).flatten(0, 1)[:a] for p, s in ((st["kp"], st["ks"]), (st["vp"], st["vs"])))
        if kept:
            k, v = torch.cat((k, kept[0][n])), torch.cat((v, kept[1][n]))
        for h in range(case["HQ"]):
            slope = None if st["slopes"] is None else st["slopes"][h].double()
            o[n, :, h] = _attend(st["q"][n, :, h].double(), k[:, h // G], v[:, h // G], case["softcap"], slope)
    return (o, *kept) if kept else o
