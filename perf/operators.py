"""The softmax layers of a hybrid model, next to its linear ones: attention over a sequence (training step and prompt),
one new token over a paged cache of keys and values, and the writing of that cache.

``listed()`` are fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds before
the call, ``run`` is one pass, ``work`` what that pass cannot do without and ``exact`` the same outputs in 64 bits.  With
``own`` false ``run`` computes the operators with elementary torch operations in 32 bits, rounded once at the end; with
``own`` true it makes the calls a user makes of the package."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _attn(name, B, T, HQ, HKV, D, dtype="bf16", causal=True, softcap=0.0, slopes=False, prefix=False, docs=0, grad=True):
    return dict(name=name, op="attn", B=B, T=T, HQ=HQ, HKV=HKV, D=D, dtype=dtype, causal=causal, softcap=softcap,
                slopes=slopes, prefix=prefix, docs=docs, grad=grad)


def _decode(name, N, L, HQ, HKV, D, page, dtype="bf16", softcap=0.0, slopes=False, append=False):
    return dict(name=name, op="decode", N=N, L=L, HQ=HQ, HKV=HKV, D=D, page=page, dtype=dtype, softcap=softcap, slopes=slopes,
                append=append)


def _append(name, N, T, HKV, D, page, dtype="bf16"):
    return dict(name=name, op="append", N=N, T=T, HKV=HKV, D=D, page=page, dtype=dtype)


def listed():
    return [
        # a prompt of a few words: nothing but latency
        _attn("attn_prompt_37", 1, 37, 16, 16, 128, grad=False),
        # a long prompt read in before generation, heads biased by distance, four query heads to a key head
        _attn("attn_prefill_slopes", 1, 8192, 32, 8, 128, slopes=True, grad=False),
        # training step of a softmax layer of a hybrid model on this package's headline shape (the largest case)
        _attn("attn_train", 4, 8192, 16, 4, 128),
        # training step on packed documents of very unequal lengths, scores capped
        _attn("attn_train_packed_cap", 1, 16384, 16, 8, 128, softcap=30.0, docs=23),
        # training step of a prefix language model (a question seen whole, an answer token by token), narrow heads, odd length
        _attn("attn_train_prefix", 4, 2011, 16, 16, 64, prefix=True),
        # a small layer in float32
        _attn("attn_train_f32", 2, 1000, 4, 2, 64, dtype="f32"),
        # one generated token of one conversation: latency
        _decode("decode_1", 1, 500, 16, 4, 128, 16, append=True),
        # one generated token of a serving batch of unequal lengths
        _decode("decode_64", 64, 4096, 32, 8, 128, 64, append=True),
        # one generated token over two very long documents
        _decode("decode_long", 2, 131072, 16, 4, 128, 128),
        # float32, biased and capped, pages of a length that is no power of two
        _decode("decode_f32", 9, 3001, 12, 3, 64, 24, dtype="f32", softcap=20.0, slopes=True),
        # the keys and values of seven prompts go into the cache
        _append("append_prompts", 7, 16384, 8, 128, 16),
        # those of one new token of each conversation
        _append("append_tokens", 64, 64, 8, 128, 64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max((work(c) for c in listed()), key=lambda w: w["flops"])
    while True:
        op = rng.choice(("attn", "attn", "decode", "append"))
        dtype = "bf16" if rng.random() < 0.8 else "f32"
        G, HKV, D = rng.choice((1, 1, 2, 4, 5, 8)), rng.choice((1, 2, 3, 4, 8)), rng.choice((64, 128, 128, 96))
        if op == "attn":
            mask = rng.choice(("causal", "causal", "whole", "prefix"))
            T = _log_int(rng, 1, 8192)
            docs = min(T, _log_int(rng, 1, 40)) if rng.random() < 0.4 else 0
            B = 1 if docs else _log_int(rng, 1, 8)
            c = _attn(None, B, T, G * HKV, HKV, D, dtype, mask != "whole", rng.choice((0.0, 0.0, 15.0, 50.0)), rng.random() < 0.3,
                      mask == "prefix", docs, rng.random() < 0.6)
            # (4-byte elements have a sixteenth of the matrix rate)
            fits = work(c)["flops"] * (16 if dtype == "f32" else 1) <= most["flops"] / 2
        elif op == "decode":
            N, L = _log_int(rng, 1, 128), _log_int(rng, 1, 65536)
            c = _decode(None, N, L, G * HKV, HKV, D, rng.choice((16, 24, 32, 64, 100, 128)), dtype, rng.choice((0.0, 0.0, 15.0, 50.0)),
                        rng.random() < 0.3, rng.random() < 0.5)
            fits = work(c)["bytes"] <= 5e8
        else:
            N = _log_int(rng, 1, 100)
            c = _append(None, N, max(N, _log_int(rng, 1, 16384)), HKV, D, rng.choice((16, 24, 32, 64, 100, 128)), dtype)
            fits = True
        if fits:
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
    """Lengths of the sequences of an attention case."""
    return _lengths(case["docs"], case["T"]) if case["docs"] else [case["T"]] * case["B"]


def _prefixes(case):
    """Prefix lengths: from none to the whole sequence, about a third of it on average."""
    lens = _documents(case)
    rng = random.Random(len(lens) * 7919 + case["T"])
    return [min(n, int(n * rng.random() ** 2 + 0.5)) for n in lens] if case["prefix"] else [0] * len(lens)


def _cached(case):
    """Tokens in the cache per sequence of a decoding case: from one to L."""
    N, L = case["N"], case["L"]
    return [max(1, round(L * (1.0 if N == 1 else 0.25 + 0.75 * i / (N - 1)))) for i in range(N)]


def _pairs(case):
    pairs = 0
    for n, p in zip(_documents(case), _prefixes(case)):
        pairs += n * (n + 1) // 2 + p * (p - 1) // 2 if case["causal"] else n * n
    return pairs


def work(case):
    size, D, HKV = DTYPES[case["dtype"]].itemsize, case["D"], case["HKV"]
    if case["op"] == "attn":
        tokens, HQ = sum(_documents(case)), case["HQ"]
        moved = tokens * D * size * (2 * HQ + 2 * HKV)              # q, k, v in, o out
        if case["grad"]:
            moved += tokens * D * size * (2 * HQ + 2 * HKV)         # do in, dq, dk, dv out
        return {"bytes": moved, "flops": _pairs(case) * HQ * D * (14 if case["grad"] else 4)}
    if case["op"] == "decode":
        tokens, new = sum(_cached(case)), case["N"] if case["append"] else 0
        moved = 2 * (tokens + 2 * new) * HKV * D * size + 2 * case["N"] * case["HQ"] * D * size
        return {"bytes": moved, "flops": 4 * (tokens + new) * case["HQ"] * D}
    return {"bytes": 4 * case["T"] * HKV * D * size, "flops": 0}


def _slopes(H, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device=device)


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    dt, D, HKV = DTYPES[case["dtype"]], case["D"], case["HKV"]
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev, dtype=dt)
    st = dict(case=case)
    if case["op"] == "attn":
        B, T, HQ = case["B"], case["T"], case["HQ"]
        lens, prefixes = _documents(case), _prefixes(case)
        order = list(range(len(lens)))
        rng.shuffle(order)
        lens, prefixes = [lens[i] for i in order], [prefixes[i] for i in order]
        st.update(q=randn(B, T, HQ, D), k=randn(B, T, HKV, D), v=randn(B, T, HKV, D), lens=lens, prefixes=prefixes, cu=None,
                  prefix=None, slopes=_slopes(HQ, dev) if case["slopes"] else None)
        if case["docs"]:
            st["cu"] = torch.tensor(_offsets(lens), dtype=torch.int32, device=dev)
        if case["prefix"]:
            st["prefix"] = torch.tensor(prefixes, dtype=torch.int32, device=dev)
        if case["grad"]:
            st["do"] = randn(B, T, HQ, D)
            for x in ("q", "k", "v"):
                st[x].requires_grad_(True)
        return st
    # a cache: the pages of all sequences, shuffled, and a few that belong to none
    S, N = case["page"], case["N"]
    if case["op"] == "decode":
        start = _cached(case)
        rng.shuffle(start)
        fresh = [1 if case["append"] else 0] * N
    else:
        fresh = _lengths(N, case["T"])
        rng.shuffle(fresh)
        start = [rng.randrange(0, 2 * S) for _ in range(N)]
    held = [(a + b + S - 1) // S for a, b in zip(start, fresh)]
    if case["op"] == "decode":
        room = held
    else:
        room = [(2 * S - 1 + b + S - 1) // S for b in fresh]        # (as many pages whatever the seed)
    ids = list(range(sum(room) + 3))
    rng.shuffle(ids)
    table, at = torch.zeros(N, max(room), dtype=torch.int32), 0
    for n, m in enumerate(held):
        table[n, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
        at += m
    st.update(k_pages=randn(len(ids), S, HKV, D), v_pages=randn(len(ids), S, HKV, D), table=table.to(dev), start=start, fresh=fresh,
              lens=torch.tensor(start, dtype=torch.int32, device=dev))
    if case["op"] == "decode":
        st.update(q=randn(N, 1, case["HQ"], D), k=None, v=None, slopes=_slopes(case["HQ"], dev) if case["slopes"] else None)
        if case["append"]:
            st.update(k=randn(N, 1, HKV, D), v=randn(N, 1, HKV, D))
    else:
        st.update(k=randn(1, case["T"], HKV, D), v=randn(1, case["T"], HKV, D),
                  cu=torch.tensor(_offsets(fresh), dtype=torch.int32, device=dev))
    return st


def run(st):
    case = st["case"]
    return (_run_own if own else _run_plain)[case["op"]](st)


# ---- the package's calls ----
def _own_attn(st):
    import linear_moe_amd as L
    c = st["case"]
    o = L.softmax_attn(st["q"], st["k"], st["v"], causal=c["causal"], softcap=c["softcap"], slopes=st["slopes"], prefix_lens=st["prefix"],
                       cu_seqlens=st["cu"], head_first=False)
    if not c["grad"]:
        return o
    return (o.detach(),) + torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"])


def _own_decode(st):
    import linear_moe_amd as L
    c = st["case"]
    o = L.paged_attn_decode(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"], k=st["k"], v=st["v"], softcap=c["softcap"],
                            slopes=st["slopes"], head_first=False)
    return (o, st["k_pages"], st["v_pages"]) if c["append"] else o


def _own_append(st):
    import linear_moe_amd as L
    L.paged_kv_append(st["k_pages"], st["v_pages"], st["k"], st["v"], st["table"], st["lens"], cu_seqlens=st["cu"], head_first=False)
    return st["k_pages"], st["v_pages"]


# ---- the plain forms ----
def _allowed(n, prefix, causal, dev):
    i = torch.arange(n, device=dev)
    return (i[None, :] <= i[:, None]) | (i[None, :] < prefix) if causal else None


def _plain_attn(st):
    c, dev = st["case"], st["q"].device
    HQ, HKV, D, cap = c["HQ"], c["HKV"], c["D"], c["softcap"]
    G, scale = HQ // HKV, c["D"] ** -0.5
    q, k, v = (st[x].detach().reshape(-1, st[x].shape[2], D).float() for x in ("q", "k", "v"))
    outs = [torch.empty_like(q)]
    if c["grad"]:
        do = st["do"].reshape(-1, HQ, D).float()
        outs += [torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)]
    at = 0
    for n, p in zip(st["lens"], st["prefixes"]):
        rows = slice(at, at + n)
        at += n
        mask = _allowed(n, p, c["causal"], dev)
        i = torch.arange(n, device=dev, dtype=torch.float32)
        for h in range(HKV):
            kh, vh = k[rows, h], v[rows, h]
            for g in range(h * G, (h + 1) * G):
                qh = q[rows, g]
                s = scale * (qh @ kh.t())
                if cap:
                    t = torch.tanh(s / cap)
                    s = cap * t
                if st["slopes"] is not None:
                    s = s - st["slopes"][g] * (i[:, None] - i[None, :]).abs()
                if mask is not None:
                    s = torch.where(mask, s, -math.inf)
                pr = torch.exp(s - s.amax(1, keepdim=True))
                pr = pr / pr.sum(1, keepdim=True)
                o = pr @ vh
                outs[0][rows, g] = o
                if not c["grad"]:
                    continue
                dh = do[rows, g]
                ds = pr * (dh @ vh.t() - (dh * o).sum(1, keepdim=True))
                if cap:
                    ds = ds * (1.0 - t * t)
                outs[1][rows, g] = scale * (ds @ kh)
                dk, dv = scale * (ds.t() @ qh), pr.t() @ dh
                if g == h * G:
                    outs[2][rows, h], outs[3][rows, h] = dk, dv
                else:
                    outs[2][rows, h] += dk
                    outs[3][rows, h] += dv
    like = [st["q"], st["q"], st["k"], st["v"]]
    outs = [x.reshape(y.shape).to(y.dtype) for x, y in zip(outs, like)]
    return tuple(outs) if c["grad"] else outs[0]


def _slots(table, pos, seq, S):
    """Row of the pages, taken as one list of slots, that holds position pos of sequence seq."""
    return table[seq, pos // S].long() * S + pos % S


def _plain_append(st):
    dev, S = st["table"].device, st["case"]["page"]
    fresh = torch.tensor(st["fresh"], device=dev)
    seq = torch.repeat_interleave(torch.arange(len(st["fresh"]), device=dev), fresh)
    pos = torch.arange(seq.numel(), device=dev) - st["cu"].long()[seq] + st["lens"].long()[seq]
    rows = _slots(st["table"], pos, seq, S)
    for pages, x in ((st["k_pages"], st["k"]), (st["v_pages"], st["v"])):
        pages.view(-1, *pages.shape[2:])[rows] = x[0]
    return st["k_pages"], st["v_pages"]


def _plain_decode(st):
    c, dev = st["case"], st["q"].device
    S, N, HQ, HKV, D, cap = c["page"], c["N"], c["HQ"], c["HKV"], c["D"], c["softcap"]
    lens = st["lens"].long()
    if c["append"]:
        rows = _slots(st["table"], lens, torch.arange(N, device=dev), S)
        for pages, x in ((st["k_pages"], st["k"]), (st["v_pages"], st["v"])):
            pages.view(-1, HKV, D)[rows] = x[:, 0]
        lens = lens + 1
    L = max(st["start"]) + (1 if c["append"] else 0)
    pos = torch.arange(L, device=dev)
    rows = _slots(st["table"], pos[None, :].expand(N, L), torch.arange(N, device=dev)[:, None], S)
    live = pos[None, :] < lens[:, None]
    o = torch.empty(N, HKV, HQ // HKV, D, device=dev)
    q = st["q"].view(N, HKV, HQ // HKV, D).float()
    for h in range(HKV):
        k, v = (x.view(-1, HKV, D)[:, h][rows].float() for x in (st["k_pages"], st["v_pages"]))        # [N, L, D]
        s = D ** -0.5 * (k @ q[:, h].transpose(1, 2).contiguous())                                         # [N, L, G]
        if cap:
            s = cap * torch.tanh(s / cap)
        if st["slopes"] is not None:
            s = s - st["slopes"].view(HKV, -1)[h] * (lens[:, None] - 1 - pos[None, :])[..., None]
        s = torch.where(live[..., None], s, -math.inf)
        p = torch.exp(s - s.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        o[:, h] = p.transpose(1, 2).contiguous() @ v
    o = o.view(N, 1, HQ, D).to(st["q"].dtype)
    return (o, st["k_pages"], st["v_pages"]) if c["append"] else o


_run_own = {"attn": _own_attn, "decode": _own_decode, "append": _own_append}
_run_plain = {"attn": _plain_attn, "decode": _plain_decode, "append": _plain_append}


# ---- 64 bits, from the definition ----
def _attend(q, k, v, scale, cap, slope, hidden):
    """softmax(scores) v of one head: q [m, D], k, v [n, D], the last of the m queries at the last of the n keys."""
    s = torch.einsum("id,jd->ij", q, k).mul_(scale) if not q.requires_grad else torch.einsum("id,jd->ij", q, k) * scale
    if cap:
        s = torch.tanh(s / cap) * cap
    if slope is not None:
        m, n = s.shape
        far = torch.arange(n, device=s.device)[None, :] - torch.arange(n - m, n, device=s.device)[:, None]
        s = s - slope * far.abs().double()
    if hidden is not None:
        s = s.masked_fill(hidden, -math.inf)
    return torch.softmax(s, dim=1) @ v


def exact(case, seed):
    st = prepare(case, seed)
    G = case["HQ"] // case["HKV"] if "HQ" in case else 0
    scale = 1.0 / math.sqrt(case["D"])
    if case["op"] == "attn":
        leaves = [st[x].detach().double() for x in ("q", "k", "v")]
        q, k, v = leaves
        o, grads = torch.zeros_like(q), [torch.zeros_like(x) for x in leaves] if case["grad"] else []
        spans, first = [], 0
        for j, (n, p) in enumerate(zip(st["lens"], st["prefixes"])):
            spans.append((0, first, n, p) if case["docs"] else (j, 0, n, p))
            first += n
        for b, t0, n, p in spans:
            hidden = None
            if case["causal"]:
                hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
                hidden[:, :p] = False
            for h in range(case["HQ"]):
                part = [x[b, t0:t0 + n, hh].clone().requires_grad_(case["grad"]) for x, hh in ((q, h), (k, h // G), (v, h // G))]
                slope = None if st["slopes"] is None else st["slopes"][h].double()
                y = _attend(*part, scale, case["softcap"], slope, hidden)
                o[b, t0:t0 + n, h] = y.detach()
                if case["grad"]:
                    got = torch.autograd.grad(y, part, st["do"][b, t0:t0 + n, h].double())
                    for acc, x, hh in zip(grads, got, (h, h // G, h // G)):
                        acc[b, t0:t0 + n, hh] += x
        return (o, *grads) if case["grad"] else o
    pages = [st["k_pages"].double(), st["v_pages"].double()]
    S, table = case["page"], st["table"].tolist()
    at = 0
    for n, (a, f) in enumerate(zip(st["start"], st["fresh"])):
        for pg, x in zip(pages, (st["k"], st["v"])):
            j = 0
            while j < f:                                  # whole runs inside a page
                slot, run_ = (a + j) % S, min(f - j, S - (a + j) % S)
                rows = x[n, j:j + run_] if case["op"] == "decode" else x[0, at + j:at + j + run_]
                pg[table[n][(a + j) // S], slot:slot + run_] = rows.double()
                j += run_
        at += f
    if case["op"] == "append":
        return tuple(pages)
    o = torch.empty(case["N"], 1, case["HQ"], case["D"], dtype=torch.float64, device=st["q"].device)
    for n, (a, f) in enumerate(zip(st["start"], st["fresh"])):
        mine = st["table"][n, :(a + f + S - 1) // S].long()
        k, v = (pg[mine].flatten(0, 1)[:a + f] for pg in pages)
        for h in range(case["HQ"]):
            slope = None if st["slopes"] is None else st["slopes"][h].double()
            o[n, :, h] = _attend(st["q"][n, :, h].double(), k[:, h // G], v[:, h // G], scale, case["softcap"], slope, None)
    return (o, *pages) if case["append"] else o
