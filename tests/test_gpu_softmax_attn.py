"""softmax_attn on the GPU against float64: the outputs and gradients element by element, within the bounds that
oracle/softmax.py derives from the kernels' roundings."""
import ctypes as C

import pytest
import torch

import linear_moe_amd as L
from linear_moe_amd import _lib
from oracle import softmax
from tests.util import gen

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def inputs(seed, B, T, HQ, HKV, K, V, dtype):
    return (gen(seed, B, T, HQ, K, dtype=dtype), gen(seed + 1, B, T, HKV, K, dtype=dtype), gen(seed + 2, B, T, HKV, V, dtype=dtype),
            gen(seed + 3, B, T, HQ, V, dtype=dtype))


def alibi(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)])


def run_and_check(cuda, q, k, v, do, cu=None, prefix=None, slopes=None, cu_on="cuda", **kw):
    want = softmax.attn(q, k, v, do=do, cu=cu, prefix_lens=prefix, slopes=slopes, **kw)
    leaves = [x.to(cuda).requires_grad_(True) for x in (q, k, v)]
    extra = dict(cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device=cu_on),
                 prefix_lens=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=cuda),
                 slopes=None if slopes is None else slopes.to(cuda))
    o = L.softmax_attn(*leaves, head_first=False, **extra, **kw)
    grads = torch.autograd.grad(o, leaves, do.to(cuda))
    for name, x in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        softmax.check(x, want[name], name)
    with torch.no_grad():                                    # forward-only calls give the same numbers
        assert torch.equal(o, L.softmax_attn(*leaves, head_first=False, **extra, **kw))
    return o, grads


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1, 2, 31, 33, 63, 64, 65, 127, 128, 129, 200, 257, 321])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(cuda, dtype, T, causal):
    run_and_check(cuda, *inputs(T, 2, T, 2, 1, 64, 64, dtype), causal=causal)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,HQ", [(129, 1), (321, 1), (321, 3), (700, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_odd_numbers_of_tiles(cuda, D, T, HQ, causal):
    run_and_check(cuda, *inputs(T + HQ, 1, T, HQ, 1, D, D, BF16), causal=causal)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["causal", "whole", "prefix", "packed", "packed_prefix", "cap_bias"])
def test_a_thousand_tokens(cuda, D, kind, dtype):
    """Several work-groups to a sequence in every kernel, the gradients of keys shared by some, unequal documents."""
    T, HQ, HKV = 1091, 2, 1
    cu = [0, 3, 3, 131, 900, 1091]
    kw = {"causal": {}, "whole": dict(causal=False), "prefix": dict(prefix=[700]), "packed": dict(cu=cu),
          "packed_prefix": dict(cu=cu, prefix=[2, 5, 128, 130, 64]), "cap_bias": dict(softcap=4.0, slopes=alibi(2))}[kind]
    run_and_check(cuda, *inputs(83, 1, T, HQ, HKV, D, D, dtype), **kw)


@pytest.mark.parametrize("kind", ["causal", "whole", "packed_prefix", "cap_bias"])
def test_float32_strips_of_32_rows(cuda, kind):
    """(16 rows to a wave where there are few, 32 where 512 such strips fill the card)"""
    B, T, H = (1, 2070, 8) if kind == "packed_prefix" else (2, 1035, 8)
    kw = {"causal": {}, "whole": dict(causal=False), "packed_prefix": dict(cu=[0, 17, 17, 1300, 2066], prefix=[20, 5, 400, 0]),
          "cap_bias": dict(softcap=4.0, slopes=alibi(8))}[kind]
    x = inputs(97, B, T, H, H, 48, 64, F32)
    if kind == "packed_prefix":
        x[3][:, 2066:] = 0
    run_and_check(cuda, *x, **kw)


@pytest.mark.parametrize("causal", [True, False])
def test_rows_far_apart(cuda, causal):
    """A row stride of 2^24 elements: the offsets inside a tile of 64 rows pass 31 bits."""
    T, D = 67, 64
    q, k, v, do = inputs(101, 1, T, 2, 1, D, D, BF16)
    far = torch.zeros(T * 2 ** 24, dtype=BF16, device=cuda).as_strided((1, T, 1, D), (T * 2 ** 24, 2 ** 24, D, 1))
    far.copy_(k)
    want = softmax.attn(q, k, v, do=do, causal=causal)
    leaves = [q.to(cuda).requires_grad_(True), far.detach().requires_grad_(True), v.to(cuda).requires_grad_(True)]
    assert leaves[1].stride(1) == 2 ** 24
    o = L.softmax_attn(*leaves, head_first=False, causal=causal)
    for name, x in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do.to(cuda)))):
        softmax.check(x, want[name], name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N", [64, 65, 256, 257])
def test_many_documents(cuda, N, dtype):
    """Up to and beyond the number of documents that a work-group looks through for its tile."""
    lens = [(7 * n) % 5 + (130 if n % 50 == 9 else 0) for n in range(N)]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    x = inputs(89, 1, cu[-1] + 3, 2, 1, 64, 64, dtype)
    x[3][:, cu[-1]:] = 0                        # (rows behind the last document)
    run_and_check(cuda, *x, cu=cu)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K,V", [(128, 128), (64, 128), (128, 64), (96, 96), (32, 8), (8, 128), (20, 13), (1, 1), (127, 72)])
def test_head_dims(cuda, dtype, K, V):
    run_and_check(cuda, *inputs(7, 1, 150, 2, 1, K, V, dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("HQ,HKV", [(1, 1), (4, 4), (4, 2), (5, 1), (6, 2), (16, 1), (9, 3)])
def test_shared_heads(cuda, dtype, HQ, HKV):
    run_and_check(cuda, *inputs(11, 2, 140, HQ, HKV, 64, 64, dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap,bias", [(3.0, False), (0.0, True), (5.0, True), (50.0, False)])
@pytest.mark.parametrize("mask", ["causal", "whole", "prefix"])
def test_scores(cuda, dtype, D, cap, bias, mask):
    q, k, v, do = inputs(13, 2, 190, 4, 2, D, D, dtype)
    run_and_check(cuda, 3 * q, k, v, do, softcap=cap, slopes=alibi(4) if bias else None, causal=mask != "whole",
                  prefix=[70, 190] if mask == "prefix" else None)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("prefix", [[0, 1], [64, 63], [65, 128], [129, 199], [200, 500], [-5, 100]])
def test_prefix(cuda, dtype, prefix):
    run_and_check(cuda, *inputs(17, 2, 200, 2, 2, 64, 64, dtype), prefix=prefix)


DOCS = [[0, 300], [0, 1, 2, 3, 300], [0, 0, 64, 64, 128, 300, 300], [0, 65, 193, 194, 300], [0, 128, 256, 300]]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cu", DOCS)
@pytest.mark.parametrize("cu_on", ["cuda", "cpu"])
def test_documents(cuda, dtype, cu, cu_on):
    run_and_check(cuda, *inputs(19, 1, 300, 4, 2, 64, 64, dtype), cu=cu, cu_on=cu_on)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_documents_with_everything(cuda, dtype):
    run_and_check(cuda, *inputs(23, 1, 300, 4, 2, 128, 96, dtype), cu=DOCS[2], prefix=[4, 10, 0, 64, 100, 3], slopes=alibi(4), softcap=4.0)
    run_and_check(cuda, *inputs(23, 1, 300, 4, 2, 128, 96, dtype), cu=DOCS[3], causal=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_behind_the_last_document_are_zero(cuda, dtype):
    q, k, v, do = inputs(29, 1, 300, 4, 2, 64, 64, dtype)
    for x in (q, k, v, do):
        x[:, 130:] = float("nan")
    leaves = [x.to(cuda).requires_grad_(True) for x in (q, k, v)]
    cu = torch.tensor([0, 70, 130], dtype=torch.int32, device=cuda)
    o = L.softmax_attn(*leaves, cu_seqlens=cu, head_first=False)
    grads = torch.autograd.grad(o, leaves, do.to(cuda))
    want = softmax.attn(q[:, :130], k[:, :130], v[:, :130], cu=[0, 70, 130], do=do[:, :130])
    for name, x in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        assert (x[:, 130:] == 0).all(), name
        softmax.check(x[:, :130], want[name], name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_document_does_not_see_what_another_holds(cuda, dtype, bad):
    q, k, v, do = (x.to(cuda) for x in inputs(31, 1, 300, 4, 2, 64, 64, dtype))
    cu = torch.tensor([0, 90, 170, 300], dtype=torch.int32, device=cuda)

    def all_of(q, k, v, do):
        leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
        o = L.softmax_attn(*leaves, cu_seqlens=cu, head_first=False)
        return (o, *torch.autograd.grad(o, leaves, do))

    clean = all_of(q, k, v, do)
    for x in (q, k, v, do):
        x[:, 90:170] = bad
    for a, b in zip(clean, all_of(q, k, v, do)):
        assert torch.equal(a[:, :90], b[:, :90]) and torch.equal(a[:, 170:], b[:, 170:])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("at", [0, 5, 64, 100, 149])
def test_a_token_reaches_no_row_before_it(cuda, dtype, at):
    """Whatever a token's key and value hold, NaN and infinities too, rows before it are the same bits."""
    q, k, v, _ = (x.to(cuda) for x in inputs(37, 1, 150, 2, 1, 64, 64, dtype))
    with torch.no_grad():
        clean = L.softmax_attn(q, k, v, head_first=False)
        for bad in (float("nan"), float("inf"), 1e30):
            k2, v2 = k.clone(), v.clone()
            k2[:, at], v2[:, at] = bad, bad
            got = L.softmax_attn(q, k2, v2, head_first=False)
            assert torch.equal(got[:, :at], clean[:, :at]), bad


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores(cuda, dtype):
    """Scores of hundreds: one key takes all, and none overflows."""
    q, k, v, do = inputs(41, 1, 130, 2, 1, 64, 64, dtype)
    o, grads = run_and_check(cuda, 30 * q, 10 * k, v, do)
    run_and_check(cuda, 30 * q, 10 * k, v, do, softcap=30.0)
    run_and_check(cuda, q, k, v, do, scale=0.0)
    run_and_check(cuda, q, k, v, do, scale=-0.5)
    run_and_check(cuda, q, k, v, do, slopes=torch.tensor([-0.01, 100.0]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts_give_the_same_bits(cuda, dtype):
    B, T, H, D = 2, 100, 4, 64
    qkv = gen(43, B, T, H, 3 * D, dtype=dtype).to(cuda)
    q, k, v = qkv.split(D, dim=-1)
    do = gen(44, B, T, H, D, dtype=dtype).to(cuda)

    def all_of(q, k, v, do, head_first):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        o = L.softmax_attn(*leaves, head_first=head_first)
        return (o, *torch.autograd.grad(o, leaves, do))

    plain = all_of(q.contiguous(), k.contiguous(), v.contiguous(), do, False)
    views = all_of(q, k, v, do, False)
    first = all_of(*(x.transpose(1, 2) for x in (q, k, v)), do.transpose(1, 2), True)
    firstc = all_of(*(x.transpose(1, 2).contiguous() for x in (q, k, v)), do.transpose(1, 2).contiguous(), True)
    odd = [torch.empty(x.numel() + 1, dtype=dtype, device=cuda)[1:].view(x.shape).copy_(x) for x in (q, k, v)]      # off 16 bytes
    for a, b, c, d, e in zip(plain, views, first, firstc, all_of(*odd, do, False)):
        assert torch.equal(a, b) and torch.equal(a, c.transpose(1, 2)) and torch.equal(a, d.transpose(1, 2)) and torch.equal(a, e)
    # one key head for all, as a broadcast view or as itself
    k1, v1 = k[:, :, :1].contiguous(), v[:, :, :1].contiguous()
    with torch.no_grad():
        assert torch.equal(L.softmax_attn(q, k1, v1, head_first=False), L.softmax_attn(q, k1.expand_as(k), v1.expand_as(v), head_first=False))
    # the gradient of a broadcast output (a sum) and of one whose rows are strided
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    o = L.softmax_attn(*leaves, head_first=False)
    ones = torch.autograd.grad(o.sum(), leaves, retain_graph=True)
    for a, b in zip(ones, torch.autograd.grad(o, leaves, torch.ones_like(o))):
        assert torch.equal(a, b)


def test_gradients_against_differences(cuda):
    """Directional differences of sum(o do) in float32: an error of h^2 times the third derivative (of order one for
    directions of unit size per element) and of the outputs' rounding over h."""
    q, k, v, do = inputs(47, 1, 70, 2, 1, 64, 64, F32)
    kw = dict(head_first=False, softcap=6.0, slopes=alibi(2).to(cuda), prefix_lens=torch.tensor([20], device=cuda))
    leaves = [x.to(cuda).requires_grad_(True) for x in (q, k, v)]
    do = do.to(cuda)
    grads = torch.autograd.grad(L.softmax_attn(*leaves, **kw), leaves, do)
    f = lambda xs: float((L.softmax_attn(*xs, **kw).double() * do.double()).sum())
    h = 2.0 ** -6
    with torch.no_grad():
        for i, g in enumerate(grads):
            for seed in range(3):
                d = gen(100 + seed, *leaves[i].shape).to(cuda)
                d /= d.norm()
                xs = [x.detach() for x in leaves]
                up, down = list(xs), list(xs)
                up[i], down[i] = xs[i] + h * d, xs[i] - h * d
                slope, want = (f(up) - f(down)) / (2 * h), float((g.double() * d.double()).sum())
                # |f| <= sum |o do| ~ 5e3, each term rounded to 2^-22 of itself at worst, over 2 h; h^2 / 6 times a third derivative of
                # at most the size of the gradient
                tol = 5e3 * 2.0 ** -22 / h + h * h * float(g.norm())
                assert abs(slope - want) < tol, (i, seed, slope, want, tol)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_repeated_calls_agree_bit_for_bit_and_on_another_stream(cuda, dtype):
    q, k, v, do = (x.to(cuda) for x in inputs(53, 2, 333, 6, 2, 128, 128, dtype))

    def all_of():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        o = L.softmax_attn(*leaves, head_first=False)
        return (o, *torch.autograd.grad(o, leaves, do))

    first = all_of()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = all_of()
    torch.cuda.current_stream().wait_stream(s)
    for a, b, c in zip(first, second, all_of()):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("backwards", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_the_library_called_for_itself(cuda, D, backwards):
    """A backward pass without o_low, and rows that lie in memory from the last to the first."""
    T, HQ, HKV = 300, 4, 2
    q, k, v, do = inputs(107, 1, T, HQ, HKV, D, D, BF16)
    want = softmax.attn(q, k, v, do=do, low=False)
    dev = [x.flip(1).contiguous().to(cuda) if backwards else x.to(cuda) for x in (q, k, v, do)]
    out = [torch.zeros_like(dev[i]) for i in (0, 0, 1, 2)]
    lse, delta = (torch.zeros(HQ, T, device=cuda) for _ in range(2))

    def rows(x):
        at = (T - 1) * x.stride(1) if backwards else 0
        return _lib.Tensor4(x.data_ptr() + 2 * at, x.stride(0), -x.stride(1) if backwards else x.stride(1), x.stride(2))

    a = _lib.AttnArgs()
    a.dtype, a.causal, a.scale = _lib.LMOE_BF16, 1, D ** -0.5
    a.B, a.T, a.HQ, a.HKV, a.K, a.V, a.N, a.NT = 1, T, HQ, HKV, D, D, 1, (T + 63) // 64
    a.q, a.k, a.v, a.d_o = map(rows, dev)
    a.o, a.dq, a.dk, a.dv = map(rows, out)
    a.lse, a.delta = lse.data_ptr(), delta.data_ptr()
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    assert lib.lmoe_softmax_attn_fwd(C.byref(a), st) == 0, lib.lmoe_last_error()
    floats = lib.lmoe_softmax_attn_bwd_floats(C.byref(a))
    assert floats > 0                                         # (few keys: their rows are shared)
    assert lib.lmoe_softmax_attn_bwd(C.byref(a), st) == -11
    ws = torch.empty(floats, device=cuda)
    a.ws = ws.data_ptr()
    assert lib.lmoe_softmax_attn_bwd(C.byref(a), st) == 0, lib.lmoe_last_error()
    for name, x in zip(("o", "dq", "dk", "dv"), out):
        softmax.check(x.flip(1) if backwards else x, want[name], name)


def test_no_tokens(cuda):
    for shape in ((0, 5), (2, 0)):
        leaves = [torch.zeros(*shape, 2, 64, dtype=BF16, device=cuda, requires_grad=True) for _ in range(3)]
        o = L.softmax_attn(*leaves, head_first=False)
        assert o.shape == (*shape, 2, 64)
        for g, x in zip(torch.autograd.grad(o.sum(), leaves), leaves):
            assert g.shape == x.shape


def test_only_the_gradients_that_are_wanted(cuda):
    q, k, v, do = (x.to(cuda) for x in inputs(59, 1, 100, 4, 2, 64, 64, BF16))
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    full = torch.autograd.grad(L.softmax_attn(*leaves, head_first=False), leaves, do)
    for i in range(3):
        xs = [q, k, v]
        xs[i] = xs[i].detach().requires_grad_(True)
        (g,) = torch.autograd.grad(L.softmax_attn(*xs, head_first=False), xs[i], do)
        assert torch.equal(g, full[i])


@pytest.mark.parametrize("odd", [False, True])
def test_saved_tensor_hooks_and_checkpoint(cuda, odd):
    """Hooks that hand back other types and strides: gradients of the same values (odd: rows off 16 bytes, which take the node in
    Python)."""
    q, k, v, do = (x.to(cuda) for x in inputs(61, 1, 130, 4, 2, 64, 64, BF16))
    if odd:
        q, k, v = (torch.empty(x.numel() + 1, dtype=BF16, device=cuda)[1:].view(x.shape).copy_(x) for x in (q, k, v))

    def all_of(f):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        return torch.autograd.grad(f(*leaves), leaves, do)

    op = lambda *xs: L.softmax_attn(*xs, head_first=False, slopes=alibi(4).to(cuda), prefix_lens=torch.tensor([9], device=cuda))
    plain = all_of(op)

    def unpack(x):
        if not x.is_floating_point():
            return x.long()
        wide = torch.empty(*x.shape, 2, dtype=torch.float64, device=x.device)[..., 0]
        return wide.copy_(x)

    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
        hooked = all_of(op)
    again = all_of(lambda *xs: torch.utils.checkpoint.checkpoint(op, *xs, use_reentrant=False))
    for a, b, c in zip(plain, hooked, again):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("D", [64, 60])              # (60: padded, 64 as it is)
def test_second_derivatives_are_refused(cuda, D):
    q, k, v, do = (x.to(cuda).requires_grad_(True) for x in inputs(67, 1, 20, 2, 2, D, D, F32))
    plain = torch.autograd.grad(L.softmax_attn(q, k, v, head_first=False), (q, k, v), do)
    grads = torch.autograd.grad(L.softmax_attn(q, k, v, head_first=False), (q, k, v), do, create_graph=True)
    for a, b in zip(plain, grads):
        assert torch.equal(a, b)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(b.sum(), q, retain_graph=True)


def test_the_node_keeps_to_the_rules_of_autograd(cuda):
    q, k, v, do = (x.to(cuda) for x in inputs(71, 1, 40, 4, 2, 64, 64, BF16))
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    op = lambda: L.softmax_attn(q * 1, k, v, head_first=False)
    o = op()
    first = torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(o, (q, k, v), do)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(o, (q, k, v), do)
    for bad in (q, o):                                # what it saved has changed: the inputs, and the output
        o = op() if bad is q else o
        x = q * 1
        o = L.softmax_attn(x, k, v, head_first=False)
        with torch.no_grad():
            (x if bad is q else o).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(o, (q, k, v), do)
    # outputs in a chain, a gradient that never arrives, and the memory of a node that goes unused
    y = L.softmax_attn(L.softmax_attn(q, q, q, head_first=False), k.expand(1, 40, 2, 64), v, head_first=False)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(y, (q, k, v), do))
    assert torch.autograd.grad(op().sum() * 0 + k.sum(), v, allow_unused=True)[0].abs().max() == 0
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    o = op()
    del o, y
    assert torch.cuda.memory_allocated() <= before


def test_a_captured_step_follows_offsets_and_prefixes(cuda):
    """Forward and backward in one graph, replayed with other inputs, offsets and prefixes, the program's own work between."""
    shape = dict(B=1, T=400, HQ=4, HKV=2, K=64, V=64)
    q, k, v, do = (x.to(cuda) for x in inputs(71, dtype=BF16, **shape))
    cu = torch.tensor([0, 100, 250, 400], dtype=torch.int32, device=cuda)
    pre = torch.tensor([10, 0, 70], dtype=torch.int32, device=cuda)

    def step():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        o = L.softmax_attn(*leaves, cu_seqlens=cu, prefix_lens=pre, head_first=False)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed, (offs, prefix) in enumerate((([0, 100, 250, 400], [10, 0, 70]), ([0, 0, 333, 400], [0, 64, 1]), ([0, 64, 128, 390], [64, 3, 262]))):
        for x, y in zip((q, k, v, do), inputs(300 + 7 * seed, dtype=BF16, **shape)):
            x.copy_(y)
        cu.copy_(torch.tensor(offs))
        pre.copy_(torch.tensor(prefix))
        graph.replay()
        got = [x.clone() for x in out]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b), seed


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (F32, 64)])
def test_a_long_sequence(cuda, dtype, D):
    """Rows of thousands of keys, checked on some of the rows against float64 (the rest of the sequence's keys and values
    are there all the same)."""
    T, HQ, HKV = 5003, 2, 1
    q, k, v, do = inputs(73, 1, T, HQ, HKV, D, D, dtype)
    o = L.softmax_attn(*(x.to(cuda) for x in (q, k, v)), head_first=False)
    for i in (0, 1, 4095, 4096, 5002):
        for h in range(HQ):
            ref = softmax.head(q[0, i:i + 1, h], k[0, :i + 1, 0], v[0, :i + 1, 0], D ** -0.5, dtype=dtype)
            softmax.check(o[0, i:i + 1, h], ref, (i, h))
