"""Norm and rotation of queries and keys on the GPU, against float64 within derived bounds (oracle/rope.py)."""
import ctypes as C

import pytest
import torch

import linear_moe_amd as L
from linear_moe_amd import _lib
from oracle import rope
from tests.util import gen

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def positions_of(B, T, offsets=None, lens=None, table=None):
    """[B, T] positions; -1 in rows behind the last sequence."""
    if table is not None:
        return table.expand(B, T).long()
    if lens is None:
        pos = torch.arange(T).expand(B, T)
        return pos + (0 if offsets is None else torch.tensor(offsets)[:, None])
    pos = torch.full((1, T), -1)
    at = 0
    for n, m in enumerate(lens):
        pos[0, at:at + m] = torch.arange(m) + (0 if offsets is None else offsets[n])
        at += m
    return pos


def check(cuda, B, T, HQ, HKV, D, dtype, R=None, interleaved=False, norm=True, wdtype=None, eps=1e-6, offsets=None, lens=None, positions=None,
          L_table=None, head_first=False, seed=7, make=None, x=None, cu_dtype=torch.int32):
    R = D if R is None else R
    lay = (lambda y: y.transpose(1, 2)) if head_first else (lambda y: y)
    q, k, dq, dk = (gen(seed + i, B, T, H, D, dtype=dtype) for i, H in enumerate((HQ, HKV, HQ, HKV)))
    if x is not None:
        q, k = x(q), x(k)
    qw, kw = (None, None) if wdtype is None else (1 + 0.3 * gen(seed + 5 + i, D, dtype=wdtype) for i in range(2))
    pos = positions_of(B, T, offsets, lens, positions)
    cos, sin = L.rope_table(int(pos.max()) + 1 if L_table is None else L_table, R) if R else (None, None)
    real = torch.ones(B, T, dtype=torch.bool) if lens is None else (torch.arange(T) < sum(lens))[None]
    c, s = rope.angles(pos, cos, sin) if R else (torch.ones(B, T, 0), torch.zeros(B, T, 0))
    c, s = c.double()[:, :, None], s.double()[:, :, None]
    make = make or (lambda y: y.to(cuda))
    leaves = [lay(make(y)).detach().requires_grad_(True) for y in (q, k)] + [w.to(cuda).requires_grad_(True) for w in (qw, kw) if w is not None]
    ints = lambda y: None if y is None else torch.tensor(y, dtype=torch.int32, device=cuda)
    cu = None
    if lens is not None:
        cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=cu_dtype, device=cuda)
    call = lambda: L.qk_norm_rope(*leaves[:2], *(leaves[2:] or (None, None)), *((cos.to(cuda), sin.to(cuda)) if R else (None, None)),
                                  positions=None if positions is None else positions.to(cuda), offsets=ints(offsets), cu_seqlens=cu, eps=eps, norm=norm,
                                  interleaved=interleaved, head_first=head_first)
    z = call()
    with torch.no_grad():
        z2 = call()
    assert all(torch.equal(a, b) for a, b in zip(z, z2))                # the path without a node: the same bits
    got = torch.autograd.grad(z, leaves, [lay(y.to(cuda)) for y in (dq, dk)])
    again = torch.autograd.grad(call(), leaves, [lay(y.to(cuda)) for y in (dq, dk)])
    assert all(torch.equal(a, b) for a, b in zip(got, again))           # no sum depends on an order that changes
    for i, (x_, w, dz) in enumerate(((q, qw, dq), (k, kw, dk))):
        dz = torch.where(real[..., None, None], dz, torch.zeros_like(dz))
        xr = torch.where(real[..., None, None], x_, torch.zeros_like(x_))
        bz, bx, bw = rope.bounds(xr, w, c, s, R, interleaved, eps, dtype, norm, dz, wdtype or F32)
        leaf = xr.double().requires_grad_(True)
        wl = None if w is None else w.double().requires_grad_(True)
        ref = rope.forward(leaf, wl, c, s, R, interleaved, eps, norm)
        grads = torch.autograd.grad(ref, [leaf] + ([] if w is None else [wl]), dz.double())
        out, dx = lay(z[i]).cpu().double(), lay(got[i]).cpu().double()
        assert z[i].dtype == dtype and z[i].shape == leaves[i].shape and z[i].is_contiguous()
        for name, a, b, tol in (("z", out, ref.detach(), bz), ("dx", dx, grads[0], bx)):
            off = (a - torch.where(real[..., None, None], b, torch.zeros_like(b))).abs()
            assert (off <= torch.where(real[..., None, None], tol, torch.zeros_like(tol))).all(), (i, name, (off / tol.clamp_min(1e-300)).max())
        if w is not None:
            off = (got[2 + i].cpu().double() - grads[1]).abs()
            assert got[2 + i].dtype == wdtype and (off <= bw).all(), (i, "dw", (off / bw).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (64, 32), (96, 96), (256, 256), (80, 40), (36, 18), (2, 2), (8, 0), (128, 16), (250, 250), (16, 16), (32, 16)])
def test_dims(cuda, dtype, interleaved, D, R):
    check(cuda, 2, 5, 6, 2, D, dtype, R, interleaved, wdtype=dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R,off", [(36, 36, 0), (80, 40, 0), (80, 40, 4), (128, 96, 2), (128, 128, 1), (200, 100, 2), (256, 64, 2), (118, 118, 0), (254, 100, 0), (64, 40, 0), (62, 2, 0)])
def test_pieces_of_a_row(cuda, dtype, interleaved, D, R, off):
    """Rows that begin anywhere and columns that no 16 bytes divide; few tokens, and enough of them for several heads at a time."""
    def shifted(y):
        out = torch.zeros(y.numel() + 8, dtype=y.dtype, device=cuda)[off:off + y.numel()].view(y.shape)
        return out.copy_(y)
    for B, T, HQ, HKV in ((2, 3, 5, 2), (1, 1501, 9, 3)):
        check(cuda, B, T, HQ, HKV, D, dtype, R, interleaved, wdtype=F32, make=shifted)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,HQ,HKV", [(1, 1, 1, 1), (1, 1, 16, 4), (3, 1, 5, 1), (1, 333, 4, 4), (2, 129, 7, 3), (1, 1111, 12, 12), (5, 64, 1, 9)])
def test_sizes(cuda, dtype, B, T, HQ, HKV):
    check(cuda, B, T, HQ, HKV, 64, dtype, wdtype=F32, head_first=T % 2 == 0)


@pytest.mark.parametrize("norm,wdtype", [(False, None), (True, None), (True, BF16), (True, F32)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_and_weights(cuda, norm, wdtype, dtype):
    check(cuda, 2, 9, 4, 2, 128, dtype, norm=norm, wdtype=wdtype)
    check(cuda, 2, 9, 4, 2, 36, dtype, norm=norm, wdtype=wdtype, interleaved=True)


@pytest.mark.parametrize("cu_dtype", [torch.int32, torch.int64])
def test_packed_documents_offsets_and_rows_behind(cuda, cu_dtype):
    check(cuda, 1, 60, 4, 2, 64, BF16, lens=[1, 0, 17, 0, 0, 30], wdtype=BF16, cu_dtype=cu_dtype)
    check(cuda, 1, 60, 4, 2, 64, BF16, lens=[0, 1, 17, 12, 30, 0], offsets=[5, 0, 1000, 3, 2, 9], wdtype=F32, cu_dtype=cu_dtype)
    check(cuda, 1, 40, 3, 1, 36, F32, lens=[0, 0], wdtype=F32, L_table=1, cu_dtype=cu_dtype)                          # nothing but rows behind
    check(cuda, 1, 300, 3, 1, 64, F32, lens=[1] * 300, offsets=list(range(300)), cu_dtype=cu_dtype)
    for n in (1023, 1024, 1025, 2100):                                                                                # as many as a work-group keeps, and more
        check(cuda, 1, n + 9, 3, 1, 64, BF16, lens=[(3 * i) % 4 and 1 for i in range(n)], offsets=[i % 50 for i in range(n)], cu_dtype=cu_dtype)


def test_rows_behind_the_last_document_do_not_spread(cuda):
    def spoilt(y):
        y = y.clone()
        y[:, 48:] = float("nan")
        return y
    check(cuda, 1, 60, 4, 2, 64, BF16, lens=[18, 30], wdtype=BF16, x=spoilt)


def test_positions(cuda):
    check(cuda, 3, 1, 4, 2, 64, BF16, offsets=[0, 7, 31000], wdtype=BF16)
    check(cuda, 2, 6, 4, 2, 64, F32, positions=torch.tensor([5, 4, 3, 2, 1, 0]))
    check(cuda, 2, 6, 4, 2, 64, F32, positions=torch.tensor([[5, 4, 3, 2, 1, 0], [9, 9, 9, 0, 0, 1]], dtype=torch.int32))
    # outside the table: normed, not turned
    check(cuda, 2, 6, 4, 2, 64, F32, positions=torch.tensor([-1, 4, 3, -2 ** 31, 2 ** 31 - 1, 2 ** 40]), L_table=4)
    check(cuda, 2, 6, 4, 2, 64, F32, offsets=[-3, 2 ** 31 - 2], L_table=4)


def test_sizes_of_numbers(cuda):
    check(cuda, 1, 8, 4, 2, 64, F32, x=lambda y: y * 1e-3, wdtype=F32)
    check(cuda, 1, 8, 4, 2, 64, F32, x=lambda y: y * 1e15, wdtype=F32)
    check(cuda, 1, 8, 4, 2, 64, F32, x=lambda y: y * 0, eps=1e-5, wdtype=F32)
    check(cuda, 1, 8, 4, 2, 64, BF16, x=lambda y: y * 1e-4, wdtype=F32, eps=1e-5)


def test_a_nan_stays_in_its_row(cuda):
    q, k = gen(1, 1, 5, 4, 64).to(cuda), gen(2, 1, 5, 2, 64).to(cuda)
    cos, sin = L.rope_table(5, 64, device=cuda)
    good = L.qk_norm_rope(q, k, cos=cos, sin=sin, head_first=False)
    q[0, 2, 1, 7], k[0, 0, 0, 0] = float("nan"), float("inf")
    z = L.qk_norm_rope(q, k, cos=cos, sin=sin, head_first=False)
    bad = [torch.zeros(x.shape[:3], dtype=torch.bool) for x in (q, k)]
    bad[0][0, 2, 1] = bad[1][0, 0, 0] = True
    for a, b, m in zip(z, good, bad):
        assert torch.equal(a.cpu()[~m], b.cpu()[~m]) and a.cpu()[m].isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views(cuda, dtype):
    """q and k as views of one projection, rows on odd addresses, a transposed and a repeated one."""
    B, T, H, D = 2, 7, 4, 64
    w = gen(11, D, dtype=dtype).to(cuda)
    cos, sin = L.rope_table(T, D, device=cuda)
    big = gen(12, B, T, 3 * H * D + 1, dtype=dtype).to(cuda)
    for first in (0, 1):
        q, k = (big[..., first + i * H * D:first + (i + 1) * H * D].view(B, T, H, D) for i in (0, 2))
        # (every other token lies on an odd address, for either first column: the rows of such views are summed in another order than those of
        # contiguous ones, so that both are held to the bound of the definition)
        c, s = (y.double()[None, :, None] for y in (cos, sin))
        for x, y in zip((q, k), L.qk_norm_rope(q, k, w, w, cos, sin, head_first=False)):
            ref, tol = rope.forward(x, w, c, s, D, False, 1e-6), rope.bounds(x, w, c, s, D, False, 1e-6, dtype)
            assert ((y.double() - ref).abs() <= tol).all()
    x = gen(13, B, T, D, H, dtype=dtype).to(cuda).transpose(2, 3)
    one = gen(14, B, T, 1, D, dtype=dtype).to(cuda).requires_grad_(True)
    k = one.expand(B, T, H, D)
    a = L.qk_norm_rope(x, k, w, w, cos, sin, head_first=False)
    b = L.qk_norm_rope(x.contiguous(), k.contiguous(), w, w, cos, sin, head_first=False)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    g = torch.autograd.grad(a[1], one, torch.ones_like(a[1]))[0]
    parts = torch.autograd.grad(b[1], one, torch.ones_like(b[1]))[0]
    assert torch.equal(g, parts)


def test_against_differences(cuda):
    """The gradients in float32 against central differences of the definition in float64: of order h^2 off, 1e-8 here, beside the kernel's 96 roundings."""
    T, H, D = 5, 2, 16
    q, k, w = gen(21, 1, T, H, D), gen(22, 1, T, H, D), 1 + 0.2 * gen(23, D)
    cos, sin = L.rope_table(T, D)
    dz = gen(24, 1, T, H, D)
    leaves = [x.to(cuda).requires_grad_(True) for x in (q, k, w)]
    z = L.qk_norm_rope(*leaves, None, cos.to(cuda), sin.to(cuda), head_first=False)
    got = torch.autograd.grad(z[0], [leaves[0], leaves[2]], dz.to(cuda))
    c, s = (x.double()[None, :, None] for x in (cos, sin))
    loss = lambda x, y: float((rope.forward(x, y, c, s, D, False, 1e-6) * dz.double()).sum())
    h = 1e-4
    for seed in range(4):
        dx, dw = gen(30 + seed, 1, T, H, D).double(), gen(40 + seed, D).double()
        slope = (loss(q.double() + h * dx, w.double() + h * dw) - loss(q.double() - h * dx, w.double() - h * dw)) / (2 * h)
        mine = float((got[0].cpu().double() * dx).sum() + (got[1].cpu().double() * dw).sum())
        size = float((got[0].cpu().double() * dx).abs().sum() + (got[1].cpu().double() * dw).abs().sum())
        assert abs(slope - mine) <= 1e-5 * size


def test_one_weight_and_one_gradient(cuda):
    q, k, w = (gen(50 + i, *s).to(cuda) for i, s in enumerate(((2, 3, 4, 64), (2, 3, 2, 64), (64,))))
    cos, sin = L.rope_table(3, 64, device=cuda)
    both = [x.clone().requires_grad_(True) for x in (q, k, w, w)]
    z = L.qk_norm_rope(*both, cos, sin, head_first=False)
    full = torch.autograd.grad(z, both, [torch.ones_like(x) for x in z])
    for i in range(4):
        xs = [x.clone().requires_grad_(j == i) for j, x in enumerate((q, k, w, w))]
        z = L.qk_norm_rope(*xs, cos, sin, head_first=False)
        assert torch.equal(torch.autograd.grad(z, xs[i], [torch.ones_like(x) for x in z])[0], full[i])
    xs = [x.clone().requires_grad_(True) for x in (q, k)]
    z = L.qk_norm_rope(*xs, w, None, cos, sin, head_first=False)
    g = torch.autograd.grad(z[0], xs, torch.ones_like(z[0]), allow_unused=True)
    assert torch.equal(g[0], full[0]) and (g[1] is None or (g[1] == 0).all())


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_rotation_alone_keeps_nothing_of_its_input(cuda, interleaved):
    """Its gradient is the gradient turned back: q and k may be overwritten in between, in the node in native code and the one in Python."""
    cos, sin = L.rope_table(7, 64, device=cuda)
    for table in ((cos, sin), (cos.double(), sin.double())):             # (a table in 64 bits takes the path in Python)
        leaf = [gen(70 + i, 2, 7, h, 64, dtype=BF16).to(cuda).requires_grad_(True) for i, h in enumerate((4, 2))]
        q, k = (x * 1.0 for x in leaf)
        z = L.qk_norm_rope(q, k, None, None, *table, norm=False, interleaved=interleaved, head_first=False)
        with torch.no_grad():
            q.zero_(), k.fill_(float("nan"))
        dz = [gen(75 + i, *x.shape, dtype=BF16).to(cuda) for i, x in enumerate(z)]
        got = torch.autograd.grad(z, leaf, dz)
        back = L.qk_norm_rope(*dz, None, None, cos, -sin, norm=False, interleaved=interleaved, head_first=False)
        assert all(torch.equal(a, b) for a, b in zip(got, back))
        z = L.qk_norm_rope(*(x * 1.0 for x in leaf), None, None, *table, norm=False, interleaved=interleaved, head_first=False)
        g = torch.autograd.grad(z[1], leaf, dz[1], allow_unused=True)
        assert torch.equal(g[1], back[1]) and (g[0] is None or (g[0] == 0).all())


def test_the_node_in_python_gives_the_same_bits(cuda):
    """A call that needs a conversion takes the steps in Python."""
    q, k, w = (gen(90 + i, *s, dtype=BF16).to(cuda) for i, s in enumerate(((2, 9, 4, 64), (2, 9, 2, 64), (64,))))
    cos, sin = L.rope_table(40, 64, device=cuda)
    offs = torch.tensor([3, 30], dtype=torch.int32, device=cuda)
    out = []
    for c, s, o in ((cos, sin, offs), (cos.double(), sin.double(), offs.long())):
        leaves = [x.clone().requires_grad_(True) for x in (q, k, w, w)]
        z = L.qk_norm_rope(*leaves, c, s, offsets=o, head_first=False)
        out.append([*z, *torch.autograd.grad(z, leaves, [torch.ones_like(x) for x in z])])
    assert type(out[0][0].grad_fn) is not type(out[1][0].grad_fn)
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_a_workspace_that_is_not_needed_is_left_alone(cuda):
    """The block of a backward pass without gradients of weights asks for no workspace; one that is given all the same is not written."""
    q, k, dq, dk = (gen(100 + i, 2, 5, h, 64, dtype=BF16).to(cuda) for i, h in enumerate((4, 2, 4, 2)))
    a, out, ws = _lib.RopeArgs(), [torch.empty_like(q), torch.empty_like(k)], torch.full((4096,), 7.0, device=cuda)
    a.dtype = a.w_dtype = _lib.LMOE_BF16
    a.B, a.T, a.HQ, a.HKV, a.D, a.N, a.norm, a.eps = 2, 5, 4, 2, 64, 2, 1, 1e-6
    for n, x in dict(q=q, k=k, dzq=dq, dzk=dk, dq=out[0], dk=out[1]).items():
        setattr(a, n, _lib.Tensor4(x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)))
    lib = _lib.load()
    assert lib.lmoe_qk_norm_rope_floats(C.byref(a)) == 0
    a.ws = ws.data_ptr()
    assert lib.lmoe_qk_norm_rope_bwd(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    assert (ws == 7).all()
    leaves = [x.clone().requires_grad_(True) for x in (q, k)]
    got = torch.autograd.grad(L.qk_norm_rope(*leaves, head_first=False), leaves, [dq, dk])
    assert all(torch.equal(x, y) for x, y in zip(got, out))


def test_no_tokens(cuda):
    cos, sin = L.rope_table(4, 64, device=cuda)
    w = torch.ones(64, device=cuda, requires_grad=True)
    for shape in ((0, 5), (2, 0)):
        q, k = (torch.empty(*shape, H, 64, device=cuda, requires_grad=True) for H in (4, 2))
        z = L.qk_norm_rope(q, k, w, None, cos, sin, head_first=False)
        assert [x.shape for x in z] == [q.shape, k.shape]
        assert (torch.autograd.grad(z, w, [torch.ones_like(x) for x in z])[0] == 0).all()


def test_graph_and_stream(cuda):
    """Captured forward and backward, replayed with other positions; the table's rows follow what offsets holds then."""
    q, k = gen(61, 3, 1, 8, 64, dtype=BF16).to(cuda), gen(62, 3, 1, 2, 64, dtype=BF16).to(cuda)
    w = [gen(63 + i, 64, dtype=BF16).to(cuda) for i in range(2)]
    cos, sin = L.rope_table(50, 64, device=cuda)
    offs = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    want = {}
    for add in (0, 5, 40):
        want[add] = L.qk_norm_rope(q, k, *w, cos, sin, offsets=offs + add, head_first=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            L.qk_norm_rope(q, k, *w, cos, sin, offsets=offs, head_first=False)
        leaves = [x.clone().requires_grad_(True) for x in (q, k, *w)]
    torch.cuda.current_stream().wait_stream(side)
    g, train = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z = L.qk_norm_rope(q, k, *w, cos, sin, offsets=offs, head_first=False)
    with torch.cuda.graph(train):
        y = L.qk_norm_rope(*leaves, cos, sin, offsets=offs, head_first=False)
        grads = torch.autograd.grad(y, leaves, [torch.ones_like(x) for x in y])
    for add in (0, 5, 40, 0):
        offs.copy_(torch.tensor([0, 1, 2], dtype=torch.int32) + add)
        g.replay()
        train.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(z, want[add])) and all(torch.equal(a, b) for a, b in zip(y, want[add]))
        eager = [x.clone().detach().requires_grad_(True) for x in (q, k, *w)]
        out = L.qk_norm_rope(*eager, cos, sin, offsets=offs, head_first=False)
        ref = torch.autograd.grad(out, eager, [torch.ones_like(x) for x in out])
        assert all(torch.equal(a, b) for a, b in zip(grads, ref))


def test_large(cuda):
    """Rows enough for every lane group to take many."""
    check(cuda, 2, 6001, 10, 3, 64, BF16, wdtype=BF16)
    check(cuda, 1, 3001, 5, 2, 36, BF16, R=20, interleaved=True, wdtype=F32)


def test_refusals(cuda):
    q, k, w = torch.zeros(2, 3, 4, 64, device=cuda), torch.zeros(2, 3, 2, 64, device=cuda), torch.ones(64, device=cuda)
    cos, sin = L.rope_table(3, 64, device=cuda)
    ok = dict(cos=cos, sin=sin, head_first=False)
    L.qk_norm_rope(q, k, w, w, **ok)
    bad = [
        dict(q=q[0]), dict(q=q.half(), k=k.half()), dict(k=k.bfloat16()), dict(k=k[:1]), dict(k=k[..., :32]), dict(q=q[..., :63], k=k[..., :63]),
        dict(q=torch.zeros(1, 1, 1, 258, device=cuda), k=torch.zeros(1, 1, 1, 258, device=cuda)), dict(q_weight=w[:32]), dict(q_weight=w.half()),
        dict(q_weight=w, k_weight=w.bfloat16()), dict(q_weight=w, norm=False), dict(cos=None), dict(cos=None, sin=None, norm=False), dict(cos=cos[:2]),
        dict(cos=cos.cpu(), sin=sin.cpu()), dict(cos=torch.zeros(3, 33, device=cuda), sin=torch.zeros(3, 33, device=cuda)), dict(cos=cos.int(), sin=sin.int()),
        dict(eps=-1.0), dict(eps=float("nan")), dict(positions=torch.zeros(3, device=cuda)), dict(positions=torch.zeros(2, dtype=torch.int32, device=cuda)),
        dict(positions=torch.zeros(3, dtype=torch.int32, device=cuda), offsets=torch.zeros(2, dtype=torch.int32, device=cuda)),
        dict(offsets=torch.zeros(3, dtype=torch.int32, device=cuda)), dict(offsets=torch.zeros(2, device=cuda)), dict(offsets=torch.zeros(2, dtype=torch.int32)),
        dict(cu_seqlens=torch.tensor([0, 3], device=cuda)), dict(cu_seqlens=torch.tensor([0, 3]), head_first=True), dict(cos=cos.clone().requires_grad_(True)),
        dict(q=q[:1], k=k[:1], cu_seqlens=torch.tensor([0, 2])), dict(q=q[:1], k=k[:1], cu_seqlens=torch.tensor([3], device=cuda)),
    ]
    for change in bad:
        with pytest.raises(ValueError):
            L.qk_norm_rope(**{**dict(q=q, k=k), **ok, **change})
    with pytest.raises(RuntimeError):
        L.qk_norm_rope(q.cpu(), k.cpu(), **ok)
    with pytest.raises(RuntimeError):
        L.qk_norm_rope(q, k.cpu(), **ok)
    leaf = q.clone().requires_grad_(True)
    z = L.qk_norm_rope(leaf, k, **ok)[0]
    g = torch.autograd.grad(z.square().sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)
    # an offset that changes between forward and backward is noticed
    offs = torch.zeros(2, dtype=torch.int32, device=cuda)
    z = L.qk_norm_rope(leaf, k, offsets=offs, **ok)[0]
    offs += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        z.sum().backward()


def test_transforms_are_refused(cuda):
    from torch.autograd import forward_ad as fw
    q, k = gen(110, 2, 3, 4, 64).to(cuda), gen(111, 2, 3, 2, 64).to(cuda)
    cos, sin = L.rope_table(3, 64, device=cuda)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: L.qk_norm_rope(x, k, None, None, cos, sin, head_first=False)[0])(q[None])
    with pytest.raises(RuntimeError), fw.dual_level():
        L.qk_norm_rope(fw.make_dual(q, torch.ones_like(q)), k, None, None, cos, sin, head_first=False)


@pytest.mark.parametrize("native", [True, False])
def test_hooks_on_what_is_saved(cuda, native):
    """What a hook hands back may lie anywhere and have another type; another shape is noticed."""
    q, k, w = gen(120, 2, 3, 4, 64).to(cuda), gen(121, 2, 3, 2, 64).to(cuda), gen(122, 64).to(cuda)
    cos, sin = L.rope_table(9, 64, device=cuda)
    offs = torch.tensor([1, 6], dtype=torch.int32 if native else torch.int64, device=cuda)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, w)]
    call = lambda: L.qk_norm_rope(*leaves, None, cos, sin, offsets=offs, head_first=False)
    ones = lambda z: [torch.ones_like(x) for x in z]
    z = call()
    want = torch.autograd.grad(z, leaves, ones(z))
    away = lambda x: (x.cpu().double() if x.is_floating_point() else x.cpu().long()).transpose(0, -1).contiguous()
    with torch.autograd.graph.saved_tensors_hooks(away, lambda x: x.transpose(0, -1).to(cuda)):
        z = call()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(z, leaves, ones(z)), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x[:1]):
        z = call()
    with pytest.raises(RuntimeError, match="came back as"):
        torch.autograd.grad(z, leaves, ones(z))


def test_two_at_once(cuda):
    """Calls on two streams at the same time, forward and backward, and in inference mode: the bits of each by itself."""
    q, k, w = gen(130, 4, 700, 8, 128, dtype=BF16).to(cuda), gen(131, 4, 700, 2, 128, dtype=BF16).to(cuda), gen(132, 128, dtype=BF16).to(cuda)
    cos, sin = L.rope_table(700, 128, device=cuda)

    def step():
        leaves = [x.clone().requires_grad_(True) for x in (q, k, w, w)]
        z = L.qk_norm_rope(*leaves, cos, sin, head_first=False)
        return [*z, *torch.autograd.grad(z, leaves, [q, k])]
    want = step()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x in got for a, b in zip(x, want))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(L.qk_norm_rope(q, k, w, w, cos, sin, head_first=False), want))
