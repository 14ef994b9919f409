"""The host side of softmax_attn and the paged cache, without a GPU: the argument blocks have the C layout, and every call that
the kernels do not take is refused before anything is launched."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

import linear_moe_amd as L
from linear_moe_amd import _lib

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "lmoe.h")
FAKE = 0x1000                                   # never dereferenced: every call below is refused, or has no tokens


@pytest.mark.parametrize("struct,cls", [("lmoe_attn_args", _lib.AttnArgs), ("lmoe_paged_args", _lib.PagedArgs)])
def test_argument_blocks_have_the_c_layout(struct, cls):
    fields = [f[0] for f in cls._fields_]
    prog = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){", f'printf("%zu\\n", sizeof({struct}));']
    prog += [f'printf("%zu\\n", offsetof({struct}, {f}));' for f in fields] + ["return 0;}"]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(src, "w").write("\n".join(prog))
        subprocess.check_call(["gcc", "-o", exe, src])
        out = [int(x) for x in subprocess.check_output([exe]).split()]
    assert out[0] == C.sizeof(cls)
    assert out[1:] == [getattr(cls, f).offset for f in fields]


def attn_args(**kw):
    a = _lib.AttnArgs()
    a.dtype, a.causal, a.B, a.T, a.HQ, a.HKV, a.K, a.V, a.N, a.NT = _lib.LMOE_BF16, 1, 2, 130, 4, 2, 64, 64, 2, 6
    a.scale = 1.0
    for n in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv"):
        setattr(a, n, _lib.Tensor4(FAKE, 130 * 256, 256, 64))
    a.lse = a.delta = FAKE
    for n, x in kw.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("code,kw", [
    (-2, dict(dtype=2)), (-3, dict(K=136)), (-3, dict(V=0)), (-3, dict(K=60)), (-3, dict(dtype=_lib.LMOE_F32, V=6)), (-4, dict(B=-1)),
    (-4, dict(HKV=0)), (-3, dict(HQ=5)), (-8, dict(HQ=65536, HKV=1)), (-4, dict(NT=5)), (-6, dict(N=1)), (-5, dict(cu_seqlens=FAKE)),
    (-5, dict(cu_seqlens=FAKE, chunk_map=FAKE)), (-4, dict(cu_seqlens=FAKE, chunk_map=FAKE, B=1, NT=6)), (-7, dict(k=_lib.Tensor4())),
    (-11, dict(dk=_lib.Tensor4())), (-15, dict(softcap=-1.0)), (-15, dict(softcap=float("nan"))), (-15, dict(softcap=float("inf"))),
    (-15, dict(causal=0, prefix_lens=FAKE)), (-9, dict(q=_lib.Tensor4(FAKE + 2, 0, 256, 64))), (-9, dict(dv=_lib.Tensor4(FAKE, 0, 260, 64))),
    (-8, dict(T=2 ** 30, NT=2 ** 25)),
    (-9, dict(o_low=FAKE + 4)), (-8, dict(dtype=_lib.LMOE_F32, T=2 ** 20, HQ=128, HKV=128, NT=2 ** 15))])
def test_softmax_attn_blocks_that_are_refused(code, kw):
    lib = _lib.load()
    for fn in (lib.lmoe_softmax_attn_fwd, lib.lmoe_softmax_attn_bwd):
        assert fn(C.byref(attn_args(**kw)), None) == code, lib.lmoe_last_error()
        assert fn(None, None) == -1


def test_softmax_attn_backward_needs_what_forward_kept():
    lib = _lib.load()
    for n in ("lse", "delta"):
        assert lib.lmoe_softmax_attn_bwd(C.byref(attn_args(**{n: None})), None) == -11
    for n in ("d_o", "dq"):
        assert lib.lmoe_softmax_attn_bwd(C.byref(attn_args(**{n: _lib.Tensor4()})), None) == -11
    for kw in (dict(T=0, NT=0), dict(B=0, N=0, NT=0)):         # no tokens: checked, and nothing launched
        assert lib.lmoe_softmax_attn_fwd(C.byref(attn_args(**kw)), None) == 0
        assert lib.lmoe_softmax_attn_bwd(C.byref(attn_args(**kw)), None) == 0


def paged_args(**kw):
    a = _lib.PagedArgs()
    a.dtype, a.N, a.HQ, a.HKV, a.K, a.V, a.P, a.S, a.M, a.B, a.T = _lib.LMOE_BF16, 3, 4, 2, 64, 64, 10, 16, 4, 3, 5
    a.scale, a.table_stride, a.table, a.lens, a.ws = 1.0, 4, FAKE, FAKE, FAKE
    for n in ("q", "o", "kp", "vp", "kn", "vn"):
        setattr(a, n, _lib.Tensor4(FAKE, 2048, 128, 64))
    for n, x in kw.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("code,kw", [
    (-2, dict(dtype=5)), (-3, dict(K=160)), (-3, dict(V=4)), (-4, dict(S=0)), (-4, dict(M=-1)), (-4, dict(HKV=0)), (-8, dict(N=70000)),
    (-8, dict(M=2 ** 20, S=2 ** 12)), (-8, dict(M=2 ** 25 + 1, S=2 ** 5)), (-7, dict(lens=None)), (-7, dict(table=None)), (-7, dict(vp=_lib.Tensor4())), (-11, dict(vn=_lib.Tensor4())),
    (-9, dict(kp=_lib.Tensor4(FAKE, 2048, 130, 64))), (-9, dict(kn=_lib.Tensor4(FAKE + 8, 2048, 128, 64)))])
def test_paged_blocks_that_are_refused(code, kw):
    lib = _lib.load()
    for fn in (lib.lmoe_paged_attn_decode, lib.lmoe_paged_kv_append):
        assert fn(C.byref(paged_args(**kw)), None) == code, lib.lmoe_last_error()
        assert fn(None, None) == -1
    assert lib.lmoe_paged_attn_floats(C.byref(paged_args(**kw))) == code


def test_paged_blocks_of_one_op_that_are_refused():
    lib = _lib.load()
    decode, append = lib.lmoe_paged_attn_decode, lib.lmoe_paged_kv_append
    assert decode(C.byref(paged_args(HQ=3)), None) == -3
    assert decode(C.byref(paged_args(HQ=65535 * 2, HKV=1)), None) == -8
    assert decode(C.byref(paged_args(HQ=60000, HKV=1, N=60000)), None) == -8
    assert decode(C.byref(paged_args(softcap=-2.0)), None) == -15
    assert decode(C.byref(paged_args(q=_lib.Tensor4())), None) == -7
    assert append(C.byref(paged_args(kn=_lib.Tensor4(), vn=_lib.Tensor4())), None) == -7
    assert append(C.byref(paged_args(B=2)), None) == -6
    assert append(C.byref(paged_args(cu_seqlens=FAKE)), None) == -6
    assert append(C.byref(paged_args(T=2 ** 26)), None) == -8
    assert append(C.byref(paged_args(T=0)), None) == 0         # no tokens, no sequences: nothing launched
    assert decode(C.byref(paged_args(N=0)), None) == 0


def test_a_call_that_is_cut_needs_its_workspace():
    lib = _lib.load()
    a = paged_args(M=1000, N=1)
    n = lib.lmoe_paged_attn_floats(C.byref(a))
    assert n > 0 and n % ((64 + 2) * 4) == 0
    for ws in (None, FAKE + 4):
        a.ws = ws
        assert lib.lmoe_paged_attn_decode(C.byref(a), None) == -11


class OnGpu:
    """What the checks see of a GPU tensor: everything but data."""

    def __init__(self, *shape, dtype=torch.bfloat16, index=0, requires_grad=False):
        self._t = torch.empty(*shape, device="meta", dtype=dtype)
        self.shape, self.dtype, self.device, self.is_cuda, self.requires_grad = self._t.shape, dtype, torch.device("cuda", index), True, requires_grad

    def __getattr__(self, n):
        return getattr(self._t, n)

    def data_ptr(self):
        return FAKE


@pytest.fixture
def device0(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr("linear_moe_amd._host.stream_ptr", lambda: 0)


def test_softmax_attn_refuses_before_any_launch(device0):
    x = torch.zeros(1, 2, 8, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        L.softmax_attn(x, x, x)
    q, k = OnGpu(1, 8, 4, 64), OnGpu(1, 8, 2, 64)
    for bad, what in ((dict(q=OnGpu(1, 8, 3, 64)), "no multiple"), (dict(q=OnGpu(8, 4, 64)), "4-dimensional"), (dict(v=OnGpu(1, 9, 2, 64)), "mismatch"),
                      (dict(k=OnGpu(1, 8, 2, 72)), "mismatch"), (dict(q=OnGpu(1, 8, 4, 64, dtype=torch.float16)), "dtype"),
                      (dict(v=OnGpu(1, 8, 2, 136)), "unsupported"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap"),
                      (dict(slopes=OnGpu(3)), "slopes must be 4"), (dict(slopes=OnGpu(4, requires_grad=True)), "constants"),
                      (dict(prefix_lens=OnGpu(1, dtype=torch.int32), causal=False), "causal"), (dict(prefix_lens=OnGpu(2, dtype=torch.int32)), "whole numbers"),
                      (dict(prefix_lens=OnGpu(1)), "whole numbers"), (dict(prefix_lens=torch.zeros(1, dtype=torch.int32)), "live on"),
                      (dict(cu_seqlens=torch.tensor([0, 8]), head_first=True, q=k, k=k), "head_first=False"), (dict(cu_seqlens=torch.tensor([0, 7])), "end at T"),
                      (dict(cu_seqlens=torch.tensor([0, 8]), q=OnGpu(2, 8, 4, 64), k=OnGpu(2, 8, 2, 64), v=OnGpu(2, 8, 2, 64)), "batch size 1")):
        with pytest.raises(ValueError, match=what):
            L.softmax_attn(**{**dict(q=q, k=k, v=k, head_first=False), **bad})
    with pytest.raises(RuntimeError, match="current device"):
        L.softmax_attn(OnGpu(1, 8, 4, 64, index=1), OnGpu(1, 8, 2, 64, index=1), OnGpu(1, 8, 2, 64, index=1), head_first=False)
    with pytest.raises(RuntimeError, match="one device"):
        L.softmax_attn(q, OnGpu(1, 8, 2, 64, index=1), k, head_first=False)


def test_the_paged_cache_refuses_before_any_launch(device0):
    pages, table, lens = OnGpu(10, 16, 2, 64), OnGpu(3, 4, dtype=torch.int32), OnGpu(3, dtype=torch.int32)
    q, new = OnGpu(3, 1, 4, 64), OnGpu(3, 1, 2, 64)
    x = torch.zeros(10, 16, 2, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        L.paged_attn_decode(x, x, x, x, x)
    decode = dict(q=q, k_pages=pages, v_pages=pages, page_table=table, lens=lens, head_first=False)
    for bad, what in ((dict(k_pages=OnGpu(10, 16, 64)), "must be"), (dict(v_pages=OnGpu(9, 16, 2, 64)), "agree"), (dict(k_pages=OnGpu(10, 16, 2, 60)), "unsupported"),
                      (dict(k_pages=OnGpu(10, 16, 2, 64, dtype=torch.float16)), "dtype"), (dict(page_table=OnGpu(3, 4)), "whole numbers"),
                      (dict(page_table=OnGpu(3, dtype=torch.int32)), "page_table"), (dict(page_table=OnGpu(3, 4, dtype=torch.int32, index=1)), "page_table"),
                      (dict(lens=OnGpu(4, dtype=torch.int32)), "lens"), (dict(lens=OnGpu(3)), "lens"), (dict(q=OnGpu(3, 1, 5, 64)), "no multiple"),
                      (dict(q=OnGpu(2, 1, 4, 64)), "q must have shape"), (dict(q=OnGpu(3, 2, 4, 64)), "q must have shape"), (dict(q=OnGpu(3, 1, 4, 64, dtype=torch.float32)), "like the pages"),
                      (dict(k=new), "go together"), (dict(k=OnGpu(3, 1, 4, 64), v=new), "k must have shape"), (dict(softcap=float("nan")), "softcap"),
                      (dict(slopes=OnGpu(2)), "slopes must be 4")):
        with pytest.raises(ValueError, match=what):
            L.paged_attn_decode(**{**decode, **bad})
    with pytest.raises(RuntimeError, match="no backward"):
        L.paged_attn_decode(**{**decode, "q": OnGpu(3, 1, 4, 64, requires_grad=True)})
    with pytest.raises(RuntimeError, match="current device"):
        L.paged_attn_decode(**{**decode, "k_pages": OnGpu(10, 16, 2, 64, index=1)})
    append = dict(k_pages=pages, v_pages=pages, k=new, v=new, page_table=table, lens=lens, head_first=False)
    for bad, what in ((dict(k=OnGpu(3, 2, 64)), "4-dimensional"), (dict(k=OnGpu(2, 1, 2, 64)), "k must have shape"), (dict(v=OnGpu(3, 2, 2, 64)), "v must have shape"),
                      (dict(cu_seqlens=torch.tensor([0, 1, 2, 3])), "batch size 1"), (dict(cu_seqlens=torch.tensor([0, 1, 2, 3]), head_first=True), "head_first=False"),
                      (dict(cu_seqlens=torch.tensor([0, 9]), k=OnGpu(1, 9, 2, 64), v=OnGpu(1, 9, 2, 64)), "4 offsets"),
                      (dict(cu_seqlens=torch.tensor([0, 5, 4, 9]), k=OnGpu(1, 9, 2, 64), v=OnGpu(1, 9, 2, 64)), "non-decreasing")):
        with pytest.raises(ValueError, match=what):
            L.paged_kv_append(**{**append, **bad})
    with pytest.raises(RuntimeError, match="no backward"):
        L.paged_kv_append(**{**append, "v": OnGpu(3, 1, 2, 64, requires_grad=True)})
