"""What softmax_attn and the paged cache make of the plain numbers of a call, without a GPU."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

import linear_moe_amd as L
from linear_moe_amd.softmax_attn import cap_of, ints_of, slopes_of


@pytest.mark.parametrize("cap,want", [(None, 0.0), (0, 0.0), (30, 30.0), (1e-20, 1e-20), (1e-41, 2.0 ** -126), (1e-60, 2.0 ** -126), (5e-324, 2.0 ** -126)])
def test_a_cap_stays_one_in_32_bits(cap, want):
    assert cap_of(cap, "op") == want and (C.c_float(cap_of(cap, "op")).value > 0) == bool(cap)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.uint8])
def test_whole_numbers_in_32_bits_keep_their_meaning(dtype):
    """What 32 bits do not hold is as far out of range as before."""
    far = [2 ** 32 + 3, -2 ** 32 + 3, 2 ** 31, -2 ** 31 - 1, 2 ** 62] if dtype == torch.int64 else []
    x = torch.tensor([0, 1, 100] + far, dtype=dtype)
    got = ints_of(x, x.numel(), x.device, "x")
    assert got.dtype == torch.int32 and got[:3].tolist() == [0, 1, 100]
    assert got[3:].tolist() == [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1][:len(far)]


def test_forward_mode_and_traces_are_refused():
    """The paged ops and slopes have no derivatives: a tangent is refused like a gradient, not dropped; so is a trace, which would hold
    none of the writes."""
    x, t, n = torch.zeros(2, 4, 1, 64), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    new, rows = torch.zeros(2, 1, 1, 64), dict(page_table=t, lens=n, head_first=False)
    decode = lambda **kw: L.paged_attn_decode(**{**dict(q=new, k_pages=x, v_pages=x, k=new, v=new, slopes=torch.zeros(1)), **rows, **kw})
    append = lambda **kw: L.paged_kv_append(**{**dict(k_pages=x, v_pages=x, k=new, v=new), **rows, **kw})
    with forward_ad.dual_level():
        dual = lambda y: forward_ad.make_dual(y, torch.ones_like(y))
        for op, names in ((decode, ("q", "k", "v", "k_pages", "v_pages", "slopes")), (append, ("k", "v", "k_pages", "v_pages"))):
            for name in names:
                like = torch.zeros(1) if name == "slopes" else x if "pages" in name else new
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    op(**{name: dual(like)})
            with pytest.raises(RuntimeError, match="GPU only"):        # (nothing wrong with a call that has none)
                op()
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            slopes_of(dual(torch.zeros(4)), 4, torch.device("cpu"), "softmax_attn")
        assert slopes_of(torch.zeros(4), 4, torch.device("cpu"), "softmax_attn").shape == (4,)
    for op in (decode, append):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(lambda q: op(k=q) if op is append else op(q=q), (new,))
