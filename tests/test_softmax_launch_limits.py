"""Calls whose launches would have 2^32 threads or more are refused before anything is launched (no GPU needed)."""
import ctypes as C

import pytest

from linear_moe_amd import _lib
from tests.test_softmax_host import FAKE, attn_args, paged_args


@pytest.mark.parametrize("HQ,HKV,refused", [(252, 252, True), (252, 126, False), (128, 128, False)])
def test_the_wide_kernel_of_the_keys_counts_twice(HQ, HKV, refused):
    """More than 256 documents of 128 columns: as many work-groups of 512 threads as chunks times key heads."""
    lib = _lib.load()
    # (an odd address of ws, which is looked at behind the sizes: nothing gets as far as a launch)
    kw = dict(cu_seqlens=FAKE, chunk_map=FAKE, B=1, N=65535, T=64, NT=65535, HQ=HQ, HKV=HKV, K=128, V=128, ws=FAKE + 4)
    if not refused:
        kw["ws"] = None
    a = attn_args(**kw)
    code = lib.lmoe_softmax_attn_bwd_floats(C.byref(a))
    assert (code == -8) == refused, code
    if refused:
        assert lib.lmoe_softmax_attn_bwd(C.byref(a), None) == -8


@pytest.mark.parametrize("T", [2 ** 26 - 3, 2 ** 26 - 1])
def test_tokens_that_are_written(T):
    assert _lib.load().lmoe_paged_kv_append(C.byref(paged_args(B=1, N=1, T=T)), None) == -8
