"""The workspace of a backward pass of softmax_attn is bounded, whatever the size of the batch (no GPU needed)."""
import ctypes as C

import pytest

from linear_moe_amd import _lib
from tests.test_softmax_host import FAKE, attn_args


def floats(T, HQ, HKV, D, docs=0, B=1, **kw):
    chunks = (T + 63) // 64
    packed = dict(cu_seqlens=FAKE, chunk_map=FAKE, N=docs, NT=chunks + docs) if docs else dict(N=B, NT=B * chunks)
    n = _lib.load().lmoe_softmax_attn_bwd_floats(C.byref(attn_args(B=B, T=T, HQ=HQ, HKV=HKV, K=D, V=D, **packed, **kw)))
    assert n >= 0 or (n == -8 and (chunks + docs) * HQ >= 2 ** 23), n      # (too many work-groups)
    return n


@pytest.mark.parametrize("T,HQ,HKV,D", [(32768, 8, 8, 128), (131072, 8, 8, 128), (131072, 32, 32, 128), (131072, 64, 8, 64), (2 ** 20, 8, 8, 64)])
@pytest.mark.parametrize("docs", [1, 23, 300, 5000])
def test_packed_calls_that_fill_the_card_many_times_have_none(T, HQ, HKV, D, docs):
    assert floats(T, HQ, HKV, D, docs) == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 4, 16])
@pytest.mark.parametrize("docs", [0, 1, 30, 400])
def test_at_most_a_gibibyte(D, G, docs):
    for HKV in (1, 3, 8, 32, 100, 512):
        for T in (1, 63, 255, 511, 1000, 4097, 16384, 16900, 40000, 131072, 300000):
            for causal in (0, 1):
                assert 4 * floats(T, HKV * G, HKV, D, docs, causal=causal) <= 2 ** 30, (T, HKV, causal)
