"""Caps of the scores from the least to the largest on the GPU: the error of a score must not grow with a cap that the scores are
far below.  Against float64, within the bounds of oracle/softmax.py."""
import pytest
import torch

import linear_moe_amd as L
from oracle import softmax
from tests.test_gpu_paged_kv import Cache, alibi, decode_and_check
from tests.test_gpu_softmax_attn import inputs, run_and_check

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

# (both sides of the border between the two forms of the kernels on 2-byte elements, and far beyond it)
CAPS = [1000.0, 1024.0, 1025.0, 1e4, 1e6, 1e8, 1e20, 1e30, 2.9e38]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("bias", [False, True])
def test_large_caps(cuda, dtype, D, cap, bias):
    q, k, v, do = inputs(113, 1, 190, 4, 2, D, D, dtype)
    run_and_check(cuda, 3 * q, k, v, do, softcap=cap, slopes=alibi(4) if bias else None, prefix=[70])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap", [1000.0, 1025.0, 1500.0, 4000.0])
def test_large_caps_that_the_scores_reach(cuda, dtype, cap):
    """Scores from a few units to several times the cap: both branches of the form for large caps."""
    q, k, v, do = inputs(127, 1, 190, 2, 1, 64, 64, dtype)
    spread = torch.logspace(-3, 2.5, 190)[None, :, None, None]
    run_and_check(cuda, (q * spread).to(dtype), (10 * k).to(dtype), v, do, softcap=cap)
    run_and_check(cuda, (q * spread).to(dtype), (10 * k).to(dtype), v, do, softcap=cap, scale=-0.25, causal=False)


@pytest.mark.parametrize("D", [64, 128])
def test_large_caps_in_long_sequences(cuda, D):
    """Two groups of waves to the rows, several work-groups to the keys, documents; and rows that take the kernels with 64-bit offsets."""
    x = inputs(131, 1, 1091, 2, 1, D, D, BF16)
    run_and_check(cuda, *x, softcap=1e6)
    run_and_check(cuda, *x, softcap=1e7, cu=[0, 3, 3, 131, 900, 1091], slopes=alibi(2))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap", [1e-12, 1e-30, 1e-41, 1e-60])
def test_least_caps(cuda, dtype, cap):
    """All scores are nothing: every row is the mean of what it sees.  (In 32 bits the last two are denormal and 0, which would be none.)"""
    x = inputs(137, 1, 130, 2, 1, 64, 64, dtype)
    run_and_check(cuda, *x, softcap=cap)
    run_and_check(cuda, *x, softcap=cap, slopes=alibi(2))
    zero = torch.zeros_like(x[0])
    run_and_check(cuda, zero, *x[1:], softcap=cap, scale=0.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap", CAPS + [1e-30, 1e-60])
@pytest.mark.parametrize("bias", [False, True])
def test_decoding(cuda, dtype, cap, bias):
    c = Cache(5, [1, 90, 1000], 32, 2, 64, 64, dtype)
    decode_and_check(cuda, c, 4, 64, 64, dtype, True, cap, alibi(4) if bias else None)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap", [1000.0, 1500.0])
def test_decoding_with_scores_that_reach_the_cap(cuda, dtype, cap):
    c = Cache(7, [40, 700], 16, 1, 64, 64, dtype)
    for n, (kk, _) in enumerate(c.rows):
        kk *= torch.logspace(0, 3.5, kk.shape[0])[:, None, None].to(dtype)
        for j in range(kk.shape[0]):
            c.put(n, j, kk[j], c.rows[n][1][j])
    decode_and_check(cuda, c, 2, 64, 64, dtype, softcap=cap)


def test_a_cap_beyond_all_scores_is_none(cuda):
    """In 2-byte elements: at 1e8 the outputs are those without a cap to the rounding of the output and of p."""
    q, k, v, _ = (x.to(cuda) for x in inputs(139, 2, 200, 4, 2, 64, 64, BF16))
    with torch.no_grad():
        plain = L.softmax_attn(q, k, v, head_first=False).double()
        capped = L.softmax_attn(q, k, v, softcap=1e8, head_first=False).double()
    bound = softmax.attn(*(x.cpu() for x in (q, k, v)))["o"][1].to(cuda)
    assert ((plain - capped).abs() <= 2 * bound).all()
