"""The paths that large training calls of softmax_attn take, all outputs and gradients against float64 (oracle/softmax.py, on the
GPU): one group of waves to the rows, tiles of keys that no, some or all work-groups share.  What a call shares is read off its
workspace, so that a rule that changes takes no path out of the tests unnoticed."""
import pytest
import torch

import linear_moe_amd as L
from oracle import softmax
from tests.test_gpu_softmax_attn import alibi, inputs
from tests.test_softmax_workspace import floats

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def check_all(cuda, x, cu=None, prefix=None, slopes=None, **kw):
    q, k, v, do = (y.to(cuda) for y in x)
    want = softmax.attn(q, k, v, do=do, cu=cu, prefix_lens=prefix, slopes=slopes, **kw)
    leaves = [y.requires_grad_(True) for y in (q, k, v)]
    o = L.softmax_attn(*leaves, head_first=False, cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device=cuda),
                       prefix_lens=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=cuda),
                       slopes=None if slopes is None else slopes.to(cuda), **kw)
    for name, y in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do))):
        softmax.check(y, want[name], name)


KINDS = ["causal", "whole", "prefix", "cap", "bias", "cap_bias"]


def options(kind, lens, H):
    kw = {"whole": dict(causal=False), "prefix": dict(prefix=[(7 * n) // 10 for n in lens])}.get(kind, {})
    if "cap" in kind:
        kw["softcap"] = 4.0
    if "bias" in kind:
        kw["slopes"] = alibi(H)
    return kw


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


LONG = [6000, 17, 4100, 0, 1200, 64, 5003]                                     # (of tiles with one, two, three and four parts)
MANY = [5000, 4097] + [(13 * n) % 50 for n in range(296)]                      # (more than a work-group looks through)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_documents_of_which_the_long_ones_are_shared(cuda, D, kind):
    T, HQ, HKV = sum(LONG), 8, 4
    assert floats(T, HQ, HKV, D, len(LONG)) == 4 * T * HKV * 2 * D
    check_all(cuda, inputs(151, 1, T, HQ, HKV, D, D, BF16), cu=offsets(LONG), **options(kind, LONG, HQ))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["causal", "cap"])
def test_many_documents_of_which_the_long_ones_are_shared(cuda, D, kind):
    T, HQ, HKV = 16384, 8, 4
    lens = MANY + [T - sum(MANY)]
    assert len(lens) > 256 and lens[-1] >= 0 and floats(T, HQ, HKV, D, len(lens)) == 4 * T * HKV * 2 * D
    check_all(cuda, inputs(157, 1, T, HQ, HKV, D, D, BF16), cu=offsets(lens), **options(kind, lens, HQ))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["causal", "whole", "cap"])
def test_documents_that_are_not_shared(cuda, D, kind):
    """Tiles for several times the card."""
    T, HQ, HKV = sum(LONG), 16, 16
    assert floats(T, HQ, HKV, D, len(LONG)) == 0
    check_all(cuda, inputs(163, 1, T, HQ, HKV, D, D, BF16), cu=offsets(LONG), **options(kind, LONG, HQ))


@pytest.mark.parametrize("D,parts", [(64, 4), (128, 2)])
@pytest.mark.parametrize("kind", KINDS)
def test_long_streams_that_are_shared(cuda, D, parts, kind):
    """A full card whose tiles of keys meet so many rows that several work-groups take them."""
    B, T, HQ, HKV = 2, 4100, 32, 8
    assert floats(T, HQ, HKV, D, B=B) == parts * B * T * HKV * 2 * D
    check_all(cuda, inputs(167, B, T, HQ, HKV, D, D, BF16), **options(kind, [T] * B, HQ))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_and_keys_that_are_not_shared(cuda, D, kind):
    B, T, H = 2, 2500, 16
    assert floats(T, H, H, D, B=B) == 0
    check_all(cuda, inputs(173, B, T, H, H, D, D, BF16), **options(kind, [T] * B, H))


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("kind", ["causal", "whole", "prefix", "cap_bias"])
def test_a_long_sequence_of_few_heads(cuda, dtype, D, kind):
    """Two groups of waves to the rows, up to 16 work-groups to a tile of keys."""
    check_all(cuda, inputs(179, 1, 5003, 2, 1, D, D, dtype), **options(kind, [5003], 2))
