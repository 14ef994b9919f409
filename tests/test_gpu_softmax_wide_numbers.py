"""Whole numbers of 64 bits that 32 do not hold: page numbers, lengths and prefixes keep their meaning."""
import pytest
import torch

import linear_moe_amd as L
from oracle import softmax
from tests.test_gpu_paged_kv import Cache, same
from tests.test_gpu_softmax_attn import inputs
from tests.util import gen

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
WIDE = 2 ** 32


def test_page_numbers_that_name_no_page(cuda):
    """A number beyond 32 bits names no page, whatever its lower half: nothing is read or written there."""
    c = Cache(29, [40, 40], 16, 1, 64, 64, BF16, spare=1)
    kp, vp, table, lens = c.to(cuda)
    table = table.long()
    table[0, 1] += WIDE
    table[1, 2] += 5 * WIDE
    q, kn, vn = (gen(30 + i, 2, 1, n, 64, dtype=BF16).to(cuda) for i, n in enumerate((2, 1, 1)))
    o = L.paged_attn_decode(q, kp, vp, table, lens, head_first=False)
    for n, gone in ((0, range(16, 32)), (1, range(32, 40))):
        live = [j for j in range(40) if j not in gone]
        kk, vv = (x[live, 0] for x in c.rows[n])
        for h in range(2):
            softmax.check(o[n, :, h], softmax.head(q[n, :, h].cpu(), kk, vv, 0.125, dtype=BF16), (n, h))
    keep = kp.clone(), vp.clone()
    table[0, 2] -= WIDE                                         # (a negative one)
    L.paged_attn_decode(q, kp, vp, table, lens, kn, vn, head_first=False)
    L.paged_kv_append(kp, vp, kn, vn, table, lens, head_first=False)
    assert same(kp, keep[0]) and same(vp, keep[1])


def test_lengths(cuda):
    c = Cache(31, [32, 32], 16, 1, 64, 64, BF16, spare=0)
    kp, vp, table, _ = c.to(cuda)
    table = table[:, :2]
    q, kn, vn = (gen(40 + i, 2, 1, n, 64, dtype=BF16).to(cuda) for i, n in enumerate((1, 1, 1)))
    lens = torch.tensor([WIDE + 3, -WIDE + 3], device=cuda)     # the whole table, and nothing
    o = L.paged_attn_decode(q, kp, vp, table, lens, head_first=False)
    kk, vv = (x[:, 0] for x in c.rows[0])
    softmax.check(o[0, :, 0], softmax.head(q[0, :, 0].cpu(), kk, vv, 0.125, dtype=BF16))
    assert (o[1] == 0).all()
    keep = kp.clone(), vp.clone()
    L.paged_kv_append(kp, vp, kn, vn, table, lens, head_first=False)
    assert same(kp, keep[0]) and same(vp, keep[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prefixes(cuda, dtype):
    q, k, v, _ = inputs(149, 2, 70, 2, 1, 64, 64, dtype)
    want = softmax.attn(q, k, v, prefix_lens=[70, 0])
    o = L.softmax_attn(*(x.to(cuda) for x in (q, k, v)), prefix_lens=torch.tensor([WIDE + 1, -WIDE + 9], device=cuda), head_first=False)
    softmax.check(o, want["o"])
