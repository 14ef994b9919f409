"""More (sequence, head) pairs than work-groups of 512 threads in a launch."""
import pytest
import torch

import linear_moe_amd as L
from oracle import softmax
from tests.util import gen

pytestmark = pytest.mark.gpu


def test_eight_million_heads(cuda):
    """2^23 of them and more with a short cache: they all read the one page."""
    N, H, D, S = 65535, 129, 8, 16
    assert N * H >= 2 ** 23
    kp, vp = (gen(i, 1, S, H, D, dtype=torch.bfloat16).to(cuda) for i in (1, 2))
    q = gen(3, 64, 1, H, D, dtype=torch.bfloat16).to(cuda).repeat(1024, 1, 1, 1)[:N]
    table, lens = torch.zeros(N, 1, dtype=torch.int32, device=cuda), torch.full((N,), 11, dtype=torch.int32, device=cuda)
    o = L.paged_attn_decode(q, kp, vp, table, lens, head_first=False)
    for n in range(0, 64, 9):
        for h in (0, 64, 128):
            softmax.check(o[n, :, h], softmax.head(q[n, :, h].cpu(), kp[0, :11, h].cpu(), vp[0, :11, h].cpu(), D ** -0.5, dtype=torch.bfloat16), (n, h))
    for n0 in range(64, N, 64):
        m = min(64, N - n0)
        assert torch.equal(o[n0:n0 + m], o[:m]), n0
