"""Tables of pages of other widths than the longest sequence needs: as wide as a server's longest context, and of no column at all."""
import pytest
import torch

import linear_moe_amd as L
from oracle import softmax
from tests.test_gpu_paged_kv import Cache, alibi, decode_and_check
from tests.util import gen

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def widened(c, cols):
    """The columns behind the cache's own hold numbers that name no page, and some that do (of positions that no length reaches)."""
    more = torch.full((c.table.shape[0], cols - c.table.shape[1]), -1, dtype=torch.int32)
    more[:, ::2] = 0
    c.table = torch.cat([c.table, more], 1)
    return c


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols", [65, 512, 8192])            # (of 16 positions: two stretches, 16 and more than the longest has use for)
@pytest.mark.parametrize("append", [False, True])
def test_short_sequences_in_a_wide_table(cuda, dtype, cols, append):
    c = widened(Cache(41, [0, 1, 500, 15, 513, 900], 16, 2, 64, 64, dtype), cols)
    decode_and_check(cuda, c, 4, 64, 64, dtype, append, slopes=alibi(4))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_and_short_sequences_in_a_wide_table(cuda, dtype):
    c = widened(Cache(43, [5000, 3], 16, 1, 128, 128, dtype), 4096)
    decode_and_check(cuda, c, 2, 128, 128, dtype, True)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_table_without_columns(cuda, dtype):
    """No position exists: a token attends to itself alone, and nothing is written."""
    kp, vp = (torch.zeros(2, 16, 1, 64, dtype=dtype, device=cuda) for _ in range(2))
    table, lens = torch.zeros(3, 0, dtype=torch.int32, device=cuda), torch.tensor([0, 5, -2], dtype=torch.int32, device=cuda)
    q, k, v = (gen(50 + i, 3, 1, h, 64, dtype=dtype).to(cuda) for i, h in enumerate((2, 1, 1)))
    assert (L.paged_attn_decode(q, kp, vp, table, lens, head_first=False) == 0).all()
    o = L.paged_attn_decode(q, kp, vp, table, lens, k, v, head_first=False)
    want = v.double().cpu().expand(3, 1, 2, 64)
    softmax.check(o, (want, want.abs() * torch.finfo(dtype).eps))
    L.paged_kv_append(kp, vp, k, v, table, lens, head_first=False)
    assert (kp == 0).all() and (vp == 0).all()
