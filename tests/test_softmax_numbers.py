"""What softmax_attn and the paged cache make of the plain numbers of a call, without a GPU."""
import ctypes as C

import pytest
import torch

from linear_moe_amd.softmax_attn import cap_of, ints_of


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
