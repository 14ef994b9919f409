"""What softmax_attn and the paged cache make of the plain numbers of a call, without a GPU."""
import ctypes as C

import pytest
import torch

from linear_moe_amd.softmax_attn import cap_of


@pytest.mark.parametrize("cap,want", [(None, 0.0), (0, 0.0), (30, 30.0), (1e-20, 1e-20), (1e-41, 2.0 ** -126), (1e-60, 2.0 ** -126), (5e-324, 2.0 ** -126)])
def test_a_cap_stays_one_in_32_bits(cap, want):
    assert cap_of(cap, "op") == want and (C.c_float(cap_of(cap, "op")).value > 0) == bool(cap)
