"""The build's check of registers and occupancy (csrc/check_resources.py), on reports written here."""
import importlib.util
import os

import pytest

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "linear_moe_amd", "csrc", "check_resources.py")
spec = importlib.util.spec_from_file_location("check_resources", PATH)
check = importlib.util.module_from_spec(spec)
spec.loader.exec_module(check)


def report(tmp_path, *kernels):
    """Every guarded kernel once, as it should be, and `kernels`: (name, scratch, spilled, waves per SIMD)."""
    rows = [(f"_ZN4lmoe{len(k)}{k}IDF16bLi128EEEv", 0, 0, 8) for k in check.GUARDED] + list(kernels)
    path = tmp_path / "unit.remarks"
    path.write_text("".join(f"x.hpp:1:0: remark: {line} [-Rpass-analysis=kernel-resource-usage]\n" for n, s, v, w in rows for line in (
        f"Function Name: {n}", "    VGPRs: 256", f"    ScratchSize [bytes/lane]: {s}", f"    Occupancy [waves/SIMD]: {w}", f"    VGPRs Spill: {v}")))
    return str(path)


FWD, DQ, DKV = "_ZN4lmoe10k_attn_fwdI", "_ZN4lmoe13k_attn_bwd_dqI", "_ZN4lmoe14k_attn_bwd_dkvI"


@pytest.mark.parametrize("name,scratch,spilled,waves,ok", [
    (FWD + "Li128ELi1E", 0, 0, 2, True), (FWD + "Li128ELi1E", 4, 1, 2, False), (FWD + "Li128ELi1E", 0, 0, 1, False), (DQ + "Li64ELi2E", 8, 0, 3, False),
    (DKV + "Li128ELi8E", 0, 0, 2, True), (DKV + "Li128ELi8E", 12, 2, 2, True), (DKV + "Li128ELi8E", 16, 2, 2, False), (DKV + "Li128ELi8E", 12, 3, 2, False),
    (DKV + "Li128ELi8E", 0, 0, 1, False), (DKV + "Li64ELi4E", 8, 1, 3, True), (DKV + "Li64ELi4E", 0, 0, 2, False)])
def test_attention_kernels_are_guarded(tmp_path, capsys, name, scratch, spilled, waves, ok):
    assert (check.main([report(tmp_path, (name, scratch, spilled, waves))]) == 0) == ok
    assert ok or name in capsys.readouterr().err


def test_a_guarded_kernel_without_a_report_is_noticed(tmp_path):
    path = tmp_path / "none.remarks"
    path.write_text("")
    assert check.main([str(path)]) == 1
