"""What the build checks in the compiler's report."""
import importlib
import os

import pytest

build = importlib.import_module("autodiff-ir-rust_b200.build")

REPORT = """ptxas info    : Compiling entry function '_ZN3adb20adb_attention_tc_dkvILi2ELb0EEEv' for 'sm_100a'
ptxas info    : Function properties for _ZN3adb20adb_attention_tc_dkvILi2ELb0EEEv
    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads
ptxas info    : Used %d registers, used 1 barriers
ptxas info    : Compiling entry function '_ZN3adb12adb_rms_normILi32EEEv' for 'sm_100a'
ptxas info    : Used 40 registers, used 1 barriers
"""


def test_the_key_gradient_kernels_have_the_registers_they_share_out():
    with open(os.path.join(build.CSRC, "adb_attention_tc.cu")) as f:
        source = f.read()
    build.check_register_shares(REPORT % 96, source)
    with pytest.raises(RuntimeError, match="88 registers"):
        build.check_register_shares(REPORT % 88, source)
    with pytest.raises(RuntimeError, match="names no"):
        build.check_register_shares(REPORT.replace("_dkv", "_dq") % 96, source)
