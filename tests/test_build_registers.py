"""The build's check of the registers that a register-trading kernel is given, on reports written here."""
import pytest

from ops_tensor_b200 import build

REPORT = """ptxas info    : 0 bytes gmem
ptxas info    : Compiling entry function '_ZN5blaze27cache_attention_join_kernelILi8ELi64ELb1EEEvNS_1PE' for 'sm_100a'
    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads
ptxas info    : Used 32 registers, used 0 barriers
ptxas info    : Compiling entry function '_ZN5blaze27cache_attention_many_kernelILi64ELb0EEEvNS_1PE' for 'sm_100a'
    24 bytes stack frame, 16 bytes spill stores, 60 bytes spill loads
ptxas info    : Used %d registers, used 1 barriers
"""


def test_enough_registers():
    build.check_registers(REPORT % 128)
    build.check_registers("")


@pytest.mark.parametrize("registers", [96, 120, 127, 129])
def test_too_few_registers_end_the_build(registers):
    with pytest.raises(RuntimeError, match="cache_attention_many_kernel.* %d registers" % registers):
        build.check_registers(REPORT % registers)


def test_the_bound_is_the_kernels_own():
    text = (build.CSRC / "cache_attention_many.cuh").read_text()
    assert "kManyLaunchRegs = %d;" % build.LAUNCH_REGISTERS["cache_attention_many_kernel"] in text
