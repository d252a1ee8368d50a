"""The build's check of the registers that the tile kernel's split counts on."""
import re

import pytest

from nml_b200 import build

SOURCE = "attention_q8_tile.cu"


def report(*counts):
    return "".join(
        f"ptxas info    : Compiling entry function '_Z11tile_kernelILi{i}E' for 'sm_100a'\n"
        f"    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads\n"
        f"ptxas info    : Used {count} registers, used 2 barriers\n"
        for i, count in enumerate(counts))


def test_other_register_counts_end_the_build():
    build.check_launch_registers(SOURCE, report(80, 80, 80, 80))
    for bad in (report(80, 78, 80, 80), report(), report(88), "nvcc: nothing to do"):
        with pytest.raises(RuntimeError, match="80 registers"):
            build.check_launch_registers(SOURCE, bad)


def test_the_count_is_the_source_s_own():
    text = (build.CSRC / SOURCE).read_text()
    assert re.findall(r"constexpr int kLaunchRegisters = (\d+);", text) == [
        str(build.LAUNCH_REGISTERS[SOURCE][1])]
