"""What the build refuses: a kernel whose split of registers does not fit the registers it was compiled to."""
import re

import pytest

from rns_llm_b200.csrc import build

SOURCE = "rns_kv_prompt_sm100.cu"


def report(*kernels):
    lines = []
    for name, registers in kernels:
        lines += [f"ptxas info    : Compiling entry function '{name}' for 'sm_100a'",
                  f"ptxas info    : Function properties for {name}",
                  "    8 bytes stack frame, 24 bytes spill stores, 32 bytes spill loads",
                  f"ptxas info    : Used {registers} registers, used 0 barriers, 8 bytes cumulative stack size"]
    return "\n".join(lines)


def test_registers_of_the_prompt_kernel():
    a, b, join = "_ZN3rns16kv_prompt_kernelILi64ELi0EEE", "_ZN3rns16kv_prompt_kernelILi128ELi1EEE", "_ZN3rns21kv_prompt_join_kernelILi64EEE"
    build.check_registers(SOURCE, report((a, 128), (join, 40), (b, 128)))
    build.check_registers("rns_aux.cu", "")
    for bad in (report((a, 128), (join, 40), (b, 120)), report((a, 126)), report((join, 40)), ""):
        with pytest.raises(RuntimeError, match="register|names no"):
            build.check_registers(SOURCE, bad)


def test_the_figure_is_the_kernel_s():
    text = (build.HERE / SOURCE).read_text()
    kernel, least = build.LEAST_REGISTERS[SOURCE]
    launch, softmax, other = map(int, re.search(r"kLaunchRegs = (\d+), kSoftmaxRegs = (\d+), kOtherRegs = (\d+);", text).groups())
    assert least == launch and 8 * softmax + 8 * other <= 16 * launch
    assert f"\n{kernel}(" in text and "kPromptThreads = 512" in text
