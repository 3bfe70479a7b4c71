"""What can be told from the CUDA sources' text alone."""
import glob
import os
import re

import pytest

from conftest import ROOT

SOURCES = sorted(glob.glob(os.path.join(ROOT, "pytorch-engine_b200", "csrc", "*.cu*")))
READ = re.compile(r"\*reinterpret_cast<const (?:uint4|float4|ulonglong2|Raw8<T>)\*>\((\w+)\)")


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_arrays_read_sixteen_bytes_at_a_time_are_aligned(path):
    """A thread's own array of small elements, read through a pointer to 16 bytes, starts on a boundary of 16: in registers that
    changes nothing, in memory an address off the boundary is a fault."""
    lines = open(path).read().split("\n")
    for i, line in enumerate(lines):
        for name in READ.findall(line):
            declared = [l for l in lines[max(0, i - 12):i] if re.search(rf"\b(?:T|__nv_bfloat16|uint8_t|float|uint32_t) {name}\[", l)]
            if declared:
                assert "alignas(16)" in declared[-1], f"{os.path.basename(path)}:{i + 1}: {declared[-1].strip()}"


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_shared_memory_is_asked_for_on_every_device(path):
    """The attribute is a device's own: who remembers that a kernel has it remembers on which device."""
    text = open(path).read()
    for once in re.findall(r"static bool (\w+(?:\[[^\]]*\])*) = ", text):
        assert "kDevices]" in once, f"{os.path.basename(path)}: static bool {once}"
