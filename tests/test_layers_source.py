"""What the compiler has to be told about the layer kernels' inline assembly, on the CPU."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "instant-ngp-rendering_amd", "csrc")


def test_inline_assembly_names_what_it_writes():
    """A block that sets m0 or loads into LDS names m0 and memory: without, accesses may be moved over it."""
    found = 0
    for name in ("linear.hip", "layer_norm.hip", "checkpoint8.hip", "layer_math.h"):
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        for block in re.findall(r"asm volatile\((.*?)\);", text, re.S):
            if "m0" not in block.split(":")[0] and " lds" not in block.split(":")[0]:
                continue
            found += 1
            clobbers = block.split(":")[-1]
            assert '"m0"' in clobbers and '"memory"' in clobbers, (name, block)
    assert found == 1
