"""Shared memory that kernels read several values at a time from is declared with the alignment that this wants."""
import os
import re

import tensornet_b200


def test_dynamic_shared_memory_that_is_used_from_its_start():
    csrc = os.path.join(os.path.dirname(tensornet_b200.__file__), "csrc")
    seen = 0
    for name in ("attention_few.cu", "layer_norm.cu"):
        with open(os.path.join(csrc, name)) as f:
            text = f.read()
        for align, kind, array in re.findall(r"extern __shared__ (__align__\(16\) )?(\w+) (\w+)\[\];", text):
            wide = kind == "uint8_t" and re.search(r"reinterpret_cast<[^>]+>\(" + array + r"\b", text)
            assert align or not wide, (name, array)
            seen += bool(wide)
    assert seen >= 2
