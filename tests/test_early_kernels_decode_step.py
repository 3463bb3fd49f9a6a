"""Row maps, shared attention, sampling rules and counts begin while the kernel before them runs, which may have written any of their inputs: a selection's ids feed the
counts, row maps the attention.  A load through a `const __restrict__` pointer may be moved up past `griddepcontrol.wait`, so only weights are passed that way."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rexl3_b200", "ops", "csrc")


@pytest.mark.parametrize("source,kernels", [("rows.cu", 1), ("logits.cu", 4), ("attention_shared.cu", 3)])
def test_inputs_are_plain_pointers(source, kernels):
    text = open(os.path.join(CSRC, source)).read()
    found = re.findall(r"__global__ void __launch_bounds__\(.*?\)\s+(\w+_kernel)\((.*?)\)\s*\{", text, re.S)
    assert len(found) == kernels
    for name, params in found:
        for p in params.split(","):
            if "__restrict__" in p and p.split()[0] == "const":
                assert re.search(r"\bsuh$", p.strip()), (name, p)
    assert "__ldg(" not in text
