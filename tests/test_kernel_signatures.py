"""The argument lists that ctypes checks against the parameters of the kernel library's entry points."""
import glob
import os
import re

import pytest

from rexl3_b200.ops import build, lib


def _entries():
    for path in sorted(glob.glob(os.path.join(build.CSRC, "*.cu"))):
        with open(path) as f:
            for m in re.finditer(r"RX_API\s+[\w\s*]+?\b(rx_\w+)\(([^)]*)\)\s*\{", f.read()):
                params = m.group(2).strip()
                yield m.group(1), 0 if params in ("", "void") else params.count(",") + 1


@pytest.mark.skipif(not os.path.exists(lib.LIB_PATH), reason="the kernel library is not built")
def test_as_many_arguments_as_parameters():
    library, seen = lib.load(), 0
    for name, params in _entries():
        declared = getattr(library, name).argtypes
        if declared is not None:
            assert len(declared) == params, name
            seen += 1
    assert seen > 100
