"""The device error flag: every translation unit has its own, so the units whose kernels record an error
are the ones whose flag is read, and each read is one for which something can be recorded."""
import os
import re

import tqkv

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(tqkv.__file__))), "csrc")


def _text(name, seen):
    """The file with the headers of this folder that it includes, each once."""
    if name in seen or not os.path.exists(os.path.join(CSRC, name)):
        return ""
    seen.add(name)
    with open(os.path.join(CSRC, name)) as f:
        own = f.read()
    return "".join(_text(h, seen) for h in re.findall(r'#include "([^"]+)"', own)) + own


def test_the_flags_that_are_read_are_those_that_are_written():
    records, reads = set(), set()
    for unit in os.listdir(CSRC):
        if unit.endswith(".cu"):
            text = _text(unit, set())
            if re.search(r"(?<!void )record_device_error\(", text):
                records.add(unit)
            if "cudaMemcpyFromSymbol" in text and "g_device_error, sizeof" in text:
                reads.add(unit)
    assert records == {"tqkv_capi.cu"}
    assert reads == records
