"""What a run cannot show: properties of the kernels' source that hold by the order of its statements."""
import os
import re

import pytest

from conftest import PKG_DIR

CSRC = os.path.join(PKG_DIR, "csrc")


def source(name):
    """The file without its comments (positions of lines kept)."""
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def functions(text, pattern):
    """(name, body) of each device function whose body matches."""
    for m in re.finditer(r"MBP_DEV \w+ (\w+)\([^;{]*\) \{\n(.*?)\n\}", text, flags=re.S):
        if re.search(pattern, m.group(2)):
            yield m.group(1), m.group(2)


def test_warp_collective_tmem_accesses_reconverge_first():
    """tcgen05.ld / st / alloc / dealloc are .sync.aligned: a warp that comes from per-lane branches meets itself first."""
    found = 0
    for name, body in functions(source("tc.cuh"), r"tcgen05\.(ld|st)\.sync\.aligned"):
        before = body[:re.search(r"tcgen05\.(ld|st)\.sync\.aligned", body).start()]
        assert "__syncwarp();" in before, name
        found += 1
    assert found == 3
    for f in ("gemm.cu", "expert_gemm.cu"):
        text = source(f)
        for m in re.finditer(r"tcgen05\.(alloc|dealloc)\.", text):
            block = text[text.rindex("if (warp == 1) {", 0, m.start()):m.start()]
            assert "__syncwarp();" in block, (f, m.group(0))
        assert not re.search(r"tcgen05\.(ld|st)\.", text)  # only through the helpers


def test_masks_are_taken_by_a_converged_warp():
    """take_mask branches per lane, and matrix instructions (.sync.aligned) follow it."""
    (_, body), = functions(source("escape.cuh"), r"tgt >> lane\) & 1u")
    assert body.rstrip().endswith("__syncwarp();")
