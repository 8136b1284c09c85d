"""max_tiles of csrc/epilogue.cuh, as the host code is compiled: the most token tiles that any distribution of the rows over
the experts makes (the grid and the list bounds of both expert kernels rest on it)."""
import itertools
import os
import re
import shutil
import subprocess

import pytest

from conftest import PKG_DIR


def test_max_tiles_is_the_most_that_any_distribution_makes(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is missing")
    text = open(os.path.join(PKG_DIR, "csrc", "epilogue.cuh")).read()
    body = re.search(r"^inline long long max_tiles\(.*?^\}", text, flags=re.S | re.M).group(0)
    cases = [(e, r, t) for e in (1, 2, 3, 4) for r in range(1, 19) for t in (2, 4, 8)]
    calls = "".join(f'printf("%lld ", max_tiles({e}, {r}, {t}));' for e, r, t in cases)
    src = tmp_path / "m.cc"
    src.write_text(f"#include <cstdio>\n{body}\nint main() {{ {calls} return 0; }}\n")
    subprocess.run([gxx, str(src), "-o", str(tmp_path / "m")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "m")], check=True, capture_output=True, text=True).stdout.split()]

    def most(experts, rows, tile):
        cuts = itertools.combinations_with_replacement(range(rows + 1), experts - 1)
        return max(sum(-(-(b - a) // tile) for a, b in zip((0,) + c, c + (rows,))) for c in cuts)
    assert got == [most(*c) for c in cases]
