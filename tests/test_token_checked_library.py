"""CPU: in the bounds-checked library each source file reads its own violation counter. A function that the files share would be
linked once and read one file's counter for all."""
import os
import subprocess

import pytest

from fused_lncc import _lib


def test_counters_are_read_by_functions_of_their_own():
    path = os.path.join(os.path.dirname(_lib.LIB_PATH), "liblncc_sm100_checked.so")
    if not os.path.exists(path):
        pytest.skip("the checked library is not built")
    out = subprocess.run(["nm", "-C", path], capture_output=True, text=True, check=True).stdout
    lines = [line.split(maxsplit=2)[-2:] for line in out.splitlines() if "g_check_violations" in line or "blk::check_" in line]
    assert sum("g_check_violations" in name for _, name in lines) >= 4
    assert all(kind in "bBtdD" for kind, _ in lines), lines
