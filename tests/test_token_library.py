"""CPU: the package and its loss import whatever state the token blocks' torch library is in, and the token-block functions say
what is wrong with it."""
import os
import shutil
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fused-lncc_b200")
OPS = "libfused_lncc_torch.so"


@pytest.fixture
def copy(tmp_path):
    """The package without its torch library and what it is built from; the C library is a link."""
    root = tmp_path / "pkg"
    shutil.copytree(os.path.join(PKG, "fused_lncc"), root / "fused_lncc", ignore=shutil.ignore_patterns("*.so", "__pycache__"))
    from fused_lncc import _lib
    _lib.load()
    os.symlink(_lib.LIB_PATH, root / "fused_lncc" / "liblncc_sm100.so")
    return root


def _run(root, code):
    return subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(root)!r})\n" + code],
                          capture_output=True, text=True)


def _bytes():
    from fused_lncc import _native
    _native.load()
    with open(_native.OPS_PATH, "rb") as f:
        return f.read()


IMPORT = """
import torch
from fused_lncc import fused_lncc_loss, fused_layer_norm, _native
print("imported")
assert _native._module is None
"""
BUILD = """
_native._build = lambda: print("built") or sys.exit(0)
fused_layer_norm(torch.zeros(2, 8))
"""


def test_broken_library_breaks_the_token_blocks_alone(copy):
    from fused_lncc import _native
    mark = _native._mark()
    assert _bytes().endswith(mark)
    (copy / "fused_lncc" / OPS).write_bytes(b"no library at all" + mark)
    r = _run(copy, IMPORT + """
try:
    fused_layer_norm(torch.zeros(2, 8))
except RuntimeError as e:
    print("says", e)
""")
    assert r.returncode == 0 and "imported" in r.stdout, r.stderr
    assert "does not load" in r.stdout and "build.py --force" in r.stdout


@pytest.mark.parametrize("state", ["missing", "cut off", "another torch"])
def test_library_that_does_not_match_is_not_loaded_but_built_again(copy, state):
    data = _bytes()
    if state == "cut off":
        (copy / "fused_lncc" / OPS).write_bytes(data[:len(data) // 2])
    if state == "another torch":
        (copy / "fused_lncc" / OPS).write_bytes(data.replace(b"for torch ", b"for torch 9"))
    r = _run(copy, IMPORT + BUILD)
    assert r.returncode == 0 and r.stdout.split() == ["imported", "built"], (r.stdout, r.stderr)


def test_matching_library_is_loaded_at_import():
    r = _run(PKG, "import fused_lncc\nassert fused_lncc._native._module is not None")
    assert r.returncode == 0, r.stderr
