"""Two copies of the library in one process (another build beside the installed one) must not share state: a function-local static of a
template would be one object for both, as the dynamic linker merges such symbols even between libraries that are loaded privately."""

import shutil
import subprocess

import pytest


def test_the_library_exports_no_merged_statics():
    from liger_kernel_b200 import _lib

    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("no nm")
    out = subprocess.run([nm, "-D", "--defined-only", _lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    merged = [line.split()[-1] for line in out.splitlines() if line.split()[-2] == "u"]
    assert not [name for name in merged if "flce" in name]
