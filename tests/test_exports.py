"""What the library exports under C names: the declared entry points and nothing else."""
from __future__ import annotations

import re
import shutil
import subprocess

import pytest

from reversability_amd import _hip


@pytest.mark.skipif(shutil.which("nm") is None, reason="needs binutils")
def test_only_entry_points_have_c_names():
    listing = subprocess.run(["nm", "-D", "--defined-only", str(_hip.LIBRARY_PATH)],
                             check=True, capture_output=True, text=True).stdout
    names = [line.split()[-1] for line in listing.splitlines()]
    # C++ names, and what the compiler adds (a unit's identity, the linker's marks)
    assert [n for n in names if not re.match(r"rv_|_Z|__hip_cuid_|_init$|_fini$", n)] == []
