"""How many workgroups the absorbed latent attention puts to work (latent_share in
helix_runtime_amd/csrc/latent.hpp), through a host build of the same function."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"


def test_row_blocks_leave_few_workgroups_idle(tmp_path):
    """At least 13 of 16 of the 256 have a row block, whatever their number; a power of two
    has multiples of the eight XCDs."""
    if not os.path.exists(HIPCC) and shutil.which("hipcc") is None:
        pytest.skip("hipcc is not available")
    exe = tmp_path / "latent_share_check"
    subprocess.run([HIPCC if os.path.exists(HIPCC) else "hipcc", "-x", "hip", "--offload-arch=gfx950",
                    "-O1", "-std=c++17", os.path.join(ROOT, "tests", "cpp", "latent_share_check.cpp"),
                    "-o", str(exe)], check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe), "300"], check=True, capture_output=True, text=True, timeout=60).stdout
    share = [int(x) for x in out.split()]
    assert len(share) == 301 and share[0] == share[1] == 0
    for n, each in enumerate(share):
        assert each == 0 or 208 <= each * n <= 256, n  # (0: one list, of which all take ranges)
    assert [share[n] for n in (2, 4, 8, 16, 32)] == [128, 64, 32, 16, 8]
