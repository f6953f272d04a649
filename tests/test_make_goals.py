"""What `make` without a goal builds, as the documentation tells a user to run it."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "iree_amd", "csrc")


def _plan(*goals):
    """The commands that make would run from scratch; nothing is run."""
    return subprocess.run(["make", "-n", "-B", "-C", CSRC, *goals], check=True, capture_output=True, text=True).stdout


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_make_without_a_goal_builds_the_library_and_the_code_object():
    plan = _plan()
    assert plan == _plan("all")
    assert "libiree_amd_uk.so" in plan and "mi355x_kernels_gfx950.co" in plan
