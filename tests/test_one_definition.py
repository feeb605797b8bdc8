"""What the library has once whatever number of its sources use it (no GPU needed)."""

import shutil
import subprocess

import pytest


@pytest.mark.skipif(shutil.which("nm") is None, reason="no nm")
def test_one_pool_of_scheduler_words():
    from bastile_b200 import _lib

    names = subprocess.run(["nm", str(_lib.lib_path())], capture_output=True, text=True, check=True).stdout
    assert names.count("g_tile_sched") == 1
