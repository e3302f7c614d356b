"""Tiles of the MXFP4 products, on the host."""
import shutil
import subprocess
from pathlib import Path

import pytest

from tilebench_amd import build

SOURCE = Path(__file__).parent / "native" / "mx_tile_shape.hip"


@pytest.mark.parametrize("shape,fits", [
    ("1, 1, 4, 8", True), ("2, 2, 2, 2", True), ("2, 2, 4, 4", True), ("2, 2, 3, 2, 4, 8", True), ("1, 1, 3, 4, 1", True),
    ("4, 2, 2, 2, 2, 8", True),
    # DMAs that the wait leaves under way would hold the scales: three stages ahead of two steps' scales; scales that
    # go out right before they are read
    ("2, 2, 4, 2", False), ("1, 1, 5, 2", False), ("2, 2, 2, 1", False)])
def test_scales_land_before_they_are_read(shape, fits):
    """Every step's wait covers its scales, or the shape does not compile."""
    if shutil.which("hipcc") is None:
        pytest.skip("no hipcc")
    res = subprocess.run(["hipcc", *build.HIPCC_FLAGS, f"-DSHAPE={shape}", "-fsyntax-only", "--cuda-host-only", str(SOURCE)],
                         capture_output=True, text=True)
    assert (res.returncode == 0) == fits, res.stderr[-2000:]
    assert fits or "scales have to have landed" in res.stderr
