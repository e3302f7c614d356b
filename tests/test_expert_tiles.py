"""Tiles of the MXFP4 products, on the host."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from tilebench_amd import build
from tilebench_amd import runtime as rt

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


# ----------------------------------------------------------------------------- what ran


def tile(op, M, N, K, experts=0):
    """(kernel, rows, columns, wavefronts, stages) of a call's tile; no GPU needed."""
    t = rt.gemm_tile(op, M, N, K, experts)
    return t["kernel"], t["BM"], t["BN"], t["waves"], t.get("stages")


def cases(test):
    """The parameters of a test's first parametrisation."""
    return next(m.args[1] for m in test.pytestmark if m.name == "parametrize")


@pytest.mark.skipif(not rt.LIB_PATH.exists(), reason="libtbhip.so is not built")
def test_a_tile_says_how_many_stages_it_holds():
    """128 x 128 has two forms, which only the stages tell apart."""
    assert tile(rt.OP_MXFP4, 3500, 3600, 96) == ("mx_tile", 128, 128, 4, 2)
    assert tile(rt.OP_MXFP4, 1801, 2001, 4128) == ("mx_tile", 128, 128, 4, 4)
    assert tile(rt.OP_MXFP4_GROUPED, 8027, 1300, 96, 8) == ("mx_tile", 128, 128, 4, 2)
    assert tile(rt.OP_MXFP4_GROUPED, 2321, 900, 1408, 8) == ("mx_tile", 128, 128, 4, 4)
    assert "stages" not in rt.gemm_tile(rt.OP_MXFP4, 1, 4096, 4096) and "stages" not in rt.gemm_tile(rt.OP_W4A16, 300, 512, 512)


@pytest.mark.skipif(not rt.LIB_PATH.exists(), reason="libtbhip.so is not built")
def test_the_gpu_tests_run_every_tile():
    import test_gpu_experts as on_gpu

    dense = {tile(rt.OP_MXFP4, M, N, K) for M, N, K, _ in cases(on_gpu.test_product_on_every_tile)}
    both = {("mx_skinny", 32, 32, 4, None), ("mx_tile", 64, 64, 4, 4), ("mx_tile", 128, 128, 4, 2), ("mx_tile", 128, 128, 4, 4),
            ("mx_tile", 256, 128, 8, 3), ("mx_tile", 256, 256, 8, 2)}
    assert dense == both | {("mx_tile", 256, 256, 4, 2)}
    grouped = set()
    for rows, N, K, _ in cases(on_gpu.test_grouped_product_on_every_tile):
        # its eight segments
        R = rows + rows // 3 + 2 * rows + rows - 1 + 300 + 257 + rows + 5 if rows > 6 else rows + 3 + 65 + 1 + 20 + 4 + 1
        grouped.add(tile(rt.OP_MXFP4_GROUPED, R, N, K, 8))
    assert grouped == both | {("mx_tile", 32, 128, 4, 3)}


@pytest.mark.skipif(not rt.LIB_PATH.exists(), reason="libtbhip.so is not built")
@pytest.mark.parametrize("E,k,groups,want", [
    (60, 4, 1, ("route_lanes", 8, 128)), (256, 8, 8, ("route_lanes", 16, 128)), (500, 8, 5, ("route_rows", 64, 256)),
    (384, 8, 8, ("route_lanes", 32, 128)), (1024, 8, 8, ("route_lanes", 64, 128)), (256, 9, 8, ("route_rows", 64, 256))])
def test_the_library_says_which_routing_kernel_it_launches(E, k, groups, want):
    """get_last_config() asks the rule that the launch follows."""
    from tilebench_amd.benchmarks.experts.moe_expert_routing import impl_hip

    lib = rt.load_library()
    kernel, lanes, threads = ctypes.c_char_p(), ctypes.c_int32(), ctypes.c_int32()
    out = tuple(map(ctypes.byref, (kernel, lanes, threads)))
    assert lib.tb_moe_expert_routing_kernel(E, k, groups, *out) == rt.TB_OK
    assert (kernel.value.decode(), lanes.value, threads.value) == want
    before, impl_hip._last_call = impl_hip._last_call, (E, k, groups)
    assert tuple(impl_hip.get_last_config().values()) == want
    impl_hip._last_call = before
    assert lib.tb_moe_expert_routing_kernel(E, 33, groups, *out) == rt.TB_E_INVALID
    assert lib.tb_moe_expert_routing_kernel(7, 1, 2, *out) == rt.TB_E_INVALID
    assert lib.tb_moe_expert_routing_kernel(E, k, groups, None, *out[1:]) == rt.TB_E_INVALID
