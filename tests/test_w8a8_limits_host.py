"""The limits of the products in 8-bit integers without a device: what they refuse, they refuse before any launch."""
import iree_amd
import test_w8a8_host as host


def test_more_tiles_than_any_grid_holds_are_refused():
    most = dict(M=(1 << 31) - 1, N=1 << 24, out_stride=1 << 24)
    assert host._call("matmul_w8a8", host.MATMUL, **most) == 12
    assert b"too many tiles" in iree_amd.load_library().iree_amd_uk_last_error()


def test_rows_to_gather_from_4_gib_are_refused():
    # (the GPU tests gather from 2^32 - 16 bytes)
    assert host._call("grouped_matmul_w8a8", host.GROUPED, lhs_rows=1 << 20, lhs_stride=1 << 12) == 12
    assert b"4 GiB" in iree_amd.load_library().iree_amd_uk_last_error()
