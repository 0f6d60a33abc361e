"""Extents that the C entries refuse before they touch a device."""
from custom_matmul_kernels_b200 import custom_kernel as ck

OK_PTR = 1 << 20  # aligned, never read: every call below is refused first


def test_block_axis_of_the_dense_products(lib):
    """A microscaled side of the 16-bit products has the quantiser's limits: 2^29 along its blocks."""
    n, big = ord("n"), (1 << 29) + 1
    for bits in (4, 8):
        rc = lib.fbmm_dense_mx_bmm_x16(None, OK_PTR, n, 64, 64, 2, OK_PTR, 256, OK_PTR, 512, bits, OK_PTR, big, big, 1, 1, big, 64, None, 0)
        assert rc == ck.FBMM_ERR_INVALID and b"too large" in lib.fbmm_last_error()
        rc = lib.fbmm_mx_dense_bmm_x16(None, OK_PTR, 256, OK_PTR, 512, bits, OK_PTR, 8, 512, 2, OK_PTR, 8, 8 * big, 1, big, 8, 64, None, 0)
        assert rc == ck.FBMM_ERR_INVALID and b"too large" in lib.fbmm_last_error()
        # and scale groups that a launch can count, as fbmm_mx_quantize has
        rows = 1 << 28
        rc = lib.fbmm_dense_mx_bmm_x16(None, OK_PTR, n, rows, rows, 2, OK_PTR, 256, OK_PTR, 512, bits, OK_PTR, 1 << 28, 1 << 28, 1, 1,
                                       1 << 28, rows, None, 0)
        assert rc == ck.FBMM_ERR_INVALID and b"too large" in lib.fbmm_last_error()
