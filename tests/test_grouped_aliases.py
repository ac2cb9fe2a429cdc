"""Grouped products with an output over an operand are refused."""
import ctypes

import bwgemm


def test_output_over_an_operand_is_refused():
    buf = ctypes.create_string_buffer(8192)
    p = (ctypes.addressof(buf) + 255) & ~255
    A, B, C, off = p, p + 1024, p + 2048, p + 4096
    L = bwgemm.lib()

    def rows(A, B, C):
        return L.bw_gemm_grouped(bwgemm.DTYPE_F16, A, 8, B, 1, off, 1, None, None, C, 8, bwgemm.OUT_BF16, 4, 8, 8, None)

    def wgrad(X, Y, D):
        return L.bw_gemm_grouped_wgrad(bwgemm.DTYPE_F16, X, 8, Y, 8, off, 1, D, bwgemm.OUT_BF16, 8, 8, 8, None)

    for call in (rows, wgrad):
        assert call(A, B, A) == bwgemm.BW_ERR_INVALID and call(A, B, B) == bwgemm.BW_ERR_INVALID
        assert call(A, B, C) != bwgemm.BW_ERR_INVALID and call(A, A, C) != bwgemm.BW_ERR_INVALID
