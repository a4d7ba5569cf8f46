"""Limits of the grouped products that the C ABI names, with addresses that are never touched."""
import ctypes


def test_tiles_of_a_call_fit_one_launch():
    """2^30 rows of 512 columns are two tiles of 512 threads per 256 rows, 2^32 threads and more."""
    from mi355moe import _lib
    L = _lib.load()
    plan = ctypes.byref(_lib.MMGroupPlan(*[256] * 6, 1 << 30, 1, 3))
    for fn, K, N in ((L.mm_group_linear, 16, 512), (L.mm_group_linear_inputs, 512, 16), (L.mm_group_linear, 16, 1024)):
        assert fn(plan, 256, 256, 1, K, N, 0, 0, 256, 1, None, 0, None) == -1 and b"too many tiles" in L.mm_last_error()


def test_least_workspace_holds_eight_columns_of_every_row():
    """fp32 rows: all columns, or for a bf16 result of many routes about half of them and at least eight, which is a band."""
    from mi355moe import _lib
    L = _lib.load()
    for cols in (8, 16, 24, 40, 72, 256, 1032, 4096, 5120, 1 << 20):
        for T, k in ((1, 16), (17, 1), (5000, 8)):
            full = 4 * T * k * cols
            for dtype in (_lib.DTYPE_F16, _lib.DTYPE_F32):
                assert L.mm_group_linear_workspace(T, k, cols, 1, dtype) == full
            least = L.mm_group_linear_workspace(T, k, cols, 1, _lib.DTYPE_BF16)
            assert least == full if T * k <= 16 else 32 * T * k <= least <= full
