"""Limits of the operators of a serving step that need no GPU to be shown: every check comes before the first CUDA call."""
import ctypes as C

from test_serving_ops_refusals import A, _cache


def test_more_rows_than_a_row_number_holds(cuda_lib):
    """One KV head of 32 elements: 2^31 rows are fewer than 2^38 elements."""
    from wick_b200 import _lib
    c = C.byref(_cache(n_kv_heads=1, head_dim=32))
    for n in (0x7FFFFF01, 0x7FFFFFFF, 0x80000000, 0xFFFFFFFF):
        assert cuda_lib.wick_cuda_kv_append_q4(c, A, 32, A, 32, 1, n, A, A, None) == _lib.ERR_BAD_ARG
        assert cuda_lib.wick_cuda_kv_read_q4(c, n, A, A, A, A, None) == _lib.ERR_BAD_ARG
