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


def _refused_for_overlap(lib, code):
    from wick_b200 import _lib
    return code == _lib.ERR_BAD_ARG and b"overlaps" in lib.wick_cuda_last_error()


# Addresses that are never followed; what does not overlap fails at its workspace, which is checked behind it.
def test_attention_prompts_refuses_an_out_over_its_inputs(cuda_lib):
    def call(out, q=A, qs=256, k=4 * A, ks=128, v=8 * A, vs=128, starts=16 * A, keys=32 * A):
        return _refused_for_overlap(cuda_lib, cuda_lib.wick_cuda_attention_prompts(q, qs, k, ks, v, vs, 0, starts, keys, 2, 9, 20, 4, 2, 64, out, 0, None, 0, None))

    size = 9 * 256 * 4
    assert not call(2 * A) and not call(A)  # (q itself)
    for at, length in ((A, size), (4 * A, 20 * 512), (8 * A, 20 * 512), (16 * A, 12), (32 * A, 12)):
        assert not call(at - size) and not call(at + (length + 15) // 16 * 16)
        assert call(at - size + 16) and call(at + (length - 1) // 16 * 16)
    # rows apart from one another: q itself only where they are dense; between the columns of a single row
    assert call(A, qs=260) and call(A + 256 * 4, qs=260)
    assert not call(4 * A + 512, ks=128 + 256 * 9)
    assert call(4 * A + 496, ks=128 + 256 * 9) and call(4 * A + 528, ks=128 + 256 * 9)


def test_attention_q4_refuses_an_out_over_its_inputs(cuda_lib):
    cache = C.byref(_cache(k_quants=4 * A, k_scales=8 * A, v_quants=12 * A, v_scales=16 * A))

    def call(out, q=A, qs=256):
        return _refused_for_overlap(cuda_lib, cuda_lib.wick_cuda_attention_q4(cache, q, qs, 0, 3, 4, 20 * A, 24 * A, out, 0, None, 0, None))

    size, rows = 3 * 256 * 4, 2 * 2 * 128
    assert not call(2 * A) and not call(A)
    for at, length in ((A, size), (4 * A, rows * 32), (8 * A, rows * 4), (12 * A, rows * 32), (16 * A, rows * 4), (20 * A, 12), (24 * A, 12)):
        assert not call(at - size) and not call(at + length)
        assert call(at - size + 4) and call(at + length - 4)
    assert call(A, qs=257)


def test_limits_of_the_hook_for_waits(cuda_lib):
    from wick_b200 import _lib
    for rounds, missing in ((100, 0), ((1 << 18) + 256, 0), (0, 2)):
        assert cuda_lib.wick_cuda_debug_serving_waits(rounds, missing) == _lib.ERR_BAD_ARG
    assert cuda_lib.wick_cuda_debug_serving_waits(0, 0) == _lib.OK


def test_calls_for_another_device_than_the_current_one(monkeypatch):
    """They are made with the tensors' device as the current one and on its stream; the old one comes back, after a failure too."""
    import pytest
    import torch
    from wick_b200 import _lib, ops
    current, calls = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *error):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 1000 + dev)
    code = _lib.OK
    monkeypatch.setattr(ops, "check", lambda c: (_ for _ in ()).throw(_lib.WickCudaError(c, "refused")))

    def fn(*args):
        calls.append((current[0], *args))
        return code

    ops._call(fn, 0, 7)
    ops._call(fn, 3, 7, 8)
    assert calls == [(0, 7, 1000), (3, 7, 8, 1003)] and current == [0]
    code = _lib.ERR_BAD_ARG
    for dev in (0, 2):
        with pytest.raises(_lib.WickCudaError):
            ops._call(fn, dev)
    assert calls[2:] == [(0, 1000), (2, 1002)] and current == [0]
