"""What the operators of a serving step refuse, through the C ABI and without a GPU: every check comes before the first CUDA call."""
import ctypes as C

import pytest

A = 1 << 20  # an address that is never followed: aligned to everything


def _cache(**kw):
    from wick_b200 import _lib
    c = dict(k_quants=A, k_scales=A, v_quants=A, v_scales=A, n_slots=2, n_kv_heads=2, max_seq=128, head_dim=64)
    c.update(kw)
    return _lib.KvQ4(*(c[f] for f, _ in _lib.KvQ4._fields_))


BAD_CACHES = [dict(k_quants=None), dict(v_scales=None), dict(n_slots=0), dict(n_kv_heads=0), dict(max_seq=0), dict(max_seq=100),
              dict(head_dim=0), dict(head_dim=48), dict(head_dim=160), dict(k_quants=A + 8), dict(k_scales=A + 2), dict(n_kv_heads=70000)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=[str(b) for b in BAD_CACHES])
def test_caches_that_do_not_fit(cuda_lib, bad):
    from wick_b200 import _lib
    c = _cache(**bad)
    assert cuda_lib.wick_cuda_kv_append_q4(C.byref(c), A, 128, A, 128, 0, 1, A, A, None) == _lib.ERR_BAD_ARG
    assert cuda_lib.wick_cuda_kv_read_q4(C.byref(c), 1, A, A, A, A, None) == _lib.ERR_BAD_ARG
    assert cuda_lib.wick_cuda_attention_q4(C.byref(c), A, 256, 0, 1, 4, A, A, A, 0, A, 1 << 30, None) == _lib.ERR_BAD_ARG


def test_append_and_read(cuda_lib):
    from wick_b200 import _lib
    c = C.byref(_cache())
    append, read = cuda_lib.wick_cuda_kv_append_q4, cuda_lib.wick_cuda_kv_read_q4
    assert append(None, A, 128, A, 128, 0, 1, A, A, None) == _lib.ERR_BAD_ARG
    assert append(c, None, 128, A, 128, 0, 1, A, A, None) == _lib.ERR_BAD_ARG
    assert append(c, A, 127, A, 128, 0, 1, A, A, None) == _lib.ERR_BAD_ARG
    assert append(c, A, 128, A + 2, 128, 0, 1, A, A, None) == _lib.ERR_BAD_ARG
    assert append(c, A, 128, A, 128, 2, 1, A, A, None) == _lib.ERR_UNSUPPORTED_DTYPE
    assert append(c, A, 128, A, 128, 0, 0, A, A, None) == _lib.OK  # no rows
    assert read(c, 1, A, None, A, A, None) == _lib.ERR_BAD_ARG
    assert read(c, 1, A, A, A + 4, A, None) == _lib.ERR_BAD_ARG
    assert read(c, 0, A, A, A, A, None) == _lib.OK


def test_attention_q4(cuda_lib):
    from wick_b200 import _lib
    c, size = C.byref(_cache()), C.c_uint64(0)
    f = cuda_lib.wick_cuda_attention_q4
    query = cuda_lib.wick_cuda_attention_q4_workspace
    assert query(64, None) == _lib.ERR_BAD_ARG
    for head_dim in (0, 40, 160):
        assert query(head_dim, C.byref(size)) == _lib.ERR_BAD_ARG
    assert query(64, C.byref(size)) == _lib.OK
    big = 1 << 30
    assert f(c, A, 256, 0, 3, 3, A, A, A, 0, A, big, None) == _lib.ERR_BAD_ARG  # 3 heads over 2 KV heads
    assert f(c, A, 256, 0, 70000, 4, A, A, A, 0, A, big, None) == _lib.ERR_BAD_ARG
    assert f(c, A, 255, 0, 3, 4, A, A, A, 0, A, big, None) == _lib.ERR_BAD_ARG
    assert f(c, A, 256, 5, 3, 4, A, A, A, 0, A, big, None) == _lib.ERR_UNSUPPORTED_DTYPE
    assert f(c, A + 2, 256, 0, 3, 4, A, A, A, 0, A, big, None) == _lib.ERR_BAD_ARG
    assert f(c, A, 256, 0, 3, 4, None, A, A, 0, A, big, None) == _lib.ERR_BAD_ARG
    assert f(c, A, 256, 0, 0, 4, None, None, None, 0, None, 0, None) == _lib.OK
    if size.value:
        assert f(c, A, 256, 0, 3, 4, A, A, A, 0, A, size.value - 1, None) == _lib.ERR_BAD_ARG
        assert f(c, A, 256, 0, 3, 4, A, A, A, 0, A + 8, size.value, None) == _lib.ERR_BAD_ARG
        assert f(c, A, 256, 0, 3, 4, A, A, A, 0, None, size.value, None) == _lib.ERR_BAD_ARG


def test_attention_prompts(cuda_lib):
    from wick_b200 import _lib
    size = C.c_uint64(0)

    def call(q=A, qs=256, k=A, ks=128, v=A, vs=128, dtype=0, starts=A, seqs=2, tokens=9, keys=9, heads=4, kv=2, hd=64, out=A, work=A, room=1 << 40):
        return cuda_lib.wick_cuda_attention_prompts(q, qs, k, ks, v, vs, dtype, starts, None, seqs, tokens, keys, heads, kv, hd, out, 0, work, room, None)

    for bad in (dict(q=None), dict(k=None), dict(starts=None), dict(out=None), dict(qs=255), dict(ks=64), dict(vs=127), dict(heads=5), dict(heads=0),
                dict(kv=0), dict(hd=0), dict(hd=4), dict(hd=136), dict(q=A + 8), dict(v=A + 4), dict(ks=129), dict(heads=514, kv=2), dict(tokens=(1 << 30) + 1),
                dict(qs=1 << 39)):
        assert call(**bad) == _lib.ERR_BAD_ARG, bad
    assert call(dtype=7) == _lib.ERR_UNSUPPORTED_DTYPE
    assert call(seqs=0) == _lib.OK and call(tokens=0) == _lib.OK
    query = cuda_lib.wick_cuda_attention_prompts_workspace
    assert query(0, 2, 9, 9, 4, 2, 64, None) == _lib.ERR_BAD_ARG
    assert query(0, 2, 9, 9, 4, 3, 64, C.byref(size)) == _lib.ERR_BAD_ARG
    assert query(0, 2, 9, 9, 4, 2, 64, C.byref(size)) == _lib.OK
    if size.value:
        assert call(room=size.value - 1) == _lib.ERR_BAD_ARG
        assert call(work=A + 64) == _lib.ERR_BAD_ARG
        assert call(work=None) == _lib.ERR_BAD_ARG


def test_token_logprobs(cuda_lib):
    from wick_b200 import _lib

    def call(x=A, dtype=0, stride=100, n=3, vocab=100, tokens=A, top=0, lp=A, ent=A, ids=A, lps=A):
        return cuda_lib.wick_cuda_token_logprobs(x, dtype, stride, n, vocab, tokens, top, lp, ent, ids, lps, None)

    for bad in (dict(x=None), dict(tokens=None), dict(lp=None), dict(ent=None), dict(top=1, ids=None), dict(top=1, lps=None), dict(vocab=0), dict(stride=99),
                dict(top=65), dict(top=101), dict(vocab=20, top=21), dict(x=A + 2)):
        assert call(**bad) == _lib.ERR_BAD_ARG, bad
    assert call(dtype=3) == _lib.ERR_UNSUPPORTED_DTYPE
    assert call(n=0) == _lib.OK


def test_wrappers_refuse_what_is_not_on_a_gpu(cuda_lib):
    import torch
    from wick_b200 import _lib, ops
    x, i = torch.zeros(2, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(_lib.WickCudaError):
        ops.token_logprobs(x, i)
    with pytest.raises(_lib.WickCudaError):
        ops.attention_prompts(x, x, x, i, 1, 1, 64)
    with pytest.raises(_lib.WickCudaError):
        ops.KvCacheQ4(*(torch.zeros(1, 1, 64, n, dtype=t) for n, t in ((16, torch.uint8), (1, torch.float16)) * 2))
