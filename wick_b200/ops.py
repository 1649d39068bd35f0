"""Operator-level entry points of libwick_cuda on torch CUDA tensors.

torch is only the device allocator here: every function hands raw device pointers to the
C ABI and launches on torch's current stream.  Names follow the wick functions they stand
in for (wick/src/backend/simd.rs, cpu.rs).
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Tuple

import numpy as np
import torch

from . import _lib
from ._lib import check

DT_Q4_0, DT_Q8_0 = 2, 8
QTYPE_ID = {"q4_0": DT_Q4_0, "q8_0": DT_Q8_0}


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor) -> int:
    assert t.is_cuda and t.is_contiguous()
    return t.data_ptr()


class QuantWeight:
    """A quantised [m, k] matrix resident on the GPU in the library's layout (WeightRef, lfm2.rs:19-25)."""

    def __init__(self, dtype: int, raw: np.ndarray, m: int, k: int):
        raw = np.ascontiguousarray(raw, dtype=np.uint8)
        bb = 18 if dtype == DT_Q4_0 else 34
        assert raw.size == m * (k // 32) * bb, "raw block bytes do not match m x k"
        self._lib = _lib.load()
        self._h = C.c_void_p()
        self.dtype, self.m, self.k = dtype, m, k
        torch.cuda.init()
        check(self._lib.wick_cuda_weight_create(dtype, raw.ctypes.data, m, k, C.byref(self._h)))

    def check_products(self):
        """Waits for the current stream; raises TIMEOUT if a product of this weight gave up on a device-side wait."""
        check(self._lib.wick_cuda_weight_status(self._h, _stream()))

    def close(self):
        if self._h.value:
            self._lib.wick_cuda_weight_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def quantize_f32_to_q8_0(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """simd.rs:255-323 over the rows of x [n, k] -> (scales [n, k/32] f32, quants [n, k] i8)."""
    x = x.contiguous()
    n, k = (1, x.shape[0]) if x.dim() == 1 else x.shape
    s = torch.empty((n, k // 32), dtype=torch.float32, device=x.device)
    q = torch.empty((n, k), dtype=torch.int8, device=x.device)
    check(_lib.load().wick_cuda_quantize_q8_0(_ptr(x), n, k, _ptr(s), _ptr(q), _stream()))
    return s, q


def gemv_q8(w: QuantWeight, xs: torch.Tensor, xq: torch.Tensor) -> torch.Tensor:
    """gemv_q4_0_q8_0_neon / gemv_q8_0_q8_0_neon (simd.rs:328-415, :440-524)."""
    y = torch.empty(w.m, dtype=torch.float32, device=xq.device)
    check(_lib.load().wick_cuda_gemv_q8(w._h, _ptr(xs), _ptr(xq), _ptr(y), _stream()))
    return y


def gemm_q8(w: QuantWeight, bs: torch.Tensor, bq: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """gemm_q*_q8_0_neon (simd.rs:696-1019) over the n rows of bq; returns token-major [n, m]."""
    n = bq.shape[0]
    if out is None:
        out = torch.empty((n, w.m), dtype=torch.float32, device=bq.device)
    check(_lib.load().wick_cuda_gemm_q8(w._h, _ptr(bs), _ptr(bq), n, _ptr(out), _stream()))
    return out


def gemm_q8_tc(w: QuantWeight, bs: torch.Tensor, bq: torch.Tensor, want_sums: bool = False):
    """The tensor-core (tcgen05) form of gemm_q8: exact int32 block sums, one fused f32 chain per output
    in block order.  Returns out [n, m] (and the block sums [n, m, k/32] when asked).  Synchronises."""
    n = bq.shape[0]
    out = torch.empty((n, w.m), dtype=torch.float32, device=bq.device)
    sums = torch.empty((n, w.m, w.k // 32), dtype=torch.int32, device=bq.device) if want_sums else None
    check(_lib.load().wick_cuda_gemm_q8_tc(w._h, _ptr(bs), _ptr(bq), n, _ptr(out), _ptr(sums) if want_sums else None,
                                           _stream()))
    return (out, sums) if want_sums else out


def gemm_q8_tc_exact(w: QuantWeight, bs: torch.Tensor, bq: torch.Tensor) -> torch.Tensor:
    """gemm_q8 on the tensor cores with the reference's accumulation order: bit-identical to gemm_q8."""
    n = bq.shape[0]
    out = torch.empty((n, w.m), dtype=torch.float32, device=bq.device)
    check(_lib.load().wick_cuda_gemm_q8_tc_exact(w._h, _ptr(bs), _ptr(bq), n, _ptr(out), _stream()))
    return out


def block_sums(w: QuantWeight, xq: torch.Tensor) -> torch.Tensor:
    s = torch.empty((w.m, w.k // 32), dtype=torch.int32, device=xq.device)
    check(_lib.load().wick_cuda_block_sums(w._h, _ptr(xq), _ptr(s), _stream()))
    return s


def rmsnorm_(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """cpu::rmsnorm (cpu.rs:577-594) on each row of x, in place."""
    n, dim = (1, x.shape[0]) if x.dim() == 1 else x.shape
    check(_lib.load().wick_cuda_rmsnorm(_ptr(x), _ptr(weight), n, dim, eps, _stream()))
    return x


def silu_mul_(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    check(_lib.load().wick_cuda_silu_mul(_ptr(gate), _ptr(up), gate.numel(), _stream()))
    return gate


def ggml_expf(x: torch.Tensor) -> torch.Tensor:
    y = torch.empty_like(x)
    check(_lib.load().wick_cuda_expf(_ptr(x), _ptr(y), x.numel(), _stream()))
    return y


def rope_(q: torch.Tensor, k: torch.Tensor, pos: int, n_heads: int, n_kv_heads: int, head_dim: int, freq_base: float):
    check(_lib.load().wick_cuda_rope(_ptr(q), _ptr(k), pos, n_heads, n_kv_heads, head_dim, freq_base, _stream()))
    return q, k


def qknorm_rope_kv_(q, k, v, q_norm, k_norm, eps: float, rope_cos, rope_sin, k_cache, v_cache, start_pos: int, n_heads: int,
                    n_kv_heads: int, head_dim: int):
    """Per-head RMSNorm of Q and K, RoPE from a (position, pair) cos / sin table, and the append of the rotated K rows
    and the V rows to the caches at rows start_pos.. (lfm2.rs:783-855) for the n rows of q [n, n_heads * head_dim]."""
    n = q.shape[0]
    check(_lib.load().wick_cuda_qknorm_rope_kv(_ptr(q), _ptr(k), _ptr(v), _ptr(q_norm), _ptr(k_norm), eps, _ptr(rope_cos), _ptr(rope_sin),
                                               _ptr(k_cache), _ptr(v_cache), n, start_pos, n_heads, n_kv_heads, head_dim, _stream()))
    return q


def attention_decode(q, k_cache, v_cache, n_heads, n_kv_heads, head_dim, seq) -> torch.Tensor:
    out = torch.empty(n_heads * head_dim, dtype=torch.float32, device=q.device)
    check(_lib.load().wick_cuda_attention_decode(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), n_heads, n_kv_heads,
                                                 head_dim, seq, _stream()))
    return out


def attention_decode_splitk(q, k_cache, v_cache, n_heads, n_kv_heads, head_dim, seq) -> torch.Tensor:
    """Opt-in split-K single-query attention (runs of 256 keys + merge); agrees with attention_decode within rounding."""
    out = torch.empty(n_heads * head_dim, dtype=torch.float32, device=q.device)
    check(_lib.load().wick_cuda_attention_decode_splitk(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), n_heads, n_kv_heads,
                                                        head_dim, seq, _stream()))
    return out


def attention_prefill(q, k_cache, v_cache, n, start_pos, n_heads, n_kv_heads, head_dim, flash: bool) -> torch.Tensor:
    out = torch.empty((n, n_heads * head_dim), dtype=torch.float32, device=q.device)
    check(_lib.load().wick_cuda_attention_prefill(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), n, start_pos, n_heads,
                                                  n_kv_heads, head_dim, int(flash), _stream()))
    return out


def shortconv(proj: torch.Tensor, conv_w: torch.Tensor, state: torch.Tensor, kernel_size: int) -> torch.Tensor:
    n, three_hs = proj.shape
    hs = three_hs // 3
    out = torch.empty((n, hs), dtype=torch.float32, device=proj.device)
    check(_lib.load().wick_cuda_shortconv(_ptr(proj), _ptr(conv_w), _ptr(state), _ptr(out), n, hs, kernel_size, _stream()))
    return out


def argmax(logits: torch.Tensor) -> torch.Tensor:
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    check(_lib.load().wick_cuda_argmax(_ptr(logits), logits.numel(), _ptr(out), _stream()))
    return out


def sample_logits(logits: torch.Tensor, temperature: float, top_k: int, top_p: float, r: float) -> int:
    """Sampler::sample (sampler.rs:64-158) on device logits with the caller's uniform draw r."""
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    check(_lib.load().wick_cuda_sample_logits(_ptr(logits), logits.numel(), temperature, top_k, top_p, r, _ptr(out), _stream()))
    return int(out.item())


ARGMAX_NOALLOC_MAX = 4096 * 1024


def argmax_noalloc(logits: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """Same result as argmax() for callers that may not allocate: the scratch is a fixed array inside
    the library and the caller supplies `out` (one int32 on the device).  At most ARGMAX_NOALLOC_MAX
    logits.  Calls share that array, so keep them on one stream."""
    lib = _lib.load()
    code = lib.wick_cuda_argmax_noalloc(_ptr(logits), logits.numel(), _ptr(out), _stream())
    if code != 0:
        raise _lib.WickCudaError(code, lib.wick_cuda_argmax_noalloc_last_error().decode())
    return out


# ── operators of a serving step beside the model's own path ────────────────────────────────────────
# f32, f16 and bf16; rows may be strided views (the last dimension dense).  Misuse raises WickCudaError (BAD_ARG or
# UNSUPPORTED_DTYPE).  They launch on the current stream of their tensors' device.  A decode step calls them between kernels of a
# few microseconds: checks compare plain numbers, and devices go by index.
DTYPE_ID = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


def _bad(message: str):
    raise _lib.WickCudaError(_lib.ERR_BAD_ARG, message)


def _dtype_id(t: torch.Tensor) -> int:
    i = DTYPE_ID.get(t.dtype)
    if i is None:
        raise _lib.WickCudaError(_lib.ERR_UNSUPPORTED_DTYPE, f"{t.dtype}: f32, f16 or bf16 is needed")
    return i


def _rows(t: torch.Tensor, name: str, dev: int) -> Tuple[torch.Tensor, int, int, int]:
    """(t with a dense last dimension and rows that do not overlap, rows, columns, elements from row to row)."""
    if dev < 0 or t.get_device() != dev:
        _bad(f"{name} must be on the same GPU as the other tensors")
    if t.dim() != 2:
        _bad(f"{name} must have two dimensions")
    n, m = t.shape
    stride, dense = t.stride()
    if (m > 1 and dense != 1) or (n > 1 and stride < m):
        t, stride = t.contiguous(), m
    return t, n, m, stride if n > 1 else m  # (torch keeps any stride for a single row)


def _ids(t: torch.Tensor, n: int, name: str, dev: int) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.get_device() != dev or t.dim() != 1 or t.shape[0] != n:
        _bad(f"{name} must hold {n} int32 numbers on the tensors' GPU")
    return t if t.is_contiguous() else t.contiguous()


def _out(out: torch.Tensor, like: torch.Tensor, shape: tuple, dev: int) -> None:
    if out.shape != shape or out.dtype is not like.dtype or out.get_device() != dev or not out.is_contiguous() or out.data_ptr() % 16:
        _bad("out must be dense, of q's shape and type and start on a 16-byte boundary")


# The current stream of a device as a number: 0.1 us where making a Stream object takes 1.5.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _call(fn, dev: int, *args) -> None:
    """A function of the library on the current stream of device `dev`."""
    if dev == torch.cuda.current_device():
        code = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            code = fn(*args, _raw_stream(dev))
    if code:
        check(code)


@functools.lru_cache(maxsize=1024)
def _workspace(name: str, *sizes) -> int:
    """What a workspace function of the library says for these sizes."""
    size = C.c_uint64(0)
    check(getattr(_lib.load(), name)(*sizes, C.byref(size)))
    return size.value


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_n: int = 0):
    """Log probability of tokens[j] under row j of logits [n, vocab], the rows' entropies (nats) and their top_n (at most 64)
    likeliest tokens: (logprob [n], entropy [n], top ids [n, top_n] int32, top logprobs [n, top_n]), f32.  Equal logits by
    ascending id; NaN counts as -inf; a token outside the vocabulary has -inf."""
    dev = logits.get_device()
    logits, n, vocab, stride = _rows(logits, "logits", dev)
    tokens = _ids(tokens, n, "tokens", dev)
    if not 0 <= top_n <= 64:
        _bad("top_n must be 0 to 64")
    device = logits.device
    logprob = torch.empty(n, dtype=torch.float32, device=device)
    entropy = torch.empty_like(logprob)
    ids = torch.empty((n, top_n), dtype=torch.int32, device=device)
    lps = torch.empty((n, top_n), dtype=torch.float32, device=device)
    _call(_lib.load().wick_cuda_token_logprobs, dev, logits.data_ptr(), _dtype_id(logits), stride, n, vocab, tokens.data_ptr(), top_n,
          logprob.data_ptr(), entropy.data_ptr(), ids.data_ptr(), lps.data_ptr())
    return logprob, entropy, ids, lps


class KvCacheQ4:
    """A K / V cache in 4 bits: Q4_0 blocks of 32 values, quants [slots, kv_heads, max_seq, head_dim / 2] uint8 and scales
    [slots, kv_heads, max_seq, head_dim / 32] f16 for each of the two sides (byte i of a block's 16 holds number i in its low and number
    i + 16 in its high half; value = scale * (number - 8)).  Holds the given tensors; max_seq is a multiple of 64, head_dim of 32 and at
    most 128."""

    def __init__(self, k_quants: torch.Tensor, k_scales: torch.Tensor, v_quants: torch.Tensor, v_scales: torch.Tensor):
        dev = k_quants.get_device()
        for t, dtype in ((k_quants, torch.uint8), (k_scales, torch.float16), (v_quants, torch.uint8), (v_scales, torch.float16)):
            if dev < 0 or t.get_device() != dev or t.dtype is not dtype or t.dim() != 4 or not t.is_contiguous():
                _bad("planes must be dense tensors of four dimensions on one GPU, quants uint8 and scales f16")
        slots, heads, rows, half = shape = k_quants.shape
        if v_quants.shape != shape or half % 16 or k_scales.shape != (slots, heads, rows, half // 16) or v_scales.shape != k_scales.shape:
            _bad("the planes' shapes do not match")
        self.k_quants, self.k_scales, self.v_quants, self.v_scales = k_quants, k_scales, v_quants, v_scales
        self.n_slots, self.n_kv_heads, self.max_seq, self.head_dim, self.dev = slots, heads, rows, half * 2, dev
        self._c = _lib.KvQ4(k_quants.data_ptr(), k_scales.data_ptr(), v_quants.data_ptr(), v_scales.data_ptr(), slots, heads, rows, half * 2)

    @classmethod
    def empty(cls, n_slots: int, max_seq: int, n_kv_heads: int, head_dim: int, device="cuda") -> "KvCacheQ4":
        """A cache of zeros for at least max_seq rows per slot."""
        if not (n_slots > 0 and max_seq > 0 and n_kv_heads > 0 and 0 < head_dim <= 128) or head_dim % 32:
            _bad("sizes must be positive, head_dim a multiple of 32 and at most 128")
        rows = -(-max_seq // 64) * 64
        planes = []
        for _ in range(2):
            planes.append(torch.full((n_slots, n_kv_heads, rows, head_dim // 2), 0x88, dtype=torch.uint8, device=device))
            planes.append(torch.zeros((n_slots, n_kv_heads, rows, head_dim // 32), dtype=torch.float16, device=device))
        return cls(*planes)


def kv_append_q4(cache: KvCacheQ4, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor) -> None:
    """Rounds the rows of k and v [n, kv_heads * head_dim] to Q4_0 and writes row j to row positions[j] of slot slots[j].  Rows whose
    slot or position the cache does not have (padding: -1) are skipped; the pairs of a call must differ."""
    dev = cache.dev
    k, n, dim, k_stride = _rows(k, "k", dev)
    v, n_v, dim_v, v_stride = _rows(v, "v", dev)
    if n_v != n or dim_v != dim or v.dtype is not k.dtype or dim != cache.n_kv_heads * cache.head_dim:
        _bad("k and v must have the same type and kv_heads * head_dim columns")
    slots, positions = _ids(slots, n, "slots", dev), _ids(positions, n, "positions", dev)
    _call(_lib.load().wick_cuda_kv_append_q4, dev, cache._c, k.data_ptr(), k_stride, v.data_ptr(), v_stride, _dtype_id(k), n, slots.data_ptr(),
          positions.data_ptr())


def kv_read_q4(cache: KvCacheQ4, slots: torch.Tensor, positions: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of row positions[j] of slot slots[j]: k and v [n, kv_heads * head_dim] f32; zeros where the cache has no such row."""
    dev, n = cache.dev, slots.numel()
    slots, positions = _ids(slots, n, "slots", dev), _ids(positions, n, "positions", dev)
    k = torch.empty((n, cache.n_kv_heads * cache.head_dim), dtype=torch.float32, device=slots.device)
    v = torch.empty_like(k)
    _call(_lib.load().wick_cuda_kv_read_q4, dev, cache._c, n, slots.data_ptr(), positions.data_ptr(), k.data_ptr(), v.data_ptr())
    return k, v


def attention_q4(q: torch.Tensor, cache: KvCacheQ4, slots: torch.Tensor, lengths: torch.Tensor, n_heads: int,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of single tokens over the cache: row j of q [n, n_heads * head_dim] attends the first lengths[j] rows of slot
    slots[j]; several rows may name one slot.  Length 0 gives zeros; rows whose slot the cache does not have (padding: -1) are left as
    they are in `out` (a new one has zeros there).  `out` overlaps no input, but may be q itself."""
    dev = cache.dev
    q, n, dim, stride = _rows(q, "q", dev)
    if dim != n_heads * cache.head_dim:
        _bad("q must have n_heads * head_dim columns")
    slots, lengths = _ids(slots, n, "slots", dev), _ids(lengths, n, "lengths", dev)
    dtype, fresh = _dtype_id(q), out is None
    if fresh:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty((n, dim), dtype=q.dtype, device=q.device)
    else:
        _out(out, q, (n, dim), dev)
    size = _workspace("wick_cuda_attention_q4_workspace", cache.head_dim)
    work = torch.empty(size, dtype=torch.uint8, device=q.device)
    _call(_lib.load().wick_cuda_attention_q4, dev, cache._c, q.data_ptr(), stride, dtype, n, n_heads, slots.data_ptr(), lengths.data_ptr(),
          out.data_ptr(), fresh, work.data_ptr(), size)
    return out


def attention_prompts(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, n_heads: int, n_kv_heads: int, head_dim: int,
                      key_starts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed prompts: sequence s has the tokens starts[s] .. starts[s + 1] of q [tokens, n_heads * head_dim] and the
    keys key_starts[s] .. key_starts[s + 1] (default: the same) of k and v [keys, n_kv_heads * head_dim]; its last key belongs to its last
    token.  Tokens without a key get zeros; rows behind the last sequence are left as they are in `out` (a new one has zeros there).
    `out` overlaps no input, but may be q itself."""
    dev = q.get_device()
    q, n, dim, q_stride = _rows(q, "q", dev)
    k, n_keys, dim_k, k_stride = _rows(k, "k", dev)
    v, n_values, dim_v, v_stride = _rows(v, "v", dev)
    if q.dtype is not k.dtype or q.dtype is not v.dtype:
        _bad("q, k and v must have the same type")
    if n_heads <= 0 or n_kv_heads <= 0 or head_dim <= 0 or dim != n_heads * head_dim or n_values != n_keys or dim_k != n_kv_heads * head_dim or dim_v != dim_k:
        _bad("q must have n_heads * head_dim columns, k and v n_kv_heads * head_dim columns and the same rows")
    n_seqs = starts.numel() - 1
    if n_seqs < 0:
        _bad("starts must hold at least one offset")
    starts = _ids(starts, n_seqs + 1, "starts", dev)
    if key_starts is not None:
        key_starts = _ids(key_starts, n_seqs + 1, "key_starts", dev)
    dtype, size, fresh = _dtype_id(q), q.element_size(), out is None
    # 16-byte loads: rows that start elsewhere are copied
    if (q.data_ptr() | q_stride * size) % 16:
        q, q_stride = q.clone(memory_format=torch.contiguous_format), dim
    if (k.data_ptr() | k_stride * size) % 16:
        k, k_stride = k.clone(memory_format=torch.contiguous_format), dim_k
    if (v.data_ptr() | v_stride * size) % 16:
        v, v_stride = v.clone(memory_format=torch.contiguous_format), dim_k
    if fresh:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty((n, dim), dtype=q.dtype, device=q.device)
    else:
        _out(out, q, (n, dim), dev)
    room = _workspace("wick_cuda_attention_prompts_workspace", dtype, n_seqs, n, n_keys, n_heads, n_kv_heads, head_dim)
    work = torch.empty(room, dtype=torch.uint8, device=q.device) if room else None
    _call(_lib.load().wick_cuda_attention_prompts, dev, q.data_ptr(), q_stride, k.data_ptr(), k_stride, v.data_ptr(), v_stride, dtype,
          starts.data_ptr(), key_starts.data_ptr() if key_starts is not None else None, n_seqs, n, n_keys, n_heads, n_kv_heads, head_dim,
          out.data_ptr(), fresh, work.data_ptr() if room else None, room)
    return out
