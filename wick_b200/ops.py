"""Operator-level entry points of libwick_cuda on torch CUDA tensors.

torch is only the device allocator here: every function hands raw device pointers to the
C ABI and launches on torch's current stream.  Names follow the wick functions they stand
in for (wick/src/backend/simd.rs, cpu.rs).
"""
from __future__ import annotations

import ctypes as C
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
# UNSUPPORTED_DTYPE).  They launch on the current stream of their tensors' device.
DTYPE_ID = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise _lib.WickCudaError(_lib.ERR_BAD_ARG, message)


def _dtype_id(t: torch.Tensor) -> int:
    if t.dtype not in DTYPE_ID:
        raise _lib.WickCudaError(_lib.ERR_UNSUPPORTED_DTYPE, f"{t.dtype}: f32, f16 or bf16 is needed")
    return DTYPE_ID[t.dtype]


def _rows(t: torch.Tensor, name: str, device: torch.device) -> torch.Tensor:
    """t as rows with a dense last dimension that do not overlap."""
    _need(t.is_cuda and t.device == device, f"{name} must be on {device}")
    _need(t.dim() == 2, f"{name} must have two dimensions")
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        return t.contiguous()
    return t


def _stride(t: torch.Tensor) -> int:
    """Elements from row to row; torch keeps any number there for a single row."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ids(t: torch.Tensor, n: int, name: str, device: torch.device) -> torch.Tensor:
    _need(t.dtype == torch.int32 and t.device == device, f"{name} must be int32 on {device}")
    _need(t.dim() == 1 and t.shape[0] == n, f"{name} must hold {n} numbers")
    return t if t.is_contiguous() else t.contiguous()


def _call(name: str, device: torch.device, *args) -> None:
    """The library's function `name` on the current stream of `device`."""
    fn = getattr(_lib.load(), name)
    stream = torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        check(fn(*args, stream))
    else:
        with torch.cuda.device(device):
            check(fn(*args, stream))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_n: int = 0):
    """Log probability of tokens[j] under row j of logits [n, vocab], the rows' entropies (nats) and their top_n (at most 64)
    likeliest tokens: (logprob [n], entropy [n], top ids [n, top_n] int32, top logprobs [n, top_n]), f32.  Equal logits by
    ascending id; NaN counts as -inf; a token outside the vocabulary has -inf."""
    device = logits.device
    logits = _rows(logits, "logits", device)
    n, vocab = logits.shape
    tokens = _ids(tokens, n, "tokens", device)
    dtype = _dtype_id(logits)
    _need(0 <= top_n <= 64, "top_n must be 0 to 64")
    out = torch.empty((2, n), dtype=torch.float32, device=device)
    ids = torch.empty((n, top_n), dtype=torch.int32, device=device)
    lps = torch.empty((n, top_n), dtype=torch.float32, device=device)
    p = out.data_ptr()
    _call("wick_cuda_token_logprobs", device, logits.data_ptr(), dtype, _stride(logits), n, vocab, tokens.data_ptr(), top_n, p, p + 4 * n,
          ids.data_ptr() if top_n else None, lps.data_ptr() if top_n else None)
    return out[0], out[1], ids, lps


class KvCacheQ4:
    """A K / V cache in 4 bits: Q4_0 blocks of 32 values, quants [slots, kv_heads, max_seq, head_dim / 2] uint8 and scales
    [slots, kv_heads, max_seq, head_dim / 32] f16 for each of the two sides (byte i of a block's 16 holds number i in its low and number
    i + 16 in its high half; value = scale * (number - 8)).  Holds the given tensors; max_seq is a multiple of 64, head_dim of 32 and at
    most 128."""

    def __init__(self, k_quants: torch.Tensor, k_scales: torch.Tensor, v_quants: torch.Tensor, v_scales: torch.Tensor):
        planes = (k_quants, k_scales, v_quants, v_scales)
        self.device = k_quants.device
        for t, dtype in zip(planes, (torch.uint8, torch.float16) * 2):
            _need(t.is_cuda and t.device == self.device and t.dtype == dtype and t.dim() == 4 and t.is_contiguous(),
                  "planes must be dense tensors of four dimensions on one GPU, quants uint8 and scales f16")
        slots, heads, rows, half = k_quants.shape
        _need(v_quants.shape == k_quants.shape and half % 16 == 0 and k_scales.shape == v_scales.shape == (slots, heads, rows, half // 16),
              "the planes' shapes do not match")
        self.k_quants, self.k_scales, self.v_quants, self.v_scales = planes
        self.n_slots, self.n_kv_heads, self.max_seq, self.head_dim = slots, heads, rows, half * 2
        self._c = _lib.KvQ4(*(t.data_ptr() for t in planes), slots, heads, rows, half * 2)

    @classmethod
    def empty(cls, n_slots: int, max_seq: int, n_kv_heads: int, head_dim: int, device="cuda") -> "KvCacheQ4":
        """A cache of zeros for at least max_seq rows per slot."""
        _need(n_slots > 0 and max_seq > 0 and n_kv_heads > 0 and head_dim > 0 and head_dim % 32 == 0 and head_dim <= 128,
              "sizes must be positive, head_dim a multiple of 32 and at most 128")
        rows = -(-max_seq // 64) * 64
        planes = []
        for _ in range(2):
            planes.append(torch.full((n_slots, n_kv_heads, rows, head_dim // 2), 0x88, dtype=torch.uint8, device=device))
            planes.append(torch.zeros((n_slots, n_kv_heads, rows, head_dim // 32), dtype=torch.float16, device=device))
        return cls(*planes)


def kv_append_q4(cache: KvCacheQ4, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor) -> None:
    """Rounds the rows of k and v [n, kv_heads * head_dim] to Q4_0 and writes row j to row positions[j] of slot slots[j].  Rows whose
    slot or position the cache does not have (padding: -1) are skipped; the pairs of a call must differ."""
    device = cache.device
    k, v = _rows(k, "k", device), _rows(v, "v", device)
    n, dim = k.shape
    _need(v.shape == k.shape and v.dtype == k.dtype, "k and v must have the same shape and type")
    _need(dim == cache.n_kv_heads * cache.head_dim, "k and v must have kv_heads * head_dim columns")
    slots, positions = _ids(slots, n, "slots", device), _ids(positions, n, "positions", device)
    _call("wick_cuda_kv_append_q4", device, C.byref(cache._c), k.data_ptr(), _stride(k), v.data_ptr(), _stride(v), _dtype_id(k), n,
          slots.data_ptr(), positions.data_ptr())


def kv_read_q4(cache: KvCacheQ4, slots: torch.Tensor, positions: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of row positions[j] of slot slots[j]: k and v [n, kv_heads * head_dim] f32; zeros where the cache has no such row."""
    device, n = cache.device, slots.shape[0]
    slots, positions = _ids(slots, n, "slots", device), _ids(positions, n, "positions", device)
    k, v = torch.empty((2, n, cache.n_kv_heads * cache.head_dim), dtype=torch.float32, device=device)
    _call("wick_cuda_kv_read_q4", device, C.byref(cache._c), n, slots.data_ptr(), positions.data_ptr(), k.data_ptr(), v.data_ptr())
    return k, v


def attention_q4(q: torch.Tensor, cache: KvCacheQ4, slots: torch.Tensor, lengths: torch.Tensor, n_heads: int,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of single tokens over the cache: row j of q [n, n_heads * head_dim] attends the first lengths[j] rows of slot
    slots[j]; several rows may name one slot.  Length 0 gives zeros; rows whose slot the cache does not have (padding: -1) are left as
    they are in `out` (a new one starts with zeros)."""
    device = cache.device
    q = _rows(q, "q", device)
    n, dim = q.shape
    _need(dim == n_heads * cache.head_dim, "q must have n_heads * head_dim columns")
    slots, lengths = _ids(slots, n, "slots", device), _ids(lengths, n, "lengths", device)
    dtype = _dtype_id(q)
    fresh = out is None
    if fresh:
        out = torch.empty((n, dim), dtype=q.dtype, device=device)
    _need(out.shape == q.shape and out.dtype == q.dtype and out.device == device and out.is_contiguous(), "out must be dense, of q's shape and type")
    size = C.c_uint64(0)
    check(_lib.load().wick_cuda_attention_q4_workspace(C.byref(cache._c), n, n_heads, C.byref(size)))
    work = torch.empty(size.value, dtype=torch.uint8, device=device)
    _call("wick_cuda_attention_q4", device, C.byref(cache._c), q.data_ptr(), _stride(q), dtype, n, n_heads, slots.data_ptr(), lengths.data_ptr(),
          out.data_ptr(), fresh, work.data_ptr(), size.value)
    return out


def attention_prompts(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, n_heads: int, n_kv_heads: int, head_dim: int,
                      key_starts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed prompts: sequence s has the tokens starts[s] .. starts[s + 1] of q [tokens, n_heads * head_dim] and the
    keys key_starts[s] .. key_starts[s + 1] (default: the same) of k and v [keys, n_kv_heads * head_dim]; its last key belongs to its last
    token.  Tokens without a key get zeros; rows behind the last sequence are left as they are in `out` (a new one starts with zeros)."""
    device = q.device
    q, k, v = _rows(q, "q", device), _rows(k, "k", device), _rows(v, "v", device)
    _need(q.dtype == k.dtype == v.dtype, "q, k and v must have the same type")
    _need(n_heads > 0 and n_kv_heads > 0 and q.shape[1] == n_heads * head_dim, "q must have n_heads * head_dim columns")
    _need(k.shape == v.shape and k.shape[1] == n_kv_heads * head_dim, "k and v must have n_kv_heads * head_dim columns")
    n_seqs = starts.shape[0] - 1
    _need(n_seqs >= 0, "starts must hold at least one offset")
    starts = _ids(starts, n_seqs + 1, "starts", device)
    if key_starts is not None:
        key_starts = _ids(key_starts, n_seqs + 1, "key_starts", device)
    dtype = _dtype_id(q)
    # 16-byte loads: rows that start elsewhere are copied
    q, k, v = (t if (t.data_ptr() | _stride(t) * t.element_size()) % 16 == 0 else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
    fresh = out is None
    if fresh:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    _need(out.shape == q.shape and out.dtype == q.dtype and out.device == device and out.is_contiguous() and out.data_ptr() % 16 == 0,
          "out must be dense, of q's shape and type and start on a 16-byte boundary")
    size = C.c_uint64(0)
    check(_lib.load().wick_cuda_attention_prompts_workspace(dtype, n_seqs, q.shape[0], k.shape[0], n_heads, n_kv_heads, head_dim, C.byref(size)))
    work = torch.empty(size.value, dtype=torch.uint8, device=device)
    if n_seqs == 0:
        return out.zero_() if fresh else out
    _call("wick_cuda_attention_prompts", device, q.data_ptr(), _stride(q), k.data_ptr(), _stride(k), v.data_ptr(), _stride(v), dtype,
          starts.data_ptr(), key_starts.data_ptr() if key_starts is not None else None, n_seqs, q.shape[0], k.shape[0], n_heads, n_kv_heads,
          head_dim, out.data_ptr(), fresh, work.data_ptr(), size.value)
    return out
