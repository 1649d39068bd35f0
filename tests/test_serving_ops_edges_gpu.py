"""Operators of a serving step where they can go wrong: small vocabularies with many alternatives, magnitudes that lie
far apart.  References and bounds are those of test_serving_ops_gpu."""
import math

import pytest
import torch

from test_serving_ops_gpu import (TYPES, _attend, _check, _check_logprobs, _gen, _i32, _prompts_ref, _q4_ref, _randn, _random_cache,  # noqa: F401
                                  _starts, ops)

pytestmark = pytest.mark.gpu


# ── log probabilities ──────────────────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [33, 40, 64, 100, 200, 255, 256, 258, 300, 511, 512, 513, 600])
def test_token_logprobs_small_vocabularies_with_many_alternatives(ops, dtype, vocab):
    """Rows with fewer 16-byte pieces than two warps, which start at every offset from a 16-byte boundary."""
    x = (_randn(_gen(vocab), 5, vocab + 3) * 3).to(dtype)
    for offset in range(4):
        for top_n in (31, 32, 33, 40, 64):
            if top_n <= vocab:
                _check_logprobs(ops, x[:, offset:offset + vocab], [0, vocab - 1, vocab // 2, -1, 7], top_n)


def test_token_logprobs_small_masked_vocabularies(ops):
    """The same where a mask leaves fewer tokens than alternatives are asked for."""
    x = torch.full((4, 100), -float("inf"), device="cuda")
    x[0, [5, 17, 99]] = torch.tensor([1.0, 3.0, 2.0], device="cuda")
    x[2, :] = 1.5
    x[3, :50] = float("nan")
    x[3, 50:] = _randn(_gen(1), 50)
    _check_logprobs(ops, x, [17, 0, 3, 70], 64)


# ── packed prompts in f32: magnitudes that differ within a tile ────────────────────────────────────
# (Rows of a tile that cannot share one power of two; heads up to 64 have tiles of 128 keys, wider ones of 64.)
def _attend_all_but(q, k, v, seen, far):
    """_attend with one key left out, whose weight is 0."""
    seen = seen.clone()
    seen[:, far] = False
    return _attend(q, k, v, seen)


SIZES = [(2, 1, 64), (3, 1, 128), (2, 2, 32)]
PLACES = [1, 60, 64, 65, 127, 128, 200, 255, 256, 298]


@pytest.mark.parametrize("factor", [1e6, 1e7, 1e10, 1e20, 1e30])
@pytest.mark.parametrize("shape", SIZES, ids=str)
def test_attention_prompts_later_keys_and_values_of_any_magnitude(ops, shape, factor):
    """A finite key or value reaches the tokens that attend it and no others, wherever in its tile it lies."""
    heads, kv, hd = shape
    n = 300
    g = _gen(n)
    q, k, v = (_randn(g, n, h * hd) for h in (heads, kv, kv))
    for at in PLACES:
        ref, tol = _prompts_ref(q[:at], k[:at], v[:at], [at], [at], heads, kv, hd)
        for far_k, far_v in ((1.0, factor), (factor, 1.0), (factor, factor)):
            k2, v2 = k.clone(), v.clone()
            k2[at] *= far_k
            v2[at] *= far_v
            out = ops.attention_prompts(q, k2, v2, _starts([n]), heads, kv, hd)
            _check(out[:at], ref, tol, v[:at].abs().max().double())


@pytest.mark.parametrize("prefix", [0, 3000])
@pytest.mark.parametrize("shape", SIZES, ids=str)
def test_attention_prompts_small_rows_before_large_ones(ops, shape, prefix):
    """The first tokens of a sequence attend keys and values that are far smaller than the rest of their tile."""
    heads, kv, hd = shape
    n, small = 200, 70
    g = _gen(n + prefix)
    q, k, v = _randn(g, n, heads * hd), _randn(g, n + prefix, kv * hd), _randn(g, n + prefix, kv * hd)
    for factor in (1e-5, 1e-9, 1e-25):
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        k2[:prefix + small] *= factor
        v2[:prefix + small] *= factor
        q2[:small] /= factor
        out = ops.attention_prompts(q2, k2, v2, _starts([n]), heads, kv, hd, key_starts=_starts([n + prefix]))
        ref, tol = _prompts_ref(q2[:small], k2[:prefix + small], v2[:prefix + small], [small], [prefix + small], heads, kv, hd)
        _check(out[:small], ref, tol, v2[:prefix + small].abs().max().double())


@pytest.mark.parametrize("prefix", [0, 3000])
@pytest.mark.parametrize("shape", SIZES, ids=str)
def test_attention_prompts_far_keys_that_are_attended(ops, shape, prefix):
    """An attended key whose score is so low that its weight is 0, and whose value is huge: the scores, weights and values of the keys
    beside it are as without it."""
    heads, kv, hd = shape
    n = 300
    g = _gen(n + 1)
    q, k, v = _randn(g, n, heads * hd), _randn(g, n + prefix, kv * hd), _randn(g, n + prefix, kv * hd)
    q.view(n, heads, hd)[:, :, 0].abs_().add_(1.0)
    seen = torch.arange(n + prefix, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + prefix
    for at, low, high in ((5, -1e4, 1e30), (64, -1e6, 1.0), (130, -1e10, 1e10), (250, -1e20, 1e37)):
        k2, v2 = k.clone(), v.clone()
        for c in range(kv):
            k2[prefix + at, c * hd] = low
        v2[prefix + at] = high
        out = ops.attention_prompts(q, k2, v2, _starts([n]), heads, kv, hd, key_starts=_starts([n + prefix]))
        for h in range(heads):
            c = h * kv // heads
            a, b = k2[:, c * hd:(c + 1) * hd].double(), v2[:, c * hd:(c + 1) * hd].double()
            ref, tol = _attend_all_but(q[:, h * hd:(h + 1) * hd].double(), a, b, seen, prefix + at)
            _check(out[:, h * hd:(h + 1) * hd], ref, tol.expand(-1, hd), 0)


def test_attention_prompts_small_weights_of_huge_values(ops):
    """Weights down to 2^-100 of values up to 2^110, beside ordinary ones: the sum of p |v| bounds the error, not the largest |v|."""
    hd, n = 64, 260
    g = _gen(3)
    q, k, v = (_randn(g, n, hd) for _ in range(3))
    q[:, 0] = 8.0
    k[:, 0] = 0.0
    for at, log2_weight, log2_value in ((3, -60, 70), (70, -100, 110), (140, -40, 36), (259, -20, 30)):
        k2, v2 = k.clone(), v.clone()
        k2[at, 0] = log2_weight * math.log(2.0)  # its score beside the others': 8 / sqrt(64) times it
        v2[at] = _randn(g, hd) * 2.0 ** log2_value
        out = ops.attention_prompts(q, k2, v2, _starts([n]), 1, 1, hd).double()
        seen = torch.arange(n, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None]
        s = (q.double() @ k2.double().T / 8).masked_fill(~seen, -math.inf)
        p = torch.softmax(s, 1)
        e = ((q.double().abs() @ k2.double().abs().T) / 8).masked_fill(~seen, 0).amax(1, keepdim=True) * 2.0 ** -21
        near = torch.where(seen.any(0)[:, None], v.double().abs(), 0).max()
        bound = (2 * e + 2.0 ** -20) * (p @ v2.double().abs() + near)
        assert torch.isfinite(out).all() and ((out - p @ v2.double()).abs() <= bound).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_prompts_values_near_the_end_of_f32(ops, hd):
    """A weighted mean of values of up to 1e37 is no larger than they are."""
    n = 20
    g = _gen(hd)
    q, k, v = _randn(g, n, hd), _randn(g, n, hd), _randn(g, n, hd).abs() * 1e36 + 8e36
    out = ops.attention_prompts(q, k, v, _starts([n]), 1, 1, hd)
    ref, tol = _prompts_ref(q, k, v, [n], [n], 1, 1, hd)
    _check(out, ref, tol, v.abs().max().double())


# ── packed prompts: infinities ─────────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SIZES, ids=str)
def test_attention_prompts_keys_of_minus_infinity(ops, dtype, shape):
    """A key whose score is -inf has no weight, also where q has no more bits than 16-bit types."""
    heads, kv, hd = shape
    n = 300
    g = _gen(hd)
    q, k, v = (_randn(g, n, h * hd).half().to(dtype) for h in (heads, kv, kv))
    q.view(n, heads, hd)[:, :, 3].abs_().add_(0.5)
    seen = torch.arange(n, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None]
    for at in (1, 10, 64, 140, 299):
        k2 = k.clone()
        k2.view(n, kv, hd)[at, :, 3] = -math.inf
        out = ops.attention_prompts(q, k2, v, _starts([n]), heads, kv, hd)
        for h in range(heads):
            c = h * kv // heads
            ref, tol = _attend_all_but(q[:, h * hd:(h + 1) * hd].double(), k[:, c * hd:(c + 1) * hd].double(), v[:, c * hd:(c + 1) * hd].double(), seen, at)
            _check(out[:, h * hd:(h + 1) * hd], ref, tol.expand(-1, hd), v.abs().max().double())


@pytest.mark.parametrize("shape", SIZES, ids=str)
def test_attention_prompts_infinite_values_in_f32(ops, shape):
    """An infinite value makes its column of the tokens that attend it infinite, whatever its weight and wherever in a tile it lies; two of
    different signs make it NaN; nothing else changes."""
    heads, kv, hd = shape
    n, inf = 700, math.inf
    g = _gen(hd + 1)
    q, k, v = (_randn(g, n, h * hd) for h in (heads, kv, kv))
    q *= 30  # (weights down to nothing)
    clean = ops.attention_prompts(q, k, v, _starts([n]), heads, kv, hd).view(n, heads, hd)
    for at, value, then in ((10, inf, 400), (64, -inf, 650), (127, inf, 128), (300, -inf, 301), (0, math.nan, 1)):
        v2 = v.clone()
        v2.view(n, kv, hd)[at, :, 5] = value
        v2.view(n, kv, hd)[then, :, 6] = value
        v2.view(n, kv, hd)[then, :, 5] = -value
        out = ops.attention_prompts(q, k, v2, _starts([n]), heads, kv, hd).view(n, heads, hd)
        want = clean.clone()
        want[at:then, :, 5] = value
        want[then:, :, 5] = math.nan
        want[then:, :, 6] = value
        assert torch.equal(out.nan_to_num(7e30, 8e30, 9e30), want.nan_to_num(7e30, 8e30, 9e30))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,prefix", [(50, 0), (200, 100), (3, 6000)])
def test_attention_prompts_tokens_whose_scores_are_all_minus_infinity(ops, dtype, tokens, prefix):
    """No weight at all: zeros, as without a key, also where the keys are cut into parts."""
    heads, kv, hd = 2, 1, 64
    g = _gen(tokens)
    q, k, v = _randn(g, tokens, heads * hd).to(dtype), _randn(g, tokens + prefix, kv * hd).to(dtype), _randn(g, tokens + prefix, kv * hd).to(dtype)
    q.view(tokens, heads, hd)[:, :, 3] = 1.0
    k[:, 3] = -math.inf
    out = ops.attention_prompts(q, k, v, _starts([tokens]), heads, kv, hd, key_starts=_starts([tokens + prefix]))
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_prompts_first_key_of_minus_infinity(ops, dtype):
    """The first token has no weight, the others those of the remaining keys."""
    n, hd = 200, 64
    g = _gen(4)
    q, k, v = (_randn(g, n, hd).half().to(dtype) for _ in range(3))
    q[:, 3], k[0, 3] = 0.5, -math.inf
    out = ops.attention_prompts(q, k, v, _starts([n]), 1, 1, hd)
    k[0, 3] = 0.0
    ref, tol = _attend_all_but(q.double(), k.double(), v.double(), torch.arange(n, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None], 0)
    assert (out[0] == 0).all()
    _check(out, ref, tol, v.abs().max().double())


# ── packed prompts in 16 bits: small weights, long sums ────────────────────────────────────────────
# 147 blocks of 256 tokens: every SM has one, so that the keys are not cut into parts.
def test_attention_prompts_many_small_weights_in_f16(ops):
    """40000 weights of 2^-25.1 beside one of 1: they are 1e-3 of the sum, of values that are all theirs.  Weights are held to 2^-32 of
    the largest (half of f16's smallest number, 2^7 lifted)."""
    hd, tokens, n = 8, 147 * 256, 40000 + 147 * 256
    q, k, v = torch.zeros(tokens, hd, device="cuda"), torch.zeros(n, hd, device="cuda"), torch.ones(n, hd, device="cuda")
    q[:, 0], k[0, 0], v[0] = 1.0, 25.1 * math.log(2.0) * math.sqrt(hd), 0.0
    q, k, v = (t.half() for t in (q, k, v))
    out = ops.attention_prompts(q, k, v, _starts([tokens]), 1, 1, hd, key_starts=_starts([n]))
    w = math.exp(-float(k[0, 0]) / math.sqrt(hd))
    seen = torch.arange(n - tokens, n, device="cuda", dtype=torch.float64)[:, None]
    ref = (seen * w / (1 + seen * w)).expand(-1, hd)
    assert ((out.double() - ref).abs() <= seen * 2.0 ** -32 + 2.0 ** -11 * ref + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_attention_prompts_of_a_million_keys(ops, dtype):
    """Sums over a million keys stay within the types' roundings: a half step of the weights, one of the result."""
    heads, kv, hd, tokens, n = 1, 1, 64, 147 * 256, 1 << 20
    g = _gen(21)
    q, k, v = _randn(g, tokens, hd).to(dtype), _randn(g, n, hd).to(dtype), (_randn(g, n, hd) * 0.25 + 1).to(dtype)
    out = ops.attention_prompts(q, k, v, _starts([tokens]), heads, kv, hd, key_starts=_starts([n]))
    some = torch.tensor([0, 1, 100, 20000, tokens - 1], device="cuda")
    seen = torch.arange(n, device="cuda")[None] <= (some + n - tokens)[:, None]
    ref, tol = _attend(q[some].double(), k.double(), v.double(), seen)
    # rounded weights err at random: beside the result's half step, a quarter of one is left for them and the sums
    assert ((out[some].double() - ref).abs() <= tol + torch.finfo(dtype).eps / 2 * 1.25 * ref.abs()).all()


# ── attention over the 4-bit cache ─────────────────────────────────────────────────────────────────
def test_attention_q4_of_huge_queries(ops):
    """Queries up to f32's largest: the key of the largest score has all the weight."""
    heads, kv, hd, n = 4, 2, 64, 200
    g = _gen(22)
    cache = _random_cache(ops, g, 1, 256, kv, hd)
    for factor in (1e20, 2.0 ** 100, 1e31, 1e36):
        q = _randn(g, 1, heads * hd) * factor
        ref, _, vmax = _q4_ref(q, cache, [0], [n], heads)
        _check(ops.attention_q4(q, cache, _i32([0]), _i32([n]), heads), ref, 2.0 ** -20 * vmax, vmax)


# ── packed prompts: the ring of K and V tiles ──────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.float32, 128), (torch.float16, 64), (torch.bfloat16, 128)], ids=str)
def test_attention_prompts_items_of_any_length_in_a_row(ops, dtype, hd):
    """Many items per SM whose tiles end anywhere in the ring (3, 5 and 6 slots): no wait takes another use of a slot for its own."""
    heads = kv = 4
    lengths = [(i * 67) % 400 + 1 for i in range(150)]
    n, g = sum(lengths), _gen(hd)
    q, k, v = (_randn(g, n, h * hd).to(dtype) for h in (heads, kv, kv))
    starts = _starts(lengths)
    want = ops.attention_prompts(q, k, v, starts, heads, kv, hd)
    for _ in range(20):
        assert torch.equal(ops.attention_prompts(q, k, v, starts, heads, kv, hd), want)
    at = starts.tolist()
    for s in (0, 1, 74, 148, 149):
        a, b = at[s], at[s + 1]
        ref, tol = _prompts_ref(q[a:b], k[a:b], v[a:b], [b - a], [b - a], heads, kv, hd)
        _check(want[a:b], ref, tol, v.abs().max().double())


# ── out that is q itself, or lies over another input ───────────────────────────────────────────────
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("prefix", [0, 4000])
def test_attention_prompts_in_place(ops, dtype, prefix):
    """Undivided and in parts; in f32 with a far key, which is scored from q itself."""
    heads, kv, hd, n = 8, 2, 64, 300
    g = _gen(prefix)
    q, k, v = _randn(g, n, heads * hd).to(dtype), _randn(g, n + prefix, kv * hd), _randn(g, n + prefix, kv * hd).to(dtype)
    k[prefix + 20] *= 1e7 if dtype == torch.float32 else 1
    k, starts, keys = k.to(dtype), _starts([200, 100]), _starts([200 + prefix, 100])
    want = ops.attention_prompts(q, k, v, starts, heads, kv, hd, key_starts=keys)
    for _ in range(5):
        at = q.clone()
        assert ops.attention_prompts(at, k, v, starts, heads, kv, hd, key_starts=keys, out=at) is at and torch.equal(at, want)


def test_attention_q4_in_place(ops):
    heads, kv, hd = 16, 2, 64
    g = _gen(30)
    cache = _random_cache(ops, g, 3, 4096, kv, hd)
    slots, lengths, q = _i32([0, 1, 2]), _i32([4000, 1, 300]), _randn(g, 3, heads * hd)
    want = ops.attention_q4(q, cache, slots, lengths, heads)
    for _ in range(5):
        at = q.clone()
        assert ops.attention_q4(at, cache, slots, lengths, heads, out=at) is at and torch.equal(at, want)


def test_out_over_another_input(ops):
    from wick_b200 import _lib
    x, i = torch.zeros(40, 64, device="cuda"), _i32([0, 9])
    q, k = x[:9], x[9:18]
    cache = ops.KvCacheQ4(*(torch.zeros(1, 1, 64, w, dtype=t, device="cuda") for w, t in ((32, torch.uint8), (2, torch.float16)) * 2))
    for f in (lambda: ops.attention_prompts(q, k, k, i, 1, 1, 64, out=k), lambda: ops.attention_prompts(q, k, k, i, 1, 1, 64, out=x[4:13]),
              lambda: ops.attention_prompts(q, x[:27:3], k, i, 1, 1, 64, out=x[20:29]),
              lambda: ops.attention_q4(q, cache, i.new_zeros(9), i.new_zeros(9), 1, out=x[1:10]),
              lambda: ops.attention_q4(q[:1], cache, i[:1], i[:1], 1, out=cache.k_quants.view(-1)[:256].view(torch.float32).view(1, 64))):
        with pytest.raises(_lib.WickCudaError, match="overlaps"):
            f()
    ops.attention_prompts(q, k, k, i, 1, 1, 64, out=x[18:27])  # beside them


# ── waits that run out ─────────────────────────────────────────────────────────────────────────────
@pytest.fixture
def expiring(cuda_lib):
    """Copies whose barriers want one arrival more than anybody makes, and waits of 1.5 ms."""
    assert cuda_lib.wick_cuda_debug_serving_waits(1024, 1) == 0
    yield
    assert cuda_lib.wick_cuda_debug_serving_waits(0, 0) == 0


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.float32, 128), (torch.float16, 64), (torch.bfloat16, 128)], ids=str)
@pytest.mark.parametrize("nq,prefix", [([300, 0, 45], 0), ([60, 7], 3000)], ids=str)
def test_attention_prompts_whose_waits_run_out(ops, cuda_lib, expiring, dtype, hd, nq, prefix):
    """Every row with a key is NaN, rows of no sequence are as they were, and the next call is right."""
    heads, kv = 4, 2
    n, nk, g = sum(nq), [m + prefix for m in nq], _gen(hd)
    q, k, v = _randn(g, n + 5, heads * hd).to(dtype), _randn(g, sum(nk), kv * hd).to(dtype), _randn(g, sum(nk), kv * hd).to(dtype)
    out = torch.full_like(q, 3.0)
    args = (q, k, v, _starts(nq), heads, kv, hd, _starts(nk), out)
    ops.attention_prompts(*args)
    torch.cuda.synchronize()
    assert torch.isnan(out[:n]).all() and (out[n:] == 3).all()
    assert cuda_lib.wick_cuda_debug_serving_waits(0, 0) == 0
    ops.attention_prompts(*args)
    ref, tol = _prompts_ref(q[:n], k, v, nq, nk, heads, kv, hd)
    _check(out[:n], ref, tol, v.abs().max().double())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (12, 2, 96), (16, 4, 128)])
def test_attention_q4_whose_waits_run_out(ops, cuda_lib, expiring, dtype, heads, kv, hd):
    """The same, for rows of one tile, of several CTAs, of no key and of no slot."""
    g = _gen(heads)
    cache = _random_cache(ops, g, 4, 8192, kv, hd)
    slots, lengths = [0, 1, 2, -1, 3], [1, 8000, 0, 5, 700]
    q = _randn(g, 5, heads * hd).to(dtype)
    out = torch.full_like(q, 3.0)
    ops.attention_q4(q, cache, _i32(slots), _i32(lengths), heads, out=out)
    torch.cuda.synchronize()
    assert torch.isnan(out[[0, 1, 4]]).all() and (out[2] == 0).all() and (out[3] == 3).all()
    assert cuda_lib.wick_cuda_debug_serving_waits(0, 0) == 0
    ops.attention_q4(q, cache, _i32(slots), _i32(lengths), heads, out=out)
    ref, tol, vmax = _q4_ref(q[[0, 1, 4]], cache, [0, 1, 3], [1, 8000, 700], heads)
    _check(out[[0, 1, 4]], ref, tol, vmax)


@pytest.mark.parametrize("seqs", [255, 256, 257, 600])
def test_attention_prompts_around_the_walk_over_sequences(ops, seqs):
    """Up to 256 sequences are walked through for every item, more are searched for; some are empty."""
    heads, kv, hd = 4, 2, 64
    lengths = [(i * 37) % 90 for i in range(seqs)]
    lengths[-1] = 400
    g, n = _gen(seqs), sum(lengths)
    q, k, v = (_randn(g, n, h * hd).half() for h in (heads, kv, kv))
    starts = _starts(lengths)
    out = ops.attention_prompts(q, k, v, starts, heads, kv, hd, out=torch.full_like(q, math.nan))
    assert torch.isfinite(out).all()
    at = starts.tolist()
    for s in {0, 1, 31, 32, 100, seqs // 2, seqs - 2, seqs - 1}:
        a, b = at[s], at[s + 1]
        if a < b:
            ref, tol = _prompts_ref(q[a:b], k[a:b], v[a:b], [b - a], [b - a], heads, kv, hd)
            _check(out[a:b], ref, tol, v.abs().max().double())


# ── scores whose own rounding is more than a power of two ──────────────────────────────────────────
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SIZES, ids=str)
@pytest.mark.parametrize("log2", [24, 27, 30, 33, 40, 60, 100])
@pytest.mark.parametrize("prefix", [0, 3000])
def test_attention_prompts_huge_scores(ops, dtype, shape, log2, prefix):
    """Scores of 2^log2, of both signs: all the weight is that of the largest, whose like the others are far from."""
    heads, kv, hd = shape
    if dtype == torch.float16 and log2 // 2 + 1 > 15:
        pytest.skip("beyond f16")  # (2^16 > 65504)
    n, size, g = 200, 2.0 ** (log2 // 2 + 1), _gen(log2)
    q = torch.where(torch.rand(n, heads, 1, generator=g, device="cuda") < 0.5, -size, size).expand(-1, -1, hd).flatten(1).to(dtype)
    v = _randn(g, n + prefix, kv * hd).to(dtype)
    if dtype == torch.float32:  # every score another, at least 2^-12 of the largest apart
        height = (torch.randperm(n + prefix, generator=g, device="cuda") + 1.0) / (n + prefix)
    else:  # a few that stand out: the first tokens' scores are all 0
        height = torch.zeros(n + prefix, device="cuda")
        height[[3, 70, 150, prefix + 130, prefix + 199]] = torch.tensor([0.5, -0.25, -0.5, 0.75, -1.0], device="cuda")
    k = (height * size)[:, None].expand(-1, kv * hd).to(dtype)
    out = ops.attention_prompts(q, k, v, _starts([n]), heads, kv, hd, key_starts=_starts([n + prefix]))
    for h in range(heads):
        rows, c = slice(h * hd, (h + 1) * hd), h * kv // heads
        s = (q[:, rows].double() @ k[:, c * hd:(c + 1) * hd].double().T).masked_fill(torch.arange(n + prefix, device="cuda")[None] > torch.arange(n, device="cuda")[:, None] + prefix, -math.inf)
        p = torch.softmax(s / math.sqrt(hd), 1)
        alone = p.amax(1) == 1.0
        assert alone.sum() > 100
        ref = p @ v[:, c * hd:(c + 1) * hd].double()
        _check(out[alone][:, rows], ref[alone], 2.0 ** -20 * v.abs().max().double(), 0)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("log2", [24, 25, 26, 27, 28, 29, 30, 31, 32, 40])
def test_attention_q4_huge_scores(ops, log2):
    """Scores of about 2^(log2 - 2): the power of two that lifts the weights, which goes by the values' scales, must not meet their rounding."""
    heads, kv, hd, n = 8, 2, 64, 700
    g = _gen(log2)
    cache = _random_cache(ops, g, 1, 704, kv, hd)
    scales = cache.v_scales.float()
    for scale in (1.0, 0.4, 0.2, 0.1, 0.05, 0.02, 0.01, 1e-3, 1e-5):
        cache.v_scales.copy_(scales * scale)
        q = _randn(g, 1, heads * hd) * 2.0 ** log2 / 20
        ref, _, vmax = _q4_ref(q, cache, [0], [n], heads)
        _check(ops.attention_q4(q, cache, _i32([0]), _i32([n]), heads), ref, 2.0 ** -20 * vmax, vmax)


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_prompts_values_near_the_end_of_bf16(ops, hd):
    """Weights that grow by less than what O is rescaled for: 300 keys, then one of 2^7.5 times their weight."""
    n = 400
    g = _gen(hd + 7)
    q, k, v = torch.zeros(n, hd, device="cuda"), torch.zeros(n, hd, device="cuda"), _randn(g, n, hd).abs() * 1e35 + 3e36
    q[:, 0] = math.sqrt(hd)
    k[350:, 0] = 7.5 * math.log(2.0)
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    out = ops.attention_prompts(q, k, v, _starts([n]), 1, 1, hd)
    some = torch.tensor([0, 10, 20, 350, 360], device="cuda")  # (more of equal weight have sums beyond f32, here and in plain f32)
    seen = torch.arange(n, device="cuda")[None] <= some[:, None]
    ref, tol = _attend(q[some].double(), k.double(), v.double(), seen)
    _check(out[some], ref, tol, v.abs().max().double())
