"""Operators of a serving step against their definitions in 64 bits: attention of packed prompts, the 4-bit K / V cache and the
attention over it, log probabilities.

Tolerances.  Attention: a score's absolute error is at most e = 2^-21 * sum |q_i k_i| / sqrt(d) (inputs held to 22 bits, products added in
f32), so a weight is off by a factor within 1 +- 2 e and an output by at most (2 e + 2^-20) max |v|, 2^-20 for the sums of weights and weighted
values.  In 16 bits each weight is rounded once more, half a step, and so is the result."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from wick_b200 import ops
    return ops


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _attend(q, k, v, seen):
    """q [m, d], k / v [t, d] in f64, seen [m, t]: (output, its tolerance without the type's roundings)."""
    d = q.shape[1]
    s = (q @ k.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, 1).nan_to_num(0.0)
    e = ((q.abs() @ k.abs().T) / math.sqrt(d)).masked_fill(~seen, 0).amax(1) * 2.0 ** -21
    top = torch.where(seen.any(1), torch.where(seen.any(0)[:, None], v.abs(), 0).max(), 0.0)
    return torch.where(seen.any(1)[:, None], p @ v, 0.0), ((2 * e + 2.0 ** -20) * top)[:, None]


def _check(out, ref, tol, vmax):
    half = torch.finfo(out.dtype).eps / 2
    if out.dtype == torch.float32:
        bound = tol + half * ref.abs()
    else:
        bound = tol + half * (ref.abs() + vmax) + 2.0 ** -24  # (f16: results below its normal range)
    off = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), f"off by {off.max().item():.3g}, {(off / bound.clamp_min(1e-300)).max().item():.3g} times the bound"


# ── packed prompts ─────────────────────────────────────────────────────────────────────────────────
def _prompts_ref(q, k, v, nq, nk, heads, kv, hd):
    out = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64, device="cuda")
    tol = torch.zeros(q.shape[0], heads, 1, dtype=torch.float64, device="cuda")
    q, k, v = q.double().view(-1, heads, hd), k.double().view(-1, kv, hd), v.double().view(-1, kv, hd)
    a = b = 0
    for m, t in zip(nq, nk):
        seen = torch.arange(t, device="cuda")[None] <= torch.arange(m, device="cuda")[:, None] + (t - m)
        for h in range(heads):
            if m and t:
                out[a:a + m, h], tol[a:a + m, h] = _attend(q[a:a + m, h], k[b:b + t, h * kv // heads], v[b:b + t, h * kv // heads], seen)
        a, b = a + m, b + t
    return out.flatten(1), tol.expand(-1, -1, hd).flatten(1)


def _starts(lengths):
    return _i32([0] + list(np.cumsum(lengths)))


PROMPTS = [  # heads, kv heads, head size, tokens, keys before them
    (1, 1, 64, [1], [0]),
    (4, 2, 64, [1, 127, 128, 129, 3], [0, 0, 0, 0, 0]),
    (16, 8, 64, [37, 0, 137, 5, 0], [0, 0, 0, 0, 0]),
    (32, 8, 64, [300, 65], [0, 0]),
    (8, 2, 64, [70, 1, 33], [500, 128, 1]),
    (8, 8, 128, [200, 17], [0, 300]),
    (6, 2, 128, [130, 64, 63], [0, 1, 64]),
    (5, 1, 96, [45, 91], [0, 10]),
    (14, 2, 80, [50], [77]),
    (16, 1, 32, [9, 150], [0, 0]),
    (3, 3, 8, [19, 260], [5, 0]),
    (128, 1, 16, [5, 4], [0, 3]),
    (24, 4, 64, [257], [255]),
    (12, 4, 64, [1], [1000]),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", PROMPTS, ids=str)
def test_attention_prompts(ops, dtype, shape):
    heads, kv, hd, nq, prefix = shape
    nk = [n + p for n, p in zip(nq, prefix)]
    g = _gen(sum(nq) * heads + hd)
    q, k, v = _randn(g, sum(nq), heads * hd).to(dtype), _randn(g, sum(nk), kv * hd).to(dtype), (_randn(g, sum(nk), kv * hd) + 0.3).to(dtype)
    out = ops.attention_prompts(q, k, v, _starts(nq), heads, kv, hd, key_starts=_starts(nk) if any(prefix) else None)
    ref, tol = _prompts_ref(q, k, v, nq, nk, heads, kv, hd)
    _check(out, ref, tol, v.abs().max().double())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_prompts_long(ops, dtype):
    """Thousands of keys, several sequences: many tiles, an uneven end, every size of tile on its diagonal."""
    heads, kv, hd, nq = 4, 2, 64, [2500, 1, 700, 129]
    g = _gen(5)
    q, k, v = _randn(g, sum(nq), heads * hd).to(dtype), _randn(g, sum(nq), kv * hd).to(dtype), (_randn(g, sum(nq), kv * hd) + 1).to(dtype)
    out = ops.attention_prompts(q, k, v, _starts(nq), heads, kv, hd)
    ref, tol = _prompts_ref(q, k, v, nq, nq, heads, kv, hd)
    _check(out, ref, tol, v.abs().max().double())


SPLIT = [  # few tokens, many keys: the keys of a block are cut into parts
    (4, 2, 64, [200, 3, 90], [3000, 2500, 4000]),
    (8, 8, 128, [70, 300], [2000, 3333]),
    (2, 1, 64, [2600], [0]),
    (6, 2, 96, [1, 1, 0, 1], [5000, 1, 7, 6001]),
    (5, 1, 32, [64, 1], [6100, 900]),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SPLIT, ids=str)
def test_attention_prompts_in_parts(ops, dtype, shape):
    heads, kv, hd, nq, prefix = shape
    nk = [n + p for n, p in zip(nq, prefix)]
    g = _gen(sum(nk))
    q, k, v = _randn(g, sum(nq), heads * hd).to(dtype), _randn(g, sum(nk), kv * hd).to(dtype), (_randn(g, sum(nk), kv * hd) + 0.3).to(dtype)
    starts, key_starts = _starts(nq), _starts(nk) if any(prefix) else None
    out = ops.attention_prompts(q, k, v, starts, heads, kv, hd, key_starts=key_starts)
    ref, tol = _prompts_ref(q, k, v, nq, nk, heads, kv, hd)
    _check(out, ref, tol, v.abs().max().double())
    # a value that only the last token of the first sequence attends, one that all of its tokens do, and padding behind the sequences
    v2 = v.clone()
    v2[nk[0] - 1, 1] = math.inf
    v2[0, 2] = math.nan
    pad = torch.full((9, kv * hd), math.nan, dtype=dtype, device="cuda")
    out2 = torch.full((sum(nq) + 5, heads * hd), 7.0, dtype=dtype, device="cuda")
    ops.attention_prompts(torch.cat([q, q[:5].expand(5, -1) if nq[0] > 5 else q[:1].expand(5, -1)]), torch.cat([k, pad]), torch.cat([v2, pad]), starts, heads, kv, hd,
                          key_starts=key_starts if key_starts is not None else starts, out=out2)
    hit = torch.zeros_like(out, dtype=torch.bool).view(-1, heads, hd)
    hit[nq[0] - 1, :heads // kv, 1] = True
    hit[:nq[0], :heads // kv, 2] = True
    hit = hit.flatten(1)
    assert (out2[sum(nq):] == 7).all() and torch.equal(out2[:sum(nq)][~hit], out[~hit])
    assert not torch.isfinite(out2[:sum(nq)][hit]).any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_prompts_fewer_keys_than_tokens(ops, dtype):
    """Tokens that have no key get zeros; a sequence without any keys, one without tokens."""
    heads, kv, hd, nq, nk = 4, 2, 64, [40, 10, 0, 150], [25, 0, 60, 149]
    g = _gen(6)
    q, k, v = _randn(g, sum(nq), heads * hd).to(dtype), _randn(g, sum(nk), kv * hd).to(dtype), _randn(g, sum(nk), kv * hd).to(dtype)
    out = ops.attention_prompts(q, k, v, _starts(nq), heads, kv, hd, key_starts=_starts(nk))
    ref, tol = _prompts_ref(q, k, v, nq, nk, heads, kv, hd)
    assert (out[:15] == 0).all() and (out[40:50] == 0).all() and (out[50] == 0).all()
    _check(out, ref, tol, v.abs().max().double())


def test_attention_prompts_no_keys_at_all(ops):
    q = torch.ones(3, 64, device="cuda")
    k = torch.ones(0, 64, device="cuda")
    out = torch.full_like(q, 7.0)
    ops.attention_prompts(q, k, k, _i32([0, 2]), 1, 1, 64, key_starts=_i32([0, 0]), out=out)
    assert (out[:2] == 0).all() and (out[2] == 7).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_prompts_padding_is_left_alone(ops, dtype):
    """Rows behind the last sequence hold NaN: results do not depend on them, and out keeps what it had there."""
    heads, kv, hd, nq = 8, 2, 64, [33, 100]
    g = _gen(7)
    n = sum(nq) + 77
    q, k, v = (_randn(g, n, h * hd).to(dtype) for h in (heads, kv, kv))
    want = ops.attention_prompts(q[:133].contiguous(), k[:133].contiguous(), v[:133].contiguous(), _starts(nq), heads, kv, hd)
    for x in (q, k, v):
        x[133:] = math.nan
    out = torch.full_like(q, 5.0)
    ops.attention_prompts(q, k, v, _starts(nq), heads, kv, hd, out=out)
    assert torch.equal(out[:133], want) and (out[133:] == 5).all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_prompts_not_finite_in_masked_places(ops, dtype, value):
    """A key or value that is not finite reaches the tokens that attend it and no others."""
    heads, kv, hd, nq = 4, 2, 64, [90, 200, 60]
    g = _gen(8)
    q, k, v = (_randn(g, sum(nq), h * hd).to(dtype) for h in (heads, kv, kv))
    clean = ops.attention_prompts(q, k, v, _starts(nq), heads, kv, hd)
    v2, k2 = v.clone(), k.clone()
    at = 90 + 140  # the second sequence's 140th token, KV head 1, dims 3 and 64 + 9
    v2[at, hd + 3] = value
    v2[at, hd + 9] = value
    out = ops.attention_prompts(q, k, v2, _starts(nq), heads, kv, hd)
    hit = torch.zeros_like(out, dtype=torch.bool).view(-1, heads, hd)
    for h in (2, 3):
        hit[at:290, h, 3] = hit[at:290, h, 9] = True
    hit = hit.flatten(1)
    assert torch.equal(out[~hit], clean[~hit])
    assert (torch.isnan(out[hit]) if math.isnan(value) else out[hit] == value).all()
    k2[at, hd + 3] = value  # a key: only rows of its own sequence at and behind it, of its heads
    out = ops.attention_prompts(q, k2, v, _starts(nq), heads, kv, hd).view(-1, heads, hd)
    assert torch.equal(out[:at], clean.view(-1, heads, hd)[:at]) and torch.equal(out[290:], clean.view(-1, heads, hd)[290:])
    assert torch.equal(out[:, :2], clean.view(-1, heads, hd)[:, :2])


@pytest.mark.parametrize("big,small", [(1.0, 1.0), (1e4, 1e-4), (1e-4, 1e4), (3e-7, 2e6)])
def test_attention_prompts_scales_of_f32(ops, big, small):
    """f32 keeps its precision whatever the magnitudes of q, k and v."""
    heads, kv, hd, nq = 4, 2, 64, [150, 40]
    g = _gen(9)
    q, k, v = _randn(g, 190, heads * hd) * big, _randn(g, 190, kv * hd) * small, _randn(g, 190, kv * hd) * big
    out = ops.attention_prompts(q, k, v, _starts(nq), heads, kv, hd)
    ref, tol = _prompts_ref(q, k, v, nq, nq, heads, kv, hd)
    _check(out, ref, tol, v.abs().max().double())


def test_attention_prompts_large_scores(ops):
    """Scores of hundreds: a weight near 1 beside weights that vanish, and maxima that grow from tile to tile."""
    heads, kv, hd, n = 2, 1, 64, 400
    g = _gen(10)
    q = _randn(g, n, heads * hd)
    k = _randn(g, n, kv * hd) * torch.linspace(0.1, 30, n, device="cuda")[:, None]
    v = _randn(g, n, kv * hd)
    for dtype in TYPES:
        a, b, c = q.to(dtype), k.to(dtype), v.to(dtype)
        out = ops.attention_prompts(a, b, c, _starts([n]), heads, kv, hd)
        ref, tol = _prompts_ref(a, b, c, [n], [n], heads, kv, hd)
        _check(out, ref, tol, c.abs().max().double())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_prompts_strided_views(ops, dtype):
    """Views of one fused projection, a transposed tensor, rows that start between 16-byte boundaries, columns taken apart."""
    heads, kv, hd, n = 4, 2, 64, 75
    g = _gen(11)
    fused = _randn(g, n, (heads + 2 * kv) * hd + 16).to(dtype)
    q, k, v = fused[:, :heads * hd], fused[:, heads * hd:(heads + kv) * hd], fused[:, (heads + kv) * hd:(heads + 2 * kv) * hd]
    want = ops.attention_prompts(q.contiguous(), k.contiguous(), v.contiguous(), _starts([n]), heads, kv, hd)
    assert torch.equal(ops.attention_prompts(q, k, v, _starts([n]), heads, kv, hd), want)
    assert torch.equal(ops.attention_prompts(q.T.contiguous().T, k, v, _starts([n]), heads, kv, hd), want)
    odd = torch.empty(n * (kv * hd + 1) + 3, dtype=dtype, device="cuda")[3:].as_strided((n, kv * hd), (kv * hd + 1, 1))
    odd.copy_(v)
    assert torch.equal(ops.attention_prompts(q, k, odd, _starts([n]), heads, kv, hd), want)


def test_attention_prompts_captured_and_replayed_with_other_lengths(ops):
    heads, kv, hd, n = 8, 2, 64, 300
    g = _gen(12)
    for dtype in TYPES:
        q, k, v = (_randn(g, n, h * hd).to(dtype) for h in (heads, kv, kv))
        starts, out = _starts([300, 0, 0]), torch.zeros_like(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.attention_prompts(q, k, v, starts, heads, kv, hd, out=out)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                ops.attention_prompts(q, k, v, starts, heads, kv, hd, out=out)
        torch.cuda.current_stream().wait_stream(side)
        for lengths in ([120, 0, 180], [1, 1, 100]):
            starts.copy_(_starts(lengths))
            q.copy_(_randn(g, n, heads * hd))
            out.fill_(9)
            graph.replay()
            m = sum(lengths)
            want = ops.attention_prompts(q[:m], k[:m], v[:m], starts, heads, kv, hd)
            assert torch.equal(out[:m], want) and (out[m:] == 9).all()


def test_attention_prompts_many_short_sequences(ops):
    heads, kv, hd = 4, 2, 64
    lengths = [(i * 7) % 11 for i in range(1500)]
    g = _gen(13)
    q, k, v = (_randn(g, sum(lengths), h * hd) for h in (heads, kv, kv))
    out = ops.attention_prompts(q, k, v, _starts(lengths), heads, kv, hd)
    some = [0, 1, 2, 700, 1498, 1499]
    at = np.concatenate([[0], np.cumsum(lengths)])
    for s in some:
        a, b = int(at[s]), int(at[s + 1])
        if a < b:
            ref, tol = _prompts_ref(q[a:b], k[a:b], v[a:b], [b - a], [b - a], heads, kv, hd)
            _check(out[a:b], ref, tol, v.abs().max().double())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
@pytest.mark.parametrize("seqs", [32, 33, 100, 1024, 1025])
def test_attention_prompts_every_way_of_counting_blocks(ops, dtype, seqs):
    """Sequences are walked through by level, one after the other, or searched for, by how many they are; some are empty."""
    heads, kv, hd = 4, 1, 32
    lengths = [(i * 37) % 90 if seqs <= 100 else (i * 5) % 7 for i in range(seqs)]
    lengths[seqs // 2] = 300
    g = _gen(seqs)
    n = sum(lengths)
    q, k, v = (_randn(g, n, h * hd).to(dtype) for h in (heads, kv, kv))
    out = torch.full_like(q, math.nan)
    ops.attention_prompts(q, k, v, _starts(lengths), heads, kv, hd, out=out)
    assert torch.isfinite(out).all()
    at = np.concatenate([[0], np.cumsum(lengths)])
    for s in {0, 1, seqs // 2 - 1, seqs // 2, seqs // 2 + 1, seqs - 1}:
        a, b = int(at[s]), int(at[s + 1])
        if a < b:
            ref, tol = _prompts_ref(q[a:b], k[a:b], v[a:b], [b - a], [b - a], heads, kv, hd)
            _check(out[a:b], ref, tol, v.abs().max().double())


def test_attention_prompts_two_graphs_in_turn(ops):
    """Two captured calls, one of them cut into parts, replayed in any order."""
    heads, kv, hd = 8, 2, 64
    g = _gen(15)
    for dtype in TYPES:
        calls = []
        for nq, nk in (([60, 70], [3000, 4000]), ([500, 300], [500, 300])):
            q, k, v = _randn(g, sum(nq), heads * hd).to(dtype), _randn(g, sum(nk), kv * hd).to(dtype), _randn(g, sum(nk), kv * hd).to(dtype)
            calls.append((q, k, v, _starts(nq), heads, kv, hd, _starts(nk), torch.zeros_like(q)))
        want = [ops.attention_prompts(*c[:8]) for c in calls]
        side, graphs = torch.cuda.Stream(), []
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for c in calls:
                graphs.append(torch.cuda.CUDAGraph())
                with torch.cuda.graph(graphs[-1], stream=side):
                    ops.attention_prompts(*c)
        torch.cuda.current_stream().wait_stream(side)
        for i in (0, 1, 1, 0, 0, 1):
            calls[i][8].fill_(3)
            graphs[i].replay()
            assert torch.equal(calls[i][8], want[i])


def test_attention_prompts_two_streams_at_once(ops):
    heads, kv, hd, n = 8, 2, 64, 900
    g = _gen(14)
    data = [[_randn(g, n, h * hd) for h in (heads, kv, kv)] for _ in range(2)]
    starts = _starts([400, 500])
    want = [ops.attention_prompts(*d, starts, heads, kv, hd) for d in data]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in data], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.attention_prompts(*data[i], starts, heads, kv, hd))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


# ── the 4-bit cache ────────────────────────────────────────────────────────────────────────────────
def _blocks(x):
    """f32 [n, dim] -> (quants [n, dim / 2], scales [n, dim / 32] as f16 bits) by the package's own writer of such blocks."""
    from wick_b200 import gguf_synth as gs
    raw = gs.quantize_q4_0(x).reshape(x.shape[0], -1, 18)
    return raw[..., 2:].reshape(x.shape[0], -1), np.ascontiguousarray(raw[..., :2]).view(np.uint16).reshape(x.shape[0], -1)


def _values(quants, scales):
    b = quants.reshape(*quants.shape[:-1], -1, 16).astype(np.int32)
    q = np.concatenate([b & 15, b >> 4], -1) - 8
    return (q * scales.view(np.float16).astype(np.float32)[..., None]).reshape(*quants.shape[:-1], -1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 1, 32), (7, 3, 8, 64), (130, 4, 2, 96), (33, 2, 5, 128)], ids=str)
def test_append_writes_the_blocks_of_the_files(ops, dtype, shape):
    n, slots, kv, hd = shape
    g = _gen(n)
    cache = ops.KvCacheQ4.empty(slots, 150, kv, hd)
    assert cache.max_seq == 192
    k, v = _randn(g, n, kv * hd).to(dtype), (_randn(g, n, kv * hd) * 1e-3).to(dtype)
    k[0, :32] = 0.0                       # a block of zeros
    k[0, kv * hd - 32:] = -0.5            # equal magnitudes
    v[n - 1, :32] = torch.tensor([(-1.0) ** i for i in range(32)])  # both signs
    order = np.random.default_rng(n).permutation(slots * 192)[:n]
    slot, pos = order // 192, order % 192
    before = [t.clone() for t in (cache.k_quants, cache.k_scales, cache.v_quants, cache.v_scales)]
    ops.kv_append_q4(cache, k, v, _i32(slot), _i32(pos))
    for x, quants, scales, q0, d0 in ((k, cache.k_quants, cache.k_scales, *before[:2]), (v, cache.v_quants, cache.v_scales, *before[2:])):
        q, d = _blocks(x.float().cpu().numpy())
        q0, d0 = q0.cpu().numpy(), d0.cpu().numpy().view(np.uint16)
        q0[slot, :, pos], d0[slot, :, pos] = q.reshape(n, kv, -1), d.reshape(n, kv, -1)
        assert np.array_equal(quants.cpu().numpy(), q0) and np.array_equal(scales.cpu().numpy().view(np.uint16), d0)
    got = ops.kv_read_q4(cache, _i32(slot), _i32(pos))
    for x, y in zip((k, v), got):
        assert np.array_equal(y.cpu().numpy(), _values(*_blocks(x.float().cpu().numpy())))


def test_append_and_read_skip_rows_that_the_cache_does_not_have(ops):
    cache = ops.KvCacheQ4.empty(2, 64, 2, 64)
    g = _gen(1)
    k, v = _randn(g, 6, 128), _randn(g, 6, 128)
    ops.kv_append_q4(cache, k, v, _i32([0, -1, 2, 1, 1, 1]), _i32([3, 0, 0, -1, 64, 63]))
    used = torch.zeros(2, 64, dtype=torch.bool)
    used[0, 3] = used[1, 63] = True
    changed = (cache.k_quants.cpu() != 0x88).flatten(3).any(3).any(1)
    assert torch.equal(changed, used)
    a, b = ops.kv_read_q4(cache, _i32([0, 5, -3, 1, 1, 0, 0]), _i32([3, 0, 0, 63, 64, -1, 3]))
    for x, y in ((a, k), (b, v)):
        want = torch.from_numpy(_values(*_blocks(y.cpu().numpy())))
        assert torch.equal(x[[0, 6]].cpu(), want[[0, 0]]) and torch.equal(x[3].cpu(), want[5]) and (x[[1, 2, 4, 5]] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_append_of_strided_rows(ops, dtype):
    g = _gen(2)
    n, kv, hd = 9, 2, 64
    fused = _randn(g, n, 2 * kv * hd + 3).to(dtype)
    k, v = fused[:, :kv * hd], fused[:, kv * hd + 1:2 * kv * hd + 1]  # rows 4 or 2 bytes off any wider boundary
    slots, pos = _i32([0] * n), _i32(range(n))
    a, b = ops.KvCacheQ4.empty(1, 64, kv, hd), ops.KvCacheQ4.empty(1, 64, kv, hd)
    ops.kv_append_q4(a, k, v, slots, pos)
    ops.kv_append_q4(b, k.contiguous(), v.contiguous(), slots, pos)
    for x, y in zip(ops.kv_read_q4(a, slots, pos), ops.kv_read_q4(b, slots, pos)):
        assert torch.equal(x, y)
    assert torch.equal(a.k_quants, b.k_quants) and torch.equal(a.v_scales, b.v_scales)


def _random_cache(ops, g, slots, rows, kv, hd):
    planes = []
    for std in (0.27, 0.2):
        shape = (slots, kv, rows)
        planes.append(torch.randint(0, 256, (*shape, hd // 2), generator=g, device="cuda", dtype=torch.uint8))
        sign = torch.randint(0, 2, (*shape, hd // 32), generator=g, device="cuda") * 2.0 - 1
        planes.append((sign * std * (0.5 + torch.rand(sign.shape, generator=g, device="cuda"))).half())
    return ops.KvCacheQ4(*planes)


def _q4_ref(q, cache, slots, lengths, heads):
    kv, hd, n = cache.n_kv_heads, cache.head_dim, q.shape[0]
    out = torch.zeros(n, heads, hd, dtype=torch.float64, device="cuda")
    tol = torch.zeros(n, heads, 1, dtype=torch.float64, device="cuda")
    vmax = 0.0
    q = q.double().view(n, heads, hd)
    for j, (s, t) in enumerate(zip(slots, lengths)):
        t = min(t, cache.max_seq)
        if s < 0 or t <= 0:
            continue
        for c in range(kv):
            k, v = (torch.from_numpy(_values(a[s, c, :t].cpu().numpy(), b[s, c, :t].cpu().numpy().view(np.uint16))).double().cuda()
                    for a, b in ((cache.k_quants, cache.k_scales), (cache.v_quants, cache.v_scales)))
            vmax = max(vmax, v.abs().max().item())
            group = heads // kv
            seen = torch.ones(group, t, dtype=torch.bool, device="cuda")
            out[j, c * group:(c + 1) * group], tol[j, c * group:(c + 1) * group] = _attend(q[j, c * group:(c + 1) * group], k, v, seen)
    return out.flatten(1), tol.expand(-1, -1, hd).flatten(1), vmax


Q4 = [  # heads, kv heads, head size, lengths
    (1, 1, 64, [1]),
    (4, 2, 64, [0, 1, 2, 63, 64, 65, 127, 129]),
    (32, 8, 64, [517, 3]),
    (16, 8, 64, [900, 1, 0, 333, 64, 2049, 15, 16, 17]),
    (8, 8, 128, [130, 1000]),
    (16, 4, 128, [77, 640]),
    (12, 2, 96, [300, 5]),
    (10, 2, 32, [40, 1500]),
    (7, 1, 64, [257]),
    (24, 2, 64, [100, 700]),
    (16, 1, 64, [511]),
    (40, 2, 32, [90, 0]),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", Q4, ids=str)
def test_attention_q4(ops, dtype, shape):
    heads, kv, hd, lengths = shape
    g = _gen(heads * hd + len(lengths))
    rows = -(-max(lengths) // 64) * 64
    cache = _random_cache(ops, g, len(lengths), rows, kv, hd)
    slots = np.random.default_rng(1).permutation(len(lengths)).tolist()
    q = _randn(g, len(lengths), heads * hd).to(dtype)
    ref, tol, vmax = _q4_ref(q, cache, slots, lengths, heads)
    for s, t in zip(slots, lengths):  # behind a row's length: scales that are not finite
        cache.k_scales[s, :, t:] = math.nan
        cache.v_scales[s, :, t:] = math.inf
    out = ops.attention_q4(q, cache, _i32(slots), _i32(lengths), heads)
    _check(out, ref, tol, vmax)
    assert all((out[j] == 0).all() for j, t in enumerate(lengths) if t == 0)


def test_attention_q4_padding_shared_slots_and_capped_lengths(ops):
    heads, kv, hd = 8, 2, 64
    g = _gen(3)
    cache = _random_cache(ops, g, 3, 128, kv, hd)
    slots, lengths = [1, -1, 1, 0, 3, 1, 2], [100, 50, 101, 5000, 7, 102, -4]
    q = _randn(g, len(slots), heads * hd)
    out = torch.full_like(q, 3.0)
    ops.attention_q4(q, cache, _i32(slots), _i32(lengths), heads, out=out)
    assert (out[[1, 4]] == 3).all() and (out[6] == 0).all()
    keep = [0, 2, 3, 5]
    ref, tol, vmax = _q4_ref(q[keep], cache, [slots[i] for i in keep], [lengths[i] for i in keep], heads)
    _check(out[keep], ref, tol, vmax)


@pytest.mark.parametrize("kscale,vscale", [(1e-3, 1e3), (30.0, 1e-4), (2e-7, 6e-8), (1.0, 3e4)])
def test_attention_q4_magnitudes(ops, kscale, vscale):
    """Scales from the smallest to the largest that f16 has, mixed within a row."""
    heads, kv, hd, n = 8, 2, 64, 300
    g = _gen(4)
    cache = _random_cache(ops, g, 1, 320, kv, hd)
    for t, s in ((cache.k_scales, kscale), (cache.v_scales, vscale)):
        t.copy_((t.float() / 0.3 * s * torch.rand(t.shape, generator=g, device="cuda")).clamp(-65504, 65504))
    q = _randn(g, 1, heads * hd) * 0.3 / max(kscale, 1e-3)
    ref, tol, vmax = _q4_ref(q, cache, [0], [n], heads)
    _check(ops.attention_q4(q, cache, _i32([0]), _i32([n]), heads), ref, tol, vmax)


def test_attention_q4_strided_queries_and_a_graph(ops):
    heads, kv, hd, n = 8, 2, 64, 5
    g = _gen(5)
    cache = _random_cache(ops, g, n, 1024, kv, hd)
    wide = _randn(g, n, heads * hd + 5)
    slots, lengths = _i32(range(n)), _i32([1000, 1, 77, 500, 0])
    want = ops.attention_q4(wide[:, 2:2 + heads * hd].contiguous(), cache, slots, lengths, heads)
    assert torch.equal(ops.attention_q4(wide[:, 2:2 + heads * hd], cache, slots, lengths, heads), want)
    q, out = wide[:, 2:2 + heads * hd].contiguous(), torch.zeros(n, heads * hd, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attention_q4(q, cache, slots, lengths, heads, out=out)
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for graph in graphs:
            with torch.cuda.graph(graph, stream=side):
                ops.attention_q4(q, cache, slots, lengths, heads, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for graph, values in zip(graphs * 2, ([3, 900, 64, 1, 1024], [1000, 1, 77, 500, 0], [5, 5, 5, 5, 5], [0, 0, 0, 0, 1])):
        lengths.copy_(_i32(values))
        graph.replay()
        assert torch.equal(out, ops.attention_q4(q, cache, slots, lengths, heads))


def test_attention_q4_offsets_beyond_32_bits(ops):
    """The last slot of a cache of more than 2^32 bytes of quants."""
    heads, kv, hd, rows = 8, 8, 64, 6400
    slots = 2 ** 32 // (kv * rows * hd // 2) + 2
    planes = [torch.empty((slots, kv, rows, w), dtype=t, device="cuda") for w, t in ((hd // 2, torch.uint8), (hd // 32, torch.float16)) * 2]
    cache = ops.KvCacheQ4(*planes)
    g = _gen(6)
    n = 200
    at, s = _i32(range(n)), _i32([slots - 1] * n)
    k, v = _randn(g, n, kv * hd), _randn(g, n, kv * hd)
    ops.kv_append_q4(cache, k, v, s, at)
    small = ops.KvCacheQ4.empty(1, n, kv, hd)
    ops.kv_append_q4(small, k, v, torch.zeros_like(s), at)
    for x, y in zip(ops.kv_read_q4(cache, s, at), ops.kv_read_q4(small, torch.zeros_like(s), at)):
        assert torch.equal(x, y)
    q = _randn(g, 1, heads * hd)
    ref, tol, vmax = _q4_ref(q, small, [0], [n], heads)
    _check(ops.attention_q4(q, cache, s[:1], _i32([n]), heads), ref, tol, vmax)


def test_attention_q4_many_rows(ops):
    """More rows than SMs, and than a block has threads."""
    heads, kv, hd, n = 4, 2, 32, 1300
    g = _gen(7)
    cache = _random_cache(ops, g, 3, 192, kv, hd)
    slots, lengths = [i % 3 for i in range(n)], [(i * 37) % 180 for i in range(n)]
    q = _randn(g, n, heads * hd)
    out = ops.attention_q4(q, cache, _i32(slots), _i32(lengths), heads)
    some = list(range(0, n, 97)) + [n - 1]
    ref, tol, vmax = _q4_ref(q[some], cache, [slots[i] for i in some], [lengths[i] for i in some], heads)
    _check(out[some], ref, tol, vmax)


def test_attention_q4_long(ops):
    heads, kv, hd = 8, 2, 64
    g = _gen(8)
    lengths = [70001, 3, 20000]
    cache = _random_cache(ops, g, 3, 70016, kv, hd)
    q = _randn(g, 3, heads * hd)
    ref, tol, vmax = _q4_ref(q, cache, [2, 0, 1], lengths, heads)
    _check(ops.attention_q4(q, cache, _i32([2, 0, 1]), _i32(lengths), heads), ref, tol, vmax)


# ── log probabilities ──────────────────────────────────────────────────────────────────────────────
def _logprobs_ref(x, tokens, top_n):
    """In f64 on the host: NaN as -inf, logits beyond +-1e30 as infinite; a stable order of (value descending, id ascending)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    x = np.where(np.abs(x) >= 1e30, np.copysign(np.inf, x), x)
    n, vocab = x.shape
    lp, ent, ids, lps = np.full(n, -np.inf), np.zeros(n), np.zeros((n, top_n), np.int32), np.full((n, top_n), -np.inf)
    for i in range(n):
        m = x[i].max()
        with np.errstate(invalid="ignore"):
            d = np.where(x[i] == m, 0.0, x[i] - m) if m > -np.inf else np.full(vocab, -np.inf)
        e = np.exp(d)
        logp = d - (np.log(e.sum()) if e.sum() else 0.0)
        if 0 <= tokens[i] < vocab:
            lp[i] = logp[tokens[i]]
        with np.errstate(invalid="ignore"):
            ent[i] = -np.nansum(np.where(e > 0, np.exp(logp) * logp, 0.0)) if e.sum() else 0.0
        ids[i] = np.argsort(-x[i], kind="stable")[:top_n]
        lps[i] = logp[ids[i]]
    return lp, ent, ids, lps


def _check_logprobs(ops, x, tokens, top_n):
    """A thread adds at most 4 + vocab / 256 terms, each off by 2^-22 (its exponential) before half a step per addition."""
    lp, ent, ids, lps = ops.token_logprobs(x, _i32(tokens), top_n)
    n, vocab = x.shape
    assert lp.shape == ent.shape == (n,) and ids.shape == lps.shape == (n, top_n) and ids.dtype == torch.int32
    want = _logprobs_ref(x.float().cpu().numpy(), tokens, top_n)
    rel = (8 + vocab / 256) * 2.0 ** -24
    for got, ref in ((lp, want[0]), (lps, want[3])):
        got = got.cpu().numpy().astype(np.float64)
        inf = np.isinf(ref)
        assert np.array_equal(got[inf], ref[inf])
        assert (np.abs(got[~inf] - ref[~inf]) <= rel + 2.0 ** -23 * np.abs(ref[~inf])).all()
    assert np.array_equal(ids.cpu().numpy(), want[2])
    got = ent.cpu().numpy()
    assert (np.abs(got - want[1]) <= 3 * rel * (1 + math.log(vocab))).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 1000, 64), (4, 4099, 5), (3, 50021, 20), (1, 65536, 5), (700, 517, 3),
                                   (1, 140001, 64), (64, 32768, 20), (2, 65536, 0)], ids=str)
def test_token_logprobs(ops, dtype, shape):
    n, vocab, top_n = shape
    g = _gen(vocab + n)
    x = (_randn(g, n, vocab) * 3).to(dtype)
    x[:, vocab // 2] += 9
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda").tolist()
    tokens[0] = vocab // 2
    _check_logprobs(ops, x, tokens, top_n)


def test_token_logprobs_masked_vocabularies(ops):
    """Rows of which a mask leaves three tokens, one, none; infinities, NaN, the type's lowest value, equal logits."""
    vocab, inf, low = 33000, math.inf, torch.finfo(torch.float32).min
    x = torch.full((9, vocab), -inf, device="cuda")
    x[0, [5, 17, 32999]] = torch.tensor([1.0, 3.0, 2.0], device="cuda")
    x[1, 31000] = -2.5
    x[3, :] = _randn(_gen(1), vocab)
    x[3, [4, 9]] = inf
    x[4, :] = math.nan
    x[4, [100, 7]] = 0.25
    x[5, :] = 1.5
    x[6, ::2], x[6, 1::2] = 0.0, -0.0
    x[7, :] = low
    x[7, 12] = 2.0
    x[8, :] = torch.arange(vocab, device="cuda") * 1e-3
    _check_logprobs(ops, x, [17, 0, 3, 9, 7, 200, 0, 12, -1], 8)
    _check_logprobs(ops, x, [0, 31000, vocab, 3, 99, 0, 1, 12, vocab - 1], 1)


def test_token_logprobs_sharp_and_flat_rows(ops):
    x = torch.zeros(3, 65536, device="cuda")
    x[0, 77] = 60.0
    x[1, 5] = 18.0
    x[2] += 1e4
    _check_logprobs(ops, x, [77, 5, 3], 4)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_token_logprobs_of_strided_rows(ops, dtype):
    """Rows of a padded vocabulary, which start at every offset from a 16-byte boundary; columns that are not dense."""
    g = _gen(4)
    x = _randn(g, 11, 2003).to(dtype)
    tokens = list(range(0, 1100, 100))
    _check_logprobs(ops, x[:, 1:1999], tokens, 5)
    _check_logprobs(ops, x[:, ::2], [t % 1002 for t in tokens], 5)
    _check_logprobs(ops, x.T.contiguous().T, tokens, 5)
    _check_logprobs(ops, x[:1], tokens[:1], 2)


def test_token_logprobs_in_a_graph_and_without_rows(ops):
    g = _gen(6)
    x, tokens = _randn(g, 4, 65536), _i32([1, 2, 3, 4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.token_logprobs(x, tokens, 5)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = ops.token_logprobs(x, tokens, 5)
    torch.cuda.current_stream().wait_stream(side)
    x.copy_(_randn(g, 4, 65536))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, ops.token_logprobs(x, tokens, 5)))
    empty = ops.token_logprobs(x[:0], tokens[:0], 2)
    assert empty[0].shape == (0,) and empty[2].shape == (0, 2)


def test_wrappers_refuse(ops):
    from wick_b200 import _lib
    x, i = torch.zeros(2, 64, device="cuda"), _i32([0, 1])
    cache = ops.KvCacheQ4.empty(1, 64, 1, 64)
    bad = [lambda: ops.token_logprobs(x, i.long()), lambda: ops.token_logprobs(x, i[:1]), lambda: ops.token_logprobs(x, i, 65),
           lambda: ops.token_logprobs(x, i, -1), lambda: ops.token_logprobs(x.double(), i), lambda: ops.token_logprobs(x[0], i),
           lambda: ops.token_logprobs(x, i.cpu()), lambda: ops.kv_append_q4(cache, x, x.half(), i, i), lambda: ops.kv_append_q4(cache, x[:, :32], x[:, :32], i, i),
           lambda: ops.attention_q4(x, cache, i, i, 2), lambda: ops.attention_q4(x, cache, i, i[:1], 1), lambda: ops.attention_q4(x, cache, i, i, 1, out=x.half()),
           lambda: ops.attention_prompts(x, x, x.half(), i, 1, 1, 64), lambda: ops.attention_prompts(x, x, x, i, 2, 1, 64),
           lambda: ops.attention_prompts(x, x, x, i, 1, 1, 64, key_starts=i[:1]), lambda: ops.attention_prompts(x, x, x, i, 1, 1, 64, out=x[:1]),
           lambda: ops.KvCacheQ4.empty(1, 64, 1, 48), lambda: ops.KvCacheQ4(cache.k_quants, cache.k_scales, cache.v_quants, cache.v_scales[:, :, :32])]
    for f in bad:
        with pytest.raises(_lib.WickCudaError):
            f()


def test_offsets_and_slots_without_a_dimension(ops):
    from wick_b200 import _lib
    x, one = torch.zeros(2, 64, device="cuda"), torch.zeros((), dtype=torch.int32, device="cuda")
    cache = ops.KvCacheQ4.empty(1, 64, 1, 64)
    for f in (lambda: ops.kv_read_q4(cache, one, one), lambda: ops.attention_prompts(x, x, x, one, 1, 1, 64),
              lambda: ops.attention_prompts(x, x, x, _i32([[0, 1], [1, 2]]), 1, 1, 64)):
        with pytest.raises(_lib.WickCudaError):
            f()


# ── together ───────────────────────────────────────────────────────────────────────────────────────
def test_a_serving_step(ops):
    """Packed prompts, their keys and values into the cache, the next tokens' attention over it, log probabilities of the choice:
    eager and as one captured graph, on a stream of its own."""
    heads, kv, hd, vocab = 8, 2, 64, 4000
    nq = [130, 1, 64, 77]
    n, seqs = sum(nq), len(nq)
    g = _gen(20)
    cache = ops.KvCacheQ4.empty(seqs + 1, 200, kv, hd)
    q, k, v = (_randn(g, n, h * hd) for h in (heads, kv, kv))
    prompt_slots = _i32(np.repeat(np.arange(seqs), nq))
    prompt_pos = _i32(np.concatenate([np.arange(m) for m in nq]))
    o = ops.attention_prompts(q, k, v, _starts(nq), heads, kv, hd)
    ref, tol = _prompts_ref(q, k, v, nq, nq, heads, kv, hd)
    _check(o, ref, tol, v.abs().max().double())
    ops.kv_append_q4(cache, k, v, prompt_slots, prompt_pos)
    # a padded batch of five rows: the last one is no sequence
    slots, pos, lengths = _i32([0, 1, 2, 3, -1]), _i32(nq + [-1]), _i32([m + 1 for m in nq] + [0])
    head = _randn(g, heads * hd, vocab) * 0.1
    q1, k1, v1 = (_randn(g, 5, h * hd) for h in (heads, kv, kv))
    out = torch.zeros(5, heads * hd, device="cuda")
    tokens = _i32([7, 8, 9, 10, -1])

    def step():
        ops.kv_append_q4(cache, k1, v1, slots, pos)
        ops.attention_q4(q1, cache, slots, lengths, heads, out=out)
        return ops.token_logprobs(out @ head, tokens, 5)

    eager = [t.clone() for t in step()]
    ref, tol, vmax = _q4_ref(q1[:4], cache, [0, 1, 2, 3], [m + 1 for m in nq], heads)
    _check(out[:4], ref, tol, vmax)
    assert (out[4] == 0).all() and eager[0][4] == -math.inf
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, eager))


def test_attention_prompts_without_sequences(ops):
    x = torch.ones(3, 64, device="cuda")
    out = torch.full_like(x, 2.0)
    assert (ops.attention_prompts(x, x, x, _i32([0]), 1, 1, 64, out=out) == 2).all()
    assert (ops.attention_prompts(x, x, x, _i32([0]), 1, 1, 64) == 0).all()
    assert (ops.attention_prompts(x, x, x, _i32([1, 2]), 1, 1, 64, key_starts=_i32([0, 3]))[[0, 2]] == 0).all()
    assert ops.attention_prompts(x[:0], x, x, _i32([0, 0]), 1, 1, 64).shape == (0, 64)
