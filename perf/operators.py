"""The operators of a serving step beside the model's own path, as cases to be timed: attention of packed prompts, the
4-bit K / V cache (append and read back, attention over it) and log probabilities.

A case is one pass: what `run` does for one prepared state.  With `own` it makes the calls of `wick_b200.ops`; without, it
computes the same in elementary torch operations in f32.  Head counts and sizes are those of the package's own model shapes
(16 or 32 query heads, 8 KV heads, head size 64) and of its wide-head test shape (128)."""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one decode step of eight sequences: their new K / V rows go into the 4-bit cache
        dict(name="append_8_rows", kind="append", n=8, slots=8, kv=8, hd=64, type="f32"),
        # the K / V rows of packed prompts
        dict(name="append_4093_rows", kind="append", n=4093, slots=6, kv=8, hd=64, type="f32"),
        # one sequence, a short chat: latency
        dict(name="q4_1x517", kind="q4", rows=1, longest=517, heads=32, kv=8, hd=64, type="f32"),
        # a serving batch with ragged lengths
        dict(name="q4_64x4100", kind="q4", rows=64, longest=4100, heads=32, kv=8, hd=64, type="f32"),
        # one very long document, wide heads
        dict(name="q4_1x131000_hd128", kind="q4", rows=1, longest=131000, heads=16, kv=4, hd=128, type="bf16"),
        # one-line prompts of a few users, small model
        dict(name="prompts_6x137_f32", kind="prompts", seqs=6, longest=137, prefix=0, heads=16, kv=8, hd=64, type="f32"),
        # pages of text packed into one step, 1.6B-class model, the package's own type
        dict(name="prompts_8x1001_f32", kind="prompts", seqs=8, longest=1001, prefix=0, heads=32, kv=8, hd=64, type="f32"),
        # one long prompt with wide heads in 16 bits
        dict(name="prompts_1x8000_bf16", kind="prompts", seqs=1, longest=8000, prefix=0, heads=32, kv=8, hd=128, type="bf16"),
        # the next chunk of prompts whose first keys are cached
        dict(name="prompts_4x512_after_3500_f16", kind="prompts", seqs=4, longest=512, prefix=3500, heads=32, kv=8, hd=64, type="f16"),
        # one decode step: the chosen token and its five alternatives
        dict(name="logprobs_1_top5", kind="logprobs", n=1, vocab=65536, top=5, type="f32"),
        # a serving batch's step with twenty alternatives
        dict(name="logprobs_64_top20", kind="logprobs", n=64, vocab=65536, top=20, type="f32"),
        # scoring of a long text, an odd vocabulary in 16 bits
        dict(name="logprobs_2500_bf16", kind="logprobs", n=2500, vocab=50021, top=0, type="bf16"),
    ]


def draw(rng):
    def logu(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["append", "q4", "q4", "prompts", "prompts", "prompts", "logprobs", "logprobs"])
    heads, kv, hd = rng.choice([(16, 8, 64), (32, 8, 64), (16, 4, 128), (24, 4, 64), (8, 8, 128), (12, 2, 96), (10, 2, 32)])
    c = dict(kind=kind, kv=kv, hd=hd, type=rng.choice(["f32", "f32", "f16", "bf16"]))
    if kind == "append":
        return dict(c, n=logu(1, 4096), slots=rng.randint(1, 32))
    if kind == "logprobs":
        return dict(kind=kind, n=logu(1, 1200), vocab=logu(500, 140000), top=rng.choice([0, 1, 5, 20]), type=c["type"])
    if kind == "q4":
        longest = logu(1, 100000)
        return dict(c, heads=heads, rows=logu(1, min(64, max(2, 260000 // longest))), longest=longest)
    longest = logu(1, 4000)
    seqs = logu(1, min(16, max(2, 8000 // longest)))
    return dict(c, heads=heads, seqs=seqs, longest=longest, prefix=rng.choice([0, 0, logu(1, 2000)]))


def _lengths(n, longest, least=1):
    """n ragged lengths that go by the case alone: the longest, and others spread between a quarter of it and it."""
    rng = random.Random(n * 1000003 + longest)
    return [longest] + [rng.randint(max(least, longest // 4), longest) for _ in range(n - 1)]


def _pairs(case):
    """(query tokens, key rows, attended pairs) of a packed prompt case."""
    nq = _lengths(case["seqs"], case["longest"])
    nk = [n + case["prefix"] for n in nq]
    return nq, nk, sum(n * case["prefix"] + n * (n + 1) // 2 for n in nq)


def _starts(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    kind, t = case["kind"], TYPES[case["type"]]
    if kind == "logprobs":
        # a model's logits: a broad bulk and a few tokens that stand out
        x = randn(case["n"], case["vocab"]) * 2.5
        hot = torch.randint(0, case["vocab"], (case["n"], 8), generator=g, device="cuda")
        x.scatter_add_(1, hot, randn(case["n"], 8).abs() * 6)
        return dict(kind=kind, logits=x.to(t), tokens=hot[:, 0].to(torch.int32).contiguous(), top=case["top"])
    kv, hd = case["kv"], case["hd"]
    if kind == "prompts":
        nq, nk, _ = _pairs(case)
        return dict(kind=kind, q=randn(sum(nq), case["heads"] * hd).to(t), k=randn(sum(nk), kv * hd).to(t), v=(randn(sum(nk), kv * hd) * 0.7 + 0.1).to(t),
                    starts=_starts(nq), key_starts=_starts(nk) if case["prefix"] else None, heads=case["heads"], kv=kv, hd=hd,
                    nq=max(nq), nk=max(nk))
    n = case["slots"] if kind == "append" else case["rows"]
    rows = -(-case["n"] // n) + 7 if kind == "append" else case["longest"]
    rows = -(-rows // 64) * 64
    planes = []
    for std in (0.27, 0.2):  # keys and values: random nibbles, scales of both signs as the rounding gives them
        sign = torch.randint(0, 2, (n, kv, rows, hd // 32), generator=g, device="cuda") * 2.0 - 1.0
        planes.append(torch.randint(0, 256, (n, kv, rows, hd // 2), generator=g, device="cuda", dtype=torch.uint8))
        planes.append((sign * std * (0.6 + 0.8 * torch.rand(sign.shape, generator=g, device="cuda"))).half())
    order = torch.randperm(n, generator=g, device="cuda")
    if kind == "append":
        j = torch.arange(case["n"], device="cuda")
        return dict(kind=kind, planes=planes, slots=order[j % n].to(torch.int32), positions=(j // n + 5).to(torch.int32),
                    k=randn(case["n"], kv * hd).to(t), v=(randn(case["n"], kv * hd) * 0.7).to(t), kv=kv, hd=hd)
    return dict(kind=kind, planes=planes, slots=order.to(torch.int32), lengths=torch.tensor(_lengths(n, case["longest"]), dtype=torch.int32).cuda(),
                q=randn(n, case["heads"] * hd).to(t), heads=case["heads"], kv=kv, hd=hd, nk=case["longest"])


# ── the plain forms ─────────────────────────────────────────────────────────────────────────────────
def _values(quants, scales):
    """Blocks of 32: byte i holds value i in its low and value i + 16 in its high bits; value = scale * (bits - 8)."""
    b = quants.unflatten(-1, (-1, 16)).int()
    return (torch.cat([b & 15, b >> 4], -1).float() - 8.0).mul_(scales.float().unsqueeze(-1)).flatten(-2)


def _blocks(x):
    """f32 [..., 32 m] -> the nearest such blocks: the value of largest magnitude becomes -8."""
    x = x.unflatten(-1, (-1, 32))
    d = x.gather(-1, x.abs().argmax(-1, keepdim=True)) / -8.0
    inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    q = (x * inv + 8.5).trunc().clamp(0, 15).to(torch.uint8)
    return (q[..., :16] | (q[..., 16:] << 4)).flatten(-2), d.squeeze(-1).half()


def _softmax_v(scores, seen, v):
    """softmax over the last axis of the scores where seen, times v; nothing seen gives zeros."""
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.clamp_min(-3e38)).exp_()
    return p @ v / p.sum(-1, keepdim=True).clamp_min(1e-38)


def _plain_prompts(s):
    heads, kv, hd, total = s["heads"], s["kv"], s["hd"], s["q"].shape[0]
    starts = s["starts"].long()
    keys = starts if s["key_starts"] is None else s["key_starts"].long()
    nq, nk = starts.diff(), keys.diff()
    at_q = (starts[:-1, None] + torch.arange(s["nq"], device="cuda")).clamp_max(total - 1)
    at_k = (keys[:-1, None] + torch.arange(s["nk"], device="cuda")).clamp_max(s["k"].shape[0] - 1)
    q = s["q"].float().view(total, kv, heads // kv, hd)[at_q].permute(0, 2, 3, 1, 4).flatten(2, 3)  # [seqs, kv, group * nq, hd]
    k = s["k"].float().view(-1, kv, hd)[at_k].transpose(1, 2)
    v = s["v"].float().view(-1, kv, hd)[at_k].transpose(1, 2)
    j, t = torch.arange(s["nq"], device="cuda"), torch.arange(s["nk"], device="cuda")
    seen = (t <= j[:, None] + (nk - nq)[:, None, None]) & (t < nk[:, None, None])  # [seqs, nq, nk]
    scores = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(hd)).unflatten(2, (heads // kv, s["nq"]))
    o = _softmax_v(scores, seen[:, None, None], v[:, :, None])  # [seqs, kv, group, nq, hd]
    token = torch.arange(total, device="cuda")
    seq = torch.searchsorted(starts, token, right=True) - 1
    return o[seq, :, :, token - starts[seq]].reshape(total, heads * hd).to(s["q"].dtype)


def _plain_q4(s):
    heads, kv, hd, n = s["heads"], s["kv"], s["hd"], s["q"].shape[0]
    slots = s["slots"].long()
    kq, kd, vq, vd = (p[slots, :, :s["nk"]] for p in s["planes"])
    q = s["q"].float().view(n, kv, heads // kv, hd)
    seen = torch.arange(s["nk"], device="cuda") < s["lengths"][:, None]
    scores = (q @ _values(kq, kd).transpose(2, 3)).mul_(1.0 / math.sqrt(hd))
    return _softmax_v(scores, seen[:, None, None], _values(vq, vd)).reshape(n, heads * hd).to(s["q"].dtype)


def _plain_append(s):
    slots, at = s["slots"].long(), s["positions"].long()
    for x, quants, scales in ((s["k"], *s["planes"][:2]), (s["v"], *s["planes"][2:])):
        q, d = _blocks(x.float().view(-1, s["kv"], s["hd"]))
        quants[slots, :, at] = q
        scales[slots, :, at] = d
    kq, kd, vq, vd = (p[slots, :, at] for p in s["planes"])
    return _values(kq, kd).flatten(1), _values(vq, vd).flatten(1)


def _plain_logprobs(s):
    x = s["logits"].float()
    n, vocab = x.shape
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    total = e.sum(1, dtype=torch.float64)
    lse = total.log()
    entropy = lse - (e.double() * d).sum(1) / total
    picked = d.gather(1, s["tokens"].long()[:, None])[:, 0] - lse
    # equal logits by ascending id: the order of (value, -id) as one whole number
    bits = (x + 0.0).view(torch.int32)
    key = ((bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32) | (0xFFFFFFFF - torch.arange(vocab, device="cuda"))
    ids = 0xFFFFFFFF - (key.topk(s["top"], dim=1).values & 0xFFFFFFFF)
    return picked.float(), entropy.float(), ids.to(torch.int32), (d.gather(1, ids) - lse[:, None]).float()


def run(s):
    kind = s["kind"]
    if not own:
        return {"prompts": _plain_prompts, "q4": _plain_q4, "append": _plain_append, "logprobs": _plain_logprobs}[kind](s)
    from wick_b200 import ops
    if kind == "prompts":
        return ops.attention_prompts(s["q"], s["k"], s["v"], s["starts"], s["heads"], s["kv"], s["hd"], key_starts=s["key_starts"])
    if kind == "logprobs":
        return ops.token_logprobs(s["logits"], s["tokens"], s["top"])
    cache = ops.KvCacheQ4(*s["planes"])
    if kind == "q4":
        return ops.attention_q4(s["q"], cache, s["slots"], s["lengths"], s["heads"])
    ops.kv_append_q4(cache, s["k"], s["v"], s["slots"], s["positions"])
    return ops.kv_read_q4(cache, s["slots"], s["positions"])


# ── what a pass cannot do without ───────────────────────────────────────────────────────────────────
def work(case):
    size = SIZE[case["type"]]
    if case["kind"] == "logprobs":
        n, vocab = case["n"], case["vocab"]
        return {"bytes": n * (vocab * size + 4 + 8 + 8 * case["top"]), "flops": 4 * n * vocab}
    kv, hd = case["kv"], case["hd"]
    if case["kind"] == "append":  # the rows in, blocks of 18 bytes out and their values back
        return {"bytes": 2 * case["n"] * kv * (hd * size + 2 * (hd // 32 * 18) + 4 * hd), "flops": 8 * case["n"] * kv * hd}
    heads = case["heads"]
    if case["kind"] == "q4":
        keys = sum(_lengths(case["rows"], case["longest"]))
        return {"bytes": 2 * keys * kv * (hd // 32) * 18 + 2 * case["rows"] * heads * hd * size, "flops": 4 * keys * heads * hd}
    nq, nk, pairs = _pairs(case)
    return {"bytes": size * hd * (2 * heads * sum(nq) + 2 * kv * sum(nk)), "flops": 4 * hd * heads * pairs}


# ── the definitions in 64 bits, one sequence or row after the other ─────────────────────────────────
def _attend(q, k, v):
    """q [m, hd] against k, v [t, hd] with the last m of the t keys the queries' own (m = 1: one query over all)."""
    m, t = q.shape[0], k.shape[0]
    w = torch.exp2((q @ k.T) * (math.log2(math.e) / math.sqrt(q.shape[1])))
    w = torch.where(torch.arange(t, device="cuda")[None] > torch.arange(t - m, t, device="cuda")[:, None], 0.0, w)
    return (w / w.sum(1, keepdim=True)) @ v


def _unpack(quants, scales):
    """Blocks [t, 16 m bytes], [t, m] -> values [t, 32 m]."""
    t, m = scales.shape
    b = quants.view(t, m, 16)
    out = torch.empty(t, m, 32, dtype=torch.float64, device="cuda")
    out[..., :16] = torch.remainder(b, 16).double() - 8
    out[..., 16:] = torch.div(b, 16, rounding_mode="floor").double() - 8
    return (out * scales.double()[..., None]).view(t, 32 * m)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return None  # the rounding itself is defined in f32, and its values go by equality
    if case["kind"] == "logprobs":
        lp, ent, tops = [], [], []
        for x, token in zip(s["logits"].double(), s["tokens"].tolist()):
            x = x - torch.logsumexp(x, 0)
            lp.append(x[token])
            ent.append(-(x.exp() * x).sum())
            tops.append(x.topk(case["top"]).values)
        return torch.stack(lp), torch.stack(ent), None, torch.stack(tops)
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    out = torch.zeros(s["q"].shape[0], heads, hd, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(-1, heads, hd)
    if case["kind"] == "q4":
        kq, kd, vq, vd = s["planes"]
        for row, (slot, t) in enumerate(zip(s["slots"].tolist(), s["lengths"].tolist())):
            for c in range(kv):
                k, v = _unpack(kq[slot, c, :t], kd[slot, c, :t]), _unpack(vq[slot, c, :t], vd[slot, c, :t])
                for h in range(c * heads // kv, (c + 1) * heads // kv):
                    out[row, h] = _attend(q[row, h][None], k, v)[0]
        return out.view(-1, heads * hd)
    nq, nk, _ = _pairs(case)
    a = b = 0
    for m, t in zip(nq, nk):
        k, v = (x[b:b + t].double().view(t, kv, hd) for x in (s["k"], s["v"]))
        for h in range(heads):
            out[a:a + m, h] = _attend(q[a:a + m, h], k[:, h * kv // heads], v[:, h * kv // heads])
        a, b = a + m, b + t
    return out.view(-1, heads * hd)
