"""Operators that serve the text model to many at once, as measured cases.

sample_tokens     the next token of each row of logits from a given random number: temperature, min-p, top-k, top-p
rope_append8      rotary positions (and the per-head norm) of new tokens, keys and values written to a cache of 8 bits
attention_paged8  attention over that cache: e4m3 values, a power of two for each block of tokens and head
linear4           products of a few rows with weights of 4 bits, a scale for each group

`own` false: plain torch forms in 32 bits (sampling in 64).  `own` true: the framework's entry points.
"""
import math
import os
import random
import sys

import torch

own = False

# The text model's own shapes (hidden 2560, 32 query heads on 8 key-value heads of 128, MLP 9728, vocabulary 151936,
# theta 1e6) are the usual ones here; the other shapes are generic.
_VOCAB = 151936
_MAX8 = 448.0  # the largest e4m3 value


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the next token of one answer, with the settings that the model's makers advise: latency
        dict(name="sample_tokens_1", op="sample", rows=1, vocab=_VOCAB, f32=True, banned=False, settings="usual"),
        # a serving batch: every answer has its own settings (greedy ones, open ones, min-p), under a grammar that forbids most
        # tokens; a small odd vocabulary (rows that start at odd addresses)
        dict(name="sample_tokens_65", op="sample", rows=65, vocab=50021, f32=False, banned=True, settings="mixed"),
        # many answers to one question at once, top-p alone over the whole vocabulary
        dict(name="sample_tokens_512", op="sample", rows=512, vocab=_VOCAB, f32=True, banned=False, settings="top_p"),
        # a serving batch of 64 sequences far into a long context, one new token each, blocks partly filled
        dict(name="rope_append8_64", op="rope", tokens=64, seqs=64, heads=32, kv_heads=8, head_dim=128, rot_dim=128,
             interleaved=False, theta=1e6, reach=131072, page=64, block=16, norm=True, f32=False, head_major=True, decode=True),
        # prompts of several sequences at once, the QKV projection's f32 output in
        dict(name="rope_append8_prompts", op="rope", tokens=8191, seqs=19, heads=32, kv_heads=8, head_dim=128, rot_dim=128,
             interleaved=False, theta=1e6, reach=512, page=16, block=16, norm=True, f32=True, head_major=False, decode=False),
        # the next token of one 512-token prompt: latency
        dict(name="attention_paged8_1", op="attention", seqs=1, new=1, heads=32, kv_heads=8, head_dim=128, shortest=512,
             longest=512, page=16, block=16, head_major=False),
        # one long document
        dict(name="attention_paged8_1_long", op="attention", seqs=1, new=1, heads=32, kv_heads=8, head_dim=128, shortest=131071,
             longest=131071, page=64, block=64, head_major=False),
        # a serving batch with sequences of every length, a scale for every token
        dict(name="attention_paged8_64", op="attention", seqs=64, new=1, heads=32, kv_heads=8, head_dim=128, shortest=1,
             longest=8192, page=16, block=1, head_major=False),
        # a prompt of odd length, every token over those before it
        dict(name="attention_paged8_prompt", op="attention", seqs=1, new=2047, heads=32, kv_heads=8, head_dim=128, shortest=2047,
             longest=2047, page=16, block=16, head_major=False),
        # one token through the model's QKV projection: latency
        dict(name="linear4_1", op="linear", rows=1, n=6144, k=2560, group=128, zeros=False, scale_f32=False, f32=False, add=False),
        # a small batch through the MLP's down projection, onto the residual stream
        dict(name="linear4_16", op="linear", rows=16, n=2560, k=9728, group=64, zeros=True, scale_f32=False, f32=True, add=True),
        # one token through the head
        dict(name="linear4_head", op="linear", rows=1, n=_VOCAB, k=2560, group=32, zeros=False, scale_f32=False, f32=True, add=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("sample", "rope", "attention", "linear"))
    if op == "sample":
        vocab = rng.choice((_VOCAB, _log(rng, 100, 260000), 32000, 65537))
        return dict(op="sample", rows=_log(rng, 1, min(512, 512 * _VOCAB // vocab)), vocab=vocab, f32=rng.random() < 0.5,
                    banned=rng.random() < 0.3, settings=rng.choice(("usual", "mixed", "top_p", "open", "min_p", "top_k")))
    if op == "linear":
        group = rng.choice((32, 64, 128))
        k = group * _log(rng, max(1, 256 // group), 16384 // group)
        rows = _log(rng, 1, 32)
        return dict(op="linear", rows=rows, n=_log(rng, 64, min(_VOCAB, _VOCAB * 2560 // (k * max(1, rows // 4)))), k=k,
                    group=group, zeros=rng.random() < 0.5, scale_f32=rng.random() < 0.3, f32=rng.random() < 0.5, add=rng.random() < 0.4)
    head_dim = rng.choice((64, 128, 128, 256))
    page, block = rng.choice(((16, 16), (16, 1), (24, 8), (32, 32), (64, 16), (64, 64), (100, 50), (1, 1)))
    kv_heads = rng.choice((1, 2, 4, 8))
    if op == "rope":
        heads = kv_heads * rng.choice((1, 2, 3, 4, 7))
        tokens = min(_log(rng, 1, 8191), 8191 * 48 * 128 // ((heads + 2 * kv_heads) * head_dim))
        decode = rng.random() < 0.5
        if decode:
            tokens = min(tokens, 512)
        seqs = tokens if decode else min(tokens, _log(rng, 1, 32))
        return dict(op="rope", tokens=tokens, seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rot_dim=rng.choice((head_dim, head_dim, head_dim // 2, head_dim * 3 // 4)), interleaved=rng.random() < 0.4,
                    theta=rng.choice((1e4, 1e6)), reach=_log(rng, 512, 131072) if decode else -(-tokens // seqs) + _log(rng, 16, 4096),
                    page=page, block=block, norm=rng.random() < 0.5, f32=rng.random() < 0.5, head_major=rng.random() < 0.5,
                    decode=decode)
    heads = kv_heads * rng.choice((1, 2, 4, 5, 7, 8, 16))
    if rng.random() < 0.3:  # prompts, or the rest of them
        seqs, new = _log(rng, 1, 4), _log(rng, 2, 1024)
        longest = new + rng.choice((0, 0, _log(rng, 1, 2048)))
        while seqs * new * longest * heads * head_dim > 2047 * 2047 * 32 * 128:
            new, longest = max(2, new // 2), max(2, longest // 2)
        return dict(op="attention", seqs=seqs, new=new, heads=heads, kv_heads=kv_heads, head_dim=head_dim, shortest=longest,
                    longest=longest, page=page, block=block, head_major=rng.random() < 0.5)
    seqs = _log(rng, 1, 256)
    longest = max(1, min(_log(rng, 16, 131072), 64 * 4096 * 8 * 128 // (seqs * kv_heads * head_dim)))
    return dict(op="attention", seqs=seqs, new=1, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                shortest=rng.choice((0, 1, longest // 2, longest)), longest=longest, page=page, block=block,
                head_major=rng.random() < 0.5)


def _lengths(case):
    """The number of keys of each sequence: spread evenly from shortest to longest, out of order."""
    lo, hi, n = case["shortest"], case["longest"], case["seqs"]
    if n == 1:
        return [hi]
    order = list(range(n))
    random.Random(n).shuffle(order)
    return [lo + (hi - lo) * i // (n - 1) for i in order]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["f32"] else 2) + case["rows"] * 36, "flops": 4 * n}
    if case["op"] == "linear":
        n, k, rows = case["n"], case["k"], case["rows"]
        groups = n * (k // case["group"])
        out = rows * n * (4 if case["f32"] else 2)
        return {"bytes": n * k // 2 + groups * ((4 if case["scale_f32"] else 2) + case["zeros"]) + rows * k * 2 + out * (1 + case["add"]),
                "flops": 2 * rows * n * k}
    if case["op"] == "rope":
        q, kv = case["tokens"] * case["heads"] * case["head_dim"], 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        size = 4 if case["f32"] else 2
        return {"bytes": q * (size + 2) + kv * (size + 1) + 8 * case["tokens"], "flops": 6 * (q + kv)}
    keys, new, nkv, hd = sum(_lengths(case)), case["new"], case["kv_heads"], case["head_dim"]
    rows = case["seqs"] * new
    seen = sum(n * new - new * (new - 1) // 2 for n in _lengths(case))
    return {"bytes": 2 * keys * nkv * hd + 2 * (keys // case["block"]) * nkv + rows * case["heads"] * hd * 4,
            "flops": 4 * seen * case["heads"] * hd}


# ------------------------------------------------------------------ inputs
def _frequencies(case):
    """Radians per position of each pair, in 64 bits (plain numbers: a model's configuration gives them)."""
    return [case["theta"] ** (-2.0 * i / case["rot_dim"]) for i in range(case["rot_dim"] // 2)]


def _pools(values, case):
    """Values [pages, slot, head, column] as a cache of 8 bits: e4m3 pools stored slot by slot or head by head, and the
    exponent (biased by 127) of each block's and head's scale, the least that brings the values within e4m3's range."""
    pages, p, h, d = values.shape
    b = case["block"]
    grouped = values.view(pages, p // b, b, h, d)
    top = grouped.abs().amax((2, 4)).clamp(min=2.0 ** -60)
    exp = torch.ceil(torch.log2(top / _MAX8))
    held = (grouped * torch.exp2(-exp)[:, :, None, :, None]).view(pages, p, h, d).to(torch.float8_e4m3fn)
    if case["head_major"]:
        held = held.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    return held, (exp + 127).to(torch.uint8)


def _settings(kind, rows, rnd):
    """Per row: temperature, top_k, top_p, min_p."""
    if kind == "usual":
        return [(0.7, 20, 0.8, 0.0)] * rows
    if kind == "top_p":
        return [(1.0, 0, 0.95, 0.0)] * rows
    if kind == "open":
        return [(rnd.uniform(0.5, 1.5), 0, 1.0, 0.0) for _ in range(rows)]
    if kind == "min_p":
        return [(rnd.uniform(0.7, 1.5), 0, 1.0, rnd.choice((0.02, 0.05, 0.1))) for _ in range(rows)]
    if kind == "top_k":
        return [(1.0, rnd.choice((1, 5, 40, 200, 1000, 5000)), 1.0, 0.0) for _ in range(rows)]
    return [rnd.choice(((0.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (1.0, 0, 1.0, 0.0), (1.2, 0, 0.9, 0.0), (1.0, 50, 1.0, 0.05),
                        (0.6, 0, 0.95, 0.02), (1.0, 300, 0.99, 0.0))) for _ in range(rows)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = random.Random(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    whole = lambda lo, hi, *s, dtype=torch.int32: torch.randint(lo, hi, s, device="cuda", generator=g, dtype=dtype)  # noqa: E731
    i32 = lambda x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
    f32 = lambda x: torch.tensor(x, device="cuda", dtype=torch.float32)  # noqa: E731
    if case["op"] == "sample":
        n, vocab = case["rows"], case["vocab"]
        x = normal(n, vocab) * 2.5
        # a few likely tokens in each row, as a trained model has them
        x.scatter_add_(1, whole(0, vocab, n, 8, dtype=torch.int64), 4 + 6 * torch.rand(n, 8, device="cuda", generator=g))
        if case["banned"]:
            x[torch.rand(n, vocab, device="cuda", generator=g) < 0.9] = -math.inf
            x[:, rnd.randrange(vocab)] = 3.0
            if n > 8:
                x[n // 2] = -math.inf  # an answer that the grammar leaves no way on
        t, k, p, m = zip(*_settings(case["settings"], n, rnd))
        return {"case": case, "logits": x if case["f32"] else x.bfloat16(), "temperature": f32(t), "top_k": i32(k), "top_p": f32(p),
                "min_p": f32(m), "uniform": torch.rand(n, device="cuda", generator=g, dtype=torch.float64),
                "ids": torch.zeros(n, device="cuda", dtype=torch.int32), "logprobs": torch.zeros(n, device="cuda"),
                "kept": torch.zeros(n, device="cuda", dtype=torch.int32)}
    if case["op"] == "linear":
        n, k, rows = case["n"], case["k"], case["rows"]
        scale = (0.5 + torch.rand(n, k // case["group"], device="cuda", generator=g)) * (0.2 / math.sqrt(k))
        out = torch.zeros(rows, n, device="cuda", dtype=torch.float32 if case["f32"] else torch.bfloat16)
        return {"case": case, "q": whole(0, 256, n, k // 2, dtype=torch.uint8),
                "scale": scale if case["scale_f32"] else scale.bfloat16(),
                "zero": whole(5, 12, n, k // case["group"], dtype=torch.uint8) if case["zeros"] else None,
                "x": normal(rows, k).bfloat16(), "add": normal(rows, n).to(out.dtype) if case["add"] else None, "out": out}
    nh, nkv, hd, ps = (case[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    if case["op"] == "rope":
        t, s = case["tokens"], case["seqs"]
        # the newest tokens of each sequence, as one run of rows: sequence i gets the positions first[i] and up
        share = [t * (i + 1) // s - t * i // s for i in range(s)]
        first = [rnd.randrange(0, max(1, case["reach"] - n + 1)) for n in share]
        seq = [i for i in range(s) for _ in range(share[i])]
        pos = [first[i] + j for i in range(s) for j in range(share[i])]
        touched = sorted({(a, b // ps) for a, b in zip(seq, pos)})
        pages = sum((n - 1) // ps + 2 for n in share) + 3  # wherever the runs begin
        ids = list(range(pages))
        rnd.shuffle(ids)
        table = whole(0, pages, s, -(-case["reach"] // ps))
        at = torch.tensor(touched, device="cuda")
        table[at[:, 0], at[:, 1]] = i32(ids[:len(touched)])
        qkv = normal(t, (nh + 2 * nkv) * hd) * 1.5
        # earlier tokens in the pools, some blocks of them much smaller than what comes
        k, k_exp = _pools(normal(pages, ps, nkv, hd) * torch.exp2(torch.randint(-6, 3, (pages, 1, nkv, 1), device="cuda", generator=g)), case)
        v, v_exp = _pools(normal(pages, ps, nkv, hd), case)
        return {"case": case, "qkv": qkv if case["f32"] else qkv.bfloat16(), "k": k, "v": v, "k_exp": k_exp, "v_exp": v_exp,
                "q_out": torch.zeros(t, nh, hd, device="cuda", dtype=torch.bfloat16), "table": table,
                "q_norm": 1 + 0.1 * normal(hd) if case["norm"] else None, "k_norm": 1 + 0.1 * normal(hd) if case["norm"] else None,
                "freqs": torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda"), "seq": i32(seq), "pos": i32(pos)}
    lens, new = _lengths(case), case["new"]
    n = len(lens)
    need = [-(-x // ps) for x in lens]
    pages = sum(need) + 3
    perm = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(n, -(-case["longest"] // ps), device="cuda", dtype=torch.int32)
    held = torch.arange(table.shape[1], device="cuda")[None, :] < i32(need)[:, None]
    table[held] = perm[:sum(need)]
    k, k_exp = _pools(normal(pages, ps, nkv, hd), case)
    v, v_exp = _pools(normal(pages, ps, nkv, hd), case)
    ahead = i32(list(range(new)))[None, :] - new
    return {"case": case, "q": (normal(n * new, nh, hd) * 2).bfloat16(), "k": k, "v": v, "k_exp": k_exp, "v_exp": v_exp, "table": table,
            "seq": i32(list(range(n)))[:, None].expand(n, new).reshape(-1).contiguous(),
            "pos": (i32(lens)[:, None] + ahead).reshape(-1).contiguous(),
            "out": torch.zeros(n * new, nh, hd, device="cuda", dtype=torch.bfloat16)}


# ------------------------------------------------------------------ one pass
def run(state):
    return {"sample": _sample, "rope": _rope, "attention": _attention, "linear": _linear}[state["case"]["op"]](state)


def _sample(s):
    if own:
        return _own_sample(s)
    # the tokens in line, likeliest first, equal ones by id; weights in 64 bits, since a token is taken by where a sum of
    # them ends
    x, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device="cuda")[None, :]
    greedy = (s["temperature"] <= 0)[:, None]
    t = torch.where(greedy, 1.0, s["temperature"].double()[:, None])
    top = x[:, :1].double()
    some = torch.isfinite(top)
    w = torch.exp((x.double() - torch.where(some, top, 0.0)) / t)
    k = s["top_k"][:, None]
    keep = (x > -math.inf) & some & (w >= s["min_p"].double()[:, None]) & ((k <= 0) | (rank < k)) & (~greedy | (rank == 0))
    w = torch.where(keep, w, 0.0)
    reached = torch.cumsum(w, 1)
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (reached - w < p * reached[:, -1:]) | (rank == 0)
    kept = keep.sum(1)
    mass = reached.gather(1, (kept - 1).clamp(min=0)[:, None])
    pick = (keep & (reached <= s["uniform"][:, None] * mass)).sum(1)
    pick = torch.minimum(pick, (keep & (w > 0)).sum(1) - 1).clamp(min=0)[:, None]
    s["ids"].copy_(torch.where(kept > 0, order.gather(1, pick)[:, 0], -1))
    logp = (x.gather(1, pick).double() - top) / t - torch.log(mass)
    s["logprobs"].copy_(torch.where(kept > 0, logp[:, 0], -math.inf))
    s["kept"].copy_(kept)
    return {k: s[k] for k in ("ids", "logprobs", "kept")}


def _turn(x, cos, sin, rd, interleaved):
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else (x[..., :rd // 2], x[..., rd // 2:rd])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, x[..., rd:]), -1)


def _rope(s):
    if own:
        return _own_rope(s)
    c = s["case"]
    t, nh, nkv, hd, rd = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"], c["rot_dim"]
    x = s["qkv"].float().view(t, nh + 2 * nkv, hd)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["q_norm"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["k_norm"]
    angle = s["pos"].double()[:, None] * s["freqs"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    s["q_out"].copy_(_turn(q, cos, sin, rd, c["interleaved"]))
    pos = s["pos"].long()
    page, slot = s["table"][s["seq"].long(), pos // c["page"]].long(), pos % c["page"]
    _append8(s["k"], s["k_exp"], _turn(k, cos, sin, rd, c["interleaved"]), page, slot, c)
    _append8(s["v"], s["v_exp"], v, page, slot, c)
    return {n: s[n] for n in ("q_out", "k", "v", "k_exp", "v_exp")}


def _append8(pool, exps, x, page, slot, c):
    """x [tokens, heads, columns] to their slots.  A block's scale grows where the new values need it, and what the block
    holds is rounded to it; a block whose first slot is written starts anew."""
    b = c["block"]
    per = c["page"] // b
    at = page * per + slot // b                       # each token's block
    top = x.abs().amax(-1).clamp(min=2.0 ** -60 * _MAX8)
    need = torch.ceil(torch.log2(top / _MAX8)) + 127  # top / 448 is exact enough: 448 is 7 times a power of two
    need += (top > _MAX8 * torch.exp2(need - 127)).float() - (top <= _MAX8 * torch.exp2(need - 128)).float()
    blocks, index = torch.unique(at, return_inverse=True)
    most = torch.zeros(blocks.numel(), x.shape[1], device="cuda").scatter_reduce(0, index[:, None].expand(-1, x.shape[1]), need, "amax")
    fresh = torch.zeros(blocks.numel(), device="cuda").scatter_reduce(0, index, (slot % b == 0).float(), "amax")[:, None] > 0
    held = exps.view(-1, x.shape[1])[blocks].float()
    now = torch.where(fresh, most, torch.maximum(most, held))
    exps.view(-1, x.shape[1])[blocks] = now.to(torch.uint8)
    lower = torch.where(fresh, 0.0, held - now)       # what the block holds comes down by so many powers of two
    slots = (blocks % per * b)[:, None] + torch.arange(b, device="cuda")[None, :]
    where = (blocks // per)[:, None].expand(-1, b)
    pool[where, slots] = (pool[where, slots].float() * torch.exp2(lower)[:, None, :, None]).to(torch.float8_e4m3fn)
    pool[page, slot] = (x * torch.exp2(127 - now[index])[..., None]).to(torch.float8_e4m3fn)


def _values(pool, exps, page, slot, block):
    return pool[page, slot].float() * torch.exp2(exps[page, slot // block].float() - 127)[..., None]


def _attention(s):
    if own:
        return _own_attention(s)
    c = s["case"]
    n, new, nh, nkv, hd, ps = c["seqs"], c["new"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    j = torch.arange(c["longest"], device="cuda")
    page, slot = s["table"].long()[:, j // ps], j % ps
    k = _values(s["k"], s["k_exp"], page, slot, c["block"])  # [sequences, keys, kv heads, columns]
    v = _values(s["v"], s["v_exp"], page, slot, c["block"])
    q = s["q"].float().view(n, new, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, hd)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1 / math.sqrt(hd))
    seen = (j <= s["pos"].view(n, new, 1)).repeat(1, nh // nkv, 1)[:, None]
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(o.view(n, nkv, nh // nkv, new, hd).permute(0, 3, 1, 2, 4).reshape(n * new, nh, hd))
    return s["out"]


def _linear(s):
    if own:
        return _own_linear(s)
    c = s["case"]
    q = torch.stack((s["q"] & 15, s["q"] >> 4), -1).view(c["n"], -1, c["group"]).float()
    w = (q - (s["zero"].float()[..., None] if c["zeros"] else 8.0)) * s["scale"].float()[..., None]
    y = torch.matmul(s["x"].float(), w.view(c["n"], c["k"]).t())
    s["out"].copy_(y + s["add"].float() if c["add"] else y)
    return s["out"]


# ------------------------------------------------------------------ the framework's calls
def _iris():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "iris.c_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import iris_cuda
    return iris_cuda


def _own_sample(s):
    if "call" not in s:
        s["call"] = _iris().sample_tokens
    s["call"](s["logits"], s["uniform"], s["ids"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
              min_p=s["min_p"], logprobs=s["logprobs"], kept=s["kept"], stream=torch.cuda.current_stream().cuda_stream)
    return {k: s[k] for k in ("ids", "logprobs", "kept")}


def _own_rope(s):
    c = s["case"]
    if "call" not in s:  # what a program keeps from step to step: the cache's description and the rotation
        ops = _iris()
        s["cache"] = ops.KvCache8.of(s["k"], s["v"], s["k_exp"], s["v_exp"], s["table"])
        s["rope"] = ops.Rope.of(c["rot_dim"], c["theta"], interleaved=c["interleaved"])
        s["call"] = ops.rope_append8
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    qkv = s["qkv"]
    s["call"](s["cache"], s["rope"], s["q_out"], qkv[:, :nh * hd], qkv[:, nh * hd:(nh + nkv) * hd], qkv[:, (nh + nkv) * hd:],
              s["seq"], s["pos"], heads=nh, q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6,
              stream=torch.cuda.current_stream().cuda_stream)
    return {n: s[n] for n in ("q_out", "k", "v", "k_exp", "v_exp")}


def _own_attention(s):
    if "call" not in s:  # kept from step to step: the cache's description and the workspace
        ops = _iris()
        s["cache"] = ops.KvCache8.of(s["k"], s["v"], s["k_exp"], s["v_exp"], s["table"])
        s["ws"] = torch.empty(ops.attention_paged8_workspace(s["cache"], s["case"]["heads"]), device="cuda", dtype=torch.uint8)
        s["call"] = ops.attention_paged8
    s["call"](s["cache"], s["out"], s["q"], s["seq"], s["pos"], scale=1 / math.sqrt(s["case"]["head_dim"]), workspace=s["ws"],
              stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_linear(s):
    if "call" not in s:  # kept from step to step: the weights' description
        ops = _iris()
        s["w"] = ops.Weights4.of(s["q"], s["scale"], s["zero"])
        s["call"] = ops.linear4
    s["call"](s["out"], s["x"], s["w"], add=s["add"], stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "rope": _exact_rope, "attention": _exact_attention, "linear": _exact_linear}[case["op"]](s, case)


def _exact_sample(s, case):
    """Row by row."""
    ids, logprobs, kept = [], [], []
    settings = zip(*(s[k].double().tolist() for k in ("temperature", "top_k", "top_p", "min_p", "uniform")))
    for r, (t, k, p, m, u) in enumerate(settings):
        x = s["logits"][r].double()
        ids_r = torch.nonzero(x > -math.inf)[:, 0]
        if not ids_r.numel():
            ids.append(-1), logprobs.append(-math.inf), kept.append(0)
            continue
        ids_r = ids_r[torch.sort(-x[ids_r], stable=True).indices]
        if t <= 0:
            ids_r, t = ids_r[:1], 1.0
        logp = (x[ids_r] - x[ids_r[0]]) / t
        logp = logp[logp.exp() >= m]
        logp = logp[:int(k)] if k > 0 else logp
        logp = logp - torch.logsumexp(logp, 0)
        if p < 1:
            ahead = logp.exp().cumsum(0) - logp.exp()
            logp = logp[:max(1, int((ahead < p).sum()))]
        logp = logp - torch.logsumexp(logp, 0)
        at = min(int((logp.exp().cumsum(0) <= u).sum()), logp.numel() - 1)
        ids.append(int(ids_r[at])), logprobs.append(float(logp[at])), kept.append(logp.numel())
    at = dict(device="cuda")
    return {"ids": torch.tensor(ids, dtype=torch.int32, **at), "logprobs": torch.tensor(logprobs, dtype=torch.float64, **at),
            "kept": torch.tensor(kept, dtype=torch.int32, **at)}


def _exact_rope(s, case):
    """The values that the 8 bits stand for, at the scales: not rounded.  The scales are whole numbers, from 64-bit values."""
    nh, nkv, hd, half, page, block = (case[k] for k in ("heads", "kv_heads", "head_dim", "rot_dim", "page", "block"))
    half //= 2
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    turns = torch.polar(torch.ones(case["tokens"], half, dtype=torch.float64, device="cuda"), s["pos"].double().outer(s["freqs"]))[:, None, :]
    heads = s["qkv"].double().view(case["tokens"], -1, hd)

    def rotated(x, w):
        y = x.clone()
        if w is not None:
            y /= ((y ** 2).sum(-1, keepdim=True) / hd + 1e-6).sqrt()
            y *= w.double()
        z = torch.complex(y[..., first], y[..., second]) * turns
        y[..., first], y[..., second] = z.real, z.imag
        return y

    tokens = {}
    table = s["table"].cpu()
    for t, (a, b) in enumerate(zip(s["seq"].tolist(), s["pos"].tolist())):
        tokens.setdefault((int(table[a, b // page]), b % page // block), []).append((b % page, t))
    if len(tokens) > 4000:
        return None
    out = {"q_out": rotated(heads[:, :nh], s["q_norm"])}
    for name, x in (("k", rotated(heads[:, nh:nh + nkv], s["k_norm"])), ("v", heads[:, nh + nkv:])):
        pool, exps = s[name].double(), s[name + "_exp"].clone()
        for (p, b), list_ in tokens.items():
            new = x[[t for _, t in list_]]
            e = torch.ceil(torch.log2(new.abs().amax((0, 2)) / _MAX8)).clamp(min=-60) + 127
            old = exps[p, b].double()
            if all(slot % block for slot, _ in list_):
                e = torch.maximum(e, old)
                pool[p, b * block:(b + 1) * block] *= torch.exp2(old - e)[None, :, None]
            pool[p, [slot for slot, _ in list_]] = new * torch.exp2(127 - e)[None, :, None]
            exps[p, b] = e.to(torch.uint8)
        out[name], out[name + "_exp"] = pool, exps
    return {n: out[n] for n in ("q_out", "k", "v", "k_exp", "v_exp")}


def _exact_attention(s, case):
    n, new, nh, nkv, hd, ps, block = (case[k] for k in ("seqs", "new", "heads", "kv_heads", "head_dim", "page", "block"))
    out = torch.zeros(n * new, nh, hd, dtype=torch.float64, device="cuda")
    for i, length in enumerate(_lengths(case)):
        if not length:
            continue
        held = s["table"][i, :(length - 1) // ps + 1].long()
        both = []
        for name in ("k", "v"):
            e = s[name + "_exp"][held].double().repeat_interleave(block, 1) - 127
            both.append((s[name][held].double() * (2.0 ** e)[..., None]).reshape(-1, nkv, hd)[:length])
        rows = slice(i * new, (i + 1) * new)
        q = s["q"][rows].double().view(new, nkv, nh // nkv, hd)
        later = torch.arange(length, device="cuda")[None, :] > s["pos"][rows, None]
        for h in range(nkv):
            x = torch.einsum("ngd,ld->gnl", q[:, h], both[0][:, h]) / math.sqrt(hd)
            p = torch.softmax(x.masked_fill(later, -math.inf), -1).nan_to_num(0.0)
            out[rows].view(new, nkv, nh // nkv, hd)[:, h] = torch.einsum("gnl,ld->ngd", p, both[1][:, h])
    return out


def _exact_linear(s, case):
    n, k, g = case["n"], case["k"], case["group"]
    parts = []
    for lo in range(0, n, 16384):  # some weights at a time: 64 bits of all of them is much memory
        q = s["q"][lo:lo + 16384]
        w = torch.empty(q.shape[0], k, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (q % 16).double(), (q // 16).double()
        zero = s["zero"][lo:lo + 16384].double() if case["zeros"] else torch.full((q.shape[0], k // g), 8.0, dtype=torch.float64, device="cuda")
        w -= zero.repeat_interleave(g, 1)
        w *= s["scale"][lo:lo + 16384].double().repeat_interleave(g, 1)
        parts.append(torch.einsum("rk,nk->rn", s["x"].double(), w))
    y = torch.cat(parts, 1)
    return y + s["add"].double() if case["add"] else y
