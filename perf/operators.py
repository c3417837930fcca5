"""Operators that run the resident text model one token at a time, as measured cases.

rope_append      rotary positions (and the per-head norm) of new tokens, keys and values written to a paged cache
attention_paged  attention of new tokens over a paged key-value cache
token_logprobs   log probabilities of given tokens, entropy and the best alternatives

`own` false: plain torch forms in 32 bits.  `own` true: the framework's entry points.
"""
import math
import os
import random
import sys

import torch

own = False

# The text model's own shape (32 query heads on 8 key-value heads of 128, vocabulary 151936, theta 1e6) is the usual
# one here; the other shapes are generic.
_VOCAB = 151936


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one sequence, one new token: the smallest call, pure latency
        dict(name="rope_append_1", op="rope", tokens=1, seqs=1, heads=32, kv_heads=8, head_dim=128, rot_dim=128,
             interleaved=False, theta=1e6, factor=1.0, original=0, reach=512, page=16, norm=True, f32=True, head_major=False,
             decode=True),
        # a serving batch of 64 sequences far into a long context (positions scaled by parts), one new token each
        dict(name="rope_append_64_far", op="rope", tokens=64, seqs=64, heads=32, kv_heads=8, head_dim=128, rot_dim=128,
             interleaved=False, theta=1e6, factor=4.0, original=32768, reach=131072, page=64, norm=True, f32=False,
             head_major=True, decode=True),
        # prompts of several sequences at once, the QKV projection's f32 output in
        dict(name="rope_append_prompts", op="rope", tokens=8191, seqs=19, heads=32, kv_heads=8, head_dim=128, rot_dim=128,
             interleaved=False, theta=1e6, factor=1.0, original=0, reach=512, page=16, norm=True, f32=True, head_major=False,
             decode=False),
        # interleaved pairs on half of each head, as many key-value heads as query heads, odd token count
        dict(name="rope_append_partial", op="rope", tokens=1031, seqs=5, heads=30, kv_heads=30, head_dim=128, rot_dim=64,
             interleaved=True, theta=1e4, factor=2.0, original=0, reach=4096, page=24, norm=False, f32=False,
             head_major=True, decode=False),
        # the next token of one 512-token prompt: latency
        dict(name="attention_paged_1", op="attention", rows=1, heads=32, kv_heads=8, head_dim=128, shortest=512,
             longest=512, page=16, head_major=False),
        # one long document
        dict(name="attention_paged_1_long", op="attention", rows=1, heads=32, kv_heads=8, head_dim=128, shortest=131071,
             longest=131071, page=64, head_major=False),
        # a serving batch with sequences of every length
        dict(name="attention_paged_64", op="attention", rows=64, heads=32, kv_heads=8, head_dim=128, shortest=1,
             longest=8192, page=16, head_major=False),
        # many short sequences, seven query heads to a key-value head of 64, odd pages stored head by head
        dict(name="attention_paged_256", op="attention", rows=256, heads=14, kv_heads=2, head_dim=64, shortest=0,
             longest=2048, page=24, head_major=True),
        # the next token of one answer, with the alternatives a user may ask for
        dict(name="token_logprobs_1", op="logprobs", rows=1, vocab=_VOCAB, top=20, f32=False, banned=False),
        # a batch of answers under a grammar that forbids most of the vocabulary
        dict(name="token_logprobs_64", op="logprobs", rows=64, vocab=_VOCAB, top=20, f32=False, banned=True),
        # a 512-token prompt scored from f32 logits
        dict(name="token_logprobs_512", op="logprobs", rows=512, vocab=_VOCAB, top=5, f32=True, banned=False),
        # a long document scored with a small odd vocabulary (rows that start at odd addresses)
        dict(name="token_logprobs_2048", op="logprobs", rows=2047, vocab=50021, top=8, f32=False, banned=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("rope", "attention", "logprobs"))
    if op == "rope":
        head_dim = rng.choice((64, 128, 128, 256))
        kv_heads = rng.choice((1, 2, 4, 8))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 7))
        tokens = min(_log(rng, 1, 8191), 8191 * 48 * 128 // ((heads + 2 * kv_heads) * head_dim))
        decode = rng.random() < 0.5
        if decode:
            tokens = min(tokens, 512)
        seqs = tokens if decode else min(tokens, _log(rng, 1, 32))
        factor = rng.choice((1.0, 2.0, 4.0, 8.0))
        return dict(op="rope", tokens=tokens, seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rot_dim=rng.choice((head_dim, head_dim, head_dim // 2, head_dim * 3 // 4)), interleaved=rng.random() < 0.4,
                    theta=rng.choice((1e4, 1e6)), factor=factor, original=rng.choice((0, 4096, 32768)) if factor > 1 else 0,
                    reach=_log(rng, 512, 131072) if decode else max(1, -(-tokens // seqs)) + _log(rng, 16, 4096),
                    page=rng.choice((1, 16, 24, 32, 64, 100)), norm=rng.random() < 0.5, f32=rng.random() < 0.5,
                    head_major=rng.random() < 0.5, decode=decode)
    if op == "attention":
        head_dim = rng.choice((64, 128, 128, 256))
        kv_heads = rng.choice((1, 2, 4, 8))
        heads = kv_heads * rng.choice((1, 2, 4, 5, 7, 8, 16))
        rows = _log(rng, 1, 256)
        longest = min(_log(rng, 16, 131072), 64 * 4096 * 8 * 128 // (rows * kv_heads * head_dim))
        return dict(op="attention", rows=rows, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    shortest=rng.choice((0, 1, longest // 2, longest)), longest=max(1, longest),
                    page=rng.choice((1, 16, 24, 32, 64, 100)), head_major=rng.random() < 0.5)
    vocab = rng.choice((_VOCAB, _log(rng, 100, 260000), 32000, 65537))
    return dict(op="logprobs", rows=_log(rng, 1, min(2047, 512 * _VOCAB // vocab)), vocab=vocab, top=rng.choice((0, 1, 5, 8, 20, 32)),
                f32=rng.random() < 0.5, banned=rng.random() < 0.3)


def _lengths(case):
    """The number of keys of each row: spread evenly from shortest to longest, out of order."""
    lo, hi, n = case["shortest"], case["longest"], case["rows"]
    if n == 1:
        return [hi]
    order = list(range(n))
    random.Random(n).shuffle(order)
    return [lo + (hi - lo) * i // (n - 1) for i in order]


def work(case):
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": n * ((4 if case["f32"] else 2) + 2) + 8 * case["tokens"], "flops": 6 * n}
    if case["op"] == "attention":
        keys = sum(_lengths(case))
        return {"bytes": keys * case["kv_heads"] * case["head_dim"] * 4 + case["rows"] * case["heads"] * case["head_dim"] * 4,
                "flops": 4 * keys * case["heads"] * case["head_dim"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (4 if case["f32"] else 2) + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}


# ------------------------------------------------------------------ inputs
def _pool(pages, case):
    """A pool of pages seen as [pages, slot, head, column], stored slot by slot or head by head."""
    p, h, d = case["page"], case["kv_heads"], case["head_dim"]
    if case["head_major"]:
        return torch.zeros(pages, h, p, d, device="cuda", dtype=torch.bfloat16).permute(0, 2, 1, 3)
    return torch.zeros(pages, p, h, d, device="cuda", dtype=torch.bfloat16)


def _frequencies(case):
    """Radians per position of each pair, in 64 bits (plain numbers: a model's configuration gives them)."""
    out = []
    for i in range(case["rot_dim"] // 2):
        f = case["theta"] ** (-2.0 * i / case["rot_dim"])
        if case["original"]:
            g = min(1.0, max(0.0, (case["original"] * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)))
            f = f * (g + (1 - g) / case["factor"])
        else:
            f = f / case["factor"]
        out.append(f)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = random.Random(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if case["op"] == "rope":
        t, s, nh, nkv, hd, ps = (case[k] for k in ("tokens", "seqs", "heads", "kv_heads", "head_dim", "page"))
        # the newest tokens of each sequence, as one run of rows: sequence i gets the positions first[i] and up
        share = [t * (i + 1) // s - t * i // s for i in range(s)]
        first = [rnd.randrange(0, max(1, case["reach"] - n + 1)) for n in share]
        seq = [i for i in range(s) for _ in range(share[i])]
        pos = [first[i] + j for i in range(s) for j in range(share[i])]
        blocks = -(-case["reach"] // ps)
        touched = sorted({(a, b // ps) for a, b in zip(seq, pos)})
        pages = sum((n - 1) // ps + 2 for n in share) + 3  # wherever the runs begin
        ids = list(range(pages))
        rnd.shuffle(ids)
        table = torch.randint(0, pages, (s, blocks), device="cuda", generator=g, dtype=torch.int32)
        at = torch.tensor(touched, device="cuda")
        table[at[:, 0], at[:, 1]] = torch.tensor(ids[:len(touched)], device="cuda", dtype=torch.int32)
        qkv = normal(t, (nh + 2 * nkv) * hd) * 1.5
        return {"case": case, "qkv": qkv if case["f32"] else qkv.bfloat16(), "k": _pool(pages, case), "v": _pool(pages, case),
                "q_out": torch.zeros(t, nh, hd, device="cuda", dtype=torch.bfloat16), "table": table,
                "q_norm": 1 + 0.1 * normal(hd) if case["norm"] else None, "k_norm": 1 + 0.1 * normal(hd) if case["norm"] else None,
                "freqs": torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda"),
                "seq": torch.tensor(seq, device="cuda", dtype=torch.int32), "pos": torch.tensor(pos, device="cuda", dtype=torch.int32)}
    if case["op"] == "attention":
        n, nh, nkv, hd, ps = (case[k] for k in ("rows", "heads", "kv_heads", "head_dim", "page"))
        lens = _lengths(case)
        need = [-(-x // ps) for x in lens]
        pages = sum(need) + 3
        perm = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        table = torch.zeros(n, -(-case["longest"] // ps), device="cuda", dtype=torch.int32)
        held = torch.arange(table.shape[1], device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
        table[held] = perm[:sum(need)]
        k, v = _pool(pages, case), _pool(pages, case)
        k.copy_(normal(pages, ps, nkv, hd))
        v.copy_(normal(pages, ps, nkv, hd))
        return {"case": case, "q": (normal(n, nh, hd) * 2).bfloat16(), "k": k, "v": v, "table": table,
                "pos": torch.tensor(lens, device="cuda", dtype=torch.int32) - 1,
                "out": torch.zeros(n, nh, hd, device="cuda", dtype=torch.bfloat16)}
    n, vocab = case["rows"], case["vocab"]
    x = normal(n, vocab) * 2.5
    # a few likely tokens in each row, as a trained model has them
    x.scatter_add_(1, torch.randint(0, vocab, (n, 8), device="cuda", generator=g), 4 + 6 * torch.rand(n, 8, device="cuda", generator=g))
    if case["banned"]:
        x[torch.rand(n, vocab, device="cuda", generator=g) < 0.9] = -math.inf
        x[:, rnd.randrange(vocab)] = 3.0
    x = x if case["f32"] else x.bfloat16()
    targets = torch.randint(0, vocab, (n,), device="cuda", generator=g, dtype=torch.int32)
    if n > 3:
        targets[-2:] = -1  # padded rows ask for no token
    e = lambda *s, dtype=torch.float32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    return {"case": case, "logits": x, "targets": targets, "logprob": e(n), "entropy": e(n),
            "top_ids": e(n, case["top"], dtype=torch.int32), "top_logprobs": e(n, case["top"])}


# ------------------------------------------------------------------ one pass
def run(state):
    return {"rope": _rope, "attention": _attention, "logprobs": _logprobs}[state["case"]["op"]](state)


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
    s["k"][page, slot] = _turn(k, cos, sin, rd, c["interleaved"]).bfloat16()
    s["v"][page, slot] = v.bfloat16()
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _turn(x, cos, sin, rd, interleaved):
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else (x[..., :rd // 2], x[..., rd // 2:rd])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, x[..., rd:]), -1)


def _attention(s):
    if own:
        return _own_attention(s)
    c = s["case"]
    n, nh, nkv, hd, ps = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    j = torch.arange(c["longest"], device="cuda")
    page, slot = s["table"].long()[:, j // ps], j % ps
    k, v = s["k"][page, slot].float(), s["v"][page, slot].float()  # [rows, keys, kv heads, columns]
    q = s["q"].float().view(n, nkv, nh // nkv, hd)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1 / math.sqrt(hd))
    x = torch.where((j[None, :] <= s["pos"][:, None])[:, None, None, :], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(o.view(n, nh, hd))
    return s["out"]


def _logprobs(s):
    if own:
        return _own_logprobs(s)
    c = s["case"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    mean = torch.where(e == 0, 0.0, e * (x - top)).sum(-1, keepdim=True) / total
    t = s["targets"].long()
    given = x.gather(1, t.clamp(min=0)[:, None]) - lse
    s["logprob"].copy_(torch.where(t < 0, 0.0, given[:, 0]))
    s["entropy"].copy_((torch.log(total) - mean)[:, 0])
    # one whole number a value, in the values' order and then from the last index to the first: no two are equal
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * (1 << 20) + (c["vocab"] - 1 - torch.arange(c["vocab"], device="cuda"))
    ids = c["vocab"] - 1 - (torch.topk(key, c["top"], dim=1).values & ((1 << 20) - 1))
    s["top_ids"].copy_(ids)
    s["top_logprobs"].copy_(x.gather(1, ids) - lse)
    return {k: s[k] for k in ("logprob", "entropy", "top_ids", "top_logprobs")}


# ------------------------------------------------------------------ the framework's calls
def _iris():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "iris.c_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import iris_cuda
    return iris_cuda


def _own_rope(s):
    if "call" not in s:  # what a program keeps from step to step: the cache's description and the rotation
        ops, c = _iris(), s["case"]
        s["cache"] = ops.KvCache.of(s["k"], s["v"], s["table"])
        scaling = dict(factor=c["factor"], original_len=c["original"], low=1.0, high=32.0)
        s["rope"] = ops.Rope.of(c["rot_dim"], c["theta"], interleaved=c["interleaved"], **scaling)
        s["call"] = ops.rope_append
    c = s["case"]
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    qkv = s["qkv"]
    s["call"](s["cache"], s["rope"], s["q_out"], qkv[:, :nh * hd], qkv[:, nh * hd:(nh + nkv) * hd], qkv[:, (nh + nkv) * hd:],
              s["seq"], s["pos"], heads=nh, q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6,
              stream=torch.cuda.current_stream().cuda_stream)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_attention(s):
    if "call" not in s:  # kept from step to step: the cache's description and the workspace
        ops, c = _iris(), s["case"]
        s["cache"] = ops.KvCache.of(s["k"], s["v"], s["table"])
        s["ws"] = torch.empty(ops.attention_paged_workspace(s["cache"], c["heads"]), device="cuda", dtype=torch.uint8)
        s["call"] = ops.attention_paged
    s["call"](s["cache"], s["out"], s["q"], None, s["pos"], scale=1 / math.sqrt(s["case"]["head_dim"]), workspace=s["ws"],
              stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_logprobs(s):
    if "call" not in s:  # kept from step to step: the workspace
        ops, c = _iris(), s["case"]
        s["ws"] = torch.empty(ops.token_logprobs_workspace(c["rows"], c["vocab"]), device="cuda", dtype=torch.uint8)
        s["call"] = ops.token_logprobs
    s["call"](s["logits"], s["targets"], s["logprob"], s["entropy"], s["top_ids"], s["top_logprobs"], workspace=s["ws"],
              stream=torch.cuda.current_stream().cuda_stream)
    return {k: s[k] for k in ("logprob", "entropy", "top_ids", "top_logprobs")}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        nh, nkv, hd, half = case["heads"], case["kv_heads"], case["head_dim"], case["rot_dim"] // 2
        i = torch.arange(half, device="cuda")
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        turns = torch.polar(torch.ones(case["tokens"], half, dtype=torch.float64, device="cuda"),
                            s["pos"].double().outer(s["freqs"]))[:, None, :]
        heads = s["qkv"].double().view(case["tokens"], -1, hd)

        def rotated(x, w):
            y = x.clone()
            if w is not None:
                y /= ((y ** 2).sum(-1, keepdim=True) / hd + 1e-6).sqrt()
                y *= w.double()
            z = torch.complex(y[..., first], y[..., second]) * turns
            y[..., first], y[..., second] = z.real, z.imag
            return y

        k, v = s["k"].double(), s["v"].double()
        seq, pos = s["seq"].tolist(), s["pos"].tolist()
        table = s["table"].tolist()
        page = torch.tensor([table[a][b // case["page"]] for a, b in zip(seq, pos)], device="cuda")
        slot = torch.tensor([b % case["page"] for b in pos], device="cuda")
        k[page, slot] = rotated(heads[:, nh:nh + nkv], s["k_norm"])
        v[page, slot] = heads[:, nh + nkv:]
        return {"q": rotated(heads[:, :nh], s["q_norm"]), "k": k, "v": v}
    if case["op"] == "attention":
        n, nh, nkv, hd, ps = (case[k] for k in ("rows", "heads", "kv_heads", "head_dim", "page"))
        out = torch.zeros(n, nh, hd, dtype=torch.float64, device="cuda")
        for r, last in enumerate(s["pos"].tolist()):
            if last < 0:
                continue
            held = s["table"][r, :last // ps + 1].long()
            k = s["k"][held].reshape(-1, nkv, hd)[:last + 1].double()
            v = s["v"][held].reshape(-1, nkv, hd)[:last + 1].double()
            q = s["q"][r].double().view(nkv, nh // nkv, hd)
            p = torch.softmax(torch.einsum("ghd,lgd->ghl", q, k) / math.sqrt(hd), -1)
            out[r] = torch.einsum("ghl,lgd->ghd", p, v).reshape(nh, hd)
        return out
    n, parts = case["rows"], ([], [], [], [])
    for lo in range(0, n, 64):  # a few rows at a time: 64 bits of all of them is much memory
        x = s["logits"][lo:lo + 64].double()
        logp = torch.log_softmax(x, -1)
        t = s["targets"][lo:lo + 64].long()
        parts[0].append(logp[torch.arange(len(t), device="cuda"), t.clamp(min=0)].masked_fill(t < 0, 0.0))
        parts[1].append(-torch.xlogy(logp.exp(), logp.exp()).sum(-1))
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        parts[2].append(ids.int())
        parts[3].append(logp.gather(1, ids))
    return dict(zip(("logprob", "entropy", "top_ids", "top_logprobs"), (torch.cat(p) for p in parts)))
