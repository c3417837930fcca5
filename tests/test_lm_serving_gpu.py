"""Sampling, the 8-bit cache and 4-bit weights on the GPU against plain 64-bit forms.

Tolerances, derived from the operators' arithmetic (u = 2^-24, half an f32 step;
2^-8 half a bf16 step, 2^-11 an f16, 2^-4 an e4m3 step, relative):

sample_tokens: ids and counts equal.  Weights and sums are 64-bit on both sides, off by
  some 2^-40 at most, so that a random number has to hit a border to 12 digits for another
  token; log probabilities are rounded to f32 once: u, and 2^-40 for what comes before.
rope_append8: K goes through the f32 arithmetic of rope_append, off by 2^-18 (|a| + |b|) of
  the pair, and one rounding to e4m3 at the scale s: 2^-4 of the value, or half the least
  step, 2^-10 s.  V and what is rounded again: equal to one rounding.  A scale may differ
  from the 64-bit one only where the largest value is within 2^-17 of 448 s.
attention_paged8: as attention_paged (2^-8 of the value and, times A = sum p |v|: 4 hd u S
  for the scores, len u, 2^-14 for the exponential), with weights in 11 bits: 2^-11 A, and
  none under 2^-25 of the largest weight times scale W: len 2^-25 448 W in the result.
  Queries under 2^-29 of the head's largest lose bits: 2^-39 of it, times a key's sum of
  magnitudes, in the score.
linear4: products of 4 (8) and 8 bits are exact; a warp adds up k / 8 of them, tensor-core
  sums drop bits instead of rounding, 2 u each, then a few additions and a product for each
  group: (k / 8 + 100) 2 u of sum |q - z| s |x|.  bf16: and 2^-8 of the value.
"""
import math

import numpy as np
import pytest

from test_lm_ops_gpu import BF, U, gen, i32, rotate64, stream

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
E4 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(iris):
    return iris


# ------------------------------------------------------------------ sample_tokens
def sample64(x, t, k, p, mp, u):
    """One row: (id, log probability, kept)."""
    x = x.astype(np.float64)
    if np.isnan(t) or np.isnan(x).any() or np.isposinf(x).any() or not np.isfinite(x).any():
        return -1, -math.inf, 0
    order = np.argsort(-x, kind="stable")
    order = order[np.isfinite(x[order])]
    if t <= 0 or p <= 0:
        return int(order[0]), 0.0, 1
    w = np.exp((x[order] - x[order[0]]) / t)
    n = len(order)
    if mp > 0:
        # w >= min_p; in logarithms, since e^(-1e-40), which is under 1, is 1 in 64 bits
        n = int(((x[order] - x[order[0]]) / t >= math.log(min(mp, 1.0))).sum())
    if 0 < k < len(x):
        n = min(n, k)
    c = np.cumsum(w[:n])
    if p < 1:
        n = max(1, int((c - w[:n] < p * c[-1]).sum()))
    u = min(max(u, 0.0), 1 - 2.0 ** -53) if u == u else 0.0
    at = min(int((c[:n] <= u * c[n - 1]).sum()), int((w[:n] > 0).sum()) - 1)
    return int(order[at]), math.log(w[at] / c[n - 1]) if w[at] > 0 else -math.inf, n


def check_samples(ops, logits, settings, uniform, **kw):
    """settings: rows of (temperature, top_k, top_p, min_p)."""
    n = logits.shape[0]
    t, k, p, mp = (list(c) for c in zip(*settings))
    f = lambda v: torch.tensor(v, device="cuda", dtype=torch.float32)  # noqa: E731
    ids, kept = i32([-7] * n), i32([-7] * n)
    lp = torch.full((n,), 7.0, device="cuda")
    ut = torch.tensor(uniform, device="cuda", dtype=torch.float64)
    args = dict(temperature=f(t), top_k=i32(k), top_p=f(p), min_p=f(mp))
    ops.sample_tokens(logits, ut, ids, logprobs=lp, kept=kept, stream=stream(), **args)
    again = torch.zeros_like(ids), torch.zeros_like(lp)
    ops.sample_tokens(logits, ut, again[0], logprobs=again[1], stream=stream(), **args)
    torch.cuda.synchronize()
    assert torch.equal(ids, again[0]) and torch.equal(lp, again[1])
    x = logits.float().cpu().numpy()
    t, p, mp = (np.float32(v).astype(np.float64) for v in (t, p, mp))
    for r in range(n):
        want = sample64(x[r], t[r], k[r], p[r], mp[r], uniform[r])
        got = int(ids[r]), float(lp[r]), int(kept[r])
        assert got[0] == want[0] and got[2] == want[2], (r, settings[r], uniform[r], got, want)
        assert got[1] == want[1] or abs(got[1] - want[1]) <= U * abs(want[1]) + 2.0 ** -40, (r, got, want)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 0.9, 0.05), (1.0, 1, 1.0, 0.0),
            (1.0, 50, 1.0, 0.1), (0.5, 300, 0.99, 0.0), (1.0, 2000, 0.999, 0.0), (2.0, 5000, 1.0, 0.0), (1.0, 0, 1.0, 0.001),
            (5.0, 0, 0.5, 0.0), (0.01, 0, 1.0, 0.0), (1.0, 256, 1.0, 0.0), (1.0, 257, 1.0, 0.0), (1.0, 512, 0.7, 0.0),
            (-1.0, 3, 0.5, 0.5), (1.0, 0, 0.0, 0.0), (1.0, -4, -1.0, -1.0), (1.0, 0, 1e-9, 0.0), (100.0, 0, 0.9, 0.0),
            (1.0, 10 ** 9, 2.0, 1.0), (1.0, 700, 1.0, 2.0), (1e6, 0, 0.6, 0.0), (1e-30, 0, 0.9, 0.0), (1.0, 0, 0.99999, 1e-6)]


@pytest.mark.parametrize("f32", (True, False))
@pytest.mark.parametrize("vocab,pad", [(1, 0), (2, 1), (7, 0), (33, 2), (100, 3), (1000, 0), (5003, 5), (16411, 1), (50021, 1), (151936, 0)])
def test_sample_tokens(ops, vocab, pad, f32):
    n = len(SETTINGS)
    x = torch.randn(n, vocab + pad, device="cuda", generator=gen(vocab)) * 2.5
    x.scatter_add_(1, torch.randint(0, vocab, (n, 4), device="cuda", generator=gen(vocab + 1)),
                   6 * torch.rand(n, 4, device="cuda", generator=gen(vocab + 2)))
    x = (x if f32 else x.bfloat16())[:, :vocab]  # rows at any alignment of the elements
    check_samples(ops, x, SETTINGS, np.random.default_rng(vocab).random(n).tolist())


@pytest.mark.parametrize("vocab", (257, 20000, 151936))
@pytest.mark.parametrize("kind", ("equal", "two", "lowest", "masked", "steps", "wide", "zeros"))
def test_sample_tokens_ties_and_masks(ops, vocab, kind):
    """Many equal logits, so that the id decides; masks of -inf and of the type's lowest value; +0 and -0."""
    n, rng = len(SETTINGS), np.random.default_rng(vocab)
    g = gen(vocab)
    x = torch.zeros(n, vocab, device="cuda")
    if kind == "two":
        x[torch.rand(n, vocab, device="cuda", generator=g) < 0.5] = 1.0
    if kind == "lowest":
        x = torch.randn(n, vocab, device="cuda", generator=g) * 3
        x[torch.rand(n, vocab, device="cuda", generator=g) < 0.9] = torch.finfo(torch.float32).min
    if kind == "masked":
        x = torch.randn(n, vocab, device="cuda", generator=g) * 3
        x[torch.rand(n, vocab, device="cuda", generator=g) < 0.995] = -math.inf
        x[3::7] = -math.inf
        x[3::7, vocab // 2] = -5.0
    if kind == "steps":
        x = torch.round(torch.randn(n, vocab, device="cuda", generator=g) * 2) / 2
    if kind == "wide":
        x = torch.randn(n, vocab, device="cuda", generator=g) * 1e4
    if kind == "zeros":
        x[torch.rand(n, vocab, device="cuda", generator=g) < 0.5] = -0.0
        x[:, ::3] = -1e-40
    check_samples(ops, x, SETTINGS, rng.random(n).tolist())


def test_sample_tokens_ends_of_the_line(ops):
    """The smallest and largest random numbers, ones outside [0, 1) and NaN."""
    us = [0.0, 2.0 ** -60, 0.5, 1 - 2.0 ** -53, 1.0, 7.0, -1.0, math.nan, math.inf]
    for vocab in (5, 5000, 151936):
        x = torch.randn(len(us), vocab, device="cuda", generator=gen(vocab))
        for s in ((1.0, 0, 1.0, 0.0), (1.0, 40, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 1000, 0.9, 0.01)):
            check_samples(ops, x, [s] * len(us), us)


def test_sample_tokens_rows_without_an_answer(ops):
    inf, nan = math.inf, math.nan
    for vocab in (9, 40000):
        x = torch.randn(8, vocab, device="cuda", generator=gen(3))
        x[0] = -inf
        x[1, vocab // 2] = nan
        x[2, vocab - 1] = inf
        x[3] = -inf
        x[3, 4] = -3.0e38
        x[4, 0] = -nan
        x[5] = torch.finfo(torch.float32).min
        for t in (1.0, 0.0):
            check_samples(ops, x, [(t, 0, 1.0, 0.0), (t, 5, 0.5, 0.0)] * 4, [0.3] * 8)
        # a setting that is not a number: of the temperature there is no answer, of the others it is as none
        check_samples(ops, x, [(nan, 0, 1.0, 0.0)] * 8, [0.3] * 8)
        check_samples(ops, x, [(1.0, 3, nan, nan)] * 8, [0.3] * 8)
        check_samples(ops, x, [(inf, 0, 0.5, 0.0), (inf, 0, 1.0, 0.5)] * 4, [0.3] * 8)


def test_sample_tokens_without_settings(ops):
    x = torch.randn(5, 3000, device="cuda", generator=gen(8))
    u = torch.rand(5, device="cuda", dtype=torch.float64, generator=gen(9))
    ids = i32([0] * 5)
    ops.sample_tokens(x, u, ids, stream=stream())
    torch.cuda.synchronize()
    want = [sample64(r, 1.0, 0, 1.0, 0.0, float(v))[0] for r, v in zip(x.cpu().numpy(), u)]
    assert ids.tolist() == want


@pytest.mark.parametrize("f32", (True, False))
def test_sample_tokens_more_logits_than_fit_on_chip(ops, f32):
    vocab = 400003 if f32 else 750001
    x = torch.randn(3, vocab + 1, device="cuda", generator=gen(1)) * 2
    x = (x if f32 else x.bfloat16())[:, 1:]
    for s in ((1.0, 0, 1.0, 0.0), (1.0, 30, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 3000, 1.0, 0.0), (0.0, 0, 1.0, 0.0)):
        check_samples(ops, x, [s] * 3, [0.1, 0.77, 0.9999])


def test_sample_tokens_follows_the_distribution(ops):
    """Evenly spread random numbers over one row: every token as often as its probability says, to one draw at each end."""
    vocab, n = 60, 4000
    x = (torch.randn(vocab, generator=torch.Generator().manual_seed(4)) * 2).to("cuda").expand(n, vocab).contiguous()
    u = (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5) / n
    ids = torch.zeros(n, device="cuda", dtype=torch.int32)
    ops.sample_tokens(x, u, ids, stream=stream())
    torch.cuda.synchronize()
    count = torch.bincount(ids.long(), minlength=vocab).double().cpu()
    assert ((count - n * torch.softmax(x[0].double().cpu(), 0)).abs() <= 1.0).all()


@pytest.mark.parametrize("top_p", (None, 0.75))
def test_sample_tokens_a_million_draws(ops, top_p):
    """Draws all along one row's line, against a search in its 64-bit sums.  A random number within 2^-30 of a token's end (the
    two sums are within 5000 * 2^-52 of each other) may go either way."""
    vocab, rows = 5000, 8192
    x = torch.randn(vocab, generator=torch.Generator().manual_seed(41)).cuda() * 2
    line = torch.argsort(x.double(), descending=True, stable=True)
    w = torch.exp(x.double() - x.double().max())[line]
    if top_p:
        w = w[:int((torch.cumsum(w, 0) - w < np.float64(np.float32(top_p)) * w.sum()).sum())]
    end = torch.cumsum(w, 0) / w.sum()
    logits, ids = x.repeat(rows, 1), torch.empty(rows, dtype=torch.int32, device="cuda")
    p = None if top_p is None else torch.full((rows,), top_p, device="cuda")
    wrong = 0
    for i in range(128):
        u = torch.rand(rows, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
        ops.sample_tokens(logits, u, ids, top_p=p)
        at = torch.searchsorted(end, u, right=True).clamp(max=w.numel() - 1)
        near = torch.minimum((end[at] - u).abs(), (end[(at - 1).clamp(min=0)] - u).abs()) < 2.0 ** -30
        wrong += int(((ids.long() != line[at]) & ~near).sum())
    assert wrong == 0



# ------------------------------------------------------------------ the 8-bit cache
def pool8(pages, page, heads, d, hm, seed, block):
    """A pool with earlier values and their exponents."""
    g = gen(seed)
    shape = (pages, heads, page, d) if hm else (pages, page, heads, d)
    b = torch.randint(0, 256, shape, device="cuda", generator=g, dtype=torch.uint8)
    b[(b & 0x7F) == 0x7F] = 0x30  # (no NaN)
    e = torch.randint(118, 126, (pages, heads, page // block), device="cuda", generator=g, dtype=torch.uint8).permute(0, 2, 1)
    return (b.permute(0, 2, 1, 3) if hm else b).view(E4), e if hm else e.contiguous()


def exponent64(top):
    """Exponents (biased) of magnitudes [...], and whether another one is as good after f32 arithmetic."""
    top = np.maximum(np.asarray(top), 448 * 2.0 ** -60)
    m, e = np.frexp(top / 448)          # top / 448 = m 2^e, 1/2 <= m < 1
    e = np.where(m == 0.5, e - 1, e)
    edge = (m >= 1 - 2.0 ** -17) | (m <= 0.5 * (1 + 2.0 ** -17))
    return np.minimum(e + 127, 187), edge & (top > 448 * 2.0 ** -60)


APPEND = [  # tokens, heads, kv heads, d, rot, interleaved, page, block, head major, f32, norm, sequences, shuffled
    (1, 32, 8, 128, 128, False, 16, 16, False, True, True, 1, False),
    (3, 4, 2, 128, 128, False, 16, 8, True, False, True, 3, False),
    (37, 6, 2, 64, 64, True, 21, 7, False, False, False, 2, True),
    (130, 7, 1, 128, 96, False, 1, 1, True, True, False, 3, False),
    (65, 5, 5, 256, 64, True, 24, 24, False, True, True, 3, True),
    (600, 16, 4, 128, 16, True, 64, 32, True, False, False, 3, False),
    (300, 0, 3, 128, 128, False, 128, 128, False, False, True, 2, True),
    (21, 4, 20, 64, 0, False, 16, 16, False, True, True, 3, False),
    (1200, 2, 1, 256, 256, False, 100, 50, True, True, True, 3, True),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c[:8])))
def test_rope_append8(ops, case):
    t, nh, nkv, d, rd, inter, page, block, hm, f32, norm, seqs, shuffled = case
    g, rng = gen(t), np.random.default_rng(t)
    qkv = torch.randn(t, (nh + 2 * nkv) * d + 8, device="cuda", generator=g) * 2
    qkv *= torch.exp2(torch.randint(-9, 6, (t, 1), device="cuda", generator=g).float())  # scales that grow and that do not
    qkv = qkv if f32 else qkv.bfloat16()
    q, k, v = (qkv[:, a * d:b * d] for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
    # runs of positions of each sequence that begin anywhere in a block
    seq = np.sort(rng.integers(0, seqs, t))
    pos = np.concatenate([rng.integers(0, 3 * page) + np.arange((seq == s).sum()) for s in range(seqs)])
    if shuffled:
        order = rng.permutation(t)
        seq, pos = seq[order], pos[order]
    blocks = int(pos.max()) // page + 2
    pages = seqs * blocks + 2
    table = torch.tensor(rng.permutation(pages)[:seqs * blocks].reshape(seqs, blocks), dtype=torch.int32, device="cuda")
    if t > 8:
        seq[1], seq[2], pos[3] = -1, seqs, -5                # padding
        table[seq[5], pos[5] // page] = pages                # a page outside the pool
    (kp, ke), (vp, ve) = pool8(pages, page, nkv, d, hm, 1, block), pool8(pages, page, nkv, d, hm, 2, block)
    before = [x.clone() for x in (kp.view(torch.uint8), ke, vp.view(torch.uint8), ve)]
    qo = torch.full((t, max(nh, 1) * d + 16), 7.0, device="cuda", dtype=torch.bfloat16)[:, :nh * d]
    qn = 1 + 0.2 * torch.randn(d, device="cuda", generator=g) if norm else None
    kn = 1 + 0.2 * torch.randn(d, device="cuda", generator=g) if norm else None
    rope = ops.Rope.of(rd, 1e4, interleaved=inter) if rd else None
    freqs = [x / 2.0 ** 64 * 2 * math.pi for x in rope.turns[:rd // 2]] if rd else []
    cache = ops.KvCache8.of(kp, vp, ke, ve, table)
    ops.rope_append8(cache, rope, qo if nh else None, q if nh else None, k, v, i32(seq), i32(pos), heads=nh, q_norm=qn, k_norm=kn,
                     stream=stream())
    torch.cuda.synchronize()
    P = torch.tensor(pos.clip(0))
    live = (seq >= 0) & (seq < seqs) & (pos >= 0)
    if nh:
        want, size = rotate64(q.reshape(t, nh, d), P, freqs, inter, 1.0, qn)
        err = (qo.reshape(t, nh, d).double().cpu() - want).abs()[live]
        assert (err <= BF * want[live].abs() + 2.0 ** -18 * size[live]).all()
        assert (qo[~torch.tensor(live)] == 7).all()
    tab = table.cpu().numpy()
    groups = {}
    for i in np.flatnonzero(live):
        p = int(tab[seq[i], pos[i] // page])
        if 0 <= p < pages:
            groups.setdefault((p, int(pos[i] % page) // block), {})[int(pos[i] % page)] = int(i)
    assert groups
    wk, size = rotate64(k.reshape(t, nkv, d), P, freqs, inter, 1.0, kn)
    wv = v.reshape(t, nkv, d).double().cpu()
    for name, pool, exps, was, was_e, want, slack in (("k", kp, ke, before[0], before[1], wk, size), ("v", vp, ve, before[2], before[3], wv, None)):
        got, got_e = pool.float().cpu().double(), exps.cpu().numpy().astype(int)
        old, old_e = was.cpu(), was_e.cpu().numpy().astype(int)
        touched = torch.zeros(pages, page, dtype=torch.bool)
        for (p, b), slots in groups.items():
            rows = list(slots.values())
            fresh = b * block in slots
            need, edge = exponent64(want[rows].abs().amax((0, 2)).numpy())
            e = got_e[p, b]
            target = need if fresh else np.maximum(need, old_e[p, b])
            assert ((e == target) | (edge & (abs(e - need) <= 1) & (slack is not None))).all(), (name, p, b, e, target)
            touched[p, b * block:(b + 1) * block] = True
            s = torch.tensor(2.0 ** (e - 127.0))[:, None]
            for slot in range(b * block, (b + 1) * block):
                if slot in slots:
                    w = want[slots[slot]]
                    if slack is None:
                        assert torch.equal(got[p, slot], (w / s).float().to(E4).double()), (name, p, slot)
                    else:
                        err = (got[p, slot] * s - w).abs()
                        assert (err <= 2.0 ** -4 * w.abs() + 2.0 ** -10 * s + 2 * 2.0 ** -18 * slack[slots[slot]]).all(), (name, p, slot)
                else:
                    x = old[p, slot].view(E4).float()
                    if not fresh:
                        x = (x * torch.tensor(2.0 ** (old_e[p, b] - e))[:, None]).float().to(E4).float()
                    assert torch.equal(got[p, slot], x.double()), (name, p, slot)
        assert torch.equal(pool.view(torch.uint8).cpu()[~touched], old[~touched])
        keep = ~touched[:, ::block]
        assert np.array_equal(got_e[keep.numpy()], old_e[keep.numpy()])


def test_rope_append8_one_token_at_a_time(ops):
    """A sequence fed token by token holds, at the last scale, what it would hold if fed whole, but for what was rounded at a
    smaller scale on the way: at most a step of the least magnitudes."""
    d, nkv, page, block, n = 128, 2, 32, 16, 77
    x = torch.randn(n, nkv * d, device="cuda", generator=gen(3)) * torch.exp2(torch.arange(n, device="cuda")[:, None] % 16 / 2.0)
    caches = []
    for step in (1, n, 5):
        pools = [torch.zeros(3, page, nkv, d, device="cuda", dtype=torch.uint8).view(E4) for _ in range(2)]
        exps = [torch.zeros(3, page // block, nkv, device="cuda", dtype=torch.uint8) for _ in range(2)]
        cache = ops.KvCache8.of(*pools, *exps, i32([[2, 0, 1]]))
        for i in range(0, n, step):
            m = min(step, n - i)
            ops.rope_append8(cache, None, None, None, x[i:i + m], x[i:i + m], i32([0] * m), i32(range(i, i + m)), heads=0, stream=stream())
        torch.cuda.synchronize()
        caches.append((pools, exps))
    (p1, e1), (pn, en), (p5, e5) = caches
    for a, b in ((p1, e1), (p5, e5)):
        for i in range(2):
            assert torch.equal(b[i], en[i])
            # twice rounded: each to half a step, 2^-4 of the value or 2^-10 at the last scale
            err = (a[i].float() - pn[i].float()).abs()
            assert (err <= 2.0 ** -3 * pn[i].float().abs() + 2.0 ** -9).all()


@pytest.mark.parametrize("n", (7, 1203))
def test_rope_append8_numbers_at_any_address(ops, n):
    """Sequence numbers that do not start at 16 bytes, tokens in any order: the same bytes."""
    d, nkv, page, block, seqs = 64, 3, 32, 16, 5
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, nkv * d, device="cuda", generator=gen(n))
    blocks = (n + seqs - 1) // seqs // page + 1
    order = torch.randperm(n, generator=g)
    seq, pos = (order % seqs).int(), (order // seqs).int()
    got = []
    for at in (0, 1, 3):
        pools = [torch.zeros(seqs * blocks, page, nkv, d, device="cuda", dtype=torch.uint8).view(E4) for _ in range(2)]
        exps = [torch.zeros(seqs * blocks, page // block, nkv, device="cuda", dtype=torch.uint8) for _ in range(2)]
        cache = ops.KvCache8.of(*pools, *exps, torch.arange(seqs * blocks, dtype=torch.int32).view(seqs, blocks).cuda())
        s = torch.full((n + 4,), -1, dtype=torch.int32, device="cuda")
        s[at:at + n] = seq.cuda()
        ops.rope_append8(cache, None, None, None, x, x, s[at:at + n], pos.cuda(), heads=0, stream=stream())
        torch.cuda.synchronize()
        got.append([p.view(torch.uint8) for p in pools] + exps)
    assert got[0][0].any()
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


def test_rope_append8_odd_values(ops):
    """Infinities and NaN are held as NaN and do not move the scale; zeros; magnitudes past the range."""
    d, page = 64, 8
    x = torch.randn(4, d, device="cuda", generator=gen(1))
    x[0, 3], x[1, 4], x[2, 5] = math.inf, -math.inf, math.nan
    pools = [torch.zeros(2, page, 1, d, device="cuda", dtype=torch.uint8).view(E4) for _ in range(2)]
    exps = [torch.zeros(2, 1, 1, device="cuda", dtype=torch.uint8) for _ in range(2)]
    cache = ops.KvCache8.of(*pools, *exps, i32([[0, 1]]))
    big = torch.full_like(x, 3e38)
    ops.rope_append8(cache, None, None, None, x, big, i32([0] * 4), i32([0, 1, 3, 2]), heads=0, stream=stream())
    ops.rope_append8(cache, None, None, None, torch.zeros_like(x), x[3:].expand(4, d).contiguous() * 1e-30, i32([0] * 4), i32(range(8, 12)), heads=0,
                     stream=stream())
    torch.cuda.synchronize()
    k, v = (p.float().cpu() for p in pools)
    fin = torch.where(torch.isfinite(x), x, 0.0).abs().max()
    assert int(exps[0][0]) == exponent64(float(fin))[0]
    s = 2.0 ** (int(exps[0][0]) - 127)
    for slot, row in ((0, 0), (1, 1), (2, 3), (3, 2)):
        want = torch.where(torch.isfinite(x[row]), x[row], math.nan).cpu()
        assert torch.equal(torch.nan_to_num(k[0, slot, 0], 777.0), torch.nan_to_num((want / s).to(E4).float(), 777.0))
    assert int(exps[1][0]) == 187 and (v[0, :4] == 448).all()
    assert int(exps[0][1]) == 67 and (k[1, :4] == 0).all() and int(exps[1][1]) == 67
    assert (v[1, :4].abs() <= 2.0 ** -9).all()


def values8(pool, exps, block):
    e = exps.cpu().double().repeat_interleave(block, 1) - 127
    return pool.float().cpu().double() * (2.0 ** e)[..., None]


def attention8_64(q, k, v, vs, scale):
    """q [heads, d], k / v [len, kv heads, d], vs [len, kv heads] scales of the values -> (out, tolerance) [heads, d]."""
    nh, d = q.shape
    n, nkv = k.shape[:2]
    if not n:
        return torch.zeros(nh, d, dtype=torch.float64), torch.zeros(nh, d, dtype=torch.float64)
    g = nh // nkv
    q = q.double().cpu()
    k, v = (x.repeat_interleave(g, 1).transpose(0, 1) for x in (k, v))
    vs = vs.repeat_interleave(g, 1).transpose(0, 1)
    p = torch.softmax(scale * torch.einsum("hd,hld->hl", q, k), -1)
    s = abs(scale) * torch.einsum("hd,hld->hl", q.abs(), k.abs()).amax(-1)
    lost = abs(scale) * 2.0 ** -39 * q.abs().amax(-1) * k.abs().sum(-1).amax(-1)
    out, a = torch.einsum("hl,hld->hd", p, v), torch.einsum("hl,hld->hd", p, v.abs())
    w = (p * vs).amax(-1)
    return out, BF * out.abs() + (4 * d * U * s + n * U + 2.0 ** -14 + 2.0 ** -11 + 2 * lost)[:, None] * a + (n * 2.0 ** -25 * 448 * w)[:, None]


def check_attention8(ops, lens, news, nh, nkv, d, page, block, hm, seed, spread=8, shuffle=False, seq_none=False, extra_seqs=0):
    """Sequences of `lens` keys, the newest `news[i]` of them as rows (one that is 0: a row that sees nothing)."""
    g = gen(seed)
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    (kp, ke), (vp, ve) = pool8(pages, page, nkv, d, hm, seed, block), pool8(pages, page, nkv, d, hm, seed + 1, block)
    for p in (kp, vp):  # values as a cache has them, not every bit pattern alike
        p.copy_((torch.randn(p.shape, device="cuda", generator=g) * 80).clamp(-440, 440).to(E4))
    for e in (ke, ve):
        e.copy_(torch.randint(122 - spread // 2, 123 + spread // 2, e.shape, device="cuda", generator=g, dtype=torch.uint8))
    ids = rng.permutation(pages)[:sum(need)]
    table = torch.full((len(lens) + extra_seqs, max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
        at += m
    seq = [i for i, m in enumerate(news) for _ in range(m)]
    pos = [lens[i] - m + j for i, m in enumerate(news) for j in range(m)]
    if shuffle:
        order = rng.permutation(len(seq))
        seq, pos = [seq[i] for i in order], [pos[i] for i in order]
    rows = len(seq)
    table = table.to("cuda")
    cache = ops.KvCache8.of(kp, vp, ke, ve, table)
    q = (torch.randn(rows, nh, d, device="cuda", generator=g) * 1.5).bfloat16()
    out = torch.full((rows, nh * d + 8), 9.0, device="cuda", dtype=torch.bfloat16)[:, :nh * d]
    ws = torch.empty(ops.attention_paged8_workspace(cache, nh), device="cuda", dtype=torch.uint8)
    scale = 1 / math.sqrt(d) / 8
    for _ in range(2):
        ops.attention_paged8(cache, out, q, None if seq_none else i32(seq), i32(pos), scale=scale, workspace=ws, stream=stream())
        first = out.clone() if _ == 0 else first
    torch.cuda.synchronize()
    assert torch.equal(first, out)
    kv, vv = values8(kp, ke, block), values8(vp, ve, block)
    vs = 2.0 ** (ve.cpu().double().repeat_interleave(block, 1) - 127)
    for r in range(rows):
        n = pos[r] + 1
        held = table[seq[r], :-(-n // page)].long().cpu() if n > 0 else torch.zeros(0, dtype=torch.long)
        cut = lambda x: x[held].flatten(0, 1)[:n]  # noqa: E731
        want, tol = attention8_64(q[r], cut(kv), cut(vv), cut(vs), scale)
        err = (out[r].view(nh, d).double().cpu() - want).abs()
        assert (err <= tol).all(), (r, n, float((err - tol).max()), float(err.max()))


ATTEND = [  # lens, new rows, heads, kv heads, d, page, block, head major
    ([1], [1], 4, 4, 128, 16, 16, False),
    ([0], [1], 8, 2, 64, 16, 8, True),
    ([512], [1], 32, 8, 128, 16, 16, False),
    ([3000], [1], 8, 2, 128, 64, 64, True),
    ([70, 0, 1, 255, 256, 257, 64, 63, 65], [1] * 9, 14, 2, 64, 24, 8, True),
    ([333, 20, 900], [1] * 3, 16, 1, 256, 16, 1, False),
    ([333, 20, 900], [1] * 3, 6, 2, 256, 100, 50, True),
    ([40, 1300, 77, 5], [1] * 4, 20, 2, 128, 1, 1, False),
    ([2000, 2001, 3], [1] * 3, 16, 1, 128, 32, 32, True),
    ([150, 130], [100, 60], 8, 2, 128, 16, 16, False),
    ([64], [64], 4, 1, 64, 24, 24, True),
    ([300], [300], 32, 8, 128, 16, 8, False),
    ([200], [150], 12, 1, 256, 100, 25, False),
    ([513, 200], [5, 9], 16, 1, 64, 7, 7, True),
    ([600, 300], [4, 8], 4, 2, 256, 16, 16, False),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{sum(c[1])}-" + "-".join(map(str, c[2:7])))
def test_attention_paged8(ops, case):
    lens, news, nh, nkv, d, page, block, hm = case
    check_attention8(ops, lens, news, nh, nkv, d, page, block, hm, sum(lens) + d)


@pytest.mark.parametrize("d,nh,nkv", [(64, 14, 2), (128, 8, 2), (256, 4, 2), (128, 16, 1)])
def test_attention_paged8_many_rows(ops, d, nh, nkv):
    """More rows than blocks run at once: equal shares of all tiles, cut units joined."""
    rng = np.random.default_rng(d)
    lens = [int(x) for x in rng.integers(0, 700, 180)]
    check_attention8(ops, lens, [1] * 180, nh, nkv, d, 16, 16, False, d)
    check_attention8(ops, lens, [1] * 180, nh, nkv, d, 32, 4, True, d + 1, seq_none=True)


@pytest.mark.parametrize("d", (64, 128, 256))
def test_attention_paged8_runs(ops, d):
    """Several rows of a sequence: in runs, in disorder, and beside single tokens."""
    check_attention8(ops, [500, 90, 260], [120, 90, 1], 8, 2, d, 16, 16, False, d)
    check_attention8(ops, [140, 90], [50, 60], 8, 2, d, 16, 2, True, d + 1, shuffle=True)
    check_attention8(ops, [1030], [900], 4, 2, d, 64, 64, False, d + 2)


def test_attention_paged8_scales_far_apart(ops):
    check_attention8(ops, [400, 33], [1, 1], 8, 2, 128, 16, 4, False, 5, spread=60)
    check_attention8(ops, [200], [120], 8, 2, 128, 16, 4, False, 6, spread=60)


def one_sequence8(ops, n, d, block, page=16, nkv=1):
    pages = -(-n // page) + 1
    k, v = (torch.randn(pages, page, nkv, d, device="cuda", generator=gen(s)).to(E4) for s in (1, 2))
    e = [torch.full((pages, page // block, nkv), 127, device="cuda", dtype=torch.uint8) for _ in range(2)]
    table = i32([list(range(pages))])
    return k, v, *e, table


@pytest.mark.parametrize("new", (1, 80))
def test_attention_paged8_not_finite(ops, new):
    """NaN in a value shows in its column of the rows that see it, in a key in all of their heads on it; in no other row."""
    n, d, block = 160, 128, 8
    k, v, ke, ve, table = one_sequence8(ops, n, d, block)
    byte = v.view(torch.uint8)
    byte[120 // 16, 120 % 16, 0, 5] = 0x7F
    byte[n // 16, n % 16, 0, 7] = 0xFF  # behind the last key
    k.view(torch.uint8)[n // 16, n % 16, 0, 3] = 0x7F
    q = torch.randn(new, 4, d, device="cuda", generator=gen(3)).bfloat16()
    q[new - 1, 2, 0] = math.nan
    pos = list(range(n - new, n))
    out = torch.zeros_like(q)
    cache = ops.KvCache8.of(k, v, ke, ve, table)
    ws = torch.empty(ops.attention_paged8_workspace(cache, 4), device="cuda", dtype=torch.uint8)

    def run():
        ops.attention_paged8(cache, out, q, i32([0] * new), i32(pos), scale=0.1, workspace=ws, stream=stream())
        torch.cuda.synchronize()
        return torch.isnan(out).cpu()

    bad = torch.zeros(new, 4, d, dtype=torch.bool)
    bad[[p >= 120 for p in pos], :, 5] = True
    bad[new - 1, 2] = True
    assert torch.equal(run(), bad)
    k.view(torch.uint8)[130 // 16, 130 % 16, 0, 9] = 0xFF
    bad[[p >= 130 for p in pos]] = True
    assert torch.equal(run(), bad)


def test_attention_paged8_queries_of_any_size(ops):
    n, d = 100, 128
    k, v, ke, ve, table = one_sequence8(ops, n, d, 16)
    cache = ops.KvCache8.of(k, v, ke, ve, table)
    ws = torch.empty(ops.attention_paged8_workspace(cache, 8), device="cuda", dtype=torch.uint8)
    base = torch.randn(1, 8, d, device="cuda", generator=gen(4))
    out = torch.zeros(1, 8, d, device="cuda", dtype=torch.bfloat16)
    for size in (1e-30, 1e-4, 1.0, 1e6, 1e30):
        q = (base * size).bfloat16()
        ops.attention_paged8(cache, out, q, i32([0]), i32([n - 1]), scale=0.05 / size, workspace=ws, stream=stream())
        torch.cuda.synchronize()
        kv, vv = (values8(p, e, 16).flatten(0, 1)[:n] for p, e in ((k, ke), (v, ve)))
        want, tol = attention8_64(q[0], kv, vv, torch.ones(n, 1, dtype=torch.float64), float(np.float32(0.05 / size)))
        assert ((out[0].double().cpu() - want).abs() <= tol).all(), size


def test_attention_paged8_leaves_other_rows(ops):
    k, v, ke, ve, table = one_sequence8(ops, 64, 64, 16)
    cache = ops.KvCache8.of(k, v, ke, ve, table)
    ws = torch.empty(ops.attention_paged8_workspace(cache, 2), device="cuda", dtype=torch.uint8)
    q = torch.ones(6, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.full((7, 2, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    ops.attention_paged8(cache, out[:6], q, i32([0, -1, 1, 0, 0, 7]), i32([3, 3, 3, -1, 2 ** 31 - 1, 3]), scale=1.0, workspace=ws,
                         stream=stream())
    torch.cuda.synchronize()
    o = out.float().cpu()
    assert (o[[1, 2, 5, 6]] == 3).all() and (o[3] == 0).all() and torch.isfinite(o).all() and (o[[0, 4]] != 3).all()


def test_a_pool_of_4_gigabytes(ops):
    """Offsets past 32 bits in a long cache."""
    d, nkv, page, block = 128, 8, 64, 64
    pages = 2 ** 32 // (page * nkv * d) + 3
    k = torch.zeros(pages, page, nkv, d, device="cuda", dtype=torch.uint8).view(E4)
    v = torch.zeros(pages, page, nkv, d, device="cuda", dtype=torch.uint8).view(E4)
    e = [torch.full((pages, 1, nkv), 127, device="cuda", dtype=torch.uint8) for _ in range(2)]
    x = torch.randn(10, nkv * d, device="cuda", generator=gen(5))
    cache = ops.KvCache8.of(k, v, *e, i32([[pages - 1]]))
    ops.rope_append8(cache, None, None, None, x, x, i32([0] * 10), i32(range(10)), heads=0, stream=stream())
    q = torch.randn(1, nkv, d, device="cuda", generator=gen(6)).bfloat16()
    out = torch.zeros_like(q)
    ws = torch.empty(ops.attention_paged8_workspace(cache, nkv), device="cuda", dtype=torch.uint8)
    ops.attention_paged8(cache, out, q, None, i32([9]), scale=0.1, workspace=ws, stream=stream())
    torch.cuda.synchronize()
    kv, vv = (values8(p[-1:], z[-1:], block).flatten(0, 1)[:10] for p, z in ((k, e[0]), (v, e[1])))
    vs = 2.0 ** (e[1][-1].cpu().double().expand(10, nkv) - 127)
    want, tol = attention8_64(q[0], kv, vv, vs, 0.1)
    assert ((out[0].double().cpu() - want).abs() <= tol).all()


# ------------------------------------------------------------------ weights of 4 bits
LINEAR = [  # rows, n, k, group, zeros, scale f32, f32 out, add, padded rows
    (1, 6144, 2560, 128, False, False, False, None, 0),
    (1, 1, 32, 32, False, True, True, None, 0),
    (3, 17, 96, 32, True, False, True, "other", 8),
    (8, 100, 64, 64, True, True, False, "other", 16),
    (9, 33, 192, 64, False, False, True, "same", 8),
    (16, 250, 9728, 64, True, False, True, "same", 0),
    (17, 40, 384, 384, True, True, True, None, 0),
    (31, 65, 1024, 256, False, False, False, "same", 0),
    (33, 300, 800, 32, True, False, True, "other", 8),
    (70, 48, 128, 128, False, True, False, None, 8),
    (5, 2560, 16384, 128, False, False, True, None, 0),
    (2, 20011, 256, 32, True, False, False, None, 0),
]


@pytest.mark.parametrize("case", LINEAR, ids=lambda c: "-".join(map(str, c)))
def test_linear4(ops, case):
    rows, n, k, group, zeros, sf, f32, add, pad = case
    g = gen(n + k)
    q = torch.randint(0, 256, (n, k // 2 + 16 * (pad > 0)), device="cuda", generator=g, dtype=torch.uint8)[:, :k // 2]
    scale = (torch.rand(n, k // group + (pad > 0), device="cuda", generator=g) - 0.3)[:, :k // group]
    scale = scale if sf else scale.bfloat16()
    zero = torch.randint(0, 128 if n % 2 else 16, (n, k // group + 3), device="cuda", generator=g, dtype=torch.uint8)[:, :k // group] if zeros else None
    x = torch.randn(rows, k + pad, device="cuda", generator=g).bfloat16()[:, :k]
    ty = torch.float32 if f32 else torch.bfloat16
    out = torch.full((rows + 1, n + 5), 7.0, device="cuda", dtype=ty)
    resid = torch.randn(rows, n + 5, device="cuda", generator=g).to(ty)
    if add == "same":
        out[:rows] = resid
    to = out[:rows, :n]
    w = ops.Weights4.of(q, scale, zero)
    ops.linear4(to, x, w, add={None: None, "same": to, "other": resid[:, :n]}[add], stream=stream())
    torch.cuda.synchronize()
    nib = torch.stack((q & 15, q >> 4), -1).reshape(n, k).double().cpu()
    z = zero.double().cpu().repeat_interleave(group, 1) if zeros else 8.0
    s = scale.double().cpu().repeat_interleave(group, 1)
    wf, xd = (nib - z) * s, x.double().cpu()
    want, size = xd @ wf.t(), xd.abs() @ wf.abs().t()
    if add:
        want = want + resid[:, :n].double().cpu()
        size = size + resid[:, :n].double().cpu().abs()
    tol = (k / 8 + 100) * 2 * U * size + (U if f32 else BF) * want.abs()
    err = (to.double().cpu() - want).abs()
    assert (err <= tol).all(), float((err - tol).max())
    rest = out[:rows, n:], out[rows:]
    assert (rest[1] == 7).all() and (add == "same" or (rest[0] == 7).all())


def test_linear4_rows_do_not_meet(ops):
    """A row of x that is not finite, or a scale, shows in its own results alone; and the same call gives the same bits."""
    n, k = 70, 512
    g = gen(1)
    q = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
    scale = torch.rand(n, k // 64, device="cuda", generator=g)
    x = torch.randn(20, k, device="cuda", generator=g).bfloat16()
    outs = []
    for bad in (False, True):
        xs, ss = x.clone(), scale.clone()
        if bad:
            xs[3, 100], xs[17, 0], ss[11, 2] = math.nan, math.inf, math.nan
        out = torch.zeros(20, n, device="cuda")
        ops.linear4(out, xs, ops.Weights4.of(q, ss), stream=stream())
        outs.append(out)
    torch.cuda.synchronize()
    a, b = (o.cpu() for o in outs)
    odd = torch.zeros(20, n, dtype=torch.bool)
    odd[3], odd[17], odd[:, 11] = True, True, True
    assert not torch.isfinite(b[odd]).any() and torch.equal(a[~odd], b[~odd])


@pytest.mark.parametrize("n,k,group,f32,sf", [(1, 32, 32, True, True), (33, 256, 64, False, False), (100, 2560, 128, False, False),
                                              (7, 1152, 384, True, False), (129, 96, 32, True, True), (300, 512, 512, False, True)])
def test_quantize4(ops, n, k, group, f32, sf):
    w = torch.randn(n, k + 8, device="cuda", generator=gen(n)) * torch.exp2(torch.randint(-20, 20, (n, 1), device="cuda", generator=gen(k)).float())
    w = w if f32 else w.bfloat16()
    w[0, :group] = 0.0
    if n > 2:
        w[1, group - 1], w[2, 0] = math.nan, -math.inf
    w = w[:, :k]
    q = torch.full((n + 1, k // 2 + 16), 0xAB, device="cuda", dtype=torch.uint8)
    scale = torch.full((n + 1, k // group + 1), 5.0, device="cuda", dtype=torch.float32 if sf else torch.bfloat16)
    ops.quantize4(ops.Weights4.of(q[:n, :k // 2], scale[:n, :k // group]), w, stream=stream())
    torch.cuda.synchronize()
    x = w.float().cpu().view(n, -1, group)
    s = (x.abs().amax(-1) / 7).to(scale.dtype)
    s[~torch.isfinite(x).all(-1)] = math.nan
    assert torch.equal(torch.nan_to_num(scale[:n, :k // group].cpu(), 777.0), torch.nan_to_num(s, 777.0))
    fine = torch.isfinite(s.float())
    sf32 = torch.where(s.float() > 0, s.float(), 1.0)[..., None]
    want = torch.clamp(torch.round(x / sf32), -8, 7) + 8
    got = torch.stack((q[:n, :k // 2] & 15, q[:n, :k // 2] >> 4), -1).reshape(n, -1, group).cpu()
    assert torch.equal(got[fine].float(), want[fine])
    assert (q[n] == 0xAB).all() and (q[:, k // 2:] == 0xAB).all() and (scale[n] == 5).all() and (scale[:, -1] == 5).all()


def test_quantize4_then_linear4(ops):
    """Weights rounded and used: off by at most half a step of the scale, and its own rounding, a weight."""
    n, k, group = 96, 1024, 128
    w = torch.randn(n, k, device="cuda", generator=gen(2)).bfloat16()
    x = torch.randn(4, k, device="cuda", generator=gen(3)).bfloat16()
    q = torch.zeros(n, k // 2, device="cuda", dtype=torch.uint8)
    scale = torch.zeros(n, k // group, device="cuda", dtype=torch.bfloat16)
    w4 = ops.Weights4.of(q, scale)
    ops.quantize4(w4, w, stream=stream())
    out = torch.zeros(4, n, device="cuda")
    ops.linear4(out, x, w4, stream=stream())
    torch.cuda.synchronize()
    s = scale.double().cpu().repeat_interleave(group, 1)
    xd = x.double().cpu()
    # the scale is rounded, so that the largest weight may lie past 7.5 steps by 2^-8 of 7
    bound = xd.abs() @ ((0.5 + 7 * 2.0 ** -8) * s).t()
    assert ((out.double().cpu() - xd @ w.double().cpu().t()).abs() <= bound).all()


# ------------------------------------------------------------------ together
class Decoder:
    """One layer and a head as a server runs them: 4-bit projections, an 8-bit cache, sampling; all buffers of its own."""

    H, NH, NKV, D, VOCAB, PAGE, BLOCK = 256, 4, 2, 64, 1000, 16, 8

    def __init__(self, ops, batch, seed=1):
        self.ops, self.batch = ops, batch
        H, NH, NKV, D = self.H, self.NH, self.NKV, self.D
        g = gen(seed)
        self.embed = torch.randn(self.VOCAB, H, device="cuda", generator=g).bfloat16()
        self.w = {}
        for name, n, k in (("qkv", (NH + 2 * NKV) * D, H), ("o", H, NH * D), ("head", self.VOCAB, H)):
            q = torch.zeros(n, k // 2, device="cuda", dtype=torch.uint8)
            w4 = ops.Weights4.of(q, torch.zeros(n, k // 64, device="cuda", dtype=torch.bfloat16))
            ops.quantize4(w4, torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k), stream=stream())
            self.w[name] = w4
        pages = batch * 8
        e = lambda *s, dtype: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
        self.kv = [e(pages, self.PAGE, NKV, D, dtype=torch.uint8).view(E4) for _ in range(2)]
        self.exps = [e(pages, self.PAGE // self.BLOCK, NKV, dtype=torch.uint8) for _ in range(2)]
        self.cache = ops.KvCache8.of(*self.kv, *self.exps, torch.randperm(pages, device="cuda", generator=g).int().view(batch, 8))
        self.rope = ops.Rope.of(D, 1e4)
        self.ids, self.seq, self.pos = i32([5] * batch), i32(range(batch)), i32([0] * batch)
        self.uniform = e(batch, dtype=torch.float64)
        self.x, self.h = e(batch, H, dtype=torch.bfloat16), e(batch, H, dtype=torch.bfloat16)
        self.qkv, self.q = e(batch, (NH + 2 * NKV) * D, dtype=torch.float32), e(batch, NH, D, dtype=torch.bfloat16)
        self.attn = e(batch, NH, D, dtype=torch.bfloat16)
        self.logits, self.logprobs = e(batch, self.VOCAB, dtype=torch.float32), e(batch, dtype=torch.float32)
        self.temperature = torch.full((batch,), 0.9, device="cuda")
        self.top_p = torch.full((batch,), 0.9, device="cuda")
        self.ws = e(ops.attention_paged8_workspace(self.cache, NH), dtype=torch.uint8)

    def step(self):
        ops, st = self.ops, stream()
        D, NH, NKV = self.D, self.NH, self.NKV
        torch.index_select(self.embed, 0, self.ids.long(), out=self.x)
        ops.linear4(self.qkv, self.x, self.w["qkv"], stream=st)
        ops.rope_append8(self.cache, self.rope, self.q, self.qkv[:, :NH * D], self.qkv[:, NH * D:(NH + NKV) * D],
                         self.qkv[:, (NH + NKV) * D:], self.seq, self.pos, heads=NH, stream=st)
        ops.attention_paged8(self.cache, self.attn, self.q, self.seq, self.pos, scale=1 / math.sqrt(D), workspace=self.ws, stream=st)
        ops.linear4(self.h, self.attn.view(self.batch, -1), self.w["o"], add=self.x, stream=st)
        ops.linear4(self.logits, self.h, self.w["head"], stream=st)
        ops.sample_tokens(self.logits, self.uniform, self.ids, temperature=self.temperature, top_p=self.top_p, logprobs=self.logprobs,
                          stream=st)
        self.pos += 1


def test_a_decoding_loop(ops):
    """The operators one behind the other, 40 tokens for three sequences: called one by one and from a captured graph, on
    streams of their own at the same time, the same tokens; and every step as the 64-bit forms of its parts have it."""
    a, b = Decoder(ops, 3), Decoder(ops, 3)
    uniform = torch.rand(40, 3, device="cuda", dtype=torch.float64, generator=gen(9))
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(sb):
        b.uniform.copy_(uniform[0])
        b.step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=sb):
        b.step()
    tokens = [], [b.ids.tolist()]
    for i in range(40):
        with torch.cuda.stream(sa):
            a.uniform.copy_(uniform[i])
            a.step()
        if i:
            with torch.cuda.stream(sb):
                b.uniform.copy_(uniform[i])
                graph.replay()
        torch.cuda.synchronize()
        tokens[0].append(a.ids.tolist())
        if i:
            tokens[1].append(b.ids.tolist())
        # this step's parts
        n = i + 1
        kv, vv = (values8(p, e, a.BLOCK) for p, e in zip(a.kv, a.exps))
        vs = 2.0 ** (a.exps[1].cpu().double().repeat_interleave(a.BLOCK, 1) - 127)
        table = a.cache.tensors[4].long().cpu()
        for r in range(3):
            cut = lambda x: x[table[r]].flatten(0, 1)[:n]  # noqa: E731
            want, tol = attention8_64(a.q[r], cut(kv), cut(vv), cut(vs), 1 / math.sqrt(a.D))
            assert ((a.attn[r].double().cpu() - want).abs() <= tol).all()
            want = sample64(a.logits[r].cpu().numpy(), float(np.float32(0.9)), 0, float(np.float32(0.9)), 0.0, float(uniform[i, r]))
            assert tokens[0][-1][r] == want[0] and abs(float(a.logprobs[r]) - want[1]) <= U * abs(want[1]) + 2.0 ** -40
    assert tokens[0] == tokens[1]
    assert len({t for step in tokens[0] for t in step}) > 20
    for x, y in zip(a.kv + a.exps + [a.logits], b.kv + b.exps + [b.logits]):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
