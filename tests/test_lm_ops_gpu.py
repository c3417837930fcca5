"""Language-model operators on the GPU against plain 64-bit forms.

Tolerances, derived from the operators' arithmetic (u = 2^-24, half an f32 step;
2^-8, half a bf16 step, relative):

rope_append: one rounding to bf16 (2^-8 of the value) after f32 arithmetic on a
  pair (a, b).  Angle: a 32-bit fraction of a half turn as f32, at most pi u;
  sincospi 2 ulp; norm: a sum of <= 256 squares over 8 lanes-serial and 5
  shuffled additions, root, quotient, two products; rotation: two products and
  an addition.  Under 40 u of |a| + |b| in all: 2^-18 (|a| + |b|) is asked.
attention_paged: 2^-8 of the value, plus, times A = sum p |v|: scores that are off
  by at most 4 hd u S, S = max over the keys of scale sum |q k| (tensor-core sums
  drop bits instead of rounding: 2 u an addition; both numerator and denominator
  see it), len u for the sums over keys, and 2^-14 for the exponential (2^-22 and
  its argument's rounding, |x| log2(e) u) and for weights carried in 16 bits (2^-16).
token_logprobs: lse = m + log S: S is a sum of V terms, at most V / 256 one after
  the other, then a tree; each term's exponential 2^-22.  (V / 256 + 100) u plus
  2^-22 of |lse| + |m|.  Entropy log S - T / S with T = sum (x - m) e^(x - m), all
  of one sign: twice that times 1 + |T / S|, plus 2^-22 (|log S| + |T / S|).  Ids: equal.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
U = 2.0 ** -24
BF = 2.0 ** -8


@pytest.fixture(scope="module")
def ops(iris):
    return iris


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def pool(pages, page, heads, d, head_major, fill=float("nan")):
    if head_major:
        return torch.full((pages, heads, page, d), fill, device="cuda", dtype=torch.bfloat16).permute(0, 2, 1, 3)
    return torch.full((pages, page, heads, d), fill, device="cuda", dtype=torch.bfloat16)


def i32(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


# ------------------------------------------------------------------ rope_append
def rotate64(x, pos, freqs, interleaved, amplitude, w, eps=1e-6):
    """64-bit norm and rotation of [T, heads, d]; also |a| + |b| of each value's pair."""
    x = x.double().cpu()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double().cpu()
    y, size = x.clone(), x.abs()
    n = len(freqs)
    if n:
        ang = pos.double().cpu()[:, None] * torch.tensor(freqs, dtype=torch.float64)
        c, s = amplitude * torch.cos(ang)[:, None], amplitude * torch.sin(ang)[:, None]
        i = torch.arange(n)
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
        size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * max(1.0, amplitude)
    return y, size


def near(got, want, slack):
    err = (got.double().cpu() - want).abs()
    bad = err > BF * want.abs() + slack
    assert not bad.any(), (float(err[bad].max()), int(bad.sum()))


ROPE = [  # tokens, heads, kv heads, d, rot, interleaved, page, head major, f32, norm, scaling, far
    (1, 32, 8, 128, 128, False, 16, False, True, True, {}, 500),
    (3, 4, 2, 128, 128, False, 16, True, False, True, {}, 2 ** 20),
    (37, 6, 2, 64, 64, True, 7, False, False, False, {}, 2 ** 30),
    (130, 7, 1, 128, 96, False, 1, True, True, False, dict(factor=4.0), 900),
    (65, 5, 5, 256, 64, True, 24, False, True, True, dict(factor=8.0, original_len=4096, low=1.0, high=4.0, amplitude=1.3), 2 ** 17),
    (17, 3, 1, 256, 256, False, 100, True, False, True, {}, 40),
    (64, 2, 2, 64, 48, False, 16, False, False, True, {}, 100000),
    (600, 16, 4, 128, 16, True, 64, True, False, False, {}, 1500),
    (9, 0, 3, 128, 128, False, 16, False, False, True, {}, 77),
    (21, 4, 4, 64, 0, False, 16, False, True, True, {}, 77),
]


@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(map(str, c[:7])))
def test_rope_append(ops, case):
    t, nh, nkv, d, rd, inter, page, hm, f32, norm, scaling, far = case
    g = gen(t)
    rng = np.random.default_rng(t)
    qkv = torch.randn(t, (nh + 2 * nkv) * d + 8, device="cuda", generator=g) * 2
    qkv = qkv if f32 else qkv.bfloat16()
    q, k, v = (qkv[:, a * d:b * d] for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
    # distinct positions anywhere below `far`, on three sequences; padding and tokens without a slot among them
    seq = rng.integers(0, 3, t)
    pos = np.array(rng.choice(far, t, replace=False) if far < 10 ** 6 else rng.integers(0, far // t, t) + np.arange(t) * (far // t))
    blocks = min(-(-far // page), 60)
    keep = pos % (blocks * page)  # the far ones beyond a table of 60 blocks have no slot
    written = [i for i in range(t) if pos[i] < blocks * page]
    touched = sorted({(int(seq[i]), int(pos[i]) // page) for i in written})
    pages = len(touched) + 5
    table = torch.full((3, blocks + 2), -7, device="cuda", dtype=torch.int32)[:, :blocks]
    ids = rng.permutation(pages)
    for (s, b), p in zip(touched, ids):
        table[s, b] = int(p)
    if t > 8:
        seq[1], seq[2], pos[3] = -1, 3, -5      # padding
        bad = next((i for i in written if i > 4), None)
        if bad is not None:                      # a page outside the pool, its neighbours stay
            table[int(seq[bad]), int(pos[bad]) // page] = pages
    kp, vp = pool(pages, page, nkv, d, hm), pool(pages, page, nkv, d, hm)
    qo = torch.full((t, max(nh, 1) * d + 16), 7.0, device="cuda", dtype=torch.bfloat16)[:, :nh * d]
    qn = 1 + 0.2 * torch.randn(d, device="cuda", generator=g) if norm else None
    kn = 1 + 0.2 * torch.randn(d, device="cuda", generator=g) if norm else None
    theta = 1e6 if d == 128 else 1e4
    rope = ops.Rope.of(rd, theta, interleaved=inter, **scaling) if rd else None
    freqs = [x / 2.0 ** 64 * 2 * math.pi for x in rope.turns[:rd // 2]] if rd else []
    cache = ops.KvCache.of(kp, vp, table)
    ops.rope_append(cache, rope, qo if nh else None, q if nh else None, k, v, i32(seq), i32(pos), heads=nh, q_norm=qn,
                    k_norm=kn, stream=stream())
    torch.cuda.synchronize()
    amp = scaling.get("amplitude", 1.0)
    P = torch.tensor(pos.clip(0))
    live = (seq >= 0) & (seq < 3) & (pos >= 0)
    if nh:
        want, size = rotate64(q.reshape(t, nh, d), P, freqs, inter, amp, qn)
        near(qo.reshape(t, nh, d)[live], want[live], 2.0 ** -18 * size[live])
        assert (qo[~torch.tensor(live)] == 7).all()
    wk, size = rotate64(k.reshape(t, nkv, d), P, freqs, inter, amp, kn)
    kc, vc = kp.cpu(), vp.cpu()
    tab = table.cpu().numpy()
    seen = np.zeros((pages, page), bool)
    for i in range(t):
        if not live[i] or pos[i] >= blocks * page:
            continue
        p, sl = int(tab[seq[i], pos[i] // page]), int(pos[i] % page)
        if p < 0 or p >= pages:
            continue
        seen[p, sl] = True
        near(kc[p, sl], wk[i], 2.0 ** -18 * size[i])
        assert torch.equal(vc[p, sl], v.reshape(t, nkv, d)[i].bfloat16().cpu())
    assert torch.isnan(kc[~torch.tensor(seen)]).all() and torch.isnan(vc[~torch.tensor(seen)]).all()
    assert seen.any() or t < 9 or far > blocks * page


def test_rope_append_in_place(ops):
    d, nh, nkv, t = 128, 4, 2, 33
    x = torch.randn(t, nh * d, device="cuda", generator=gen(5)).bfloat16()
    kv = torch.randn(t, nkv * d, device="cuda", generator=gen(6)).bfloat16()
    for inter in (False, True):
        rope = ops.Rope.of(128, 1e4, interleaved=inter)
        outs = []
        for place in (False, True):
            src = x.clone()
            dst = src if place else torch.empty_like(src)
            kp, vp = pool(4, 16, nkv, d, False, 0.0), pool(4, 16, nkv, d, False, 0.0)
            cache = ops.KvCache.of(kp, vp, i32([[0, 1, 2]]))
            ops.rope_append(cache, rope, dst, src, kv, kv, i32([0] * t), i32(range(t)), heads=nh, stream=stream())
            outs.append((dst, kp, vp))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(*outs))


# ------------------------------------------------------------------ attention_paged
def attention64(q, k, v, scale):
    """q [heads, d], k / v [len, kv heads, d] -> (out, tolerance) [heads, d] in 64 bits."""
    nh, d = q.shape
    n, nkv = k.shape[:2]
    if not n:
        return torch.zeros(nh, d, dtype=torch.float64), torch.zeros(nh, d, dtype=torch.float64)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    k, v = (x.repeat_interleave(nh // nkv, 1).transpose(0, 1) for x in (k, v))
    p = torch.softmax(scale * torch.einsum("hd,hld->hl", q, k), -1)
    s = abs(scale) * torch.einsum("hd,hld->hl", q.abs(), k.abs()).amax(-1)
    out, a = torch.einsum("hl,hld->hd", p, v), torch.einsum("hl,hld->hd", p, v.abs())
    return out, BF * out.abs() + (4 * d * U * s + n * U + 2.0 ** -14)[:, None] * a


def paged(lens, page, nkv, d, hm, seed, spare=3, blocks=None):
    """Pools of NaN with the given sequences' keys in them, and the sequences."""
    g = gen(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    kp, vp = pool(pages, page, nkv, d, hm), pool(pages, page, nkv, d, hm)
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), blocks or max(need + [1])), -1, dtype=torch.int32)
    ks, vs = [], []
    for i, n in enumerate(lens):
        ks.append(torch.randn(n, nkv, d, device="cuda", generator=g).bfloat16())
        vs.append(torch.randn(n, nkv, d, device="cuda", generator=g).bfloat16())
        for b in range(need[i]):
            p = ids.pop()
            table[i, b] = p
            m = min(page, n - b * page)
            kp[p, :m], vp[p, :m] = ks[i][b * page:b * page + m], vs[i][b * page:b * page + m]
    return kp, vp, table.cuda(), ks, vs


def attend(ops, kp, vp, table, q, pos, seq=None, scale=None, out=None):
    d = kp.shape[3]
    nh = q.shape[1]
    cache = ops.KvCache.of(kp, vp, table)
    ws = torch.full((ops.attention_paged_workspace(cache, nh),), 255, device="cuda", dtype=torch.uint8)
    out = torch.full_like(q, 9.0) if out is None else out
    ops.attention_paged(cache, out, q, seq, pos, scale=1 / math.sqrt(d) if scale is None else scale, workspace=ws,
                        stream=stream())
    torch.cuda.synchronize()
    return out


ATT = [  # lengths, heads, kv heads, d, page, head major
    ([1], 4, 1, 128, 16, False),
    ([0], 4, 2, 128, 16, False),
    ([512], 32, 8, 128, 16, False),
    ([17, 0, 1, 63, 64, 65, 200], 8, 2, 128, 16, True),
    ([5000, 3, 1200], 32, 8, 128, 24, False),
    ([9, 31, 129, 257], 7, 1, 64, 7, False),
    ([33, 700], 16, 1, 128, 100, True),
    ([300, 15], 24, 1, 64, 1, True),
    ([40, 1000], 5, 5, 256, 32, False),
    ([4097], 2, 2, 64, 64, True),
    ([129, 2, 77, 500], 40, 4, 256, 16, True),
    ([20000], 4, 1, 128, 16, False),
    (list(range(0, 300)), 6, 2, 64, 16, False),
]


@pytest.mark.parametrize("lens,nh,nkv,d,page,hm", ATT, ids=lambda c: str(c)[:24])
def test_attention_paged(ops, lens, nh, nkv, d, page, hm):
    kp, vp, table, ks, vs = paged(lens, page, nkv, d, hm, len(lens) + d)
    q = (2 * torch.randn(len(lens), nh, d, device="cuda", generator=gen(3))).bfloat16()
    # tables with room for much longer sequences are worked on in another way
    roomy = torch.full((len(lens), table.shape[1] + 40000 // page), -1, device="cuda", dtype=torch.int32)
    roomy[:, :table.shape[1]] = table
    want = [attention64(q[i], ks[i], vs[i], 1 / math.sqrt(d)) for i in range(len(lens))]
    for tab in (table, roomy):
        out = attend(ops, kp, vp, tab, q, i32(lens) - 1)
        assert torch.equal(out, attend(ops, kp, vp, tab, q, i32(lens) - 1))
        for i, (w, tol) in enumerate(want):
            err = (out[i].double().cpu() - w).abs()
            assert (err <= tol).all(), (i, float((err - tol).max()))


def test_attention_paged_rows_of_sequences(ops):
    """A run of tokens of one sequence (causal), rows in any order, padding rows, the same row twice."""
    kp, vp, table, ks, vs = paged([70, 200, 9], 16, 2, 128, False, 11)
    seq = [1] * 40 + [0, 2, 2, -1, 3, 1, 1, -5]
    pos = list(range(120, 160)) + [69, 8, 8, 5, 5, 0, -1, 3]
    q = torch.randn(len(seq), 6, 128, device="cuda", generator=gen(4)).bfloat16()
    q[42] = q[41]
    wide = torch.full((len(seq), 6 * 128 + 24), 9.0, device="cuda", dtype=torch.bfloat16)
    out = attend(ops, kp, vp, table, q, i32(pos), i32(seq), out=wide[:, :768])
    for i, (s, p) in enumerate(zip(seq, pos)):
        got = out[i].view(6, 128)
        if not 0 <= s < 3:
            assert (got == 9).all()
            continue
        want, tol = attention64(q[i], ks[s][:p + 1], vs[s][:p + 1], 1 / math.sqrt(128))
        assert ((got.double().cpu() - want).abs() <= tol).all(), i
    assert torch.equal(out[41], out[42])
    assert (wide[:, 768:] == 9).all()


def test_attention_paged_few_rows_cut_into_many_pieces(ops):
    """One long sequence among rows that see nothing, see one key or are padding, in every order."""
    kp, vp, table, ks, vs = paged([9000, 1, 40], 16, 1, 128, False, 17)
    q = torch.randn(6, 12, 128, device="cuda", generator=gen(10)).bfloat16()
    at = {0: (0, 8999), 1: (-1, 50), 2: (1, 0), 3: (2, -4), 4: (2, 39), 5: (7, 3)}
    for order in ((0, 1, 2, 3, 4, 5), (5, 1, 3, 2, 4, 0), (3, 0, 5, 1, 4, 2)):
        seq, pos = [at[r][0] for r in order], [at[r][1] for r in order]
        out = attend(ops, kp, vp, table, q, i32(pos), i32(seq))
        for i, (s, p) in enumerate(zip(seq, pos)):
            if not 0 <= s < 3:
                assert (out[i] == 9).all()
                continue
            want, tol = attention64(q[i], ks[s][:max(0, p + 1)], vs[s][:max(0, p + 1)], 1 / math.sqrt(128))
            assert ((out[i].double().cpu() - want).abs() <= tol).all(), (order, i)


def test_attention_paged_positions_and_pages_out_of_range(ops):
    """Positions past the table see the table's keys; pages outside the pool are not seen."""
    page, d = 16, 128
    kp, vp, table, ks, vs = paged([128, 128, 128], page, 1, d, False, 12)
    table[1, 2], table[1, 5], table[2, :] = -3, 2 ** 31 - 1, kp.shape[0]
    q = torch.randn(3, 4, d, device="cuda", generator=gen(5)).bfloat16()
    out = attend(ops, kp, vp, table, q, i32([2 ** 31 - 1, 127, 127]))
    keep = torch.tensor([b not in (2, 5) for b in range(8)]).repeat_interleave(page)
    for i, sel in ((0, slice(None)), (1, keep)):
        want, tol = attention64(q[i], ks[i].cpu()[sel], vs[i].cpu()[sel], 1 / math.sqrt(d))
        assert ((out[i].double().cpu() - want).abs() <= tol).all(), i
    assert (out[2] == 0).all()


@pytest.mark.parametrize("scale,size", [(0.0, 1.0), (1.0, 30.0), (-0.2, 3.0), (1e-3, 1e4)])
def test_attention_paged_scales_and_peaks(ops, scale, size):
    """One key takes all of a row (scores in the thousands), all alike, negative scales."""
    kp, vp, table, ks, vs = paged([300, 90], 16, 2, 128, True, 13)
    q = (size * torch.randn(2, 8, 128, device="cuda", generator=gen(6))).bfloat16()
    out = attend(ops, kp, vp, table, q, i32([299, 89]), scale=scale)
    for i in range(2):
        want, tol = attention64(q[i], ks[i], vs[i], scale)
        assert ((out[i].double().cpu() - want).abs() <= tol).all(), i


def test_attention_paged_shared_pages(ops):
    """Two sequences whose tables begin with the same pages."""
    kp, vp, table, ks, vs = paged([96, 40], 16, 1, 64, False, 14)
    both = torch.full((2, 8), -1, device="cuda", dtype=torch.int32)
    both[0, :6] = table[0, :6]
    both[1, :4], both[1, 4:7] = table[0, :4], table[1, :3]
    q = torch.randn(2, 4, 64, device="cuda", generator=gen(7)).bfloat16()
    out = attend(ops, kp, vp, both, q, i32([95, 103]))
    k1, v1 = (torch.cat((a[0][:64], a[1])) for a in (ks, vs))
    for i, (k, v) in enumerate(((ks[0], vs[0]), (k1, v1))):
        want, tol = attention64(q[i], k, v, 1 / 8)
        assert ((out[i].double().cpu() - want).abs() <= tol).all(), i


def test_offsets_past_32_bits(ops):
    """A pool of more than 2^32 values: keys written to its last pages and read back."""
    page, nkv, d = 64, 8, 128
    pages = 2 ** 32 // (page * nkv * d) + 5
    kp = torch.empty(pages, page, nkv, d, device="cuda", dtype=torch.bfloat16)
    vp = torch.empty(pages, page, nkv, d, device="cuda", dtype=torch.bfloat16)
    t, nh = 150, 16
    table = i32([[pages - 2, 1, pages - 1]])
    qkv = torch.randn(t, (nh + 2 * nkv) * d, device="cuda", generator=gen(8)).bfloat16()
    q, k, v = qkv[:, :nh * d], qkv[:, nh * d:(nh + nkv) * d], qkv[:, (nh + nkv) * d:]
    cache = ops.KvCache.of(kp, vp, table)
    qo = torch.empty(t, nh, d, device="cuda", dtype=torch.bfloat16)
    ops.rope_append(cache, None, qo, q, k, v, i32([0] * t), i32(range(t)), heads=nh, stream=stream())
    out = attend(ops, kp, vp, table, qo[-1:], i32([t - 1]))
    want, tol = attention64(qo[-1], k.reshape(t, nkv, d), v.reshape(t, nkv, d), 1 / math.sqrt(d))
    assert torch.equal(qo.view(t, -1), q.contiguous())
    assert ((out[0].double().cpu() - want).abs() <= tol).all()


# ------------------------------------------------------------------ token_logprobs
def answers(ops, x, targets, k, which="leit"):
    n, vocab = x.shape
    ws = torch.full((ops.token_logprobs_workspace(n, vocab),), 255, device="cuda", dtype=torch.uint8)
    lp = torch.full((n,), 9.0, device="cuda")
    en = torch.full((n,), 9.0, device="cuda")
    ids = torch.full((n, k), -9, device="cuda", dtype=torch.int32)
    tl = torch.full((n, k), 9.0, device="cuda")
    ops.token_logprobs(x, targets, lp if "l" in which else None, en if "e" in which else None, ids if "i" in which else None,
                       tl if "t" in which else None, workspace=ws, stream=stream())
    torch.cuda.synchronize()
    return lp, en, ids, tl


def check_answers(x, targets, k, got):
    """Rows of finite or -inf logits, at least one finite."""
    n, vocab = x.shape
    x, t = x.double().cpu(), targets.cpu().long()
    m = x.amax(-1)
    e = torch.exp(x - m[:, None])
    s = e.sum(-1)
    lse = m + torch.log(s)
    mean = torch.where(e == 0, 0.0, e * (x - m[:, None])).sum(-1) / s
    base = (vocab / 256 + 100) * U
    tol = base + 2.0 ** -22 * (lse.abs() + m.abs())
    tol_h = 2 * base * (1 + mean.abs()) + 2.0 ** -22 * (torch.log(s).abs() + mean.abs())
    lp, en, ids, tl = (g.cpu() for g in got)
    ok = (t >= 0) & (t < vocab)
    want = torch.where(ok, x.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0] - lse, 0.0)
    gone = want == -math.inf
    assert (lp[gone] == -math.inf).all() and (lp[~ok] == 0).all()
    err = (lp.double() - want).abs()[~gone]
    assert (err <= (tol + 2 * U * want.abs())[~gone]).all(), float(err.max())
    err = (en.double() - (torch.log(s) - mean)).abs()
    assert (err <= tol_h).all(), float(err.max())
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(ids.long(), order)
    want = x.gather(1, order) - lse[:, None]
    gone = want == -math.inf
    assert (tl[gone] == -math.inf).all()
    err = (tl.double() - want).abs()
    assert (err <= tol[:, None] + 2 * U * want.abs())[~gone].all(), float(err[~gone].max())


LP = [  # rows, vocab, k, f32, ld beyond vocab
    (1, 151936, 20, False, 0), (1, 151936, 20, True, 0), (3, 151936, 32, False, 8), (5, 1, 1, False, 0), (4, 2, 2, True, 3),
    (2, 7, 7, False, 0), (300, 31, 31, False, 0), (9, 256, 32, True, 0), (17, 257, 5, False, 0), (6, 2047, 8, False, 1),
    (40, 50021, 8, False, 0), (3, 65537, 1, True, 5), (2, 200003, 0, False, 2), (700, 1000, 20, True, 0), (2, 1000003, 20, False, 0),
]


@pytest.mark.parametrize("rows,vocab,k,f32,extra", LP)
def test_token_logprobs(ops, rows, vocab, k, f32, extra):
    x = 3 * torch.randn(rows, vocab + extra, device="cuda", generator=gen(rows + vocab))
    x = (x if f32 else x.bfloat16())[:, :vocab]
    targets = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(1), dtype=torch.int32)
    if rows > 3:
        targets[0], targets[1], targets[2] = -1, vocab, 2 ** 31 - 1
    got = answers(ops, x, targets, k)
    check_answers(x, targets, k, got)
    assert all(torch.equal(a, b) for a, b in zip(got, answers(ops, x, targets, k)))


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("vocab", [100, 4096, 151936])
def test_token_logprobs_hard_rows(ops, f32, vocab):
    """Ties, signed zeros, rising and falling rows, one token left, banned targets, huge spreads."""
    g = gen(vocab)
    ty = torch.float32 if f32 else torch.bfloat16
    rows = [torch.zeros(vocab, device="cuda"), torch.full((vocab,), -3.25, device="cuda"),
            torch.arange(vocab, device="cuda") * (8.0 / vocab), torch.arange(vocab, device="cuda") * (-8.0 / vocab),
            torch.randn(vocab, device="cuda", generator=g) * 1e-3, torch.randn(vocab, device="cuda", generator=g) * 1000,
            torch.randint(-2, 3, (vocab,), device="cuda", generator=g).float()]
    z = torch.zeros(vocab, device="cuda")
    z[1::2] = -0.0
    rows.append(z)
    one = torch.full((vocab,), -math.inf, device="cuda")
    one[vocab // 3] = -1000.0
    rows.append(one)
    few = torch.full((vocab,), -math.inf, device="cuda")
    few[[5, 50, vocab - 1]] = torch.tensor([1.0, 2.0, 1.0], device="cuda")
    rows.append(few)
    low = torch.randn(vocab, device="cuda", generator=g)
    low[::3] = torch.finfo(ty).min
    rows.append(low)
    peak = torch.randn(vocab, device="cuda", generator=g)
    peak[vocab - 2] = 3e38
    rows.append(peak)
    block = torch.randn(vocab, device="cuda", generator=g)
    block[8:48] = 20 + torch.arange(40, device="cuda") * 0.25
    rows.append(block)
    x = torch.stack(rows).to(ty)
    t = torch.full((len(rows),), vocab // 3, device="cuda", dtype=torch.int32)
    t[9] = 6
    check_answers(x, t, 20, answers(ops, x, t, 20))
    x, t = x.repeat(5, 1), t.repeat(5)  # many rows go another way
    check_answers(x, t, 32, answers(ops, x, t, 32))


@pytest.mark.parametrize("many", [1, 10])
def test_token_logprobs_rows_without_an_answer(ops, many):
    """-inf everywhere, NaN, +inf: the documented values, and neighbours that do not notice."""
    vocab, k = 5000, 6
    x = torch.randn(6, vocab, device="cuda", generator=gen(2))
    plain = x[5].clone()
    x[0] = -math.inf
    x[1, 4000], x[1, 77] = math.nan, -math.nan
    x[2, 123] = math.inf
    x[3] = math.nan
    x[4, 9], x[4, 8], x[4, 3000] = math.nan, math.inf, math.inf
    for ty in (torch.float32, torch.bfloat16):
        y = x.to(ty).repeat(many, 1)
        t = i32([3, 3, 3, 3, 3, 3])
        got = answers(ops, y, t.repeat(many), k)
        for part in range(1, many):  # (bits: a NaN is not itself)
            assert all(torch.equal(g[:6].view(torch.int32), g[6 * part:6 * part + 6].view(torch.int32)) for g in got)
        lp, en, ids, tl = (g[:6] for g in got)
        assert lp[0] == -math.inf and en[0] == 0 and (tl[0] == -math.inf).all()
        assert ids[0].tolist() == list(range(k))
        assert torch.isnan(lp[1:5]).all() and torch.isnan(en[1:5]).all() and torch.isnan(tl[1:5]).all()
        assert ids[1, :2].tolist() == [77, 4000] and ids[2, 0] == 123 and ids[3].tolist() == list(range(k))
        assert ids[4, :3].tolist() == [9, 8, 3000]
        check_answers(plain[None].to(ty), t[5:], k, (lp[5:], en[5:], ids[5:], tl[5:]))
        lp, en, ids, tl = answers(ops, y, i32([-1] * 6 * many), k)
        assert (lp == 0).all()


def test_token_logprobs_outputs_are_optional(ops):
    x = torch.randn(5, 3001, device="cuda", generator=gen(3)).bfloat16()
    t = i32([1, 2, 3, 4, 5])
    full = answers(ops, x, t, 7)
    for which in ("l", "e", "i", "t", "le", "it", "ei"):
        part = answers(ops, x, t, 7, which)
        for name, a, b in zip("leit", part, full):
            if name in which:
                assert torch.equal(a, b), which
            else:
                assert ((a == 9) | (a == -9)).all()


def test_token_logprobs_rows_far_apart(ops):
    """Row offsets past 2^31 values."""
    vocab, ld = 40000, 1200000007
    buf = torch.empty(2 * ld + vocab, device="cuda", dtype=torch.bfloat16)
    x = buf.as_strided((3, vocab), (ld, 1))
    x.copy_(torch.randn(3, vocab, device="cuda", generator=gen(4)))
    t = i32([1, 39999, 7])
    check_answers(x, t, 5, answers(ops, x, t, 5))


# ------------------------------------------------------------------ as they are used
def test_refuses_memory_that_is_not_the_devices(ops):
    kp, vp, table, _, _ = paged([20], 16, 1, 64, False, 1)
    cache = ops.KvCache.of(kp, vp, table)
    q = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    ws = torch.zeros(ops.attention_paged_workspace(cache, 2), device="cuda", dtype=torch.uint8)
    with pytest.raises(ops.IrisCudaError, match="not memory of device"):
        ops.attention_paged(cache, q, q.cpu(), None, i32([3]), scale=1.0, workspace=ws)
    with pytest.raises(ops.IrisCudaError, match="workspace of"):
        ops.attention_paged(cache, q, q, None, i32([3]), scale=1.0, workspace=ws[:0 if len(ws) <= 16 else 16].new_zeros(8))
    x = torch.zeros(2, 100)
    with pytest.raises(ops.IrisCudaError, match="not memory of device"):
        ops.token_logprobs(x, None, None, torch.zeros(2, device="cuda"), None, None, workspace=ws.new_zeros(1 << 20))
    kv = torch.zeros(1, 64, device="cuda")
    with pytest.raises(ops.IrisCudaError, match="not memory of device"):
        ops.rope_append(cache, None, None, None, kv, kv, i32([0]).cpu(), i32([0]), heads=0)


class Tiny:
    """One attention layer and a head on it, over the operators and in 64 bits."""

    def __init__(self, ops, seqs, longest, seed):
        g = gen(seed)
        self.ops, self.nh, self.nkv, self.d, self.hid, self.vocab = ops, 6, 2, 64, 96, 701
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.emb = r(self.vocab, self.hid)
        self.wqkv = r(self.hid, (self.nh + 2 * self.nkv) * self.d) / self.hid ** 0.5
        self.wo = (2 * r(self.nh * self.d, self.vocab) / (self.nh * self.d) ** 0.5)
        self.qn, self.kn = 1 + 0.1 * r(self.d), 1 + 0.1 * r(self.d)
        self.rope = ops.Rope.of(self.d, 1e4)
        page, blocks = 16, -(-longest // 16)
        self.kp, self.vp = (pool(seqs * blocks, page, self.nkv, self.d, False) for _ in range(2))
        table = torch.randperm(seqs * blocks, generator=torch.Generator().manual_seed(seed)).view(seqs, blocks).int().cuda()
        self.cache = ops.KvCache.of(self.kp, self.vp, table)
        self.ws = torch.empty(ops.attention_paged_workspace(self.cache, self.nh), device="cuda", dtype=torch.uint8)

    def buffers(self, n):
        e = lambda *s, t=torch.float32: torch.zeros(*s, device="cuda", dtype=t)  # noqa: E731
        return dict(q=e(n, self.nh, self.d, t=torch.bfloat16), o=e(n, self.nh, self.d, t=torch.bfloat16), lp=e(n), en=e(n),
                    ids=e(n, 4, t=torch.int32), tl=e(n, 4),
                    ws=torch.empty(self.ops.token_logprobs_workspace(n, self.vocab), device="cuda", dtype=torch.uint8))

    def step(self, ids, seq, pos, targets, b, st=None):
        st = stream() if st is None else st
        nh, nkv, d = self.nh, self.nkv, self.d
        qkv = self.emb[ids.long()] @ self.wqkv
        q, k, v = qkv[:, :nh * d], qkv[:, nh * d:(nh + nkv) * d], qkv[:, (nh + nkv) * d:]
        self.ops.rope_append(self.cache, self.rope, b["q"], q, k, v, seq, pos, heads=nh, q_norm=self.qn, k_norm=self.kn, stream=st)
        self.ops.attention_paged(self.cache, b["o"], b["q"], seq, pos, scale=d ** -0.5, workspace=self.ws, stream=st)
        logits = b["o"].view(len(ids), -1).float() @ self.wo
        self.ops.token_logprobs(logits, targets, b["lp"], b["en"], b["ids"], b["tl"], workspace=b["ws"], stream=st)
        return b

    def logprobs64(self, ids):
        """log softmax after every token of one sequence."""
        nh, nkv, d = self.nh, self.nkv, self.d
        qkv = self.emb[ids.long()].double().cpu() @ self.wqkv.double().cpu()
        t = len(ids)
        x = qkv.view(t, nh + 2 * nkv, d)
        freqs = [z / 2.0 ** 64 * 2 * math.pi for z in self.rope.turns[:d // 2]]
        P = torch.arange(t)
        q, _ = rotate64(x[:, :nh], P, freqs, False, 1.0, self.qn)
        k, _ = rotate64(x[:, nh:nh + nkv], P, freqs, False, 1.0, self.kn)
        k, v = (y.repeat_interleave(nh // nkv, 1) for y in (k, x[:, nh + nkv:]))
        s = torch.einsum("ihd,jhd->hij", q, k) * d ** -0.5
        s = s.masked_fill(torch.triu(torch.ones(t, t, dtype=torch.bool), 1), -math.inf)
        o = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(t, nh * d)
        return torch.log_softmax(o @ self.wo.double().cpu(), -1)


def test_a_run_together(ops):
    """Prompts of three sequences in one call, then tokens one at a time, captured and replayed.

    Logits are sums of 384 products of an output (bf16: q, k, v, o rounded, 2^-8 each) and weights of size
    2 / sqrt(384): independent errors of about 3 * 2^-9 of an output of size < 1 give a log probability within
    about 2 * 2^-8 standard deviations; 0.06 is some 8 of them."""
    lens, new = [37, 5, 64], 12
    m = Tiny(ops, 3, 96, 21)
    toks = [torch.randint(0, m.vocab, (n + new + 1,), device="cuda", generator=gen(n), dtype=torch.int32) for n in lens]
    seq = i32([i for i, n in enumerate(lens) for _ in range(n)] + [-1, -1])  # two padding rows behind the last sequence
    pos = i32([p for n in lens for p in range(n)] + [0, 0])
    ids = torch.cat([t[:n] for t, n in zip(toks, lens)] + [toks[0][:2]])
    targets = torch.cat([t[1:n + 1] for t, n in zip(toks, lens)] + [i32([-1, -1])])
    b = m.step(ids, seq, pos, targets, m.buffers(len(ids)))
    torch.cuda.synchronize()
    want = [m.logprobs64(t[:-1]) for t in toks]
    at = 0
    for t, n, w in zip(toks, lens, want):
        ref = w[:n].gather(1, t[1:n + 1].long().cpu()[:, None])[:, 0]
        assert (b["lp"][at:at + n].cpu() - ref).abs().max() < 0.06
        ent = -(w[:n].exp() * w[:n]).sum(-1)
        assert (b["en"][at:at + n].cpu() - ent).abs().max() < 0.06
        top = w[:n].gather(1, b["ids"][at:at + n].long().cpu())
        assert (b["tl"][at:at + n].cpu() - top).abs().max() < 0.06
        at += n
    assert (b["lp"][at:] == 0).all() and (b["q"][at:] == 0).all() and (b["o"][at:] == 0).all()
    # one token at a time on a side stream, as a captured step
    d = m.buffers(3)
    cid, ctg, cpos, cseq = i32([0] * 3), i32([0] * 3), i32(lens) - 1, i32([0, 1, 2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(cid, i32([-1] * 3), cpos, ctg, d)  # warm up on padding: writes nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            m.step(cid, cseq, cpos, ctg, d)
        for j in range(new):
            cid.copy_(torch.stack([t[n + j] for t, n in zip(toks, lens)]))
            ctg.copy_(torch.stack([t[n + j + 1] for t, n in zip(toks, lens)]))
            cpos += 1
            g.replay()
            ref = torch.stack([w[n + j, int(t[n + j + 1])] for t, n, w in zip(toks, lens, want)])
            side.synchronize()
            assert (d["lp"].cpu() - ref).abs().max() < 0.06, j


def test_two_streams_at_once(ops):
    """Independent calls on two streams, each with its own workspace."""
    kp, vp, table, ks, vs = paged([900, 300], 16, 2, 128, False, 31)
    q = torch.randn(2, 8, 128, device="cuda", generator=gen(9)).bfloat16()
    cache = ops.KvCache.of(kp, vp, table)
    pos = i32([899, 299])
    first = attend(ops, kp, vp, table, q, pos)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(q) for _ in range(2)]
    wss = [torch.empty(ops.attention_paged_workspace(cache, 8), device="cuda", dtype=torch.uint8) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, o, ws in zip(streams, outs, wss):
            ops.attention_paged(cache, o, q, None, pos, scale=128 ** -0.5, workspace=ws, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
