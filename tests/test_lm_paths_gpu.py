"""Each way of working of the paged-cache attention by itself: a call's way goes by
its counts and the room of its table, so that a small test takes the kernel of
few rows whatever it was written for.  A table with room for many more keys
(entries of no page behind the sequence's own) takes the two-kernel ways: the
number of kernels of every call is checked.  Cases and tolerances are those of
the tests of runs of rows, with such tables."""
import math

import pytest
import torch

import test_lm_runs_gpu as runs
from test_lm_ops_gpu import attention64, gen, i32, ops, paged, stream  # noqa: F401

pytestmark = pytest.mark.gpu


def with_room(table, page, keys=40000):
    """The same pages in a table with room for `keys` more keys a sequence (over 72 tiles: no way of few rows)."""
    roomy = torch.full((table.shape[0], table.shape[1] + keys // page), -1, device="cuda", dtype=torch.int32)
    roomy[:, :table.shape[1]] = table
    return roomy


def roomy_paged(lens, page, nkv, d, hm, seed):
    kp, vp, table, ks, vs = paged(lens, page, nkv, d, hm, seed)
    return kp, vp, with_room(table, page), ks, vs


class Counted:
    """The binding, every attention call of which has to take `kernels` kernels."""

    def __init__(self, ops, kernels):
        self.ops, self.kernels = ops, kernels

    def __getattr__(self, name):
        return getattr(self.ops, name)

    def attention_paged(self, *args, **kw):
        n = self.ops.lib().iris_cuda_kernel_launches()
        self.ops.attention_paged(*args, **kw)
        assert self.ops.lib().iris_cuda_kernel_launches() - n == self.kernels


@pytest.fixture
def two_kernels(ops, monkeypatch):
    monkeypatch.setattr(runs, "paged", roomy_paged)
    return Counted(ops, 2)


@pytest.mark.parametrize("lens,new,nh,nkv,d,page,hm", runs.RUNS)
def test_runs(two_kernels, lens, new, nh, nkv, d, page, hm):
    assert sum(new) >= 4 * len(lens)
    runs.test_attention_paged_runs(two_kernels, lens, new, nh, nkv, d, page, hm)


@pytest.mark.parametrize("d", (64, 128, 256))
def test_runs_in_any_order(two_kernels, d):
    runs.test_attention_paged_runs_in_any_order(two_kernels, d)


@pytest.mark.parametrize("d", (64, 128, 256))
@pytest.mark.parametrize("value", (float("nan"), float("inf"), -float("inf")))
def test_runs_see_nothing_of_later_tokens(two_kernels, d, value):
    runs.test_attention_paged_runs_see_nothing_of_later_tokens(two_kernels, d, value)


def test_runs_pages_out_of_range(two_kernels):
    runs.test_attention_paged_runs_pages_out_of_range(two_kernels)


def test_runs_captured(two_kernels):
    runs.test_attention_paged_runs_captured(two_kernels)


def test_a_run_with_holes_at_every_width(two_kernels):
    """Pages outside the pool among those of a run, at every head_dim."""
    for d in (64, 128, 256):
        kp, vp, table, ks, vs = roomy_paged([200], 16, 2, d, False, 41)
        table[0, 3], table[0, 4], table[0, 9] = -1, kp.shape[0], -2 ** 31
        keep = torch.tensor([b not in (3, 4, 9) for b in range(13)]).repeat_interleave(16)
        pos = list(range(30, 200))
        q = torch.randn(len(pos), 8, d, device="cuda", generator=gen(42)).bfloat16()
        out = runs.attend(two_kernels, kp, vp, table, q, i32(pos), i32([0] * len(pos)))
        for i, p in enumerate(pos):
            sel = keep[:p + 1]
            want, tol = attention64(q[i], ks[0].cpu()[:p + 1][sel], vs[0].cpu()[:p + 1][sel], 1 / math.sqrt(d))
            assert ((out[i].double().cpu() - want).abs() <= tol).all(), (d, i)


def test_streams_at_once(ops):
    """Calls that leave pieces in their workspaces, on three streams at once: rows by themselves of two kinds, runs."""
    kp, vp, table, ks, vs = paged([9000, 700, 3000], 16, 2, 128, False, 43)
    calls = []
    for seed, seq, pos in ((44, [0, 1, 2], [8999, 699, 2999]), (45, [2, 0], [2500, 8000]), (46, [0] * 40, list(range(8900, 8940)))):
        q = torch.randn(len(seq), 8, 128, device="cuda", generator=gen(seed)).bfloat16()
        tab = with_room(table, 16)
        cache = ops.KvCache.of(kp, vp, tab)
        ws = torch.full((ops.attention_paged_workspace(cache, 8),), 255, device="cuda", dtype=torch.uint8)
        calls.append((Counted(ops, 2), cache, torch.zeros_like(q), q, i32(seq), i32(pos), ws, torch.cuda.Stream(), seq, pos))
    torch.cuda.synchronize()
    for _ in range(20):
        for o, cache, out, q, seq, pos, ws, st, *_ in calls:
            o.attention_paged(cache, out, q, seq, pos, scale=128 ** -0.5, workspace=ws, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for o, cache, out, q, seq, pos, ws, st, hs, hp in calls:
        runs.check(out, q, hs, hp, ks, vs)
        alone = torch.zeros_like(q)
        o.attention_paged(cache, alone, q, seq, pos, scale=128 ** -0.5, workspace=ws, stream=stream())
        assert torch.equal(out, alone)


WAYS = [  # way, rows' positions, query heads on one key-value head, kernels
    ("few", [511, 140, 69], 4, 1), ("few", [511, 320, 140], 12, 1), ("line", [511, 320, 250, 132, 100, 69], 4, 2),
    ("line", [511, 140, 69], 12, 2), ("runs", [511, 132, 250, 69], 4, 2), ("runs", [511, 505, 400, 140, 69, 320, 132, 250], 12, 2),
    ("runs", [511, 460, 500, 448], 4, 2), ("runs", [511, 460, 455, 450, 449, 448, 500, 501], 12, 2),
]


@pytest.mark.parametrize("d", (64, 128, 256))
@pytest.mark.parametrize("way,pos,nh,kernels", WAYS)
def test_values_that_are_not_finite(ops, way, pos, nh, kernels, d):
    """A value that is an infinity or NaN, under an ordinary weight, one of 2^-40 to 2^-90 of the largest, one that is 0 in f32, and a score of
    -inf: its column of the rows that see it is not finite, and is the infinity where the weight is 2^-100 or more; every
    other column is as without it (keys whose weight is 0 add nothing there, so that they are left out of the 64-bit form)."""
    seqs = len(pos) if way == "line" else 1   # with as many sequences as rows no runs
    lens = [512] + [1] * (seqs - 1)
    kp, vp, table, ks, vs = paged(lens, 16, 1, d, False, 47)
    if way != "few":
        table = with_room(table, 16)
    cell = lambda x, p: x[int(table[0, p // 16]), p % 16, 0]  # noqa: E731
    odd = {3: (70, math.inf), 6: (130, -math.inf), 8: (135, -math.inf), 9: (200, math.inf), 11: (300, math.nan)}
    q = torch.randn(len(pos), nh, d, device="cuda", generator=gen(48)).bfloat16()
    q[:, :, 0] = 8.0  # column 0 makes keys lighter: scores in powers of 2 of 8 * -50 / sqrt(d) log2(e) = -72, -51, -36
    keep = torch.ones(512, dtype=torch.bool)
    for p in range(512):
        if p in (130, 135) or 192 <= p < 256:
            cell(kp, p)[0] = {130: -4000.0, 135: -50.0}.get(p, -math.inf)  # -4000: weight 0; 192 ..: four units' whole tile
            keep[p] = p == 135
        else:
            cell(kp, p)[0] = 0.0
        ks[0][p, 0] = cell(kp, p)
    for col, (p, x) in odd.items():
        cell(vp, p)[col] = x
    seq = [0] * len(pos)
    out = torch.full_like(q, 9.0)
    cache = ops.KvCache.of(kp, vp, table)
    ws = torch.full((ops.attention_paged_workspace(cache, nh),), 255, device="cuda", dtype=torch.uint8)
    Counted(ops, kernels).attention_paged(cache, out, q, i32(seq), i32(pos), scale=1 / math.sqrt(d), workspace=ws, stream=stream())
    torch.cuda.synchronize()
    for i, n in enumerate(pos):
        got = out[i].double().cpu()
        sel = keep[:n + 1]
        want, tol = attention64(q[i], ks[0].cpu()[:n + 1][sel], vs[0].cpu()[:n + 1][sel], 1 / math.sqrt(d))
        seen = [c for c, (p, _) in odd.items() if p <= n]
        rest = [c for c in range(d) if c not in seen]
        assert ((got - want).abs() <= tol)[:, rest].all(), (i, n)
        assert not torch.isfinite(got[:, seen]).any(), (i, n, got[0, seen])
        for c in (3, 8):
            assert odd[c][0] > n or (got[:, c] == odd[c][1]).all(), (i, n, c)
        assert 11 not in seen or torch.isnan(got[:, 11]).all()


@pytest.mark.parametrize("way,pos,nh,kernels", WAYS)
def test_scores_that_are_not_finite(ops, way, pos, nh, kernels):
    """Scores of -inf alone: zeros.  One of +inf or NaN: the head is NaN in the rows that see the key."""
    d = 128
    for value, at in ((-math.inf, 0), (math.inf, 100), (math.nan, 100)):
        seqs = len(pos) if way == "line" else 1
        kp, vp, table, ks, vs = paged([512] + [1] * (seqs - 1), 16, 1, d, False, 49)
        if way != "few":
            table = with_room(table, 16)
        q = torch.randn(len(pos), nh, d, device="cuda", generator=gen(50)).bfloat16()
        q[:, :, 0] = 1.0
        for p in range(512) if at == 0 else (at,):
            kp[int(table[0, p // 16]), p % 16, 0, 0] = value
        cache = ops.KvCache.of(kp, vp, table)
        ws = torch.full((ops.attention_paged_workspace(cache, nh),), 255, device="cuda", dtype=torch.uint8)
        out = torch.full_like(q, 9.0)
        Counted(ops, kernels).attention_paged(cache, out, q, i32([0] * len(pos)), i32(pos), scale=1 / math.sqrt(d), workspace=ws,
                                              stream=stream())
        torch.cuda.synchronize()
        for i, n in enumerate(pos):
            got = out[i].double().cpu()
            if at == 0:
                assert (got == 0).all(), (i, n)
            elif n >= at:
                assert torch.isnan(got).all(), (i, n)
            else:
                want, tol = attention64(q[i], ks[0][:n + 1], vs[0][:n + 1], 1 / math.sqrt(d))
                assert ((got - want).abs() <= tol).all(), (i, n)
