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
