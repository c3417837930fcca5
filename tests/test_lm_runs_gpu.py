"""Attention of several rows of a sequence over the paged cache (the tokens of
prompts), which takes runs of rows together: against the plain form in 64 bits
with the tolerance derived beside it."""
import math

import pytest
import torch

from test_lm_ops_gpu import attend, attention64, gen, i32, ops, paged, stream  # noqa: F401

pytestmark = pytest.mark.gpu


def check(out, q, seq, pos, ks, vs, scale=None, rows=None):
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    for i in range(len(seq)) if rows is None else rows:
        s, n = seq[i], max(0, pos[i] + 1)
        got = out[i].view(q.shape[1], -1)
        if not 0 <= s < len(ks):
            assert (got == 9).all(), i
            continue
        want, tol = attention64(q[i], ks[s][:n], vs[s][:n], scale)
        assert ((got.double().cpu() - want).abs() <= tol).all(), (i, s, n)


RUNS = [  # lengths, new tokens of each, heads, kv heads, d, page, head major
    ([16], [16], 32, 8, 128, 16, False),
    ([4], [4], 4, 4, 128, 16, True),
    ([4000], [4], 4, 4, 128, 16, True),         # four pairs a unit
    ([129], [129], 8, 8, 128, 7, False),        # 64 rows of one head
    ([300, 65, 1, 64], [300, 65, 1, 64], 8, 2, 128, 16, True),
    ([1000, 1500], [3, 5], 12, 2, 128, 33, False),
    ([700], [75], 10, 2, 64, 16, False),        # 5 heads: 12 rows
    ([200, 90], [130, 90], 34, 2, 64, 1, True),  # 17 heads: 16 and 1
    ([150], [150], 14, 1, 64, 64, False),
    ([260], [70], 9, 1, 256, 16, True),         # 9 heads: 7 rows
    ([100, 333], [100, 40], 4, 2, 256, 50, False),
    ([5000], [9], 16, 1, 128, 16, False),       # one unit, cut into many pieces
    ([6000], [33], 3, 1, 64, 16, False),
    ([3000], [10], 32, 1, 256, 16, False),
]


@pytest.mark.parametrize("lens,new,nh,nkv,d,page,hm", RUNS)
def test_attention_paged_runs(ops, lens, new, nh, nkv, d, page, hm):
    kp, vp, table, ks, vs = paged(lens, page, nkv, d, hm, 21)
    seq = [s for s, m in enumerate(new) for _ in range(m)]
    pos = [p for n, m in zip(lens, new) for p in range(n - m, n)]
    q = torch.randn(len(seq), nh, d, device="cuda", generator=gen(22)).bfloat16()
    out = attend(ops, kp, vp, table, q, i32(pos), i32(seq))
    check(out, q, seq, pos, ks, vs)
    assert torch.equal(out, attend(ops, kp, vp, table, q, i32(pos), i32(seq)))


@pytest.mark.parametrize("d", (64, 128, 256))
def test_attention_paged_runs_in_any_order(ops, d):
    """Rows of sequences and positions in any order, rows that see nothing, padding, the same row twice, row strides."""
    kp, vp, table, ks, vs = paged([170, 1, 90], 16, 2, d, False, 23)
    g = torch.Generator().manual_seed(24)
    seq = torch.randint(0, 3, (40,), generator=g).tolist() + [0] * 30 + [-1, 3, 2, 2, 2, 2 ** 31 - 1, -2 ** 31, 1, 0, 0]
    n = [170, 1, 90]
    pos = [int(torch.randint(-2, n[s], (1,), generator=g)) if 0 <= s < 3 else 7 for s in seq]
    pos[-1] = pos[-2] = 100
    q = torch.randn(len(seq), 6, d, device="cuda", generator=gen(25)).bfloat16()
    q[-1] = q[-2]
    wide = torch.full((len(seq), 6 * d + 24), 9.0, device="cuda", dtype=torch.bfloat16)
    wq = torch.full((len(seq), 6 * d + 8), float("nan"), device="cuda", dtype=torch.bfloat16)
    wq[:, :6 * d] = q.view(len(seq), -1)
    cache = ops.KvCache.of(kp, vp, table)
    ws = torch.full((ops.attention_paged_workspace(cache, 6),), 255, device="cuda", dtype=torch.uint8)
    ops.attention_paged(cache, wide[:, :6 * d], wq[:, :6 * d], i32(seq), i32(pos), scale=-0.05, workspace=ws, stream=stream())
    check(wide[:, :6 * d], q, seq, pos, ks, vs, scale=-0.05)
    assert torch.equal(wide[-1], wide[-2])
    assert (wide[:, 6 * d:] == 9).all()


@pytest.mark.parametrize("d", (64, 128, 256))
@pytest.mark.parametrize("value", (float("nan"), float("inf"), -float("inf")))
def test_attention_paged_runs_see_nothing_of_later_tokens(ops, d, value):
    """A key or value that is an infinity or NaN shows in the rows that see it, and in no other."""
    kp, vp, table, ks, vs = paged([150], 16, 2, d, False, 26)
    at = lambda x, p: x[int(table[0, p // 16]), p % 16]  # noqa: E731
    at(vp, 100)[0, 3], at(vp, 101)[1, d - 1], at(kp, 120)[0] = value, value, float("nan")
    pos = list(range(60, 150))
    q = torch.randn(len(pos), 8, d, device="cuda", generator=gen(27)).bfloat16()
    out = attend(ops, kp, vp, table, q, i32(pos), i32([0] * len(pos))).float()
    clean = [p for p in range(len(pos)) if pos[p] < 100]
    check(out, q, [0] * len(pos), pos, ks, vs, rows=clean)
    bad = torch.zeros(len(pos), 8, d, dtype=torch.bool)
    bad[40:, :4, 3], bad[41:, 4:, d - 1], bad[60:, :4] = True, True, True
    assert torch.equal(torch.isfinite(out).cpu(), ~bad)
    if not math.isnan(value):
        assert (out[40:60, :4, 3] == value).all() and (out[41:, 4:, d - 1] == value).all()
    else:
        assert torch.isnan(out[40:, :4, 3]).all()


def test_attention_paged_runs_pages_out_of_range(ops):
    """Positions past the table see the table's keys; pages outside the pool are not seen, and hold nothing."""
    page, d = 16, 128
    kp, vp, table, ks, vs = paged([128, 128], page, 1, d, False, 28)
    table[0, 2], table[0, 5], table[1, :] = -3, 2 ** 31 - 1, kp.shape[0]
    pos = [2 ** 31 - 1, 127, 90, 47, 40, 20, 5, 127, 3]
    seq = [0] * 7 + [1, 1]
    q = torch.randn(9, 4, d, device="cuda", generator=gen(29)).bfloat16()
    out = attend(ops, kp, vp, table, q, i32(pos), i32(seq))
    keep = torch.tensor([b not in (2, 5) for b in range(8)]).repeat_interleave(page)
    for i in range(7):
        n = min(128, pos[i] + 1)
        want, tol = attention64(q[i], ks[0].cpu()[:n][keep[:n]], vs[0].cpu()[:n][keep[:n]], 1 / math.sqrt(d))
        assert ((out[i].double().cpu() - want).abs() <= tol).all(), i
    assert (out[7:] == 0).all()


@pytest.mark.parametrize("rows,nh,nkv,d,longest", [(30, 32, 8, 128, 256), (37, 8, 8, 128, 500), (70, 8, 4, 64, 130), (12, 16, 8, 256, 300), (9, 32, 8, 128, 512)])
def test_attention_paged_a_block_a_unit(ops, rows, nh, nkv, d, longest):
    """As many units as the device holds blocks or half of them, short tables: sequences of no key to all, padding."""
    lens = [(i * 37) % (longest + 1) for i in range(rows - 2)] + [longest, 1]
    kp, vp, table, ks, vs = paged(lens, 16, nkv, d, False, 32)
    pos = [n - 1 for n in lens]
    seq = list(range(rows))
    seq[3], seq[5] = -1, rows
    q = torch.randn(rows, nh, d, device="cuda", generator=gen(33)).bfloat16()
    out = attend(ops, kp, vp, table, q, i32(pos), i32(seq))
    check(out, q, seq, pos, ks, vs)
    assert torch.equal(out, attend(ops, kp, vp, table, q, i32(pos), i32(seq)))


def test_attention_paged_runs_captured(ops):
    """A captured call sees the positions, sequences and pages of its replay."""
    kp, vp, table, ks, vs = paged([400, 200], 16, 2, 128, False, 30)
    q = torch.randn(64, 8, 128, device="cuda", generator=gen(31)).bfloat16()
    seq, pos = i32([0] * 64), i32(list(range(64)))
    cache = ops.KvCache.of(kp, vp, table)
    ws = torch.full((ops.attention_paged_workspace(cache, 8),), 255, device="cuda", dtype=torch.uint8)
    out = torch.full_like(q, 9.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        ops.attention_paged(cache, out, q, seq, pos, scale=0.1, workspace=ws, stream=side.cuda_stream)
    for s, p in (([0] * 64, list(range(64))), ([0] * 40 + [1] * 20 + [-1] * 4, list(range(300, 364))),
                 ([1, 0] * 32, list(range(100, 164)))):
        p = [min(x, 199) if y == 1 else x for x, y in zip(p, s)]
        seq.copy_(i32(s)), pos.copy_(i32(p)), out.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(out, q, s, p, ks, vs, scale=0.1)
