"""Sampling, the 8-bit cache and 4-bit weights on the GPU against plain 64-bit forms: small weights, the kernels that
large calls get, magnitudes at the ends of the range.

Tolerances (u = 2^-24, half an f32 step; 2^-8 half a bf16 step, relative):

attention_paged8: 2^-8 of the value and, times A = sum p |v|: 4 hd u S for the scores (S the largest sum of scale |q k|), len u
  for the sums, 8 u (T + 15) for the rounding of the exponent, which has five roundings of numbers up to T + 15 (T the largest
  magnitude of a key's score and scale in powers of two, 15 what they are raised by; numerator and denominator see them) times
  ln 2, and 2^-21 for the exponential (2^-22) and weights of 22 bits.  Weights under 2^-25 of the largest weight times scale W
  come in steps of 2^-39 of it (their second part is a multiple of 2^-24 where the largest is 2^15), rounded: 2^-40 448 W a
  key.
Products with 4-bit weights and appends: as in test_lm_serving_gpu, whose checks they go through.
"""
import ctypes
import math

import numpy as np
import pytest

import test_lm_serving_gpu as serving
from test_lm_ops_gpu import BF, U, gen, i32, stream
from test_lm_serving_gpu import E4, one_sequence8, ops, values8  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def attention8_fine64(q, k, v, vs, scale):
    """q [heads, d], k / v [len, d], vs [len] scales of the values -> (out, tolerance) [heads, d]."""
    n, d = k.shape
    q = q.double().cpu()
    s = scale * q @ k.t()
    p = torch.softmax(s, -1)
    size = abs(scale) * (q.abs() @ k.abs().t()).amax(-1)
    t = (s * math.log2(math.e) + torch.log2(vs)).abs().amax(-1)
    out, a = p @ v, p @ v.abs()
    slack = (4 * d * U * size + n * U + 8 * U * (t + 15) + 2.0 ** -21)[:, None] * a
    return out, BF * out.abs() + slack + (n * 2.0 ** -40 * 448 * (p * vs).amax(-1))[:, None]


def check_one_sequence8(ops, n, new, q, k, v, ke, ve, table, block, scale):  # noqa: F811
    """The newest `new` rows of a sequence of n keys, all heads on one."""
    cache = ops.KvCache8.of(k, v, ke, ve, table)
    heads, d = q.shape[1:]
    out = torch.zeros_like(q)
    ws = torch.empty(ops.attention_paged8_workspace(cache, heads), device="cuda", dtype=torch.uint8)
    ops.attention_paged8(cache, out, q, i32([0] * new), i32(range(n - new, n)), scale=scale, workspace=ws, stream=stream())
    torch.cuda.synchronize()
    kv, vv = (values8(p, e, block).flatten(0, 2) for p, e in ((k, ke), (v, ve)))
    vs = 2.0 ** (ve.cpu().double().repeat_interleave(block, 1).flatten() - 127)
    scale = float(np.float32(scale))
    for r in range(new):
        at = n - new + r + 1
        want, tol = attention8_fine64(q[r], kv[:at], vv[:at], vs[:at], scale)
        err = (out[r].double().cpu() - want).abs()
        assert (err <= tol).all(), (r, float(err.max()), float(want.abs().max()), float((err / tol).max()))


@pytest.mark.parametrize("d", (64, 128, 256))
@pytest.mark.parametrize("n,new,heads", [(300, 1, 4), (5000, 1, 16), (300, 90, 4), (200, 130, 16)])
@pytest.mark.parametrize("kind", ("cancel", "steps", "many", "scales"))
def test_attention_paged8_small_weights(ops, kind, n, new, heads, d):  # noqa: F811
    """Weights that differ in their 13th bit and cancel; light ones beside a key of weight 1 that is 0 in half the columns:
    between two steps of an f16 at 2^-20, all under 2^-28, and as light by the values' scales alone."""
    block = 16
    k, v, ke, ve, table = one_sequence8(ops, n, d, block)
    pages, page = k.shape[:2]
    k.zero_()
    flat_k, flat_v = k.view(pages * page, d), v.view(pages * page, d)
    q = torch.randn(new, heads, d, device="cuda", generator=gen(7)).bfloat16()
    q[..., 0] = 1.0
    one = torch.ones(d, device="cuda")
    scale = 1.0
    if kind == "cancel":
        flat_k[1::2, 0] = (-one[:1]).to(E4)
        flat_v[0::2], flat_v[1::2] = one.to(E4), (-one).to(E4)
        scale = 2.0 ** -13
    else:
        flat_v.copy_(one.expand(pages * page, d).to(E4))
        flat_v[0, :d // 2] = torch.zeros(d // 2, device="cuda").to(E4)
        flat_k[0, 0] = (one[0] * {"steps": 14.0, "many": 20.0, "scales": 1.0}[kind]).to(E4)
        if kind == "steps":
            scale = math.log(2) * (24 - math.log2(10.5)) / 14  # the others weigh 10.5 * 2^-24
        if kind == "scales":
            scale = 0.3
            ve[1:] = 127 - 25
            flat_v[1:block] = torch.zeros(d, device="cuda").to(E4)
    check_one_sequence8(ops, n, new, q, k, v, ke, ve, table, block, scale)


@pytest.mark.parametrize("d", (64, 128, 256))
@pytest.mark.parametrize("n,new,heads", [(300, 1, 4), (200, 130, 16)])
def test_attention_paged8_large_queries_on_columns_of_zeros(ops, n, new, heads, d):  # noqa: F811
    """A query of 2^120 on a column in which keys of scale 2^33 are 0: scores of 0, all keys weigh alike."""
    k, v, ke, ve, table = one_sequence8(ops, n, d, 16)
    k.view(-1, d)[:, 0] = torch.zeros(1, device="cuda").to(E4)
    ke.fill_(127 + 33)
    q = torch.zeros(new, heads, d, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 2.0 ** 120
    check_one_sequence8(ops, n, new, q, k, v, ke, ve, table, 16, 1 / math.sqrt(d))


def kernels_of(call):
    """Names of the kernels that a call launches, from the graph that it is captured into (and that is not run)."""
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    cu, raw, n = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert cu.cuGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert cu.cuGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    names = []
    for node in nodes:
        params, name = (ctypes.c_void_p * 32)(), ctypes.c_char_p()  # the first member is the function
        assert cu.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), params) == 0
        assert cu.cuFuncGetName(ctypes.byref(name), ctypes.c_void_p(params[0])) == 0
        names.append(name.value.decode())
    return names


class Named:
    """The binding, each call `what` of which has to launch one kernel with `kernel` in its mangled name."""

    def __init__(self, ops, what, kernel):  # noqa: F811
        self.ops, self.what, self.kernel = ops, what, kernel

    def __getattr__(self, name):
        call = getattr(self.ops, name)
        if name != self.what:
            return call

        def checked(*args, **kw):
            names = kernels_of(lambda: call(*args, **{**kw, "stream": stream()}))
            assert len(names) == 1 and self.kernel in names[0], (names, self.kernel)
            call(*args, **kw)
        return checked


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


# Every kernel of the products: rows of x, then n of the weights by the number of SMs, so that each rule of the launch is met: many
# rows of the weights; five and three parts of k in a cluster where one warp a strip lets more blocks be there at once; few.
LINEAR_WAYS = {
    "few": ("linear4_kernelILi1ELi8E", (1, 5, 8), lambda: 300, 1),
    "few_head": ("linear4_kernelILi2ELi2E", (1, 3, 8), lambda: 512 * sms() + 1, 0),
    "rows16_one": ("linear4_rows_kernelILi2ELi1E", (9, 12, 16), lambda: 128 * (sms() * 7 // 4 // 5) - 126, 1),
    "rows16_one_3": ("linear4_rows_kernelILi2ELi1E", (16,), lambda: 128 * (sms() * 7 // 4 // 3) - 127, 1),
    "rows16_head": ("linear4_rows_kernelILi2ELi1E", (10,), lambda: 512 * sms() + 77, 0),
    "rows16_two": ("linear4_rows_kernelILi2ELi2E", (9, 13, 16), lambda: 250, 2),
    "rows32_one": ("linear4_rows_kernelILi4ELi1E", (17, 31, 33), lambda: 128 * (sms() * 7 // 4 // 5) - 126, 1),
    "rows32_one_3": ("linear4_rows_kernelILi4ELi1E", (32,), lambda: 128 * (sms() * 7 // 4 // 3) - 127, 1),
    "rows32_head": ("linear4_rows_kernelILi4ELi1E", (32,), lambda: 512 * sms() + 77, 0),
    "rows32_two": ("linear4_rows_kernelILi4ELi2E", (17, 32, 70), lambda: 250, 2),
}


@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 384))
@pytest.mark.parametrize("way", LINEAR_WAYS)
def test_linear4_each_kernel(ops, way, group, zeros):  # noqa: F811
    kernel, rows, n, deep = LINEAR_WAYS[way]
    k = {32: (160, 1440, 4128), 64: (192, 1472, 4160), 384: (384, 1536, 4224)}[group][deep]
    kernel += f"Li{ {32: 1, 64: 2, 384: 4}[group] }ELb{int(zeros)}E"
    for i, r in enumerate(rows):
        f32, add = (i + zeros) % 2 == 0, (None, "same", "other")[(i + group // 32) % 3]
        serving.test_linear4(Named(ops, "linear4", kernel), (r, n(), k, group, zeros, i % 2 == 0, f32, add, 8 * (i % 2)))


# rows beyond 8 an SM, then as test_lm_serving_gpu's: heads, kv heads, d, rot, interleaved, page, block, head major, f32, norm,
# sequences, shuffled
APPEND_MANY = [
    (17, 4, 2, 128, 128, False, 16, 16, False, True, True, 3, False),
    (1, 2, 1, 128, 128, True, 16, 16, True, False, True, 3, True),
    (30, 1, 3, 128, 64, True, 20, 4, False, False, False, 4, True),
    (5, 3, 1, 128, 128, False, 8, 1, True, False, True, 2, False),
    (60, 0, 2, 128, 32, False, 64, 64, False, True, False, 3, True),
    (9, 2, 2, 64, 64, False, 64, 32, False, False, True, 3, True),
    (44, 7, 1, 64, 32, True, 48, 16, True, True, False, 5, False),
    (21, 2, 1, 256, 256, False, 24, 24, False, False, True, 2, False),
    (12, 1, 2, 256, 64, True, 7, 7, True, True, True, 3, True),
]


@pytest.mark.parametrize("case", APPEND_MANY, ids=lambda c: "-".join(map(str, c[:8])))
def test_rope_append8_of_many_tokens(ops, case):  # noqa: F811
    more, nh, nkv, d, f32 = *case[:4], case[9]
    kernel = f"rope_append8_kernelI{'f' if f32 else '13__nv_bfloat16'}Li{d}ELb1E"
    serving.test_rope_append8(Named(ops, "rope_append8", kernel), (8 * sms() + more, *case[1:]))


@pytest.mark.parametrize("rows,vocab,f32", [(3, 1024, True), (3, 1025, False), (500, 1500, False), (450, 16001, True), (200, 40001, False),
                                            (40, 40000, True)])
@pytest.mark.parametrize("steps", (0, 2))
def test_sample_tokens_top_k_in_shares(ops, rows, vocab, f32, steps):  # noqa: F811
    """Top-k around the largest share of a block, with one to eight blocks a row; with steps many tokens are equal."""
    ks = (1, 128, 199, 200, 201, 255, 256, 257, 400, 401, 511, 512, 513)
    x = torch.randn(rows, vocab, device="cuda", generator=gen(vocab)) * 2.5
    if steps:
        x = torch.round(x * steps) / steps
    settings = [(1.0, ks[r % len(ks)], (1.0, 0.97)[r // len(ks) % 2], (0.0, 0.0, 1e-3)[r % 3]) for r in range(rows)]
    serving.check_samples(ops, x if f32 else x.bfloat16(), settings, np.random.default_rng(rows).random(rows).tolist())


@pytest.mark.parametrize("d", (64, 128, 256))
@pytest.mark.parametrize("new,heads", [(1, 4), (80, 4), (80, 16)])
def test_attention_paged8_pages_outside_the_pool(ops, new, heads, d):  # noqa: F811
    """Pages that the pool does not have, in the middle of a sequence and at its ends: their keys are not seen."""
    n, block = 300, 8
    k, v, ke, ve, table = one_sequence8(ops, n, d, block)
    pages, page = k.shape[:2]
    table[0, 0], table[0, 3], table[0, 9], table[0, 18] = -1, pages, 2 ** 31 - 1, -2 ** 31
    q = torch.randn(new, heads, d, device="cuda", generator=gen(3)).bfloat16()
    out = torch.zeros_like(q)
    cache = ops.KvCache8.of(k, v, ke, ve, table)
    ws = torch.empty(ops.attention_paged8_workspace(cache, heads), device="cuda", dtype=torch.uint8)
    scale = 2.0 ** -4
    ops.attention_paged8(cache, out, q, i32([0] * new), i32(range(n - new, n)), scale=scale, workspace=ws, stream=stream())
    torch.cuda.synchronize()
    kv, vv = (values8(p, e, block).flatten(0, 2) for p, e in ((k, ke), (v, ve)))
    held = ((table[0] >= 0) & (table[0] < pages)).cpu().repeat_interleave(page)
    for r in range(new):
        seen = held.clone()
        seen[n - new + r + 1:] = False
        want, tol = attention8_fine64(q[r], kv[seen], vv[seen], torch.ones(int(seen.sum()), dtype=torch.float64), scale)
        assert ((out[r].double().cpu() - want).abs() <= tol).all(), r
