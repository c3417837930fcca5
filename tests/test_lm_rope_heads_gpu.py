"""The rotary append with more heads than a block's lanes take at once: every head
of every token is written, whether a block has one slice of them or several."""
import pytest
import torch

from test_lm_ops_gpu import gen, i32, near, ops, pool, rotate64, stream  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", (1, 30, 400))
@pytest.mark.parametrize("heads,kv_heads,d", [(129, 3, 64), (37, 37, 128), (250, 5, 256), (0, 41, 128)])
def test_many_heads(ops, tokens, heads, kv_heads, d):
    x = torch.randn(tokens, (heads + 2 * kv_heads) * d, device="cuda", generator=gen(heads + tokens)).bfloat16()
    q, k, v = x[:, :heads * d], x[:, heads * d:(heads + kv_heads) * d], x[:, (heads + kv_heads) * d:]
    kp, vp = pool(tokens, 1, kv_heads, d, False), pool(tokens, 1, kv_heads, d, False)
    out = torch.full((tokens, heads, d), 7.0, device="cuda", dtype=torch.bfloat16)
    rope = ops.Rope.of(d, 1e4)
    freqs = [t / 2.0 ** 64 * 2 * torch.pi for t in rope.turns[:d // 2]]
    cache = ops.KvCache.of(kp, vp, i32([list(range(tokens))]))
    ops.rope_append(cache, rope, out if heads else None, q if heads else None, k, v, i32([0] * tokens), i32(range(tokens)),
                    heads=heads, stream=stream())
    torch.cuda.synchronize()
    pos = torch.arange(tokens)
    if heads:
        want, size = rotate64(q.reshape(tokens, heads, d), pos, freqs, False, 1.0, None)
        near(out, want, 2.0 ** -18 * size)
    want, size = rotate64(k.reshape(tokens, kv_heads, d), pos, freqs, False, 1.0, None)
    near(kp[:, 0], want, 2.0 ** -18 * size)
    assert torch.equal(vp[:, 0], v.reshape(tokens, kv_heads, d))
