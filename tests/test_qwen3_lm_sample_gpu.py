"""Sessions of the text model that draw their next tokens, against the likeliest
tokens that the same session's steps give.

With top_k = 4 the kept probabilities are those of the step's four likeliest
values, renormalised.  Their f32 log probabilities, of size 2^7 at most, are
within 2^-17 (half a unit of the last place, twice for sum and difference: 2^-16),
so a draw may differ from the one worked out here where the random number lies
within 2^-14 of a step of the cumulated probabilities (four terms of 2^-16), and
the log probabilities are within 2^-14 plus their own rounding.
"""
import numpy as np
import pytest

from test_qwen3_lm_gpu import model, texts  # noqa: F401

pytestmark = pytest.mark.gpu


def test_draws_are_of_the_steps_likeliest(iris, model):  # noqa: F811
    m, _, _ = model
    (t,) = texts([40], 21)
    u = np.random.default_rng(22).random(40)
    lm = iris.Qwen3Lm(m, num_seqs=2, max_len=64, max_tokens=40)
    ref = lm.step(t, [0] * 40, np.arange(40), top_k=4)
    got = lm.sample(t, [1] * 40, np.arange(40), u, top_k=4)
    lp = ref["top_logprobs"].astype(np.float64)
    p = np.exp(lp - lp[:, :1])
    cum = np.cumsum(p / p.sum(1, keepdims=True), 1)
    pick = (cum <= u[:, None]).sum(1)
    sure = np.abs(cum - u[:, None]).min(1) > 2.0 ** -14
    assert sure.any()
    np.testing.assert_array_equal(got["next"][sure], ref["top_ids"][np.arange(40), pick][sure])
    want = np.log(p / p.sum(1, keepdims=True))[np.arange(40), pick]
    assert np.all(np.abs(got["logprobs"] - want)[sure] <= 2.0 ** -14 + np.abs(want[sure]) * 2.0 ** -23)
    lm.close()


def test_greedy_and_settings_of_each_token(iris, model):  # noqa: F811
    """Temperature 0 is the likeliest; one row's settings leave the others'."""
    m, _, _ = model
    (t,) = texts([9], 23)
    lm = iris.Qwen3Lm(m, num_seqs=3, max_len=32, max_tokens=16)
    best = lm.step(t, [0] * 9, np.arange(9), top_k=1)["top_ids"][:, 0]
    a = lm.sample(t, [1] * 9, np.arange(9), [0.5] * 9, temperature=0)
    np.testing.assert_array_equal(a["next"], best)
    assert not a["logprobs"].any()
    b = lm.sample(t, [2] * 9, np.arange(9), [0.999] * 9, temperature=[0, 30] * 4 + [0], top_p=[1, 0.9] * 4 + [1],
                  min_p=[0, 0.01] * 4 + [0])
    np.testing.assert_array_equal(b["next"][::2], best[::2])
    assert np.all(b["logprobs"][1::2] < 0)
    lm.close()


def text_of(iris, m, prompt, u, n):
    lm = iris.Qwen3Lm(m, num_seqs=1, max_len=64, max_tokens=16)
    out = [int(lm.sample(prompt, [0] * len(prompt), np.arange(len(prompt)), u[:1].repeat(len(prompt)), temperature=8.0,
                         top_p=0.95)["next"][-1])]
    for i in range(1, n):
        at = len(prompt) + i - 1
        out.append(int(lm.sample([out[-1]], [0], [at], u[i:i + 1], temperature=8.0, top_p=0.95)["next"][0]))
        if i == n // 2:
            lm.step([out[-1]], [0], [at + 1], top_k=2)  # another kind of step between; the next one feeds its token again
    assert lm.length(0) == len(prompt) + n - 1
    lm.close()
    return out


def test_captured_steps_draw_as_queued_ones(iris, model, monkeypatch):  # noqa: F811
    m, _, _ = model
    (t,) = texts([7], 24)
    u = np.random.default_rng(25).random(24)
    a = text_of(iris, m, t, u, 24)
    assert a == text_of(iris, m, t, u, 24)
    monkeypatch.setenv("IRIS_CUDA_NO_GRAPH", "1")
    assert a == text_of(iris, m, t, u, 24)
    assert len(set(a)) > 1


def test_arguments(iris, model):  # noqa: F811
    m, _, _ = model
    E = iris.IrisCudaError
    lm = iris.Qwen3Lm(m, num_seqs=1, max_len=16, max_tokens=4)
    lm.sample([1, 2], [0, 0], [0, 1], [0.1, 0.2])
    for args, kw in ((([], [], [], []), {}), (([1], [1], [0], [0.5]), {}), (([1], [0], [4], [0.5]), {}), (([1] * 5, [0] * 5, range(5), [0.5] * 5), {}),
                     (([1], [0], [2], [0.5, 0.5]), {}), (([1], [0, 0], [2], [0.5]), {}), (([1], [0], [2], [0.5]), dict(top_k=[1, 2]))):
        with pytest.raises(E):
            lm.sample(*args, **kw)
        assert lm.length(0) == 2
    lm.close()
