"""Sessions of the text model whose steps change their size: prompts and single
tokens in turn, more sizes than a session remembers."""
import os
import time

import numpy as np
import pytest

from test_qwen3_lm_gpu import model, texts  # noqa: F401

pytestmark = pytest.mark.gpu


def feed(lm, t, sizes, seq=0):
    """The text in steps of the given sizes: log probabilities, likeliest ids of the steps that ask for them, milliseconds."""
    lp, top, ms, at = [], [], [], 0
    for i, n in enumerate(sizes):
        k = 3 if i % 3 == 0 else 0
        start = time.perf_counter()
        o = lm.step(t[at:at + n], [seq] * n, np.arange(at, at + n), targets=t[at + 1:at + n + 1], top_k=k)
        ms.append((time.perf_counter() - start) * 1e3)
        lp += list(o["logprob"])
        top += o["top_ids"].ravel().tolist()
        at += n
    return np.array(lp), top, ms


def test_changing_sizes_give_what_any_session_gives(iris, model, monkeypatch):  # noqa: F811
    """Queued, captured and replayed steps, 20 sizes with and without alternatives, one behind the other, again and thrown
    out in between: the same bits as without graphs."""
    m, _, _ = model
    sizes = [1, 5, 1, 1, 5, 5] + list(range(1, 21)) + list(range(20, 0, -1)) + [1, 5] * 10
    (t,) = texts([sum(sizes) + 1], 11)
    lm = iris.Qwen3Lm(m, num_seqs=2, max_len=768, max_tokens=32)
    a = feed(lm, t, sizes, 0)
    again = feed(lm, t, sizes, 1)
    lm.close()
    monkeypatch.setenv("IRIS_CUDA_NO_GRAPH", "1")
    lm = iris.Qwen3Lm(m, num_seqs=2, max_len=768, max_tokens=32)
    b = feed(lm, t, sizes, 0)
    lm.close()
    for x in (again, b):
        np.testing.assert_array_equal(a[0], x[0])
        assert a[1] == x[1]


def test_two_sizes_in_turn_are_not_captured_again(iris, model):  # noqa: F811
    """Two sizes in turn take no longer than the same steps queued without graphs (a capture at each took over 1.2 times that)."""
    m, _, _ = model
    sizes = [8, 9] * 30
    (t,) = texts([sum(sizes) + 1], 12)

    def median():
        lm = iris.Qwen3Lm(m, num_seqs=1, max_len=768, max_tokens=32)
        ms = feed(lm, t, sizes)[2][20:]
        lm.close()
        return float(np.median(ms))

    with_graphs = median()
    os.environ["IRIS_CUDA_NO_GRAPH"] = "1"
    try:
        without = median()
    finally:
        del os.environ["IRIS_CUDA_NO_GRAPH"]
    print(f"two sizes in turn {with_graphs:.2f} ms a step, without graphs {without:.2f}")
    assert with_graphs < 1.1 * without
