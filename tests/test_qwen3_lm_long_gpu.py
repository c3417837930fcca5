"""Sessions of the text model with room for many tokens: prompts long enough for
runs of rows, a few tokens behind one, single tokens over a long table, against
the numpy oracle's decoder layers with the tolerance of test_qwen3_lm_gpu."""
import numpy as np
import pytest

from gpu_util import rel_l2
from test_qwen3_lm_gpu import TOL, logprobs_ref, model, rows, texts  # noqa: F401

pytestmark = pytest.mark.gpu


def test_long_prompts_and_continuations(iris, model):  # noqa: F811
    m, _, w = model
    ids = texts([231, 41], 7)
    ref = [logprobs_ref(w, t[:-1]) for t in ids]
    lm = iris.Qwen3Lm(m, num_seqs=2, max_len=8192, max_tokens=256)
    got, want, at = [], [], [0, 0]
    # 190 + 20 rows, 12 and 8 rows, single tokens of both, one alone
    for new in ((190, 20), (12, 8), (1, 1), (1, 1), (1, 0), (25, 10)):
        parts = [(s, at[s], ids[s][at[s]:at[s] + n]) for s, n in enumerate(new) if n]
        tg = np.concatenate([ids[s][at[s] + 1:at[s] + n + 1] for s, n in enumerate(new) if n])
        got += list(lm.step(*rows(parts), targets=tg)["logprob"])
        want += [ref[s][at[s] + j, ids[s][at[s] + j + 1]] for s, n in enumerate(new) for j in range(n)]
        at = [a + n for a, n in zip(at, new)]
    assert [lm.length(s) for s in (0, 1)] == at == [230, 40]
    assert rel_l2(got, want) < TOL
    lm.close()


def test_sessions_of_the_longest_length(iris, model):  # noqa: F811
    """Lengths up to the end of int are counted in pages without wrapping: refused by their number of pages."""
    m, _, _ = model
    for n in (2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 16):
        with pytest.raises(iris.IrisCudaError, match=f"9 sequences of {n}"):
            iris.Qwen3Lm(m, num_seqs=9, max_len=n, max_tokens=8)


def test_after_a_session_that_does_not_fit(iris, model):  # noqa: F811
    """A session whose cache no device holds is refused, and the next calls do not report its error."""
    m, _, _ = model
    lm = iris.Qwen3Lm(m, num_seqs=1, max_len=64, max_tokens=8)
    with pytest.raises(iris.IrisCudaError, match="language model session"):
        iris.Qwen3Lm(m, num_seqs=1, max_len=2 ** 24, max_tokens=8)  # 28 layers, 2 heads: 481 GB
    assert np.isfinite(lm.step([1, 2, 3], [0] * 3, [0, 1, 2])["entropy"]).all()
    lm.close()


def test_a_model_freed_before_its_sessions(iris):
    """Its weights stay until the last session is freed (the steps would read freed memory)."""
    cfg = iris.Qwen3Config(256, 512, 4, 2, 128, 1000, 2, 1e6)
    want = None
    for close_first in (False, True):
        m = iris.Qwen3.random_lm(cfg, 3)
        a, b = (iris.Qwen3Lm(m, num_seqs=1, max_len=64, max_tokens=8) for _ in range(2))
        a.step([1, 2], [0, 0], [0, 1])
        if close_first:
            m.close()
            a.close()
        ids, got = list(range(8)), []
        for j in range(3):  # queued, captured, replayed
            got.append(b.step(ids, [0] * 8, range(8 * j, 8 * j + 8), targets=ids, top_k=2))
        b.close(), a.close(), m.close()
        if want is None:
            want = got
        for x, y in zip(want, got):
            for key in x:
                np.testing.assert_array_equal(x[key], y[key])
