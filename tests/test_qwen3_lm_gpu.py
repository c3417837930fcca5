"""The text model as a language model (iris_cuda_qwen3_lm_*) against the numpy
oracle's decoder layers, and its sessions against themselves.

Against the oracle: the hidden states agree to 1e-2 relative L2 (the gate of the
encoder's tests, same layers).  Logits are products of them with embeddings
N(0, 1) of width 256, so of size 16 with errors of 0.16, and a random target's
log probability is about -(3 * 16) +- 16: relative L2 of the log probabilities
within (0.16 + 0.16) / 48 * 2 = 1.4e-2; 2e-2 is asked.  A single one of some
hundred: within 1.5, five times 0.16 for the logit and for the sum; the entropy,
at most some units with such logits, within 0.5; and where two logits lie closer
than that their ids may change places (the picked ones' values within 0.2).

Against itself: prompts whole or token by token take other GEMM splits and
attention shares, f32 sums that differ in their last bits and now and then round
an activation the other way (2^-8): the same 2e-2.
"""
import numpy as np
import pytest

from gpu_util import rel_l2
from oracle import model_gen as mg
from oracle import qwen3_oracle as qo
from test_qwen3_oracle import CFG, SEED

pytestmark = pytest.mark.gpu
TOL = 2e-2


def logprobs_ref(w, ids, head="model.embed_tokens.weight"):
    """log softmax after every token of one sequence, f64 from the oracle's f32 hidden states."""
    x = w["model.embed_tokens.weight"][np.asarray(ids)].astype(np.float32)
    cos, sin = qo.rope_tables(len(ids), 128, CFG["rope_theta"])
    for i in range(CFG["num_hidden_layers"]):
        x = qo.layer(w, i, x, cos, sin, np.ones(len(ids), np.int32), CFG)
    z = qo.rms_norm(x, w["model.norm.weight"]).astype(np.float64) @ w[head].astype(np.float64).T
    m = z.max(1, keepdims=True)
    return z - m - np.log(np.exp(z - m).sum(1, keepdims=True))


@pytest.fixture(scope="module")
def model(iris, tmp_path_factory):
    d = mg.make_qwen3_model(str(tmp_path_factory.mktemp("q3lm")), CFG, SEED)
    m = iris.Qwen3.load_lm(d)
    yield m, d, mg.qwen3_weights(CFG, SEED)
    m.close()


def texts(lens, seed=1):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, CFG["vocab_size"], n).astype(np.int32) for n in lens]


def rows(parts):
    """(ids, seq, pos) of [(sequence, first position, ids)]."""
    return (np.concatenate([p[2] for p in parts]), np.concatenate([np.full(len(p[2]), p[0], np.int32) for p in parts]),
            np.concatenate([p[1] + np.arange(len(p[2]), dtype=np.int32) for p in parts]))


def test_prompts_then_tokens_match_the_oracle(iris, model):
    m, _, w = model
    lens, new = [33, 1, 70], 6
    ids = texts([n + new + 1 for n in lens])
    ref = [logprobs_ref(w, t[:-1]) for t in ids]
    lm = iris.Qwen3Lm(m, num_seqs=3, max_len=96, max_tokens=128)
    parts = rows([(s, 0, t[:n]) for s, (t, n) in enumerate(zip(ids, lens))])
    tg = np.concatenate([t[1:n + 1] for t, n in zip(ids, lens)])
    out = lm.step(*parts, targets=tg, top_k=8)
    want = np.concatenate([r[np.arange(n), t[1:n + 1]] for r, t, n in zip(ref, ids, lens)])
    assert rel_l2(out["logprob"], want) < TOL
    allr = np.concatenate([r[:n] for r, n in zip(ref, lens)])
    picked = np.take_along_axis(allr, out["top_ids"], 1)
    # likeliest values: of the same size as the oracle's, in order, and the ids' own
    assert np.all(np.diff(out["top_logprobs"], axis=1) <= 0)
    best = -np.sort(-allr, axis=1)[:, :8]
    assert np.abs(out["top_logprobs"] - best).max() < 1.5 and rel_l2(picked, best) < 0.2
    ent = -(np.exp(allr) * allr).sum(1)
    assert np.abs(out["entropy"] - ent).max() < 0.5
    assert [lm.length(s) for s in range(3)] == lens
    got, exp = [], []
    for j in range(new):
        o = lm.step([t[n + j] for t, n in zip(ids, lens)], [0, 1, 2], [n + j for n in lens],
                    targets=[t[n + j + 1] for t, n in zip(ids, lens)])
        got += list(o["logprob"])
        exp += [r[n + j, t[n + j + 1]] for r, t, n in zip(ref, ids, lens)]
    assert rel_l2(got, exp) < TOL
    lm.close()


def test_token_by_token_is_the_prompt(iris, model):
    """The same text whole, in uneven pieces and one token at a time; twice the same bits."""
    m, _, _ = model
    (t,) = texts([41], 2)
    runs = []
    for cuts in ([40], [40], [1] * 40, [7, 16, 17]):
        lm = iris.Qwen3Lm(m, num_seqs=2, max_len=48, max_tokens=40)
        lp, at = [], 0
        for n in cuts:
            o = lm.step(t[at:at + n], [1] * n, np.arange(at, at + n), targets=t[at + 1:at + n + 1])
            lp += list(o["logprob"])
            at += n
        runs.append(np.array(lp))
        lm.close()
    np.testing.assert_array_equal(runs[0], runs[1])
    assert rel_l2(runs[2], runs[0]) < TOL and rel_l2(runs[3], runs[0]) < TOL


def test_cut_off_and_continue(iris, model):
    """A smaller position cuts a sequence off there: what follows is as if the rest had never been."""
    m, _, _ = model
    (t,), (u,) = texts([31], 3), texts([12], 4)
    lm = iris.Qwen3Lm(m, num_seqs=2, max_len=64, max_tokens=64)
    lm.step(t[:30], [0] * 30, np.arange(30))
    a = lm.step(u[:11], [0] * 11, 10 + np.arange(11), targets=u[1:12])["logprob"]
    assert lm.length(0) == 21
    lm.step(t[:10], [1] * 10, np.arange(10))
    b = lm.step(u[:11], [1] * 11, 10 + np.arange(11), targets=u[1:12])["logprob"]
    assert rel_l2(a, b) < TOL
    lm.close()


def test_arguments(iris, model):
    m, d, _ = model
    E = iris.IrisCudaError
    enc = iris.Qwen3.load(d)
    with pytest.raises(E, match="load_lm"):
        iris.Qwen3Lm(enc)
    enc.close()
    for bad in (dict(num_seqs=0), dict(max_len=0), dict(max_tokens=0), dict(max_tokens=8193)):
        with pytest.raises(E, match="session"):
            iris.Qwen3Lm(m, **bad)
    lm = iris.Qwen3Lm(m, num_seqs=2, max_len=20, max_tokens=8)
    lm.step([1, 2, 3], [0, 0, 0], [0, 1, 2])
    for ids, seq, pos in (([1], [2], [0]), ([1], [-1], [0]), ([1], [0], [4]), ([1], [1], [1]), ([1], [0], [-1]), ([1], [0], [20]),
                          ([1, 1], [0, 0], [3, 3]), ([1, 1], [0, 0], [3, 5]), ([1, 1], [0, 0], [2, 1]), ([1] * 9, [0] * 9, range(9)),
                          ([], [], [])):
        with pytest.raises(E):
            lm.step(ids, seq, pos)
        assert lm.length(0) == 3 and lm.length(1) == 0
    for k in (-1, 33):
        with pytest.raises((E, ValueError)):
            lm.step([1], [0], [3], top_k=k)
    with pytest.raises(E):
        lm.length(2)
    o = lm.step([5, 10 ** 6], [0, 1], [3, 0], targets=[-1, 10 ** 6], top_k=3)  # unknown ids embed as zeros, ask for nothing
    assert (o["logprob"] == 0).all() and np.isfinite(o["entropy"]).all()
    lm.close()


def test_a_language_model_still_encodes(iris, model):
    m, d, _ = model
    enc = iris.Qwen3.load(d)
    (t,) = texts([50], 5)
    np.testing.assert_array_equal(m.forward(t), enc.forward(t))
    enc.close()


def test_own_head_and_odd_vocabulary(iris, tmp_path):
    """lm_head.weight where the file has one; a vocabulary that is no multiple of the GEMM's tile."""
    import json
    import os
    cfg = dict(CFG, vocab_size=333, num_hidden_layers=2)
    d = mg.make_qwen3_model(str(tmp_path), cfg, 9)
    w = mg.qwen3_weights(cfg, 9)
    (t,) = [np.random.default_rng(1).integers(0, 333, 25).astype(np.int32)]

    def ref(head):
        x = w["model.embed_tokens.weight"][t]
        cos, sin = qo.rope_tables(len(t), 128, CFG["rope_theta"])
        for i in range(2):
            x = qo.layer(w, i, x, cos, sin, np.ones(len(t), np.int32), cfg)
        z = qo.rms_norm(x, w["model.norm.weight"]).astype(np.float64) @ w[head].astype(np.float64).T
        return z - z.max(1, keepdims=True) - np.log(np.exp(z - z.max(1, keepdims=True)).sum(1, keepdims=True))

    def check(head):
        m = iris.Qwen3.load_lm(d)
        lm = iris.Qwen3Lm(m, max_len=32, max_tokens=32)
        o = lm.step(t[:24], [0] * 24, np.arange(24), targets=t[1:], top_k=32)
        assert rel_l2(o["logprob"], ref(head)[np.arange(24), t[1:]]) < TOL
        assert o["top_ids"].max() < 333 and o["top_ids"].min() >= 0
        lm.close()
        m.close()

    check("model.embed_tokens.weight")
    w["lm_head.weight"] = mg.bf16_bits_to_f32(mg._qwen3_tensor(9, "lm_head.weight", (333, 256), "embed"))
    shard = "model-00002-of-00002.safetensors"
    mg.write_safetensors(os.path.join(d, shard), {"lm_head.weight": mg._qwen3_tensor(9, "lm_head.weight", (333, 256), "embed")})
    idx = os.path.join(d, "model.safetensors.index.json")
    j = json.load(open(idx))
    j["weight_map"]["lm_head.weight"] = shard
    json.dump(j, open(idx, "w"))
    check("lm_head.weight")
