"""Sampling, the 8-bit cache and 4-bit weights, what needs no GPU: every refusal
of arguments (refused before the device is touched), and what the binding reads."""
import math

import pytest

import iris_cuda
from iris_cuda import KvCache8, Rope, Weights4
from test_lm_ops_host import A, BAD_CACHES, Fake, cache, refused


def cache8(pages=None, **kw):
    d = dict(k_exp=A + 1, v_exp=A + 3, block=8, exp_page_stride=4, exp_block_stride=2, exp_head_stride=1)
    return KvCache8(pages or cache(), *{**d, **kw}.values())


def append8(c, **kw):
    d = dict(rope=Rope.of(128, 1e4), q_out=4 * A, ldq_out=512, q=A, k=A, v=A, ldq=512, ldk=256, ldv=256, f32=0, q_norm=A,
             k_norm=A, eps=1e-6, seq=A, pos=A, tokens=5, heads=4)
    d.update(kw)
    return iris_cuda.lib().iris_gpu_rope_append8(c, *d.values(), None)


def attend8(c, **kw):
    d = dict(out=A, q=A, ldo=512, ldq=512, seq=A, pos=A, rows=5, heads=4, scale=0.1, ws=A, ws_bytes=1 << 40)
    d.update(kw)
    return iris_cuda.lib().iris_gpu_attention_paged8(c, *d.values(), None)


def sample(**kw):
    d = dict(logits=A, f32=0, ld=1000, rows=5, vocab=1000, temperature=A, top_k=A, top_p=A, min_p=A, uniform=A, ids=A,
             logprobs=A, kept=A)
    d.update(kw)
    return iris_cuda.lib().iris_gpu_sample_tokens(*d.values(), None)


def weights(**kw):
    d = dict(q=A, scale=A, zero=A, n=100, k=256, group=64, scale_f32=0, q_stride=128, scale_stride=4, zero_stride=4)
    return Weights4(*{**d, **kw}.values())


def linear(w, **kw):
    d = dict(x=A, ldx=256, rows=3, out=2 * A, ldo=100, add=None, ldadd=0, f32=0)
    d.update(kw)
    return iris_cuda.lib().iris_gpu_linear4(w, *d.values(), None)


def quantize(weights, **kw):
    d = dict(w=A, f32=0, ldw=256)
    d.update(kw)
    return iris_cuda.lib().iris_gpu_quantize4(weights, *d.values(), None)


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_pages_are_refused(bad):
    c = cache8(cache(**bad))
    refused(append8(c), "rope_append8")
    refused(attend8(c), "attention_paged8")
    assert iris_cuda.lib().iris_gpu_attention_paged8_workspace(c, 4) == 0


@pytest.mark.parametrize("bad", [
    dict(k_exp=None), dict(v_exp=None), dict(block=0), dict(block=-1), dict(block=5), dict(block=32), dict(exp_page_stride=0),
    dict(exp_page_stride=-4), dict(exp_block_stride=0), dict(exp_block_stride=-1), dict(exp_head_stride=0), dict(exp_head_stride=-1),
    dict(pages=cache(page_size=256, page_stride=256 * 256), block=256), dict(pages=cache(token_stride=264)),
    dict(pages=cache(head_stride=136)), dict(pages=cache(page_stride=4104)), dict(pages=cache(page_stride=1 << 34)),
    dict(pages=cache(page_stride=1 << 60)), dict(pages=cache(token_stride=1 << 62))])
def test_bad_8_bit_caches_are_refused(bad):
    c = cache8(**bad)
    refused(append8(c), "rope_append8")
    refused(attend8(c), "attention_paged8")
    assert iris_cuda.lib().iris_gpu_attention_paged8_workspace(c, 4) == 0


def test_null_caches_and_no_rows():
    refused(append8(None), "rope_append8")
    refused(attend8(None), "attention_paged8")
    assert append8(cache8(), tokens=0, q=None, k=None, v=None, q_out=None, seq=None, pos=None) == 0
    assert attend8(cache8(), rows=0, out=None, q=None, pos=None, ws=None, ws_bytes=0) == 0
    assert sample(rows=0, logits=None, uniform=None, ids=None) == 0
    assert linear(weights(), rows=0, x=None, out=None) == 0
    # one page, block or head needs no stride
    one = cache(num_pages=1, kv_heads=1, page_stride=0, head_stride=0)
    assert append8(cache8(one, block=16, exp_page_stride=0, exp_block_stride=0, exp_head_stride=0), tokens=0) == 0


@pytest.mark.parametrize("bad", [
    dict(tokens=-1), dict(heads=-1), dict(k=None), dict(seq=None), dict(q_out=None), dict(ldq=511), dict(ldk=248), dict(eps=math.nan),
    dict(q=A + 2), dict(k_norm=A + 8), dict(seq=A + 1), dict(rope=Rope.of(256, 1e4)), dict(rope=Rope(layout=0, rot_dim=24)),
    dict(q_out=2 * A, q=2 * A, f32=1)])
def test_rope_append8_refusals(bad):
    refused(append8(cache8(), **bad), "rope_append8")


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(rows=4, seq=None), dict(heads=3), dict(heads=0), dict(out=None), dict(ws=None), dict(ldo=511),
    dict(scale=math.inf), dict(out=A + 8), dict(q=A + 2), dict(ws=A + 8), dict(pos=A + 1)])
def test_attention_paged8_refusals(bad):
    refused(attend8(cache8(), **bad), "attention_paged8")


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(rows=(1 << 24) + 1), dict(vocab=0), dict(vocab=(1 << 30) + 1, ld=1 << 31), dict(ld=999), dict(logits=None),
    dict(uniform=None), dict(ids=None), dict(logits=A + 1), dict(f32=1, logits=A + 2), dict(temperature=A + 2), dict(top_k=A + 1),
    dict(top_p=A + 2), dict(min_p=A + 2), dict(uniform=A + 4), dict(ids=A + 2), dict(logprobs=A + 2), dict(kept=A + 2)])
def test_sample_tokens_refusals(bad):
    refused(sample(**bad), "sample_tokens")


BAD_WEIGHTS = [dict(n=(1 << 30) + 1), dict(k=(1 << 30) + 64, q_stride=1 << 30, scale_stride=1 << 30), dict(q=None), dict(scale=None), dict(n=0), dict(k=0), dict(group=0), dict(group=16), dict(group=96), dict(group=192),
               dict(group=512), dict(k=288), dict(q_stride=120), dict(q_stride=136), dict(q_stride=-128), dict(scale_stride=3),
               dict(q=A + 8), dict(scale=A + 1), dict(scale_f32=1, scale=A + 2)]


@pytest.mark.parametrize("bad", BAD_WEIGHTS)
def test_bad_weights_are_refused(bad):
    refused(linear(weights(**bad)), "linear4")
    refused(quantize(weights(zero=None, **bad)), "quantize4")


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(rows=(1 << 19) + 1), dict(x=None), dict(out=None), dict(ldx=255), dict(ldx=260), dict(ldo=99),
    dict(add=3 * A, ldadd=99), dict(x=A + 8), dict(out=A + 1), dict(f32=1, out=A + 2), dict(add=A + 1, ldadd=100),
    dict(add=2 * A, ldadd=104)])
def test_linear4_refusals(bad):
    refused(linear(weights(), **bad), "linear4")


def test_linear4_zero_stride():
    refused(linear(weights(zero_stride=3)), "linear4")


@pytest.mark.parametrize("bad", [dict(w=None), dict(w=A + 8), dict(ldw=255), dict(ldw=260)])
def test_quantize4_refusals(bad):
    refused(quantize(weights(zero=None), **bad), "quantize4")
    refused(quantize(weights()), "quantize4")  # zeros of their own


def fake_cache8(**kw):
    d = dict(k=Fake("uint8", 8, 16, 2, 128), v=Fake("uint8", 8, 16, 2, 128), k_exp=Fake("uint8", 8, 2, 2),
             v_exp=Fake("uint8", 8, 2, 2), table=Fake("int32", 3, 4))
    return KvCache8.of(*{**d, **kw}.values())


def test_binding_reads_8_bit_caches():
    c = fake_cache8()
    assert (c.block, c.exp_page_stride, c.exp_block_stride, c.exp_head_stride) == (8, 4, 2, 1)
    assert (c.pages.page_size, c.pages.page_stride, c.pages.token_stride, c.pages.head_stride) == (16, 4096, 256, 128)
    assert append8(c, tokens=0) == 0
    by_head = dict(k_exp=Fake("uint8", 8, 2, 2, stride=[4, 1, 2]), v_exp=Fake("uint8", 8, 2, 2, stride=[4, 1, 2]))
    assert fake_cache8(**by_head).exp_head_stride == 2


@pytest.mark.parametrize("bad", [
    dict(k=Fake("bfloat16", 8, 16, 2, 128)), dict(v=Fake("uint8", 8, 16, 2, 64)), dict(k_exp=Fake("int32", 8, 2, 2)),
    dict(v_exp=Fake("uint8", 8, 1, 2)), dict(k_exp=Fake("uint8", 8, 3, 2), v_exp=Fake("uint8", 8, 3, 2)),
    dict(k_exp=Fake("uint8", 7, 2, 2), v_exp=Fake("uint8", 7, 2, 2)), dict(k_exp=Fake("uint8", 8, 2, 2, stride=[4, 1, 2])),
    dict(table=Fake("int64", 3, 4)), dict(k_exp=Fake("uint8", 8, 4), v_exp=Fake("uint8", 8, 4)),
    dict(k_exp=Fake("uint8", 8, 0, 2), v_exp=Fake("uint8", 8, 0, 2))])
def test_binding_refuses_other_8_bit_caches(bad):
    with pytest.raises(iris_cuda.IrisCudaError, match="KvCache8"):
        fake_cache8(**bad)


def test_binding_reads_weights():
    w = Weights4.of(Fake("uint8", 100, 128), Fake("float32", 100, 4), Fake("uint8", 100, 4))
    assert (w.n, w.k, w.group, w.scale_f32, w.q_stride, w.scale_stride, w.zero_stride) == (100, 256, 64, 1, 128, 4, 4)
    for bad in ((Fake("int32", 100, 128), Fake("float32", 100, 4)), (Fake("uint8", 100, 128), Fake("float16", 100, 4)),
                (Fake("uint8", 100, 128), Fake("float32", 99, 4)), (Fake("uint8", 100, 128), Fake("float32", 100, 3)),
                (Fake("uint8", 100, 128), Fake("float32", 100, 4), Fake("uint8", 100, 2)), (Fake("uint8", 100, 128), Fake("float32", 400)),
                (Fake("uint8", 100, 128, stride=[1, 100]), Fake("float32", 100, 4)), (Fake("uint8", 100, 128), Fake("float32", 100, 0))):
        with pytest.raises(iris_cuda.IrisCudaError, match="Weights4"):
            Weights4.of(*bad)


def test_binding_refuses_other_tensors():
    E, c, i = iris_cuda.IrisCudaError, fake_cache8(), Fake("int32", 5)
    q = Fake("bfloat16", 5, 4, 128)
    with pytest.raises(E):
        iris_cuda.attention_paged8(c, q, q, i, Fake("int64", 5), scale=0.1, workspace=Fake("uint8", 16))
    with pytest.raises(E):
        iris_cuda.rope_append8(c, None, q, Fake("float16", 5, 512), q, q, i, i, heads=4)
    good = dict(logits=Fake("float32", 5, 100), uniform=Fake("float64", 5), ids=i)
    for bad in (dict(logits=Fake("float16", 5, 100)), dict(logits=Fake("float32", 5, 100, stride=[1, 5])),
                dict(uniform=Fake("float32", 5)), dict(uniform=Fake("float64", 4)), dict(ids=Fake("int64", 5)),
                dict(temperature=Fake("float64", 5)), dict(top_k=Fake("float32", 5)), dict(top_p=Fake("float32", 1)),
                dict(min_p=Fake("bfloat16", 5)), dict(logprobs=Fake("float64", 5)), dict(kept=Fake("int64", 5))):
        with pytest.raises(E):
            iris_cuda.sample_tokens(**{**good, **bad})
    w = Weights4.of(Fake("uint8", 100, 128), Fake("float32", 100, 4))
    good = dict(out=Fake("float32", 3, 100, at=4 * A), x=Fake("bfloat16", 3, 256))
    for bad in (dict(out=Fake("float16", 3, 100)), dict(out=Fake("float32", 3, 99)), dict(x=Fake("float32", 3, 256)),
                dict(x=Fake("bfloat16", 3, 128)), dict(add=Fake("bfloat16", 3, 100)), dict(add=Fake("float32", 2, 100))):
        with pytest.raises(E):
            iris_cuda.linear4(w=w, **{**good, **bad})
    for bad in (Fake("float16", 100, 256), Fake("float32", 100, 255), Fake("float32", 100, 256, stride=[1, 100])):
        with pytest.raises(E):
            iris_cuda.quantize4(w, bad)
