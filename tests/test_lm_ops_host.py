"""Language-model operators, what needs no GPU: the rotation's frequencies and
every refusal of arguments (refused before the device is touched)."""
import ctypes as C
import math

import numpy as np
import pytest

import iris_cuda
from iris_cuda import ERR_ARG, KvCache, Rope, RopeScaling

HALF, INTERLEAVED = 0, 1


def radians(rope):
    """Frequencies held by a rotation, radians per position, from their 64-bit turns."""
    return np.array([t / 2.0 ** 64 * 2 * math.pi for t in rope.turns[:rope.rot_dim // 2]])


def close(a, b):
    # turns are the double f / (2 pi) cut to 64 bits: a few 2^-53 relative, 2^-64 turns absolute
    np.testing.assert_allclose(a, b, rtol=1e-15, atol=1e-18)


@pytest.mark.parametrize("rot_dim,theta", [(16, 1e4), (96, 1e4), (128, 1e6), (256, 5e5)])
def test_rope_frequencies(rot_dim, theta):
    r = Rope.of(rot_dim, theta)
    want = [theta ** (-2.0 * i / rot_dim) for i in range(rot_dim // 2)]
    close(radians(r), want)
    assert r.amplitude == 1.0 and r.layout == HALF
    assert Rope.of(rot_dim, theta, interleaved=True).layout == INTERLEAVED
    close(radians(Rope.of(rot_dim, theta, factor=4.0)), np.array(want) / 4)


def test_rope_scaled_by_parts():
    r = Rope.of(128, 1e6, factor=8.0, original_len=32768, low=1.0, high=4.0, amplitude=1.25)
    f = np.array([1e6 ** (-2.0 * i / 128) for i in range(64)])
    turns = 32768 * f / (2 * math.pi)
    g = np.clip((turns - 1.0) / 3.0, 0, 1)
    assert (g == 0).any() and (g == 1).any() and ((g > 0) & (g < 1)).any()
    close(radians(r), f * (g + (1 - g) / 8))
    assert r.amplitude == 1.25


def test_rope_own_frequencies_drop_whole_turns():
    f = np.array([0.0, 0.5, 2 * math.pi + 0.5, 7.0, 1e-9, 3.0, 0.25, 1e-3])
    got = radians(Rope.of_freqs(f))
    # a whole turn per position never shows at whole positions; 4e-15: the double's own step at 7 radians
    np.testing.assert_allclose(got, f % (2 * math.pi), rtol=1e-15, atol=4e-15)


@pytest.mark.parametrize("args", [
    dict(rot_dim=0), dict(rot_dim=8), dict(rot_dim=20), dict(rot_dim=272), dict(rot_dim=-16), dict(theta=0.0),
    dict(theta=-1.0), dict(theta=math.inf), dict(theta=math.nan), dict(factor=0.0), dict(factor=-2.0), dict(factor=math.nan),
    dict(original_len=-1.0), dict(original_len=4096, low=4.0, high=4.0), dict(original_len=4096, low=math.nan),
    dict(amplitude=0.0), dict(amplitude=math.nan)])
def test_rope_refusals(args):
    with pytest.raises(iris_cuda.IrisCudaError, match="rope_init"):
        Rope.of(**{**dict(rot_dim=128, theta=1e4), **args})


def test_rope_refusals_at_the_c_entry():
    L = iris_cuda.lib()
    r = Rope()
    f = (C.c_double * 64)(*([0.1] * 64))
    before = L.iris_gpu_op_failures()
    assert L.iris_gpu_rope_init(None, HALF, 128, 1e4, None) == ERR_ARG
    assert L.iris_gpu_rope_init(C.byref(r), 2, 128, 1e4, None) == ERR_ARG
    assert L.iris_gpu_rope_init_freqs(C.byref(r), HALF, 128, None, 1.0) == ERR_ARG
    f[3] = math.inf
    assert L.iris_gpu_rope_init_freqs(C.byref(r), HALF, 128, f, 1.0) == ERR_ARG
    f[3] = -0.5
    assert L.iris_gpu_rope_init_freqs(C.byref(r), HALF, 128, f, 1.0) == ERR_ARG
    assert L.iris_gpu_op_failures() == before + 5
    assert L.iris_gpu_rope_init(C.byref(r), HALF, 128, 1e4, None) == 0


# addresses that are never followed: every call below is refused by its arguments
A = 1 << 20


def cache(**kw):
    d = dict(k=A, v=A, table=A, num_pages=8, page_size=16, kv_heads=2, head_dim=128, num_seqs=3, max_blocks=4,
             table_stride=4, page_stride=16 * 256, token_stride=256, head_stride=128)
    return KvCache(**{**d, **kw})


BAD_CACHES = [dict(k=None), dict(v=None), dict(table=None), dict(num_pages=0), dict(page_size=0), dict(kv_heads=0),
              dict(kv_heads=70000), dict(head_dim=96), dict(head_dim=0), dict(num_seqs=0), dict(max_blocks=0),
              dict(k=A + 8), dict(v=A + 2), dict(table=A + 2), dict(table_stride=3), dict(table_stride=-4),
              dict(page_stride=4100), dict(page_stride=0), dict(page_stride=-4096), dict(token_stride=0),
              dict(token_stride=250), dict(head_stride=0), dict(head_stride=-128), dict(head_stride=4)]


def append(c, **kw):
    d = dict(rope=Rope.of(128, 1e4), q_out=4 * A, ldq_out=512, q=A, k=A, v=A, ldq=512, ldk=256, ldv=256, f32=0, q_norm=A,
             k_norm=A, eps=1e-6, seq=A, pos=A, tokens=5, heads=4)
    d.update(kw)
    return iris_cuda.lib().iris_gpu_rope_append(c, *d.values(), None)


def attend(c, **kw):
    d = dict(out=A, q=A, ldo=512, ldq=512, seq=A, pos=A, rows=5, heads=4, scale=0.1, ws=A, ws_bytes=1 << 40)
    d.update(kw)
    return iris_cuda.lib().iris_gpu_attention_paged(c, *d.values(), None)


def logprobs(**kw):
    d = dict(logits=A, f32=0, ld=1000, rows=5, vocab=1000, targets=A, logprob=A, entropy=A, top_k=4, top_ids=A,
             top_logprobs=A, ws=A, ws_bytes=1 << 40)
    d.update(kw)
    return iris_cuda.lib().iris_gpu_token_logprobs(*d.values(), None)


def refused(rc, name):
    assert rc == ERR_ARG
    assert name in iris_cuda.last_error()


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches_are_refused(bad):
    refused(append(cache(**bad)), "rope_append")
    refused(attend(cache(**bad)), "attention_paged")
    assert iris_cuda.lib().iris_gpu_attention_paged_workspace(cache(**bad), 4) == 0


def test_null_cache_is_refused():
    refused(append(None), "rope_append")
    refused(attend(None), "attention_paged")


@pytest.mark.parametrize("bad", [
    dict(tokens=-1), dict(heads=-1), dict(heads=70000), dict(k=None), dict(v=None), dict(seq=None), dict(pos=None),
    dict(q=None), dict(q_out=None), dict(ldq=511), dict(ldq=504), dict(ldq_out=516), dict(ldk=248), dict(ldv=255), dict(eps=-1.0),
    dict(eps=math.nan), dict(q=A + 2), dict(k=A + 8), dict(v=A + 4), dict(q_out=A + 8), dict(q_norm=A + 4),
    dict(k_norm=A + 8), dict(seq=A + 1), dict(pos=A + 2), dict(rope=Rope.of(256, 1e4)), dict(rope=Rope(layout=7, rot_dim=64)),
    dict(rope=Rope(layout=0, rot_dim=24)), dict(q_out=2 * A, q=2 * A, f32=1), dict(q_out=2 * A, q=2 * A, ldq_out=520)])
def test_rope_append_refusals(bad):
    refused(append(cache(), **bad), "rope_append")


def test_rope_append_f32_rows_may_be_multiples_of_four():
    refused(append(cache(), f32=0, ldk=260), "row strides")
    refused(append(cache(), f32=1, ldk=258), "row strides")
    assert append(cache(), f32=1, ldk=260, tokens=0) == 0


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(rows=4, seq=None), dict(heads=3), dict(heads=0), dict(heads=131072), dict(out=None), dict(q=None),
    dict(pos=None), dict(ws=None), dict(ldo=511), dict(ldq=504), dict(scale=math.nan), dict(scale=math.inf), dict(out=A + 8),
    dict(q=A + 2), dict(ws=A + 8), dict(seq=A + 2), dict(pos=A + 1)])
def test_attention_paged_refusals(bad):
    refused(attend(cache(), **bad), "attention_paged")


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(ld=999), dict(top_k=-1), dict(top_k=33),
    dict(vocab=3, top_k=4), dict(logits=None), dict(ws=None), dict(targets=None), dict(top_ids=None, top_logprobs=None),
    dict(logits=A + 1), dict(f32=1, logits=A + 2), dict(targets=A + 2), dict(logprob=A + 1), dict(entropy=A + 2),
    dict(top_ids=A + 2), dict(top_logprobs=A + 1), dict(ws=A + 8), dict(ws_bytes=0)])
def test_token_logprobs_refusals(bad):
    refused(logprobs(**bad), "token_logprobs")


def test_nothing_to_do_needs_no_device():
    assert append(cache(), tokens=0) == 0
    assert attend(cache(), rows=0) == 0
    assert logprobs(rows=0) == 0


class Fake:
    """What the binding reads of a device tensor."""

    def __init__(self, dtype, *shape, stride=None, at=A):
        self.dtype, self.shape, self.at = "torch." + dtype, shape, at
        s, st = 1, []
        for n in reversed(shape):
            st.insert(0, s)
            s *= n
        self.st = stride or st

    def stride(self, i=None):
        return self.st if i is None else self.st[i]

    def data_ptr(self):
        return self.at

    def numel(self):
        return int(np.prod(self.shape))

    def element_size(self):
        return {"bfloat16": 2, "float16": 2, "float32": 4, "int32": 4, "int64": 8, "uint8": 1}[self.dtype[6:]]


def fake_cache(**kw):
    d = dict(k=Fake("bfloat16", 8, 16, 2, 128), v=Fake("bfloat16", 8, 16, 2, 128), table=Fake("int32", 3, 4))
    d.update(kw)
    return KvCache.of(d["k"], d["v"], d["table"])


def test_binding_reads_layouts():
    c = fake_cache()
    assert (c.num_pages, c.page_size, c.kv_heads, c.head_dim, c.num_seqs, c.max_blocks) == (8, 16, 2, 128, 3, 4)
    assert (c.table_stride, c.page_stride, c.token_stride, c.head_stride) == (4, 4096, 256, 128)
    one = dict(k=Fake("bfloat16", 8, 16, 1, 64, stride=[1024, 64, 3, 1]), v=Fake("bfloat16", 8, 16, 1, 64, stride=[1024, 64, 5, 1]))
    assert fake_cache(**one).head_stride == 0  # the stride of an axis of one says nothing
    assert append(fake_cache(**one), rope=None, ldq=256, ldq_out=256, ldk=64, ldv=64, tokens=0) == 0
    by_head = [4096, 128, 2048, 1]
    c = fake_cache(k=Fake("bfloat16", 8, 16, 2, 128, stride=by_head), v=Fake("bfloat16", 8, 16, 2, 128, stride=by_head))
    assert (c.page_stride, c.token_stride, c.head_stride) == (4096, 128, 2048)


@pytest.mark.parametrize("bad", [
    dict(k=Fake("float16", 8, 16, 2, 128)), dict(v=Fake("bfloat16", 9, 16, 2, 128)), dict(table=Fake("int64", 3, 4)),
    dict(k=Fake("bfloat16", 8, 16, 256)), dict(v=Fake("bfloat16", 8, 16, 2, 128, stride=[4096, 128, 2048, 1])),
    dict(table=Fake("int32", 3, 4, stride=[1, 3]))])
def test_binding_refuses_other_caches(bad):
    with pytest.raises(iris_cuda.IrisCudaError, match="KvCache"):
        fake_cache(**bad)


def test_binding_refuses_other_tensors():
    E, c = iris_cuda.IrisCudaError, fake_cache()
    i = Fake("int32", 5)
    qkv = dict(q=Fake("float32", 5, 512), k=Fake("float32", 5, 256), v=Fake("float32", 5, 256))

    def call(**kw):
        d = {**qkv, **dict(q_out=Fake("bfloat16", 5, 4, 128), seq=i, pos=i, heads=4), **kw}
        iris_cuda.rope_append(c, None, d["q_out"], d["q"], d["k"], d["v"], d["seq"], d["pos"], heads=d["heads"],
                              q_norm=d.get("q_norm"))

    for bad in (dict(k=Fake("float16", 5, 256)), dict(q=Fake("bfloat16", 5, 512)), dict(v=Fake("float32", 4, 256)),
                dict(q_out=Fake("float32", 5, 4, 128)), dict(heads=3), dict(pos=Fake("int64", 5)), dict(pos=Fake("int32", 4)),
                dict(q_norm=Fake("float32", 64)), dict(q_norm=Fake("bfloat16", 128))):
        with pytest.raises(E):
            call(**bad)
    q = Fake("bfloat16", 5, 4, 128)
    for bad in (dict(out=Fake("bfloat16", 5, 4, 64)), dict(q=Fake("float32", 5, 4, 128)), dict(pos=Fake("int32", 6)),
                dict(seq=Fake("int64", 5)), dict(q=Fake("bfloat16", 5, 4, 128, stride=[512, 1, 4]))):
        d = {**dict(out=q, q=q, seq=i, pos=i), **bad}
        with pytest.raises(E):
            iris_cuda.attention_paged(c, d["out"], d["q"], d["seq"], d["pos"], scale=0.1, workspace=Fake("uint8", 16))
    f = Fake("float32", 5)
    for bad in (dict(logits=Fake("float16", 5, 100)), dict(logits=Fake("float32", 5, 100, stride=[1, 5])),
                dict(targets=Fake("int64", 5)), dict(entropy=Fake("float32", 4)), dict(top_ids=Fake("int64", 5, 3)),
                dict(top_logprobs=Fake("float32", 5, 2)), dict(top_ids=Fake("int32", 5, 3, stride=[6, 1])),
                dict(top_ids=Fake("int32", 5, 1, stride=[4, 1]), top_logprobs=None)):
        d = {**dict(logits=Fake("float32", 5, 100), targets=i, logprob=f, entropy=f, top_ids=Fake("int32", 5, 3),
                    top_logprobs=Fake("float32", 5, 3)), **bad}
        with pytest.raises(E):
            iris_cuda.token_logprobs(*d.values(), workspace=Fake("uint8", 1 << 20))


@pytest.mark.parametrize("amplitude", (1e300, 1e-60, 0.0, -1.0, float("nan"), float("inf")))
def test_rope_amplitude_outside_f32(amplitude):
    with pytest.raises(iris_cuda.IrisCudaError, match="amplitude"):
        Rope.of(64, 1e4, amplitude=amplitude)
