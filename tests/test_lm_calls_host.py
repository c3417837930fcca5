"""Calls of the language-model operators that need no GPU: batches of no rows,
shapes that no device holds."""
import iris_cuda
from test_lm_ops_host import Fake, append, attend, cache, fake_cache, logprobs, refused


def none(dtype, *shape):
    """An empty tensor, which has no address."""
    return Fake(dtype, *shape, at=0)


def test_batches_of_no_rows():
    c, i = fake_cache(), none("int32", 0)
    for ty in ("float32", "bfloat16"):
        iris_cuda.rope_append(c, None, none("bfloat16", 0, 4, 128), none(ty, 0, 512), none(ty, 0, 256), none(ty, 0, 256), i, i, heads=4)
        for k in (0, 3):
            iris_cuda.token_logprobs(none(ty, 0, 100), i, none("float32", 0), none("float32", 0), none("int32", 0, k),
                                     none("float32", 0, k), workspace=none("uint8", 0))
    for seq in (i, None):
        iris_cuda.attention_paged(c, none("bfloat16", 0, 4, 128), none("bfloat16", 0, 4, 128), seq, i, scale=0.1, workspace=none("uint8", 0))
    assert append(cache(), tokens=0, q=None, k=None, v=None, q_out=None, seq=None, pos=None) == 0
    assert attend(cache(), rows=0, out=None, q=None, pos=None, ws=None, ws_bytes=0) == 0
    assert logprobs(rows=0, logits=None, targets=None, top_ids=None, top_logprobs=None, ws=None, ws_bytes=0) == 0
    # what is wrong whatever the rows is still refused
    assert append(cache(), tokens=0, ldk=255) and attend(cache(), rows=0, heads=3) and logprobs(rows=0, top_k=33)


def test_more_logits_than_any_device_holds():
    """Refused as an argument, in the call and by its workspace's size."""
    L = iris_cuda.lib()
    for rows, vocab in ((2 ** 31 - 1, 2 ** 30), (2 ** 31 - 1, 513), (1025, 2 ** 30)):
        assert L.iris_gpu_token_logprobs_workspace(rows, vocab) == 0
        refused(logprobs(rows=rows, vocab=vocab, ld=vocab, ws_bytes=2 ** 63), "rows of")
    for rows, vocab in ((2 ** 31 - 1, 1), (2 ** 31 - 1, 512), (1024, 2 ** 30), (8192, 151936)):
        # at least the largest values of blocks of 256, four bytes each
        assert L.iris_gpu_token_logprobs_workspace(rows, vocab) >= rows * -(-vocab // 256) * 4
