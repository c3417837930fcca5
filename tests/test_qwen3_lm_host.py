"""What iris_cuda_qwen3_load_lm refuses before it touches the device: models
whose config.json asks for what the decoder layers do not do."""
import json

import pytest

import iris_cuda
from test_qwen3_oracle import CFG


def load(tmp_path, lm, **more):
    (tmp_path / "config.json").write_text(json.dumps(dict(CFG, **more), indent=1))
    with pytest.raises(iris_cuda.IrisCudaError) as e:  # without weights in the directory every load ends in some error
        (iris_cuda.Qwen3.load_lm if lm else iris_cuda.Qwen3.load)(str(tmp_path)).close()
    return str(e.value)


REFUSED = [
    (dict(rope_scaling=dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)), "scales rotary"),
    (dict(rope_scaling=dict(type="linear", factor=2.0)), "scales rotary"),
    (dict(rope_parameters=dict(rope_theta=1e6, rope_type="llama3", factor=8.0)), "scales rotary"),
    (dict(rms_norm_eps=1e-5), "rms_norm_eps"),
    (dict(use_sliding_window=True, sliding_window=4096), "use_sliding_window"),
    (dict(attention_bias=True), "attention_bias"),
]


@pytest.mark.parametrize("more,why", REFUSED)
def test_configs_a_language_model_is_refused_for(tmp_path, more, why):
    assert why in load(tmp_path, True, **more)
    assert why not in load(tmp_path, False, **more)  # the encoder reads prompts as ever


@pytest.mark.parametrize("more", [
    {}, dict(rope_scaling=None, use_sliding_window=False, attention_bias=False, rms_norm_eps=1e-6, sliding_window=None),
    dict(rope_parameters=dict(rope_theta=1e6, rope_type="default")), dict(rope_scaling=dict(rope_type="default"))])
def test_configs_a_language_model_takes(tmp_path, more):
    e = load(tmp_path, True, **more)
    assert not any(why in e for _, why in REFUSED)
