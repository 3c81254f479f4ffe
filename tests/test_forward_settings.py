"""What ``LlamaB200Model.forward`` takes from a file and a configuration, on the CPU: it applies a
setting or a tensor, or it refuses it before the first kernel."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import gguf_oracle as O

gguf = pytest.importorskip("gguf")

HID, HEADS, KV, D, INTER, VOCAB = 64, 2, 1, 32, 96, 40
TENSORS = {"token_embd.weight": (VOCAB, HID), "output.weight": (VOCAB, HID)}
for _l in range(2):
    TENSORS |= {f"blk.{_l}.attn_q.weight": (HEADS * D, HID), f"blk.{_l}.attn_k.weight": (KV * D, HID),
                f"blk.{_l}.attn_v.weight": (KV * D, HID), f"blk.{_l}.attn_output.weight": (HID, HEADS * D),
                f"blk.{_l}.ffn_gate.weight": (INTER, HID), f"blk.{_l}.ffn_up.weight": (INTER, HID),
                f"blk.{_l}.ffn_down.weight": (HID, INTER)}
NORMS = ["output_norm.weight"] + [f"blk.{_l}.{n}_norm.weight" for _l in range(2) for n in ("attn", "ffn")]


def write_gguf(path, arch="llama", more=None, **fields):
    """A whole small model as a GGUF file: all that a Llama layer has, and ``more`` ({name: array}).
    ``fields``: metadata below the architecture's prefix, dots as two underscores."""
    w = gguf.GGUFWriter(str(path), arch)
    w.add_block_count(2)
    w.add_embedding_length(HID)
    w.add_feed_forward_length(INTER)
    w.add_head_count(HEADS)
    w.add_head_count_kv(KV)
    w.add_key_length(D)
    w.add_context_length(4096)
    w.add_rope_freq_base(500000.0)
    for name, value in fields.items():
        key = f"{arch}.{name.replace('__', '.')}"
        if isinstance(value, str):
            w.add_string(key, value)
        elif isinstance(value, int):
            w.add_uint32(key, value)
        else:
            w.add_float32(key, value)
    for i, (name, (n, k)) in enumerate(TENSORS.items()):
        w.add_tensor(name, O.make_weights(n, k, O.Q8_0, seed=i), raw_dtype=gguf.GGMLQuantizationType(O.Q8_0))
    for name in NORMS:
        w.add_tensor(name, np.ones(HID, np.float32))
    for name, value in (more or {}).items():
        w.add_tensor(name, value)
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()
    return str(path)


def _model(path, cfg=None):
    from vllm_webgpu_b200.models.llama import LlamaB200Model
    from vllm_webgpu_b200.quant.gguf_loader import gguf_read_config
    model = LlamaB200Model(gguf_read_config(path) if cfg is None else cfg, device="cpu")
    model.load_weights(path)
    return model


def _forward(model):
    from vllm_webgpu_b200.kv_cache import PagedKVCache
    cache = PagedKVCache(2, 4, KV, D, 16, torch.float16, "cpu")
    return model.forward(torch.zeros(3, dtype=torch.int64), None, cache.extend(["a"], [3]))


def test_a_plain_file_gets_as_far_as_the_kernels(tmp_path):
    with pytest.raises(ValueError, match="CUDA"):
        _forward(_model(write_gguf(tmp_path / "m.gguf")))


@pytest.mark.parametrize("name,size", [("blk.1.attn_q.bias", HEADS * D), ("blk.0.attn_k.bias", KV * D),
                                       ("blk.0.attn_v.bias", KV * D), ("blk.1.attn_output.bias", HID),
                                       ("blk.0.ffn_gate.bias", INTER), ("blk.1.ffn_up.bias", INTER),
                                       ("blk.0.ffn_down.bias", HID), ("blk.0.attn_norm.bias", HID),
                                       ("blk.0.post_ffw_norm.weight", HID), ("blk.1.layer_output_scale.weight", 1),
                                       ("blk.1.attn_sinks.weight", HEADS), ("output.bias", VOCAB),
                                       ("rope_factors_long.weight", D // 2)])
def test_a_file_with_a_tensor_that_forward_leaves_out_is_refused(tmp_path, name, size):
    model = _model(write_gguf(tmp_path / "m.gguf", arch="qwen2", more={name: np.zeros(size, np.float32)}))
    with pytest.raises(NotImplementedError, match="tensors"):
        _forward(model)


def test_a_bias_is_loaded_under_its_name(tmp_path):
    bias = np.arange(HEADS * D, dtype=np.float32)
    model = _model(write_gguf(tmp_path / "m.gguf", arch="qwen2", more={"blk.1.attn_q.bias": bias}))
    assert torch.equal(model.weights["model.layers.1.self_attn.q_proj.bias"], torch.from_numpy(bias))
    with pytest.raises(NotImplementedError, match="bias"):
        model.transformer_layer(1, torch.zeros(3, HID), None, type("Step", (), {"cache": type("Cache", (), {"dtype": torch.float16})}))


def test_a_safetensors_bias_is_refused(tmp_path):
    import json
    import struct
    header, data = {}, b""
    for name, n in (("model.norm.weight", HID), ("model.layers.0.self_attn.q_proj.bias", HEADS * D)):
        header[name] = {"dtype": "F16", "shape": [n], "data_offsets": [len(data), len(data) + 2 * n]}
        data += np.ones(n, np.float16).tobytes()
    head = json.dumps(header).encode()
    p = tmp_path / "m.safetensors"
    p.write_bytes(struct.pack("<Q", len(head)) + head + data)
    with pytest.raises(NotImplementedError, match="q_proj.bias"):
        _forward(_model(str(p), cfg={"num_hidden_layers": 2}))


def test_weights_that_change_are_looked_over_again(tmp_path):
    model = _model(write_gguf(tmp_path / "m.gguf"))
    with pytest.raises(ValueError, match="CUDA"):
        _forward(model)
    model.weights["model.layers.0.self_attn.v_proj.bias"] = torch.zeros(KV * D)
    with pytest.raises(NotImplementedError, match="v_proj.bias"):
        _forward(model)
    model.load_weights(write_gguf(tmp_path / "n.gguf", more={"blk.0.attn_k.bias": np.zeros(KV * D, np.float32)}))
    with pytest.raises(NotImplementedError, match="k_proj.bias"):
        _forward(model)


@pytest.mark.parametrize("arch,eps", [("qwen3", 1e-6), ("llama", 1e-5), ("qwen2", 3e-6)])
def test_the_file_gives_the_norms_eps(tmp_path, arch, eps):
    from vllm_webgpu_b200.quant.gguf_loader import gguf_read_config
    model = _model(write_gguf(tmp_path / "m.gguf", arch, attention__layer_norm_rms_epsilon=eps))
    assert model._cfg("rms_norm_eps") == np.float32(eps)
    assert gguf_read_config(write_gguf(tmp_path / "n.gguf"))["rms_norm_eps"] is None


def _turns(model):
    """Radians per position of each pair as forward turns them, and the factor."""
    steps, factor, _ = model._rope_plan()
    turns = steps.numpy().view(np.uint64).astype(np.float64) * 2.0 ** -64
    return np.minimum(turns, 1 - turns) * 2 * np.pi, factor


def _plain(n=D, theta=500000.0):
    return theta ** (-2.0 * np.arange(n // 2) / n)


def _same(got, want):  # steps are rounded to 2^-64 of a turn, the file's numbers to 32 bits
    assert np.allclose(got, want, rtol=1e-6, atol=1e-15)


def test_the_file_gives_the_stretch_of_positions(tmp_path):
    got, factor = _turns(_model(write_gguf(tmp_path / "plain.gguf")))
    _same(got, _plain())
    assert factor == 1.0
    for name, fields in (("new", {"rope__scaling__type": "linear", "rope__scaling__factor": 4.0}),
                         ("old", {"rope__scale_linear": 4.0})):
        got, factor = _turns(_model(write_gguf(tmp_path / f"{name}.gguf", **fields)))
        _same(got, _plain() / 4)
        assert factor == 1.0
    none = {"rope__scaling__type": "none", "rope__scaling__factor": 4.0}
    _same(_turns(_model(write_gguf(tmp_path / "none.gguf", **none)))[0], _plain())


@pytest.mark.parametrize("more,by,fast,slow", [
    ({}, 1.0, 32.0, 1.0),
    ({"rope__scaling__attn_factor": 0.75}, 0.75, 32.0, 1.0),
    ({"rope__scaling__yarn_beta_fast": 16.0, "rope__scaling__yarn_beta_slow": 2.0}, 1.0, 16.0, 2.0),
])
def test_the_file_gives_yarn(tmp_path, more, by, fast, slow):
    fields = {"rope__scaling__type": "yarn", "rope__scaling__factor": 8.0, "rope__scaling__original_context_length": 2048}
    got, factor = _turns(_model(write_gguf(tmp_path / "m.gguf", **fields, **more)))
    f = _plain()
    # a pair that makes more than ``fast`` turns over the old context stays, below ``slow`` it is
    # stretched whole; between the two by its index
    pair = [D * np.log(2048 / (t * 2 * np.pi)) / (2 * np.log(500000.0)) for t in (fast, slow)]
    low, high = max(np.floor(pair[0]), 0), min(np.ceil(pair[1]), D - 1)
    ramp = np.clip((np.arange(D // 2) - low) / (high - low), 0, 1)
    _same(got, f * (1 - ramp) + f / 8 * ramp)
    assert factor == pytest.approx(by * (0.1 * np.log(8.0) + 1), rel=1e-6)


def test_a_stretch_that_is_not_there_is_refused(tmp_path):
    model = _model(write_gguf(tmp_path / "m.gguf", rope__scaling__type="longrope", rope__scaling__factor=4.0))
    with pytest.raises(ValueError, match="longrope"):
        model._rope_plan()


def test_the_file_gives_the_rotary_width(tmp_path):
    got, _ = _turns(_model(write_gguf(tmp_path / "m.gguf", rope__dimension_count=20)))
    assert got.shape == (10,)
    _same(got, _plain(20))


def test_llama3_frequencies_are_stretched_once(tmp_path):
    """A Hugging Face configuration with llama3 scaling beside a GGUF file that carries the same
    stretch as divisors."""
    f = _plain()
    turns = 512 * f / (2 * np.pi)
    keep = np.clip((turns - 1) / (4 - 1), 0, 1)
    want = keep * f + (1 - keep) * f / 8
    divisors = (f / want).astype(np.float32)
    assert divisors.max() == 8 and divisors.min() == 1
    path = write_gguf(tmp_path / "m.gguf", more={"rope_freqs.weight": divisors})
    scaling = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 512}
    cfg = {"hidden_size": HID, "num_attention_heads": HEADS, "head_dim": D, "rope_theta": 500000.0}
    _same(_turns(_model(path))[0], want)
    for key in ("rope_type", "type"):
        other = {(key if k == "rope_type" else k): v for k, v in scaling.items()}
        _same(_turns(_model(path, {**cfg, "rope_scaling": other}))[0], want)
    _same(_turns(_model(write_gguf(tmp_path / "n.gguf"), {**cfg, "rope_scaling": scaling}))[0], want)
    # another stretch beside divisors is one more: both hold
    linear = {"rope_type": "linear", "factor": 2.0}
    _same(_turns(_model(path, {**cfg, "rope_scaling": linear}))[0], want / 2)


def test_the_order_of_pairs_is_the_weights(tmp_path):
    """GGUF files of the llama architecture hold q and k for pairs (2i, 2i + 1), whatever
    configuration stands beside them; other files for pairs (i, i + half)."""
    from vllm_webgpu_b200.models.llama import LlamaB200Model
    from vllm_webgpu_b200.quant.gguf_loader import FileWeights, gguf_read_config
    llama, qwen = write_gguf(tmp_path / "l.gguf"), write_gguf(tmp_path / "q.gguf", "qwen3")
    hf = {"hidden_size": HID, "num_attention_heads": HEADS, "head_dim": D, "rope_theta": 500000.0}

    def order(path, cfg):
        return _model(path, cfg)._rope_plan()[2]
    assert order(llama, None) is True and order(qwen, None) is False
    assert order(llama, hf) is True and order(qwen, hf) is False
    assert order(qwen, gguf_read_config(llama)) is False
    assert order(llama, {**hf, "rope_interleaved": False}) is False  # said outright
    model = LlamaB200Model(gguf_read_config(llama), device="cpu")
    model.weights = FileWeights()  # of safetensors
    assert model._rope_plan()[2] is False
    model = LlamaB200Model(gguf_read_config(llama), device="cpu")
    model.weights = {}             # put together by hand: the configuration's file
    assert model._rope_plan()[2] is True


@pytest.mark.parametrize("cfg,want", [
    ({}, [0, 0, 0]),
    ({"sliding_window": None}, [0, 0, 0]),
    ({"sliding_window": 48}, [48, 48, 48]),                                                   # Mistral
    ({"sliding_window": 48, "use_sliding_window": False, "max_window_layers": 1}, [0, 0, 0]),  # Qwen2, off
    ({"sliding_window": 48, "use_sliding_window": True, "max_window_layers": 1}, [0, 48, 48]),
    ({"sliding_window": 48, "layer_types": ["full_attention", "sliding_attention", "full_attention"]}, [0, 48, 0]),
])
@pytest.mark.parametrize("counts", [[1, 1], [5, 1]], ids=["single", "mixed"])
def test_the_window_reaches_attention(tmp_path, monkeypatch, cfg, want, counts):
    """A layer's call of attention is given the configuration's window (the kernels stand aside)."""
    from vllm_webgpu_b200 import ops
    from vllm_webgpu_b200.kv_cache import PagedKVCache
    model = _model(write_gguf(tmp_path / "m.gguf"),
                   {"hidden_size": HID, "num_attention_heads": HEADS, "num_key_value_heads": KV, "head_dim": D, **cfg})
    model._w = lambda layer, proj: torch.zeros(INTER if proj in ("gate", "up") else HID, HID)
    seen = []

    def attention(q, *rest, window=0, **kw):
        seen.append(window)
        return q
    monkeypatch.setattr(ops, "paged_attention", attention)
    monkeypatch.setattr(ops, "paged_prompt_attention", attention)
    monkeypatch.setattr(ops, "rope_append", lambda q, *rest, **kw: q.contiguous())
    monkeypatch.setattr(ops, "rms_norm", lambda x, w, eps, residual=None, out_dtype=None: (x, residual) if residual is not None else x)
    for name in ("project_qkv", "project_ffn_act"):
        monkeypatch.setattr(type(model), name, lambda self, *a: None)
    for name in ("project_o", "project_down"):
        monkeypatch.setattr(type(model), name, lambda self, layer, x, out: out)
    cache = PagedKVCache(3, 4, KV, D, 16, torch.float16, "cpu")
    step = cache.extend(["a", "b"], counts)
    model.weights = {**model.weights, **{f"model.layers.2.{n}_layernorm.weight": torch.ones(HID)
                                         for n in ("input", "post_attention")}}
    for layer in range(3):
        model.transformer_layer(layer, torch.zeros(sum(counts), HID), None, step)
    assert seen == want


def test_the_file_gives_the_window(tmp_path):
    model = _model(write_gguf(tmp_path / "m.gguf", attention__sliding_window=48))
    assert [model._window(layer) for layer in range(2)] == [48, 48]
    assert _model(write_gguf(tmp_path / "n.gguf"))._window(0) == 0


def test_rotary_settings_of_newer_configurations(tmp_path):
    """Configurations that hold theta, the stretch and the rotary part together, as a dict or as
    the installed transformers' objects."""
    from types import SimpleNamespace
    path = write_gguf(tmp_path / "m.gguf")
    base = {"hidden_size": HID, "num_attention_heads": HEADS, "head_dim": D}

    def turns(**params):
        cfg = {**base, "rope_parameters": params}
        got = _turns(_model(path, cfg))[0]
        assert np.array_equal(got, _turns(_model(path, SimpleNamespace(**cfg)))[0])
        return got
    _same(turns(rope_type="default", rope_theta=500000.0), _plain())
    _same(turns(rope_type="linear", factor=4.0, rope_theta=500000.0), _plain() / 4)
    _same(turns(rope_type="default", rope_theta=500000.0, partial_rotary_factor=0.5), _plain(D // 2))
    transformers = pytest.importorskip("transformers")
    cfg = transformers.LlamaConfig(hidden_size=HID, num_attention_heads=HEADS, num_key_value_heads=KV, head_dim=D,
                                   rope_parameters={"rope_type": "linear", "factor": 4.0, "rope_theta": 500000.0})
    _same(_turns(_model(path, cfg))[0], _plain() / 4)
    cfg = transformers.MistralConfig(hidden_size=HID, num_attention_heads=HEADS, head_dim=D, sliding_window=48)
    model = _model(path, cfg)
    assert model._window(0) == 48
    _same(_turns(model)[0], _plain(theta=10000.0))
    cfg = transformers.Qwen2Config(hidden_size=HID, num_attention_heads=HEADS, num_hidden_layers=3, sliding_window=48,
                                   use_sliding_window=True, max_window_layers=2)
    assert [_model(path, cfg)._window(layer) for layer in range(3)] == [0, 0, 48]
    assert _model(path, transformers.Qwen2Config(sliding_window=48))._window(0) == 0


@pytest.mark.parametrize("arch", ["granite", "phi3", "gemma2", "olmo2"])
def test_files_of_other_architectures_are_refused(tmp_path, arch):
    path = write_gguf(tmp_path / "m.gguf", arch)
    hf = {"hidden_size": HID, "num_attention_heads": HEADS, "head_dim": D, "num_hidden_layers": 2}
    for cfg in (None, hf):
        with pytest.raises(NotImplementedError, match=arch):
            _forward(_model(path, cfg))


@pytest.mark.parametrize("setting", [{"final_logit_softcapping": 30.0}, {"attn_logit_softcapping": 50.0},
                                     {"hidden_act": "gelu_pytorch_tanh"},
                                     {"layer_types": ["full_attention", "chunked_attention"]},
                                     {"rope_parameters": {"full_attention": {"rope_theta": 1e6},
                                                          "sliding_attention": {"rope_theta": 1e4}}}])
def test_settings_that_forward_leaves_out_are_refused(tmp_path, setting):
    hf = {"hidden_size": HID, "num_attention_heads": HEADS, "num_key_value_heads": KV, "head_dim": D,
          "num_hidden_layers": 2, "hidden_act": "silu"}
    model = _model(write_gguf(tmp_path / "m.gguf"), hf)
    with pytest.raises(ValueError, match="CUDA"):
        _forward(model)
    model.model_config = {**hf, **setting}  # looked over again
    with pytest.raises(NotImplementedError):
        _forward(model)


def test_other_weights_bring_their_own_rotary_plan(tmp_path):
    model = _model(write_gguf(tmp_path / "a.gguf"))
    first = model._rope_plan()
    assert model._rope_plan() is first
    divisors = np.full(D // 2, 2.0, np.float32)
    model.load_weights(write_gguf(tmp_path / "b.gguf", more={"rope_freqs.weight": divisors}))
    _same(_turns(model)[0], _plain() / 2)
    model.weights["rope_freqs.weight"] = torch.full((D // 2,), 4.0)
    _same(_turns(model)[0], _plain() / 4)
    model.model_config = {**model.model_config, "rope_theta": 10000.0}
    _same(_turns(model)[0], _plain(theta=10000.0) / 4)
    model.load_weights(write_gguf(tmp_path / "c.gguf", "qwen3"))
    assert model._rope_plan()[2] is False


@pytest.mark.parametrize("more", [{"mscale": 0.7}, {"mscale_all_dim": 1.0}, {"truncate": False}])
def test_yarn_options_that_rope_steps_leaves_out_are_refused(more):
    from vllm_webgpu_b200 import ops
    yarn = {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 2048}
    want, factor = ops.rope_steps(D, 10000.0, yarn, device="cpu")
    same, _ = ops.rope_steps(D, 10000.0, {**yarn, "truncate": True, "mscale": None}, device="cpu")
    assert torch.equal(want, same) and factor > 1
    with pytest.raises(ValueError, match=next(iter(more))):
        ops.rope_steps(D, 10000.0, {**yarn, **more}, device="cpu")
