"""From a GGUF file to logits on the GPU: the file's configuration and tensors through
``gguf_read_config``, ``build_model`` and ``load_weights`` into ``forward``, against the definition in
64 bits with the settings that the file was written with."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import gguf_oracle as O
from tests.test_gpu_forward import _check

pytestmark = pytest.mark.gpu
gguf = pytest.importorskip("gguf")

HID, HEADS, KV, D, INTER, VOCAB, LAYERS = 512, 8, 2, 64, 768, 320, 2
THETA = 500000.0
PROJ = {"attn_q": (HEADS * D, HID, O.Q4_K), "attn_k": (KV * D, HID, O.Q4_K), "attn_v": (KV * D, HID, O.Q6_K),
        "attn_output": (HID, HEADS * D, O.Q4_0), "ffn_gate": (INTER, HID, O.Q4_K), "ffn_up": (INTER, HID, O.Q4_K),
        "ffn_down": (HID, INTER, O.Q6_K)}
F = THETA ** (-2.0 * np.arange(D // 2) / D)
# name: architecture, metadata, what it means: eps, window, radians per position, factor on the turned values
FILES = {
    "llama with divisors": ("llama", {"attention.layer_norm_rms_epsilon": 1e-5}, 1e-5, 0, F / np.linspace(1, 8, D // 2), 1.0),
    "qwen3 with yarn": ("qwen3", {"attention.layer_norm_rms_epsilon": 1e-6, "rope.scaling.type": "yarn",
                                  "rope.scaling.factor": 4.0, "rope.scaling.original_context_length": 64},
                        1e-6, 0, None, 0.1 * math.log(4.0) + 1),
    "llama with a window": ("llama", {"attention.layer_norm_rms_epsilon": 2e-4, "attention.sliding_window": 24,
                                      "rope.scaling.type": "linear", "rope.scaling.factor": 2.0}, 2e-4, 24, F / 2, 1.0),
    "part of the head": ("llama", {"attention.layer_norm_rms_epsilon": 1e-5, "rope.dimension_count": 32}, 1e-5, 0,
                         THETA ** (-2.0 * np.arange(16) / 32), 1.0),
}


def _yarn():
    pair = [D * math.log(64 / (t * 2 * math.pi)) / (2 * math.log(THETA)) for t in (32.0, 1.0)]
    low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), D - 1)
    ramp = np.clip((np.arange(D // 2) - low) / max(high - low, 0.001), 0, 1)
    return F * (1 - ramp) + F / 4 * ramp


def _write(path, name):
    """The file, and its tensors as 64-bit matrices by their GGUF names."""
    arch, fields, eps, window, radians, factor = FILES[name]
    w, dense = gguf.GGUFWriter(str(path), arch), {}
    w.add_block_count(LAYERS)
    w.add_embedding_length(HID)
    w.add_feed_forward_length(INTER)
    w.add_head_count(HEADS)
    w.add_head_count_kv(KV)
    w.add_key_length(D)
    w.add_context_length(4096)
    w.add_rope_freq_base(THETA)
    for key, value in fields.items():
        add = w.add_string if isinstance(value, str) else w.add_uint32 if isinstance(value, int) else w.add_float32
        add(f"{arch}.{key}", value)

    def quant(tensor, n, k, qt, seed):
        raw = O.make_weights(n, k, qt, seed=seed)
        w.add_tensor(tensor, np.ascontiguousarray(raw).reshape(n, -1), raw_dtype=gguf.GGMLQuantizationType(qt))
        dense[tensor] = O.dequantize(raw, qt, n, k).astype(np.float64)

    def vector(tensor, value):
        w.add_tensor(tensor, value.astype(np.float32))
        dense[tensor] = value.astype(np.float32).astype(np.float64)
    rng = np.random.RandomState(5)
    for layer in range(LAYERS):
        for i, (nm, (n, k, qt)) in enumerate(PROJ.items()):
            quant(f"blk.{layer}.{nm}.weight", n, k, qt, 100 * layer + i)
        for nm in ("attn_norm", "ffn_norm"):
            vector(f"blk.{layer}.{nm}.weight", 1 + 0.1 * rng.randn(HID))
        if arch == "qwen3":
            for nm in ("attn_q_norm", "attn_k_norm"):
                vector(f"blk.{layer}.{nm}.weight", 1 + 0.1 * rng.randn(D))
    quant("token_embd.weight", VOCAB, HID, O.Q8_0, 998)
    quant("output.weight", VOCAB, HID, O.Q6_K, 999)
    vector("output_norm.weight", 1 + 0.1 * rng.randn(HID))
    if name == "llama with divisors":
        vector("rope_freqs.weight", np.linspace(1, 8, D // 2))
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()
    return dense


def _logits(w, ids, name):
    """The definition in 64 bits: logits after every token of one sequence."""
    arch, _, eps, window, radians, factor = FILES[name]
    radians = _yarn() if radians is None else radians
    t, rot = len(ids), 2 * len(radians)

    def norm(x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * g

    def turned(x):
        z = factor * np.exp(1j * np.arange(t)[:, None] * radians[None])[:, None]
        y = x.copy()
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if arch == "llama" else (slice(0, rot // 2), slice(rot // 2, rot))
        c = (x[..., a] + 1j * x[..., b]) * z
        y[..., a], y[..., b] = c.real, c.imag
        return y
    i, j = np.arange(t)[:, None], np.arange(t)[None]
    hidden = (j > i) | ((j <= i - window) if window else False)
    h = w["token_embd.weight"][ids]
    for layer in range(LAYERS):
        def p(nm):
            return w[f"blk.{layer}.{nm}.weight"]
        x = norm(h, p("attn_norm"))
        q, k, v = ((x @ p(f"attn_{c}").T).reshape(t, -1, D) for c in "qkv")
        if arch == "qwen3":
            q, k = norm(q, p("attn_q_norm")), norm(k, p("attn_k_norm"))
        q, k = turned(q), turned(k)
        k, v = k.repeat(HEADS // KV, axis=1), v.repeat(HEADS // KV, axis=1)
        s = np.where(hidden[None], -np.inf, np.einsum("thd,jhd->htj", q, k) / math.sqrt(D))
        e = np.exp(s - s.max(-1, keepdims=True))
        h = h + np.einsum("htj,jhd->thd", e / e.sum(-1, keepdims=True), v).reshape(t, -1) @ p("attn_output").T
        x = norm(h, p("ffn_norm"))
        g, u = x @ p("ffn_gate").T, x @ p("ffn_up").T
        h = h + (g / (1 + np.exp(-g)) * u) @ p("ffn_down").T
    return norm(h, w["output_norm.weight"]) @ w["output.weight"].T


@pytest.mark.parametrize("name", FILES)
def test_logits_of_a_file(cuda, tmp_path, name):
    from vllm_webgpu_b200.kv_cache import PagedKVCache
    from vllm_webgpu_b200.models.gemma4 import build_model
    from vllm_webgpu_b200.quant.gguf_loader import gguf_read_config
    path = str(tmp_path / "model.gguf")
    dense = _write(path, name)
    cfg = gguf_read_config(path)
    model = build_model(cfg["architectures"][0], cfg, "cuda:0")
    model.load_weights(path)
    rng = np.random.RandomState(3)
    texts = {"a": rng.randint(0, VOCAB, 90), "b": rng.randint(0, VOCAB, 33)}
    want = {s: _logits(dense, ids, name) for s, ids in texts.items()}
    cache = PagedKVCache(LAYERS, 16, KV, D, 16, torch.float16, "cuda:0")
    done = dict.fromkeys(texts, 0)
    for counts in ({"a": 60, "b": 7}, {"b": 1, "a": 1}, {"a": 1, "b": 20}, {"a": 20, "b": 1}, {"a": 1, "b": 1}):
        ids = np.concatenate([texts[s][done[s]:done[s] + n] for s, n in counts.items()])
        got = model.forward(torch.from_numpy(ids).cuda(), None, cache.extend(list(counts), list(counts.values())))
        for row, (s, n) in enumerate(counts.items()):
            done[s] += n
            _check(got[row], want[s][done[s] - 1])
