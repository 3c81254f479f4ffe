"""Whole layers on the GPU: a small random quantized model's forward pass over the paged cache
(prompts, single tokens, several sequences at once) against its definition in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import gguf_oracle as O

pytestmark = pytest.mark.gpu

HID, HEADS, KV, D, INTER, VOCAB, LAYERS = 512, 8, 2, 64, 768, 320, 2
NAMES = {"self_attn.q_proj": (HEADS * D, HID), "self_attn.k_proj": (KV * D, HID), "self_attn.v_proj": (KV * D, HID),
         "self_attn.o_proj": (HID, HEADS * D), "mlp.gate_proj": (INTER, HID), "mlp.up_proj": (INTER, HID),
         "mlp.down_proj": (HID, INTER)}


def _model(interleaved, qk_norm):
    from vllm_webgpu_b200.formats import GGUFQuantTensor
    from vllm_webgpu_b200.models.llama import LlamaB200Model
    cfg = {"hidden_size": HID, "num_attention_heads": HEADS, "num_key_value_heads": KV, "head_dim": D,
           "num_hidden_layers": LAYERS, "rope_theta": 10000.0, "rope_interleaved": interleaved, "rms_norm_eps": 1e-5}
    model, dense = LlamaB200Model(cfg, device="cuda:0"), {}

    def quant(name, n, k, qt, seed):
        raw = O.make_weights(n, k, qt, seed=seed)
        model.weights[name] = GGUFQuantTensor(torch.from_numpy(np.ascontiguousarray(raw).reshape(n, -1)).cuda(), qt, (n, k))
        dense[name] = O.dequantize(raw, qt, n, k).astype(np.float64)

    def vector(name, n, seed):
        w = 1 + 0.1 * np.random.RandomState(seed).randn(n).astype(np.float32)
        model.weights[name], dense[name] = torch.from_numpy(w).cuda(), w.astype(np.float64)
    for layer in range(LAYERS):
        for i, (nm, (n, k)) in enumerate(NAMES.items()):
            quant(f"model.layers.{layer}.{nm}.weight", n, k, O.Q6_K if nm == "mlp.down_proj" else O.Q4_K, 100 * layer + i)
        vector(f"model.layers.{layer}.input_layernorm.weight", HID, 7 + layer)
        vector(f"model.layers.{layer}.post_attention_layernorm.weight", HID, 17 + layer)
        if qk_norm:
            vector(f"model.layers.{layer}.self_attn.q_norm.weight", D, 27 + layer)
            vector(f"model.layers.{layer}.self_attn.k_norm.weight", D, 37 + layer)
    quant("model.embed_tokens.weight", VOCAB, HID, O.Q8_0, 998)
    quant("lm_head.weight", VOCAB, HID, O.Q6_K, 999)
    vector("model.norm.weight", HID, 47)
    return model, dense


def _norm(x, w):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * w


def _turned(x, interleaved):
    t = x.shape[0]
    phi = np.arange(t)[:, None] * 10000.0 ** (-2 * np.arange(D // 2) / D)[None]
    c, s = np.cos(phi)[:, None], np.sin(phi)[:, None]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :D // 2], x[..., D // 2:])
    y = np.empty_like(x)
    if interleaved:
        y[..., 0::2], y[..., 1::2] = a * c - b * s, a * s + b * c
    else:
        y[..., :D // 2], y[..., D // 2:] = a * c - b * s, a * s + b * c
    return y


def _logits(w, ids, interleaved):
    """The definition in 64 bits: logits after every token of one sequence."""
    h, t = w["model.embed_tokens.weight"][ids], len(ids)
    for layer in range(LAYERS):
        def p(name):
            return w[f"model.layers.{layer}.{name}.weight"]
        x = _norm(h, p("input_layernorm"))
        q, k, v = ((x @ p(f"self_attn.{n}_proj").T).reshape(t, -1, D) for n in "qkv")
        if f"model.layers.{layer}.self_attn.q_norm.weight" in w:
            q, k = _norm(q, p("self_attn.q_norm")), _norm(k, p("self_attn.k_norm"))
        q, k = _turned(q, interleaved), _turned(k, interleaved)
        k, v = k.repeat(HEADS // KV, axis=1), v.repeat(HEADS // KV, axis=1)
        s = np.einsum("thd,jhd->htj", q, k) / math.sqrt(D)
        s = np.where(np.tril(np.ones((t, t), bool))[None], s, -np.inf)
        e = np.exp(s - s.max(-1, keepdims=True))
        a = np.einsum("htj,jhd->thd", e / e.sum(-1, keepdims=True), v).reshape(t, -1)
        h = h + a @ p("self_attn.o_proj").T
        x = _norm(h, p("post_attention_layernorm"))
        g, u = x @ p("mlp.gate_proj").T, x @ p("mlp.up_proj").T
        h = h + (g / (1 + np.exp(-g)) * u) @ p("mlp.down_proj").T
    return _norm(h, w["model.norm.weight"]) @ w["lm_head.weight"].T


def _check(got, want):
    # About ten roundings to f16 (2^-11) a layer and projections within 2e-3 of their rms, over
    # two layers: about 20 independent parts of 5e-4 to 1e-3, 4e-3 of the rms together; the
    # largest of a few hundred logits within 5 times that.
    err = np.abs(got.double().cpu().numpy() - want).max() / np.sqrt((want ** 2).mean())
    assert err <= 2e-2, err


@pytest.mark.parametrize("interleaved,qk_norm", [(True, False), (False, True)], ids=["pairs", "half with head norms"])
def test_forward_over_the_cache(cuda, interleaved, qk_norm):
    from vllm_webgpu_b200.kv_cache import PagedKVCache
    model, w = _model(interleaved, qk_norm)
    rng = np.random.RandomState(3)
    texts = {"a": rng.randint(0, VOCAB, 75), "b": rng.randint(0, VOCAB, 10), "c": rng.randint(0, VOCAB, 40)}
    want = {s: _logits(w, ids, interleaved) for s, ids in texts.items()}
    cache = PagedKVCache(LAYERS, 20, KV, D, 16, torch.float16, "cuda:0")
    done = dict.fromkeys(texts, 0)

    def step(counts):
        names = list(counts)
        ids = np.concatenate([texts[s][done[s]:done[s] + n] for s, n in counts.items()])
        got = model.forward(torch.from_numpy(ids).cuda(), None, cache.extend(names, list(counts.values())))
        for s, n in counts.items():
            done[s] += n
        for i, s in enumerate(names):
            _check(got[i], want[s][done[s] - 1])
        return got
    step({"a": 70, "b": 5})          # two prompts together
    step({"b": 1, "a": 1})           # single tokens, the order changed
    step({"c": 33, "a": 1, "b": 2})  # a prompt beside continuing sequences
    for _ in range(2):
        step({"a": 1, "b": 1, "c": 1})
    for s in texts:
        cache.release(s)
    assert cache.free_pages == 20
    first = step_again = None
    for _ in range(2):               # the same prompt in other pages gives the same bits
        cache.extend(["x"], [17])
        got = model.forward(torch.from_numpy(texts["c"]).cuda(), None, cache.extend(["y"], [40]))
        first, step_again = (got, None) if first is None else (first, got)
        cache.release("y")
    assert torch.equal(first, step_again)


def test_forward_refusals(cuda):
    from vllm_webgpu_b200.kv_cache import PagedKVCache
    from vllm_webgpu_b200.models.gemma4 import Gemma4B200Model
    model, _ = _model(True, False)
    cache = PagedKVCache(LAYERS, 4, KV, D, 16, torch.bfloat16, "cuda:0")
    with pytest.raises(ValueError, match="2 tokens"):
        model.forward(torch.zeros(2, dtype=torch.int64, device="cuda"), None, cache.extend(["a"], [3]))
    model.weights["model.layers.0.self_attn.q_proj.bias"] = torch.zeros(HEADS * D, device="cuda")
    with pytest.raises(NotImplementedError, match="bias"):
        model.forward(torch.zeros(3, dtype=torch.int64, device="cuda"), None, cache.extend(["b"], [3]))
    with pytest.raises(NotImplementedError):
        Gemma4B200Model(None, device="cuda:0").forward(None, None, None)
