"""The host side of the operators between the projections, on the CPU: the paged cache's
bookkeeping, the rotary frequencies, the packed arguments and the entry points' refusals."""
from __future__ import annotations

import math
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _cache(pages=6, page=8):
    from vllm_webgpu_b200.kv_cache import PagedKVCache
    return PagedKVCache(2, pages, 2, 16, page, torch.float16, "cpu")


def test_extend_lays_tokens_out_in_pages():
    c = _cache()
    step = c.extend(["a", "b"], [11, 8])
    assert c.free_pages == 3 and not step.decode and step.max_q == 11
    assert step.positions.tolist() == list(range(11)) + list(range(8))
    assert step.lens.tolist() == [11, 8] and step.q_starts.tolist() == [0, 11, 19]
    assert step.block_tables.shape == (2, 2) and step.block_tables.dtype == torch.int32
    tab = step.block_tables.tolist()
    assert step.slots.tolist() == [tab[0][i // 8] * 8 + i % 8 for i in range(11)] + [tab[1][0] * 8 + i for i in range(8)]
    step = c.extend(["b", "a"], [1, 1])
    assert step.decode and step.positions.tolist() == [8, 11] and step.lens.tolist() == [9, 12]
    assert step.block_tables.tolist()[1] == tab[0] and step.block_tables.tolist()[0][0] == tab[1][0]
    assert len(set(step.slots.tolist())) == 2


def test_a_full_cache_refuses_and_changes_nothing():
    c = _cache()
    c.extend(["a"], [40])
    with pytest.raises(RuntimeError, match="1 free pages, 2"):
        c.extend(["b", "a"], [3, 1])
    assert c.free_pages == 1 and c.length("a") == 40 and c.length("b") == 0
    c.release("a")
    c.release("unknown")
    assert c.free_pages == 6 and c.length("a") == 0
    assert sorted(c.extend(["b"], [48]).block_tables.flatten().tolist()) == list(range(6))


def test_cache_refusals():
    from vllm_webgpu_b200.kv_cache import PagedKVCache
    for bad in (dict(page_size=12), dict(page_size=0), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            PagedKVCache(1, 4, 1, 64, **{"device": "cpu", **bad})
    for dim in (4, 60, 264):
        with pytest.raises(ValueError):
            PagedKVCache(1, 4, 1, dim, device="cpu")
    c = _cache()
    for seqs, counts in ((["a", "a"], [1, 1]), (["a"], [0]), (["a"], [1, 2])):
        with pytest.raises(ValueError):
            c.extend(seqs, counts)
    assert c.free_pages == 6


def _turns(steps):
    return [(s % 2 ** 64) / 2.0 ** 64 for s in steps.tolist()]


def test_rope_steps_default_linear_and_factors():
    from vllm_webgpu_b200 import ops
    for kw, by in ((dict(), 1.0), (dict(scaling={"rope_type": "linear", "factor": 4.0}), 4.0),
                   (dict(freq_factors=[2.0] * 32), 2.0), (dict(scaling={"type": "linear", "factor": 2}), 2.0)):
        steps, factor = ops.rope_steps(64, 10000.0, device="cpu", **kw)
        assert steps.dtype == torch.int64 and factor == 1.0
        for i, t in enumerate(_turns(steps)):
            assert t == pytest.approx(10000.0 ** (-i / 32) / (2 * math.pi) / by, rel=1e-15)


def test_rope_steps_llama3_and_yarn():
    """Against the published formulas, pair by pair."""
    from vllm_webgpu_b200 import ops
    s = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
             original_max_position_embeddings=8192)
    got = _turns(ops.rope_steps(128, 500000.0, s, device="cpu")[0])
    kinds = set()
    for i in range(64):
        f = 500000.0 ** (-2 * i / 128)
        wave = 2 * math.pi / f
        if wave < 8192 / 4.0:
            want, kind = f, "kept"
        elif wave > 8192 / 1.0:
            want, kind = f / 8, "stretched"
        else:
            m = (8192 / wave - 1.0) / 3.0
            want, kind = (1 - m) * f / 8 + m * f, "between"
        kinds.add(kind)
        assert got[i] == pytest.approx(want / (2 * math.pi), rel=1e-14)
    assert kinds == {"kept", "stretched", "between"}
    y = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)
    steps, factor = ops.rope_steps(128, 10000.0, y, device="cpu")
    assert factor == pytest.approx(0.1 * math.log(4.0) + 1.0)
    got = _turns(steps)
    assert got[0] == pytest.approx(1 / (2 * math.pi), rel=1e-14)                       # fast pairs stay
    assert got[63] == pytest.approx(10000.0 ** (-126 / 128) / 4 / (2 * math.pi), rel=1e-14)  # slow ones stretch
    assert ops.rope_steps(128, 1e4, {**y, "attention_factor": 0.5}, device="cpu")[1] == 0.5


def test_rope_steps_refusals():
    from vllm_webgpu_b200 import ops
    for args in ((3,), (0,), (64, 0.0), (64, 1e4, {"rope_type": "dynamic"}), (64, 1e4, None, [1.0] * 31),
                 (64, 1e4, None, [0.0] * 32)):
        with pytest.raises(ValueError):
            ops.rope_steps(*args, device="cpu")


def test_packed_arguments_match_the_header():
    """The struct formats name the header's fields one for one: all of 8 bytes, in order."""
    from vllm_webgpu_b200 import ops
    text = open(os.path.join(ROOT, "include", "ggufmm.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, fmt in (("ggufmm_norm_args", ops._NORM_ARGS), ("ggufmm_rope_args", ops._ROPE_ARGS),
                      ("ggufmm_attention_args", ops._ATTENTION_ARGS)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        kinds = ""
        for decl in body.split(";"):
            decl = decl.strip()
            if not decl:
                continue
            if "*" in decl:
                kinds += "Q"
            else:
                kinds += {"int64_t": "q", "double": "d"}[decl.split()[0]] * (decl.count(",") + 1)
        flat = re.sub(r"(\d+)([Qqd])", lambda m: m.group(2) * int(m.group(1)), fmt.format)
        assert flat == kinds, name


def _attention(**other):
    from vllm_webgpu_b200 import _lib, ops
    p = 1 << 20
    f = dict(q=p, q_row=1024, q_head=128, out=p, o_row=1024, o_head=128, k=p, k_page=16384, k_head=2048, k_slot=128, v=p,
             v_page=16384, v_head=2048, v_slot=128, tables=p, table_row=4, table_width=4, lens=p, q_starts=p, batch=2,
             total_q=2, max_q=1, q_heads=8, kv_heads=8, head_dim=128, page_size=16, num_pages=9, dtype=2, window=0,
             scale=0.1)
    f.update(other)
    args = ops._ATTENTION_ARGS.pack(*f.values())
    lib = _lib.lib()
    return (lib.ggufmm_paged_attention(args, p, 1 << 40, None), lib.ggufmm_paged_prompt_attention(args, None, 0, None))


def test_attention_refuses_on_the_host():
    from vllm_webgpu_b200 import _lib as L
    both = ((L.ERR_ARG, ("q", "out", "k", "v", "tables", "lens"), 0),
            (L.ERR_DTYPE, ("dtype",), 0),
            (L.ERR_SHAPE, ("kv_heads", "num_pages", "page_size", "head_dim", "q_heads"), 0),
            (L.ERR_SHAPE, ("window", "batch", "total_q"), -1),
            (L.ERR_SHAPE, ("q_heads",), 9), (L.ERR_SHAPE, ("head_dim",), 132), (L.ERR_SHAPE, ("head_dim",), 264),
            (L.ERR_SHAPE, ("page_size",), 12), (L.ERR_SHAPE, ("table_row",), 3), (L.ERR_SHAPE, ("table_width",), 1 << 28),
            (L.ERR_SHAPE, ("k_slot", "v_head", "o_head", "q_row"), 120),
            (L.ERR_ALIGN, ("k_page", "v_slot", "q_row", "o_head"), 2052), (L.ERR_ALIGN, ("q", "k", "out"), (1 << 20) + 8),
            (L.ERR_ALIGN, ("lens", "tables"), (1 << 20) + 2), (L.ERR_ARG, ("scale",), float("nan")))
    for status, names, value in both:
        for name in names:
            assert _attention(**{name: value}) == (status, status), (name, value)
    assert _attention(q_starts=0)[1] == L.ERR_ARG
    assert _attention(max_q=3)[1] == L.ERR_SHAPE
    assert _attention(total_q=3)[0] == L.ERR_SHAPE
    assert _attention(q_heads=8 * 65) == (L.ERR_SHAPE, L.ERR_SHAPE)
    lib = L.lib()
    assert lib.ggufmm_paged_attention(None, None, 0, None) == L.ERR_ARG
    assert lib.ggufmm_paged_prompt_attention(None, None, 0, None) == L.ERR_ARG
    assert lib.ggufmm_paged_attention_workspace_size(0, 8, 8, 128) == 0
    assert lib.ggufmm_paged_attention_workspace_size(2, 8, 8, 128) > 0


def test_norm_and_rope_refuse_on_the_host():
    from vllm_webgpu_b200 import _lib as L
    from vllm_webgpu_b200 import ops
    lib, p = L.lib(), 1 << 20

    def norm(x=p, xt=2, m=1, n=64, ldx=64, r=p, rt=2, ldr=64, ro=p, ldro=64, w=p, wt=0, add=0.0, eps=1e-5, y=p, yt=2, ldy=64):
        return lib.ggufmm_rms_norm(ops._NORM_ARGS.pack(x or 0, r or 0, ro, w, y or 0, ldx, ldr, ldro, ldy, m, n, xt, rt, wt, yt,
                                                       add, eps), None)
    assert lib.ggufmm_rms_norm(None, None) == L.ERR_ARG
    assert norm(m=0) == L.OK
    assert norm(x=None) == L.ERR_ARG and norm(y=None) == L.ERR_ARG and norm(r=None) == L.ERR_ARG
    assert norm(eps=-1.0) == L.ERR_ARG and norm(eps=float("nan")) == L.ERR_ARG
    assert norm(xt=3) == L.ERR_DTYPE and norm(yt=-1) == L.ERR_DTYPE and norm(wt=9) == L.ERR_DTYPE and norm(rt=5) == L.ERR_DTYPE
    for bad in (dict(m=-1), dict(n=0), dict(n=65537, ldx=1 << 20, ldr=1 << 20, ldro=1 << 20, ldy=1 << 20), dict(ldx=63),
                dict(ldy=63), dict(ldr=63), dict(ldro=63)):
        assert norm(**bad) == L.ERR_SHAPE, bad
    assert norm(x=p + 1) == L.ERR_ALIGN and norm(w=p + 2) == L.ERR_ALIGN

    def rope(**other):
        f = dict(q=p, q_row=512, q_head=128, q_out=p, qo_row=512, qo_head=128, k=p, k_row=256, k_head=128, v=p, v_row=256,
                 v_head=128, k_cache=p, kc_page=4096, kc_head=2048, kc_slot=128, v_cache=p, vc_page=4096, vc_head=2048,
                 vc_slot=128, positions=p, slots=p, steps=p, tokens=3, q_heads=4, kv_heads=2, head_dim=128, rot_dim=128,
                 interleaved=0, x_dtype=2, q_out_dtype=2, cache_dtype=2, page_size=16, num_pages=5, factor=1.0)
        f.update(other)
        return lib.ggufmm_rope_append(ops._ROPE_ARGS.pack(*f.values()), None)
    assert lib.ggufmm_rope_append(None, None) == L.ERR_ARG
    assert rope(tokens=0) == L.OK
    for name in ("q", "q_out", "v", "k_cache", "v_cache", "positions", "slots", "steps"):
        assert rope(**{name: 0}) == L.ERR_ARG, name
    for name, value in (("tokens", -1), ("q_heads", 0), ("kv_heads", 0), ("head_dim", 120), ("head_dim", 12), ("rot_dim", 130),
                        ("rot_dim", 7), ("page_size", 20), ("num_pages", 0), ("kc_slot", 120), ("q_row", -1), ("v_head", -8)):
        assert rope(**{name: value}) == L.ERR_SHAPE, (name, value)
    for name in ("x_dtype", "q_out_dtype", "cache_dtype"):
        assert rope(**{name: 4}) == L.ERR_DTYPE
    assert rope(cache_dtype=0) == L.ERR_DTYPE
    for name, value in (("q", p + 1), ("k_cache", p + 8), ("positions", p + 4), ("vc_page", 4100)):
        assert rope(**{name: value}) == L.ERR_ALIGN, (name, value)


def test_the_operators_refuse_cpu_tensors():
    from vllm_webgpu_b200 import ops
    x, i = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.rms_norm(x), lambda: ops.rope(x, i, i), lambda: ops.rope_append(x, x, x, i, i, i, x, x),
                 lambda: ops.paged_attention(x, x, x, i, i), lambda: ops.paged_prompt_attention(x, i, 1, x, x, i, i)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
