"""The operators between a layer's projections, as cases to measure: the root-mean-square norm with
the residual's addition, the rotary positions with the append to a paged key-value cache, and the
attention over that cache, for one new token per sequence and for ragged causal prompts.

``own`` false: ``run`` computes them with elementary torch operations in 32 bits. ``own`` true: it
calls ``vllm_webgpu_b200.ops``. ``exact`` computes them from their definitions in 64 bits.

Caches are [pages, kv heads, page size, head dim]; a sequence's tokens lie in the pages that its
row of the block table names, in order.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _ops():
    """The framework's operators (its package folder lies beside this one)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-webgpu_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from vllm_webgpu_b200 import ops
    return ops


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _norm(rows, width, x, res, out, w="f32", eps=1e-5):
    return {"op": "norm", "rows": rows, "width": width, "x": x, "res": res, "out": out, "w": w, "eps": eps}


def _rope(tokens, hq, hkv, dim, rot, inter, x, cache, page, first, scaling="none", theta=500000.0, skip=0):
    return {"op": "rope", "tokens": tokens, "hq": hq, "hkv": hkv, "dim": dim, "rot": rot, "interleaved": inter, "x": x,
            "cache": cache, "page": page, "first": first, "scaling": scaling, "theta": theta, "skip": skip}


def _decode(batch, longest, spread, hq, hkv, dim, dtype, page, window=0):
    return {"op": "decode", "batch": batch, "longest": longest, "spread": spread, "hq": hq, "hkv": hkv, "dim": dim,
            "dtype": dtype, "page": page, "window": window}


def _prompt(batch, longest, spread, before, hq, hkv, dim, dtype, page, window=0):
    return {"op": "prompt", "batch": batch, "longest": longest, "spread": spread, "before": before, "hq": hq, "hkv": hkv,
            "dim": dim, "dtype": dtype, "page": page, "window": window}


def listed():
    return [
        # the norm after the o projection of one decoded token: 32-bit GEMV sums onto a bf16 stream
        dict(_norm(1, 4096, "f32", "bf16", "bf16"), name="norm, one token"),
        # the same for an 8192-token prompt, the longest batch of the prefill workloads
        dict(_norm(8192, 4096, "f32", "bf16", "bf16"), name="norm, prompt"),
        # a norm without a residual, of an odd width that no vector load fits
        dict(_norm(333, 2815, "f16", "none", "f16", "f16"), name="norm, odd width"),
        # eight sequences decoding with the 8B layer's heads, pairs as GGUF files of the Llama family order them
        dict(_rope(8, 32, 8, 128, 128, True, "bf16", "bf16", 16, 4001), name="rope, decode"),
        # a long prompt late in a long context, frequencies scaled for it
        dict(_rope(8192, 32, 8, 128, 128, True, "bf16", "bf16", 16, 100003, "llama3"), name="rope, long prompt"),
        # wide heads turned in half of their width, 32-bit projections into an f16 cache, padding tokens among them
        dict(_rope(1023, 16, 8, 256, 128, False, "f32", "f16", 32, 17, "yarn", 10000.0, 7), name="rope, part of the head"),
        # one user's chat: the smallest attention call, where latency counts
        dict(_decode(1, 513, 0, 32, 8, 128, "bf16", 16), name="attention, one short"),
        # a small batch of ordinary lengths
        dict(_decode(16, 2048, 1500, 32, 8, 128, "bf16", 16), name="attention, small batch"),
        # a full server: many ragged sequences
        dict(_decode(64, 8192, 7000, 32, 8, 128, "bf16", 16), name="attention, full batch"),
        # one very long context with the 70B layer's heads
        dict(_decode(1, 131035, 0, 64, 8, 128, "f16", 64), name="attention, long context"),
        # a few short prompts of different lengths arriving together, some of them continuing a cached text
        dict(_prompt(5, 301, 280, 77, 32, 8, 128, "bf16", 16), name="prompts, short"),
        # the 8192-token prompt
        dict(_prompt(1, 8192, 0, 0, 32, 8, 128, "bf16", 16), name="prompt, long"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["norm", "rope", "decode", "decode", "prompt"])
    if op == "norm":
        rows = _log(rng, 1, 8192)
        width = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        rows = min(rows, 8192 * 4096 // width)
        return _norm(rows, width, rng.choice(["f32", "f16", "bf16"]), rng.choice(["none", "f32", "f16", "bf16"]),
                     rng.choice(["f32", "f16", "bf16"]), rng.choice(["f32", "bf16"]), rng.choice([1e-5, 1e-6]))
    if op == "rope":
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 3, 4, 7, 8])
        dim = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        most = max(1, min(8192, 8192 * 48 * 128 // ((hq + 2 * hkv) * dim)))
        x = rng.choice(["f32", "f16", "bf16"])
        return _rope(_log(rng, 1, most if x != "f32" else max(1, most // 2)), hq, hkv, dim, rot, rng.random() < 0.5, x,
                     rng.choice(["f16", "bf16"]), rng.choice([8, 16, 24, 64]), _log(rng, 1, 1000000),
                     rng.choice(["none", "llama3", "yarn", "linear"]), rng.choice([10000.0, 500000.0]), rng.choice([0, 3]))
    dim = rng.choice([64, 128, 128, 128, 96, 256])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 4, 5, 8])
    dtype = rng.choice(["f16", "bf16"])
    page = rng.choice([8, 16, 16, 24, 64])
    window = rng.choice([0, 0, 0, 1024])
    if op == "decode":
        batch = _log(rng, 1, 64)
        # at most half of the cached bytes of a full batch of longest sequences, for room in the plain form
        longest = _log(rng, 1, min(131072, max(64, 64 * 8192 * 8 * 128 // (2 * batch * hkv * dim))))
        return _decode(batch, longest, rng.randint(0, longest), hq, hkv, dim, dtype, page, window)
    batch = _log(rng, 1, 8)
    before = rng.choice([0, _log(rng, 1, 2000)])
    longest = _log(rng, 1, 8192)
    # no more score values than half of the long prompt's
    while batch * hq * longest * (longest + before) > 32 * 8192 * 8192 // 2:
        longest = max(1, longest * 3 // 4)
    return _prompt(batch, longest, rng.randint(0, longest - 1), before, hq, hkv, dim, dtype, page, window)


# ---------------------------------------------------------------------------------------------
# what a case's sizes mean
# ---------------------------------------------------------------------------------------------
def _spread(n, top, spread):
    """n lengths between top - spread and top, the first of them top."""
    return [top - (i * 2654435761 % (spread + 1)) for i in range(n)]


def _lengths(case):
    """The new tokens and the length of each sequence, the new ones included."""
    if case["op"] == "decode":
        lens = _spread(case["batch"], case["longest"], case["spread"])
        return [1] * len(lens), lens
    new = _spread(case["batch"], case["longest"], case["spread"])
    return new, [n + (case["before"] if i % 2 else 0) for i, n in enumerate(new)]


def _pairs(new, lens, window):
    """How many (query, key) pairs the causal mask leaves."""
    total = 0
    for n, length in zip(new, lens):
        seen = np.arange(length - n + 1, length + 1, dtype=np.int64).clip(min=0)
        total += int((np.minimum(seen, window) if window else seen).sum())
    return total


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        per = _BYTES[case["x"]] + _BYTES[case["out"]] + (2 * _BYTES[case["res"]] if case["res"] != "none" else 0)
        return {"bytes": n * per + case["width"] * _BYTES[case["w"]], "flops": 5 * n}
    if case["op"] == "rope":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
        kept = t - (t // case["skip"] if case["skip"] else 0)
        xb = _BYTES[case["x"]]
        return {"bytes": t * (2 * hq * d * xb + 8 + 8) + kept * 2 * hkv * d * (xb + 2), "flops": 3 * t * (hq + hkv) * case["rot"]}
    new, lens = _lengths(case)
    hq, hkv, d, window = case["hq"], case["hkv"], case["dim"], case["window"]
    seen = sum(min(length, window + n - 1) if window else length for n, length in zip(new, lens))
    return {"bytes": seen * 2 * hkv * d * 2 + sum(new) * hq * d * 2 * 2, "flops": 4 * d * hq * _pairs(new, lens, window)}


def _angles(case):
    """Radians per position of each pair, in 64 bits, and the factor on the turned values."""
    n, theta = case["rot"], case["theta"]
    f = theta ** (-np.arange(0, n, 2, dtype=np.float64) / n)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "llama3":  # factor 8 over an original context of 8192, bands at 1 and 4 turns
        turns = 8192 * f / (2 * math.pi)
        smooth = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return (1 - smooth) * f / 8.0 + smooth * f, 1.0
    if case["scaling"] == "yarn":  # factor 4 over an original context of 4096, ramp between 32 turns and 1
        def pair_of(turns):
            return n * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), n - 1)
        ramp = np.clip((np.arange(n // 2) - low) / max(high - low, 0.001), 0.0, 1.0)
        return f / 4.0 * ramp + f * (1 - ramp), 0.1 * math.log(4.0) + 1.0
    return f, 1.0


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, dtype, gain=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32 if dtype == "f32" else _DTYPES[dtype]).mul_(gain)

    s = {"case": dict(case)}
    if case["op"] == "norm":
        m, n = case["rows"], case["width"]
        s["x"] = normal(m, n, dtype=case["x"])
        s["res"] = normal(m, n, dtype=case["res"], gain=3.0) if case["res"] != "none" else None
        s["weight"] = (1.0 + normal(n, dtype="f32", gain=0.1)).to(_DTYPES[case["w"]])
        return s
    page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["dim"]
    if case["op"] == "rope":
        t, dtype = case["tokens"], _DTYPES[case["cache"]]
        # q, k and v side by side, as a grouped projection leaves them
        qkv = normal(t, (hq + 2 * hkv) * d, dtype=case["x"])
        s["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        s["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        s["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
        s["positions"] = torch.arange(case["first"], case["first"] + t, device=dev, dtype=torch.int64)
        pages = -(-t // page) + 2
        order = torch.randperm(pages, generator=g, device=dev)
        at = torch.arange(t, device=dev)
        slots = order[at // page] * page + at % page
        if case["skip"]:
            slots = torch.where(at % case["skip"] == case["skip"] - 1, -1, slots)
        s["slots"] = slots
        radians, s["factor"] = _angles(case)
        turns = radians / (2 * math.pi)
        s["steps"] = torch.from_numpy(np.array([int(round(float(x) * 2.0 ** 64)) for x in turns], dtype=np.uint64).view(np.int64).copy()).to(dev)
        s["k_cache"] = torch.zeros(pages, hkv, page, d, dtype=dtype, device=dev)
        s["v_cache"] = torch.zeros(pages, hkv, page, d, dtype=dtype, device=dev)
        return s
    new, lens = _lengths(case)
    widest = max(1, -(-max(lens) // page))
    counts = [-(-length // page) for length in lens]
    pages = sum(counts) + 1
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), widest, dtype=torch.int32, device=dev)
    first = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[first:first + c]
        first += c
    s["table"] = table
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["k_cache"] = normal(pages, hkv, page, d, dtype=case["dtype"])
    s["v_cache"] = normal(pages, hkv, page, d, dtype=case["dtype"])
    s["q"] = normal(sum(new), hq, d, dtype=case["dtype"], gain=2.0)
    s["scale"] = d ** -0.5
    if case["op"] == "prompt":
        s["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev)
        s["most"] = max(new)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    return _PLAIN[op](s)


def _own_norm(s):
    c = s["case"]
    got = _ops().rms_norm(s["x"], s["weight"], eps=c["eps"], residual=s["res"], out_dtype=_DTYPES[c["out"]])
    return {"out": got} if s["res"] is None else {"out": got[0], "res": got[1]}


def _own_rope(s):
    q = _ops().rope_append(s["q"], s["k"], s["v"], s["positions"], s["steps"], s["slots"], s["k_cache"], s["v_cache"],
                           interleaved=s["case"]["interleaved"], factor=s["factor"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_decode(s):
    return _ops().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], scale=s["scale"],
                                  window=s["case"]["window"])


def _own_prompt(s):
    return _ops().paged_prompt_attention(s["q"], s["starts"], s["most"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                         scale=s["scale"], window=s["case"]["window"])


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float()
    if s["res"] is not None:
        x = x + s["res"].float()
    y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + c["eps"]) * s["weight"].float()
    y = y.to(_DTYPES[c["out"]])
    return {"out": y} if s["res"] is None else {"out": y, "res": x.to(s["res"].dtype)}


def _plain_rope(s):
    c = s["case"]
    n = c["rot"]
    # the turn of each (token, pair): an exact product modulo one turn in 64-bit integers
    turn = (s["positions"][:, None] * s["steps"][None, :]).float() * 2.0 ** -64
    angle = turn * (2 * math.pi)
    cos, sin = torch.cos(angle)[:, None, :] * s["factor"], torch.sin(angle)[:, None, :] * s["factor"]

    def turned(x):
        x = x.float()
        r, rest = x[..., :n], x[..., n:]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            y = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
        else:
            a, b = r[..., :n // 2], r[..., n // 2:]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
        return torch.cat([y, rest], dim=-1)

    keep = s["slots"] >= 0
    slots = s["slots"][keep]
    pages, offsets = slots // c["page"], slots % c["page"]
    s["k_cache"][pages, :, offsets] = turned(s["k"])[keep].to(s["k_cache"].dtype)
    s["v_cache"][pages, :, offsets] = s["v"][keep].to(s["v_cache"].dtype)
    return {"q": turned(s["q"]).to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s, q, at):
    """q [B, n, Hq, D] at positions at [B, n] (negative: no query) over each sequence's cached tokens, in 32 bits."""
    c = s["case"]
    b, n, hq, d = q.shape
    hkv = c["hkv"]
    table = s["table"].long()

    def cached(cache):
        return cache[table].transpose(1, 2).flatten(2, 3).float()  # [B, Hkv, tokens, D]

    scores = (q.float() * s["scale"]).unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3) @ cached(s["k_cache"]).transpose(2, 3)
    scores = scores.unflatten(2, (hq // hkv, n))
    j = torch.arange(scores.shape[-1], device=q.device)
    seen = j[None, None, :] <= at[:, :, None]
    if c["window"]:
        seen = seen & (j[None, None, :] > at[:, :, None] - c["window"])
    seen = seen[:, None, None]
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(dim=-1, keepdim=True).clamp_min(-3.0e38)
    p = scores.sub_(top).exp_()
    p = p.div_(p.sum(dim=-1, keepdim=True).clamp_min(1e-37))
    v = cached(s["v_cache"])
    v = v.masked_fill_((j[None, :] >= s["lens"][:, None])[:, None, :, None], 0.0)
    o = (p.flatten(2, 3) @ v).unflatten(2, (hq // hkv, n))
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3).to(q.dtype)  # [B, n, Hq, D]


def _plain_decode(s):
    return _plain_attention(s, s["q"][:, None], s["lens"].long()[:, None] - 1)[:, 0]


def _plain_prompt(s):
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(s["most"], device=starts.device)
    there = i[None, :] < new[:, None]
    row = torch.where(there, starts[:-1, None] + i[None, :], 0)
    at = torch.where(there, lens[:, None] - new[:, None] + i[None, :], -1)
    o = _plain_attention(s, s["q"][row], at)
    out = torch.empty_like(s["q"])
    out[row[there]] = o[there]
    return out


_OWN = {"norm": _own_norm, "rope": _own_rope, "decode": _own_decode, "prompt": _own_prompt}
_PLAIN = {"norm": _plain_norm, "rope": _plain_rope, "decode": _plain_decode, "prompt": _plain_prompt}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        total = s["x"].double() if s["res"] is None else s["x"].double().add(s["res"].double())
        size = torch.linalg.vector_norm(total, dim=1).square() / case["width"]
        out = total / torch.sqrt(size + case["eps"])[:, None] * s["weight"].double()
        return {"out": out} if s["res"] is None else {"out": out, "res": total}
    if case["op"] == "rope":
        radians, factor = _angles(case)
        phi = s["positions"].double()[:, None] * torch.from_numpy(radians).to(s["q"].device)
        spin = torch.polar(torch.full_like(phi, factor), phi)[:, None, :]
        n, half = case["rot"], case["rot"] // 2
        pairs = torch.arange(n, device=phi.device)
        first, second = (pairs[0::2], pairs[1::2]) if case["interleaved"] else (pairs[:half], pairs[half:])

        def spun(x):
            y = x.double().clone()
            z = torch.complex(y[..., first], y[..., second]) * spin
            y[..., first], y[..., second] = z.real, z.imag
            return y
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        flat_k, flat_v = (c.transpose(1, 2).reshape(-1, case["hkv"], case["dim"]) for c in (k_cache, v_cache))
        flat_k, flat_v = flat_k.clone(), flat_v.clone()
        stored = torch.nonzero(s["slots"] >= 0).flatten()
        flat_k[s["slots"][stored]] = spun(s["k"])[stored]
        flat_v[s["slots"][stored]] = s["v"].double()[stored]
        shape = (-1, case["page"], case["hkv"], case["dim"])
        return {"q": spun(s["q"]), "k_cache": flat_k.reshape(shape).transpose(1, 2).contiguous(),
                "v_cache": flat_v.reshape(shape).transpose(1, 2).contiguous()}
    new, lens = _lengths(case)
    hq, hkv, window = case["hq"], case["hkv"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    first = 0
    for b, (n, length) in enumerate(zip(new, lens)):
        if length > 0:
            rows = s["table"][b, :-(-length // case["page"])].long()
            keys, values = (torch.cat([c[rows, h].reshape(1, -1, case["dim"]) for h in range(hkv)])[:, :length].double()
                            for c in (s["k_cache"], s["v_cache"]))
            for i in range(0, n, 512):  # blocks of queries
                m = min(512, n - i)
                at = torch.arange(length - n + i, length - n + i + m, device=out.device)
                j = torch.arange(length, device=out.device)
                hidden = j[None, :] > at[:, None]
                if window:
                    hidden |= j[None, :] <= at[:, None] - window
                for h in range(hkv):
                    for head in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                        logits = s["q"][first + i:first + i + m, head].double() @ keys[h].T * s["scale"]
                        weights = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=1)
                        out[first + i:first + i + m, head] = weights @ values[h]
        first += n
    return out
