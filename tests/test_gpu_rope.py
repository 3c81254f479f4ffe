"""ggufmm_rope_append against the definition in 64 bits: pair orders, part of the head,
large positions, scaled frequencies, cache layouts, dropped slots and refusals."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


def _turned(x, positions, radians, interleaved, factor):
    """The definition in 64 bits."""
    x = x.double().cpu().clone()
    n = 2 * len(radians)
    phi = positions.double().cpu()[:, None] * radians[None, :]
    c, s = (torch.cos(phi) * factor)[:, None], (torch.sin(phi) * factor)[:, None]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    ra, rb = a * c - b * s, a * s + b * c
    if interleaved:
        x[..., 0:n:2], x[..., 1:n:2] = ra, rb
    else:
        x[..., :n // 2], x[..., n // 2:n] = ra, rb
    return x


def _check(got, want, dtype, size):
    # The angle is exact to a turn's 2^-24 half (3e-7 radians with the store to 32 bits and
    # the sine's own error), times the pair's size; two products and a sum of 32 bits.
    tol = (5e-7 + 4 * UNIT[F32]) * size + UNIT[dtype] * want.abs() + TINY[dtype]
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def _radians(n, theta):
    return torch.tensor([theta ** (-2 * i / n) for i in range(n // 2)], dtype=torch.float64)


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (80, 20), (96, 24), (256, 128), (8, 2), (24, 24), (128, 0)])
@pytest.mark.parametrize("xt,ct", [(F32, F16), (BF16, BF16), (F16, BF16)])
def test_append_matches_the_definition(cuda, interleaved, dim, rot, xt, ct):
    from vllm_webgpu_b200 import ops
    torch.manual_seed(dim + rot)
    t, hq, hkv, page, pages = 13, 6, 2, 8, 5
    factor = 1.25
    qkv = torch.randn(t, (hq + 2 * hkv) * dim).to(xt).cuda()  # side by side: strided views
    q = qkv[:, :hq * dim].view(t, hq, dim)
    k = qkv[:, hq * dim:(hq + hkv) * dim].view(t, hkv, dim)
    v = qkv[:, (hq + hkv) * dim:].view(t, hkv, dim)
    positions = torch.tensor([0, 1, 2, 77, 4095, 131071, 1000003, 2 ** 31, 5, 6, 7, 8, 9], device="cuda")
    slots = torch.randperm(pages * page)[:t].cuda()
    slots[4] = -1
    kc = torch.full((pages, hkv, page, dim), 7.0, dtype=ct, device="cuda")
    vc = torch.full_like(kc, -7.0)
    kc0, vc0 = kc.clone(), vc.clone()
    rad = _radians(rot, 10000.0) if rot else torch.zeros(0, dtype=torch.float64)
    steps = ops.rope_steps(rot, 10000.0)[0] if rot else torch.zeros(0, dtype=torch.int64, device="cuda")
    qkv0 = qkv.clone()
    got = ops.rope_append(q, k, v, positions, steps, slots, kc, vc, interleaved=interleaved, factor=factor)
    assert torch.equal(qkv, qkv0) and got.dtype == xt
    # where positions are large, the 64-bit reference's own angle is off by pos * 2^-53: no matter
    size = 8.0  # above the size of any pair drawn, times the factor
    _check(got, _turned(q, positions, rad, interleaved, factor), xt, size)
    want_k, want_v = kc0.double().cpu(), vc0.double().cpu()
    tk = _turned(k, positions, rad, interleaved, factor)
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            want_k[s // page, :, s % page] = tk[i]
            want_v[s // page, :, s % page] = v[i].double().cpu().to(F32).to(ct).double()
    _check(kc, want_k, ct, size)
    assert torch.equal(vc.double().cpu(), want_v)


@pytest.mark.parametrize("layout", ["pages-heads", "pages-slots", "pairs of caches"])
def test_cache_strides(cuda, layout):
    """The cache by other strides: [pages, page size, heads, dim] storage, k and v interleaved by page."""
    from vllm_webgpu_b200 import ops
    t, h, d, page, pages = 30, 3, 64, 16, 4
    if layout == "pages-heads":
        kc, vc = (torch.zeros(pages, h, page, d, dtype=BF16, device="cuda") for _ in range(2))
    elif layout == "pages-slots":
        kc, vc = (torch.zeros(pages, page, h, d, dtype=BF16, device="cuda").transpose(1, 2) for _ in range(2))
    else:
        both = torch.zeros(pages, 2, h, page, d + 8, dtype=BF16, device="cuda")[..., :d]
        kc, vc = both[:, 0], both[:, 1]
    k, v = (torch.randn(t, h, d, device="cuda").to(BF16) for _ in range(2))
    q = torch.randn(t, h, d, device="cuda").to(BF16)
    steps, _ = ops.rope_steps(d)
    pos, slots = torch.arange(t, device="cuda"), torch.arange(5, 5 + t, device="cuda")
    q2 = ops.rope_append(q, k, v, pos, steps, slots, kc, vc)
    flat_k, flat_v = (c.transpose(1, 2).reshape(pages * page, h, d) for c in (kc, vc))
    assert torch.equal(flat_k[5:5 + t], ops.rope(k, pos, steps)) and torch.equal(flat_v[5:5 + t], v)
    assert int(flat_k[:5].count_nonzero()) == 0 and int(flat_k[5 + t:].count_nonzero()) == 0
    assert torch.equal(q2, ops.rope(q, pos, steps))


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_other_dtypes(cuda, interleaved):
    from vllm_webgpu_b200 import ops
    x = torch.randn(9, 5, 128, device="cuda")
    pos = torch.arange(100, 109, device="cuda")
    steps, _ = ops.rope_steps(64)
    want = ops.rope(x, pos, steps, interleaved)
    as16 = ops.rope(x, pos, steps, interleaved, out=torch.empty(9, 5, 128, dtype=F16, device="cuda"))
    assert torch.equal(as16, want.half())
    y = x.clone()
    assert ops.rope(y, pos, steps, interleaved, out=y).data_ptr() == y.data_ptr() and torch.equal(y, want)
    back = ops.rope(want, -pos, steps, interleaved)  # turning back: the inverse
    assert torch.allclose(back, x, atol=4e-6)


def test_a_long_way_out_is_exact(cuda):
    """Relative positions hold at any distance: <R(a) q, R(b) k> depends on a - b alone."""
    from vllm_webgpu_b200 import ops
    q, k = torch.randn(1, 1, 128, device="cuda"), torch.randn(1, 1, 128, device="cuda")
    steps, _ = ops.rope_steps(128, 500000.0)

    def dot(a, b):
        pa, pb = (torch.tensor([p], device="cuda") for p in (a, b))
        return float((ops.rope(q, pa, steps).double() * ops.rope(k, pb, steps).double()).sum())
    near = dot(40, 3)
    for far in (1 << 20, (1 << 31) - 100, 1 << 40):
        assert abs(dot(40 + far, 3 + far) - near) < 2e-4  # 128 products of angles good to 5e-7
    assert math.isfinite(near)


def test_empty_and_dropped(cuda):
    from vllm_webgpu_b200 import _lib, ops
    steps, _ = ops.rope_steps(64)
    kc, vc = (torch.zeros(2, 2, 8, 64, dtype=F16, device="cuda") for _ in range(2))
    z = torch.zeros(0, 2, 64, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert ops.rope_append(z, z, z, none, steps, none, kc, vc).shape == (0, 2, 64)
    _lib.lib().ggufmm_device_status(1, None)
    x = torch.randn(3, 2, 64, device="cuda")
    pos = torch.arange(3, device="cuda")
    ops.rope_append(x, x, x, pos, steps, torch.tensor([-1, -5, -(1 << 40)], device="cuda"), kc, vc)
    assert int(kc.count_nonzero()) == 0 and _lib.lib().ggufmm_device_status(1, None) == 0
    ops.rope_append(x, x, x, pos, steps, torch.tensor([16, 3, 1 << 40], device="cuda"), kc, vc)
    assert _lib.lib().ggufmm_device_status(1, None) == 2
    assert torch.equal(vc[0, :, 3], x[1].half()) and int(vc.count_nonzero()) == int(vc[0, :, 3].count_nonzero())


def test_refusals(cuda):
    from vllm_webgpu_b200 import ops
    steps, _ = ops.rope_steps(64)
    x = torch.zeros(3, 2, 64, device="cuda")
    pos = torch.arange(3, device="cuda")
    kc = torch.zeros(2, 2, 8, 64, dtype=F16, device="cuda")
    args = dict(q=x, k=x, v=x, positions=pos, steps=steps, slots=pos, k_cache=kc, v_cache=kc.clone())

    def refused(**other):
        with pytest.raises(ValueError):
            ops.rope_append(**{**args, **other})
    refused(k=x[:, :1], v=x[:, :1])                               # one head for a cache of two
    refused(v=x[:2])
    refused(k=x.half(), v=x.half())                                # not q's dtype
    refused(positions=pos[:2])
    refused(slots=None)
    refused(steps=steps.float())
    refused(steps=ops.rope_steps(66)[0])                           # wider than the head
    refused(k_cache=kc.float(), v_cache=kc.float())                # f32 cache
    refused(k_cache=kc, v_cache=kc[:1])
    odd = torch.zeros(2, 2, 9, 64, dtype=F16, device="cuda")
    refused(k_cache=odd, v_cache=odd.clone())                      # a page of 9 slots
    refused(q_out=torch.zeros(3, 2, 63, device="cuda"))
    refused(q=x.cpu())
    with pytest.raises(ValueError):
        ops.rope(torch.zeros(3, 64, device="cuda"), pos, steps)
    with pytest.raises(ValueError):
        ops.rope(torch.zeros(3, 2, 260, device="cuda"), pos, steps)  # over the widest head, no multiple of 8
