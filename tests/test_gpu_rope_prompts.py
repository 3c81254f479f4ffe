"""Rotary positions and the cache append for prompts, where a CTA takes two tokens: lengths about the
point where that begins, an odd last token, every width of a group, tokens of a pair that are dropped
one by one."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_rope import BF16, F16, F32, _check, _radians, _turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [591, 592, 593, 1023])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (24, 24), (96, 24), (80, 20), (64, 0)])
@pytest.mark.parametrize("xt,ct", [(F32, F16), (BF16, BF16), (F16, BF16)])
def test_a_prompt_matches_the_definition(cuda, tokens, interleaved, dim, rot, xt, ct):
    from vllm_webgpu_b200 import _lib, ops
    g = torch.Generator().manual_seed(tokens + dim + rot)
    hq, hkv, page, factor = 3, 2, 16, 1.25
    pages = -(-tokens // page) + 2
    qkv = torch.randn(tokens, (hq + 2 * hkv) * dim, generator=g).to(xt).cuda()
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([hq * dim, hkv * dim, hkv * dim], dim=1))
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g).cuda()
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    # of each four pairs of tokens one loses its first, one its second, one both
    pair, second = torch.arange(tokens) // 2, torch.arange(tokens) % 2
    slots[((pair % 4 == 1) & (second == 0)) | ((pair % 4 == 2) & (second == 1)) | (pair % 4 == 3)] = -1
    kc = torch.full((pages, hkv, page, dim), 7.0, dtype=ct, device="cuda")
    vc = torch.full_like(kc, -7.0)
    want_k, want_v = kc.double().cpu(), vc.double().cpu()
    rad = _radians(rot, 10000.0) if rot else torch.zeros(0, dtype=torch.float64)
    steps = ops.rope_steps(rot, 10000.0)[0] if rot else torch.zeros(0, dtype=torch.int64, device="cuda")
    _lib.lib().ggufmm_device_status(1, None)
    got = ops.rope_append(q, k, v, positions, steps, slots.cuda(), kc, vc, interleaved=interleaved, factor=factor)
    size = 8.0  # above the size of any pair drawn, times the factor
    _check(got, _turned(q, positions, rad, interleaved, factor), xt, size)
    tk, kept = _turned(k, positions, rad, interleaved, factor), slots >= 0
    at = slots[kept]
    want_k[at // page, :, at % page] = tk[kept]
    want_v[at // page, :, at % page] = v.cpu()[kept].float().to(ct).double()
    _check(kc, want_k, ct, size)
    assert torch.equal(vc.double().cpu(), want_v)
    assert _lib.lib().ggufmm_device_status(1, None) == 0


def test_a_token_does_not_depend_on_its_neighbour(cuda):
    """The same bits alone, in a short call and in a prompt; in place too."""
    from vllm_webgpu_b200 import ops
    x = torch.randn(700, 4, 128, device="cuda").to(BF16)
    pos = torch.randint(0, 100000, (700,), device="cuda")
    steps, _ = ops.rope_steps(128, 500000.0)
    want = ops.rope(x, pos, steps, True)
    assert torch.equal(ops.rope(x[100:107], pos[100:107], steps, True), want[100:107])
    y = x.clone()
    ops.rope(y, pos, steps, True, out=y)
    assert torch.equal(y, want)


def test_a_slot_past_the_last_page_in_a_prompt(cuda):
    from vllm_webgpu_b200 import _lib, ops
    t, page, pages = 601, 16, 40
    x = torch.randn(t, 2, 64, device="cuda")
    kc, vc = (torch.zeros(pages, 2, page, 64, dtype=F16, device="cuda") for _ in range(2))
    slots = torch.arange(t, device="cuda")
    slots[::7] = pages * page + torch.arange(len(slots[::7]), device="cuda")
    steps, _ = ops.rope_steps(64)
    _lib.lib().ggufmm_device_status(1, None)
    ops.rope_append(x, x, x, torch.arange(t, device="cuda"), steps, slots, kc, vc)
    assert _lib.lib().ggufmm_device_status(1, None) == 2
    flat = vc.transpose(1, 2).reshape(-1, 2, 64)[:t]
    want = x.half()
    want[::7] = 0
    assert torch.equal(flat, want)
