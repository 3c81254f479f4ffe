"""Tensors that a caller may hand the norm, rotary and attention operators in other forms than the
plain one: taken for what they hold, or refused before a launch."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _cache(pages=4, hkv=2, page=16, d=64, dtype=BF16):
    g = torch.Generator().manual_seed(7)
    return [torch.randn(pages, hkv, page, d, generator=g).to(dtype).cuda() for _ in range(2)]


def test_a_workspace_without_its_bytes_is_refused(cuda):
    """One byte seen many times over, a view with gaps or of wider values is no workspace."""
    from vllm_webgpu_b200 import ops
    kc, vc = _cache()
    q = torch.randn(1, 4, 64, device="cuda").to(BF16)
    table, lens = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([20], dtype=torch.int32, device="cuda")
    good = ops.attention_workspace(1, 4, 2, 64, "cuda")
    want = ops.paged_attention(q, kc, vc, table, lens)
    assert torch.equal(ops.paged_attention(q, kc, vc, table, lens, workspace=good), want)
    n = good.numel()
    for bad in (torch.zeros(1, dtype=torch.uint8, device="cuda").expand(n),
                torch.zeros(2 * n, dtype=torch.uint8, device="cuda")[::2],
                torch.zeros(n, dtype=torch.float32, device="cuda"), good.cpu(), good[:n - 1]):
        with pytest.raises(ValueError):
            ops.paged_attention(q, kc, vc, table, lens, workspace=bad)
    assert torch.equal(ops.paged_attention(q, kc, vc, table, lens, workspace=good), want)
