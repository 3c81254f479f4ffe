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


def test_rows_that_lie_over_one_another(cuda):
    """Expanded inputs: one row for all tokens, one table for several continuations of a text."""
    from vllm_webgpu_b200 import ops
    x, r = torch.randn(1, 96, device="cuda"), torch.randn(1, 96, device="cuda")
    want, res = ops.rms_norm(x.repeat(5, 1), None, residual=r.repeat(5, 1))
    got, res2 = ops.rms_norm(x.expand(5, 96), None, residual=r.expand(5, 96))
    assert torch.equal(got, want) and torch.equal(res2, res)
    kc, vc = _cache()
    q = torch.randn(3, 4, 64, device="cuda").to(BF16)
    table, lens = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda"), torch.tensor([40, 9, 33], dtype=torch.int32, device="cuda")
    want = ops.paged_attention(q, kc, vc, table.repeat(3, 1), lens)
    assert torch.equal(ops.paged_attention(q, kc, vc, table.expand(3, 3), lens), want)
    starts = torch.arange(4, dtype=torch.int32, device="cuda")
    want = ops.paged_prompt_attention(q, starts, 1, kc, vc, table.repeat(3, 1), lens)
    assert torch.equal(ops.paged_prompt_attention(q, starts, 1, kc, vc, table.expand(3, 3), lens), want)
    for one in (q[:1].expand(3, 4, 64), q[:, :1].expand(3, 4, 64)):
        want = ops.paged_attention(one.contiguous(), kc, vc, table.repeat(3, 1), lens)
        assert torch.equal(ops.paged_attention(one, kc, vc, table.repeat(3, 1), lens), want)
    with pytest.raises(ValueError):  # an output has to have its rows apart
        ops.rms_norm(x.repeat(5, 1), None, out=torch.zeros(1, 96, device="cuda").expand(5, 96))
    with pytest.raises(ValueError):
        ops.paged_attention(q, kc, vc, table.repeat(3, 1), lens, out=torch.zeros_like(q)[:1].expand(3, 4, 64))
