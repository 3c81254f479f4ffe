"""Prompt attention whose waits run out: the limit on polls is lowered until the wait for another
unit of work gives up, with copies and products of the last one under way. The call then reports it
through ggufmm_device_status and leaves (its own copies and products waited for, its tensor memory
given back), and the context and the next call are as before."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_attention import BF16, F16, Case

pytestmark = pytest.mark.gpu

# two and one query tiles a CTA, every padded head width, pages as wide as a tile and less, lengths
# that end inside a page, keys shared out over CTAs and joined, more units than CTAs
CASES = {
    "two tiles": ([300, 517, 40], [300, 200, 40], 8, 2, 128, BF16, 16),
    "many units": ([700] * 12, [700] * 12, 16, 8, 128, BF16, 16),
    "narrow": ([900, 333], [900, 333], 4, 4, 64, F16, 8),
    "wide heads": ([400, 77], [400, 60], 8, 2, 256, BF16, 24),
    "padded heads": ([260, 131], [200, 131], 6, 2, 80, F16, 64),
    "shared keys": ([9001], [5], 8, 2, 128, BF16, 16),
}


@pytest.mark.parametrize("name", CASES)
def test_a_wait_that_runs_out_is_reported(cuda, name):
    from vllm_webgpu_b200 import _lib, ops
    lib = _lib.lib()
    lens, new, hq, hkv, d, dtype, page = CASES[name]
    c = Case(lens, hq, hkv, d, dtype, page, seed=len(name))
    starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    q, held = c.q(sum(new)), c.device_lens()

    def call():
        out = torch.full_like(q, 7.0)
        ops.paged_prompt_attention(q, starts, max(new), c.kc, c.vc, c.table, held, out=out)
        torch.cuda.synchronize()
        return out
    lib.ggufmm_device_status(1, None)
    want = call()
    assert lib.ggufmm_device_status(1, None) == 0
    ran_out = []
    for polls in (1, 10, 40, 160, 640, 2560):
        assert lib.ggufmm_set_wait_limit(polls) == 0
        try:
            got = call()
        finally:
            assert lib.ggufmm_set_wait_limit(0) == 0
        ran_out.append(lib.ggufmm_device_status(1, None))
        assert ran_out[-1] in (0, 1)
        assert ran_out[-1] or torch.equal(got, want)  # reported, or right
        assert torch.equal(call(), want)              # and nothing of it is left behind
        assert lib.ggufmm_device_status(1, None) == 0
    print(f"{name}: ran out at {ran_out}")
    assert ran_out[0] == 1
