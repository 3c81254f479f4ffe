"""The operators between the projections inside CUDA graphs and on other streams than the default
one, their workspaces included: new inputs in the same buffers, replayed, against plain calls."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
PAGE, HQ, HKV, D = 16, 8, 2, 128


class Layer:
    """The buffers of one step of a layer between its projections."""

    def __init__(self, new, lens, seed=0):
        from vllm_webgpu_b200 import ops
        g = torch.Generator().manual_seed(seed)
        t, counts = sum(new), [-(-n // PAGE) for n in lens]
        order, at = torch.randperm(sum(counts), generator=g).int(), 0
        self.table = torch.zeros(len(lens), max(counts), dtype=torch.int32)
        slots, positions = [], []
        for b, c in enumerate(counts):
            self.table[b, :c] = order[at:at + c]
            at += c
            for p in range(lens[b] - new[b], lens[b]):
                positions.append(p)
                slots.append(int(self.table[b, p // PAGE]) * PAGE + p % PAGE)
        self.table = self.table.cuda()
        self.slots, self.positions = (torch.tensor(x, device="cuda") for x in (slots, positions))
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        self.most, self.steps, self.g = max(new), ops.rope_steps(D)[0], g
        self.kc, self.vc = (torch.empty(sum(counts), HKV, PAGE, D, dtype=BF16, device="cuda") for _ in range(2))
        self.delta, self.stream = (torch.empty(t, 512, device="cuda", dtype=x) for x in (torch.float32, BF16))
        self.qkv = torch.empty(t, (HQ + 2 * HKV) * D, dtype=BF16, device="cuda")
        self.refill()

    def refill(self):
        for x in (self.kc, self.vc, self.delta, self.stream, self.qkv):
            x.copy_(torch.randn(x.shape, generator=self.g))

    def run(self):
        from vllm_webgpu_b200 import ops
        normed, stream = ops.rms_norm(self.delta, None, residual=self.stream, out_dtype=BF16)
        q, k, v = (x.unflatten(1, (-1, D)) for x in self.qkv.split([HQ * D, HKV * D, HKV * D], dim=1))
        q = ops.rope_append(q, k, v, self.positions, self.steps, self.slots, self.kc, self.vc, interleaved=True)
        if self.most == 1:
            o = ops.paged_attention(q, self.kc, self.vc, self.table, self.lens)
        else:
            o = ops.paged_prompt_attention(q, self.starts, self.most, self.kc, self.vc, self.table, self.lens)
        return normed, stream, q, o


# a decode step; prompts; few new tokens on a long text (keys shared out: a workspace and a second
# kernel); a prompt long enough for two tokens a CTA in the append
SHAPES = {"single": ([1] * 5, [1, 17, 300, 64, 2000]), "prompts": ([70, 33], [70, 200]), "shared": ([4], [6000]),
          "long": ([700], [700])}


@pytest.mark.parametrize("shape", SHAPES)
def test_replayed_from_a_graph(cuda, shape):
    from vllm_webgpu_b200 import _lib
    layer = Layer(*SHAPES[shape], seed=1)
    layer.run()
    _lib.lib().ggufmm_device_status(1, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        first = layer.run()
        second = layer.run()  # again behind it, in memory that the first may have given back
    for _ in range(3):
        layer.refill()
        kc, vc = layer.kc.clone(), layer.vc.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*first, *second)]
        layer.kc.copy_(kc), layer.vc.copy_(vc)
        want = layer.run()
        torch.cuda.synchronize()
        for i, x in enumerate(got):
            assert torch.equal(x, want[i % len(want)]), i
    assert _lib.lib().ggufmm_device_status(1, None) == 0


@pytest.mark.parametrize("shape", SHAPES)
def test_on_two_streams_at_once(cuda, shape):
    layers = [Layer(*SHAPES[shape], seed=s) for s in (2, 3)]
    want = [layer.run() for layer in layers]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (layer, s) in enumerate(zip(layers, streams)):
            with torch.cuda.stream(s):
                got[i].append(layer.run())
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(outs, want[i]))


def test_the_current_stream_counts_not_the_inputs(cuda):
    """Inputs made on one stream, used on another that waits for it."""
    from vllm_webgpu_b200 import ops
    side = torch.cuda.Stream()
    x = torch.zeros(4000, 4096, device="cuda")
    torch.cuda.synchronize()
    for i in range(5):
        x.fill_(float(i + 1))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = ops.rms_norm(x, None, eps=0.0)
        torch.cuda.current_stream().wait_stream(side)
        x.fill_(0.0)
        y.record_stream(torch.cuda.current_stream())
        assert torch.allclose(y, torch.ones_like(y), rtol=1e-6)
