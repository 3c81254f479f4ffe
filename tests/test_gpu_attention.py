"""Attention over the paged cache against the definition in 64 bits: one new token per
sequence and ragged causal prompts, at the lengths, groups, head widths, page sizes, windows
and strides where it can go wrong."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _reference(q, starts, kc, vc, table, lens, scale, window):
    """(out, A) in 64 bits: A = sum of p |v|, the size that the products' roundings are of."""
    q, kc, vc, table = (t.double().cpu() if t.is_floating_point() else t.cpu() for t in (q, kc, vc, table))
    page, hkv, g = kc.shape[2], kc.shape[1], q.shape[1] // kc.shape[1]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for b, length in enumerate(lens):
        rows = range(starts[b], starts[b + 1])
        n = len(rows)
        if length <= 0 or n == 0:
            continue
        pages = table[b, :-(-length // page)].long()
        k = kc[pages].transpose(1, 2).reshape(-1, hkv, kc.shape[3])[:length]
        v = vc[pages].transpose(1, 2).reshape(-1, hkv, kc.shape[3])[:length]
        for i, row in enumerate(rows):
            pos = length - n + i
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                continue
            for h in range(q.shape[1]):
                s = (k[lo:pos + 1, h // g] @ q[row, h]) * scale
                p = torch.softmax(s, 0)
                out[row, h] = p @ v[lo:pos + 1, h // g]
                size[row, h] = p @ v[lo:pos + 1, h // g].abs()
    return out, size


def _check(got, want, size, dtype):
    # The weights may be rounded to the cache's type before their product with v (one unit of
    # A, twice where the sum is of unrounded ones); a score of sum |q k| scale < 64 and 256
    # terms in 32 bits is off by at most 2^-10.5 of a weight and mostly far less; then the store.
    u = UNIT[dtype]
    tol = (2 * u + 2.0 ** -10) * size + u * want.abs() + 2.0 ** -24
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), int((err > tol).sum()))


class Case:
    """A cache whose unused slots and pages hold NaN, and sequences scattered over it."""

    def __init__(self, lens, hq, hkv, d, dtype, page, seed=0, slots_first=False, gain=2.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.dtype, self.page = lens, dtype, page
        counts = [-(-max(0, n) // page) for n in lens]
        pages = sum(counts) + 3
        order = torch.randperm(pages, generator=g)
        shape = (pages, page, hkv, d) if slots_first else (pages, hkv, page, d)
        caches = []
        self.table = torch.full((len(lens), max(counts + [1]) + 2), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(counts):
            self.table[b, :c] = order[at:at + c].int()
            at += c
        for _ in range(2):
            c = torch.full(shape, float("nan"))
            c = c.transpose(1, 2) if slots_first else c
            for b, n in enumerate(lens):
                for j in range(0, max(0, n), page):
                    m = min(page, n - j)
                    c[int(self.table[b, j // page]), :, :m] = torch.randn(hkv, m, d, generator=g)
            base = c.transpose(1, 2) if slots_first else c
            base = base.to(dtype).cuda()
            caches.append(base.transpose(1, 2) if slots_first else base)
        self.kc, self.vc = caches
        self.table = self.table.cuda()
        self.g, self.hq, self.d, self.gain = g, hq, d, gain

    def q(self, tokens):
        return (torch.randn(tokens, self.hq, self.d, generator=self.g) * self.gain).to(self.dtype).cuda()

    def device_lens(self):
        return torch.tensor(self.lens, dtype=torch.int32, device="cuda")


def _decode(c, window=0, scale=None, q=None, **kw):
    from vllm_webgpu_b200 import _lib, ops
    q = c.q(len(c.lens)) if q is None else q
    _lib.lib().ggufmm_device_status(1, None)
    got = ops.paged_attention(q, c.kc, c.vc, c.table, c.device_lens(), scale=scale, window=window, **kw)
    want, size = _reference(q, list(range(len(c.lens) + 1)), c.kc, c.vc, c.table, c.lens,
                            c.d ** -0.5 if scale is None else scale, window)
    _check(got, want, size, c.dtype)
    assert _lib.lib().ggufmm_device_status(1, None) == 0
    return got


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 8, 64), (4, 1, 256), (5, 1, 96), (14, 2, 80), (3, 3, 8),
                                      (16, 1, 128), (24, 1, 64), (64, 1, 128), (33, 1, 256)])
def test_decode_heads(cuda, dtype, hq, hkv, d):
    _decode(Case([1, 0, 37, 16, 255, 301], hq, hkv, d, dtype, 16, seed=hq + d))


@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 33, 1000])
def test_decode_pages_and_windows(cuda, page, window):
    _decode(Case([1, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 129, 500], 8, 2, 64, BF16, page, seed=page), window)


@pytest.mark.parametrize("batch,longest", [(1, 1), (1, 5000), (2, 3001), (70, 90), (300, 40), (1, 20011)])
def test_decode_splits(cuda, batch, longest):
    """From many short sequences to one long one: every way the work is cut and joined."""
    lens = [max(0, longest - (i * 37) % (longest + 1)) for i in range(batch)]
    _decode(Case(lens, 4, 1, 64, F16, 16, seed=batch))


def test_decode_is_the_same_on_every_call(cuda):
    from vllm_webgpu_b200 import ops
    c = Case([4000, 3, 1999, 0, 700], 32, 8, 128, BF16, 16, seed=5)
    q = c.q(5)
    lens = c.device_lens()
    first = ops.paged_attention(q, c.kc, c.vc, c.table, lens)
    for _ in range(20):
        assert torch.equal(first, ops.paged_attention(q, c.kc, c.vc, c.table, lens))


def test_decode_peaked_and_flat_scores(cuda):
    """One weight near 1 far from the others; all weights equal; scores of large size."""
    c = Case([900, 77], 8, 2, 128, F16, 16, seed=6)
    _decode(c, q=torch.zeros(2, 8, 128, dtype=F16, device="cuda"))          # uniform weights
    c.kc[:, :, :, 0] = 0
    page, at = int(c.table[0, 600 // 16]), 600 % 16
    c.kc[page, :, at, 0] = 100.0
    q = torch.zeros(2, 8, 128, dtype=F16, device="cuda")
    q[:, :, 0] = 20.0                                                       # a score of 177, the rest 0
    got = _decode(c, q=q)
    assert torch.equal(got[0], c.vc[page, :, at].repeat_interleave(4, 0))
    q[:, :, 0] = -20.0                                                      # and of -177
    _decode(c, q=q)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("kind", ["single", "prompt"])
def test_a_long_tail_of_small_weights(cuda, dtype, kind):
    """One weight of 1 and 60000 of 2^-24.5, below the smallest 16-bit float: together 0.25%."""
    from vllm_webgpu_b200 import ops
    n = 60001
    c = Case([n], 4, 1, 64, dtype, 64, seed=13)
    top = 24.5 * 0.6931471805599453
    c.kc.zero_()
    c.vc.fill_(1.0)
    page, at = int(c.table[0, 700]), 33
    c.kc[page, 0, at, 0] = 1.0
    c.vc[page, 0, at] = 0.0
    q = torch.zeros(1, 4, 64, dtype=dtype, device="cuda")
    q[..., 0] = 17.0
    scale = top / 17.0
    if kind == "single":
        got = ops.paged_attention(q, c.kc, c.vc, c.table, c.device_lens(), scale=scale)
    else:
        got = ops.paged_prompt_attention(q, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1, c.kc, c.vc, c.table,
                                         c.device_lens(), scale=scale)
    tail = (n - 1) * 2.0 ** -24.5
    want = torch.full((1, 4, 64), tail / (1 + tail), dtype=torch.float64)
    # the bound of _check, with A = the result itself (v is not negative); the prompt's running
    # maximum may stand 2^8 below, which the weights' range takes up
    _check(got, want, want, dtype)


def test_decode_strides_and_scale(cuda):
    from vllm_webgpu_b200 import ops
    c = Case([33, 260], 8, 2, 128, BF16, 16, seed=7, slots_first=True)
    wide = c.q(2).repeat(1, 3, 1)
    q = wide[:, 5:13]
    out = torch.zeros(2, 16, 128, dtype=BF16, device="cuda")
    got = _decode(c, q=q, scale=0.05, out=out[:, 4:12])
    assert int(out[:, :4].count_nonzero()) == 0 and int(out[:, 12:].count_nonzero()) == 0
    assert torch.equal(got, ops.paged_attention(q.contiguous(), c.kc.contiguous(), c.vc.contiguous(), c.table.long(),
                                                c.device_lens().long(), scale=0.05))


def test_decode_bad_pages_and_lengths(cuda):
    """A page outside the cache reads as zeros, a length past the table is cut: flagged, no fault."""
    from vllm_webgpu_b200 import _lib, ops
    c = Case([64, 64], 4, 1, 64, F16, 16, seed=8)
    q = c.q(2)
    table = c.table.clone()
    table[0, 1], table[1, 2] = -7, 1 << 30
    _lib.lib().ggufmm_device_status(1, None)
    got = ops.paged_attention(q, c.kc, c.vc, table, c.device_lens())
    assert _lib.lib().ggufmm_device_status(1, None) == 2
    kc, vc = (torch.cat([x, torch.zeros_like(x[:1])]) for x in (c.kc, c.vc))
    table[0, 1] = table[1, 2] = kc.shape[0] - 1
    want, size = _reference(q, [0, 1, 2], kc, vc, table, [64, 64], 0.125, 0)
    _check(got, want, size, F16)
    cut = c.table[:, :2].contiguous()
    got = ops.paged_attention(q, c.kc, c.vc, cut, c.device_lens())
    assert _lib.lib().ggufmm_device_status(1, None) == 2
    want, size = _reference(q, [0, 1, 2], c.kc, c.vc, cut, [32, 32], 0.125, 0)
    _check(got, want, size, F16)
    zero = ops.paged_attention(q, c.kc, c.vc, c.table, torch.tensor([-5, 0], dtype=torch.int32, device="cuda"))
    assert int(zero.count_nonzero()) == 0


def test_decode_on_streams_and_in_a_graph(cuda):
    from vllm_webgpu_b200 import ops
    c = Case([2000, 1500], 32, 8, 128, BF16, 16, seed=9)
    qs = [c.q(2) for _ in range(4)]
    lens = c.device_lens()
    want = [ops.paged_attention(q, c.kc, c.vc, c.table, lens) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [torch.empty_like(q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(5):
        for q, s, o in zip(qs, streams, got):
            with torch.cuda.stream(s):
                ops.paged_attention(q, c.kc, c.vc, c.table, lens, out=o)
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert torch.equal(w, o)
    q, out = qs[0].clone(), torch.empty_like(qs[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.paged_attention(q, c.kc, c.vc, c.table, lens, out=out)
    for i in (1, 2, 3):
        q.copy_(qs[i])
        g.replay()
        g.replay()
        assert torch.equal(out, want[i])
    lens.copy_(torch.tensor([100, 0], dtype=torch.int32))  # other lengths in the same graph
    g.replay()
    ref, size = _reference(q, [0, 1, 2], c.kc, c.vc, c.table, [100, 0], 128 ** -0.5, 0)
    _check(out, ref, size, BF16)


# ---- prompts ------------------------------------------------------------------------------------
def _prompt(c, new, window=0, scale=None, extra_max=0):
    from vllm_webgpu_b200 import _lib, ops
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = c.q(starts[-1])
    _lib.lib().ggufmm_device_status(1, None)
    got = ops.paged_prompt_attention(q, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                                     min(max(new) + extra_max, starts[-1]), c.kc, c.vc, c.table, c.device_lens(),
                                     scale=scale, window=window)
    want, size = _reference(q, starts, c.kc, c.vc, c.table, c.lens, c.d ** -0.5 if scale is None else scale, window)
    _check(got, want, size, c.dtype)
    assert _lib.lib().ggufmm_device_status(1, None) == 0
    return got


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (3, 3, 64), (4, 1, 256), (5, 1, 96), (7, 1, 80), (2, 1, 8), (64, 1, 64),
                                      (33, 1, 128), (12, 2, 192)])
def test_prompt_heads(cuda, dtype, hq, hkv, d):
    _prompt(Case([70, 1, 33, 140], hq, hkv, d, dtype, 16, seed=hq + d), [70, 1, 20, 3])


@pytest.mark.parametrize("page", [8, 24, 64, 128])
@pytest.mark.parametrize("window", [0, 1, 50, 127, 128, 129])
def test_prompt_pages_and_windows(cuda, page, window):
    _prompt(Case([5, 127, 128, 129, 300, 257], 4, 2, 64, BF16, page, seed=page), [5, 127, 128, 129, 44, 1], window)


@pytest.mark.parametrize("new,lens", [([1], [1]), ([1, 0, 2], [1, 50, 2]), ([513], [513]), ([40], [1200]),
                                      ([4, 4, 4], [700, 4, 128]), ([31, 33, 64], [31, 33, 64]), ([200], [1000])])
def test_prompt_lengths(cuda, new, lens):
    _prompt(Case(lens, 8, 2, 128, BF16, 16, seed=len(new)), new, extra_max=3)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, BF16), (3, 1, 64, F16), (4, 1, 256, BF16), (5, 1, 96, F16)])
@pytest.mark.parametrize("new,lens,window", [([3], [5000], 0), ([1, 40, 7], [4100, 40, 0], 0), ([2, 2], [9000, 3000], 2500),
                                             ([130], [3000], 0)])
def test_prompt_keys_shared_out(cuda, hq, hkv, d, dtype, new, lens, window):
    """A few new tokens on a long cache: several CTAs take shares of the keys, some of them none."""
    from vllm_webgpu_b200 import ops
    c = Case(lens, hq, hkv, d, dtype, 16, seed=sum(new))
    wide = torch.full((len(lens), 2000), -1, dtype=torch.int32, device="cuda")  # a table for long texts
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide
    first = _prompt(c, new, window)
    q = c.q(sum(new))
    starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    a, b = (ops.paged_prompt_attention(q, starts, max(new), c.kc, c.vc, c.table, c.device_lens(), window=window)
            for _ in range(2))
    assert torch.equal(a, b) and first.shape == a.shape


@pytest.mark.parametrize("batch", [3, 40, 70])
def test_prompt_mixed_lengths(cuda, batch):
    """One long run of new tokens beside many short and empty ones, more work than SMs."""
    new = [700 if b == batch // 2 else b % 4 for b in range(batch)]
    lens = [n + (b * 37) % 300 for b, n in enumerate(new)]
    _prompt(Case(lens, 8, 8, 64, BF16, 16, seed=batch), new, extra_max=5)


def test_prompt_many_units_for_each_sm(cuda):
    """Every CTA takes several pieces of work: a repeat gives the same bits."""
    from vllm_webgpu_b200 import ops
    n, b = 260, 48
    c = Case([n] * b, 8, 4, 128, BF16, 16, seed=11)
    new = [n] * b
    first = _prompt(c, new)
    q = c.q(n * b)
    starts = torch.arange(0, n * b + 1, n, dtype=torch.int32, device="cuda")
    x, y = (ops.paged_prompt_attention(q, starts, n, c.kc, c.vc, c.table, c.device_lens()) for _ in range(2))
    assert torch.equal(x, y) and first.shape == x.shape


def test_prompt_masked_out_rows(cuda):
    """More new tokens than the length holds: the queries before position 0 see nothing."""
    from vllm_webgpu_b200 import ops
    c = Case([10, 0], 4, 1, 64, F16, 16, seed=3)
    q = c.q(20)
    starts = torch.tensor([0, 15, 20], dtype=torch.int32, device="cuda")
    got = ops.paged_prompt_attention(q, starts, 15, c.kc, c.vc, c.table, c.device_lens())
    want, size = _reference(q, [0, 15, 20], c.kc, c.vc, c.table, [10, 0], 0.125, 0)
    _check(got, want, size, F16)
    assert int(got[:5].count_nonzero()) == 0 and int(got[15:].count_nonzero()) == 0


def test_prompt_widest_window(cuda):
    """A window past every length hides nothing, at positions before 0 either."""
    from vllm_webgpu_b200 import ops
    c = Case([10, 300], 4, 1, 64, F16, 16, seed=5)
    q = c.q(30)
    starts = torch.tensor([0, 15, 30], dtype=torch.int32, device="cuda")
    a, b = (ops.paged_prompt_attention(q, starts, 15, c.kc, c.vc, c.table, c.device_lens(), window=w) for w in (0, 2 ** 31 - 1))
    assert torch.equal(a, b) and int(a[5:].count_nonzero()) > 0


def test_prompt_agrees_with_single_tokens(cuda):
    from vllm_webgpu_b200 import ops
    c = Case([300], 8, 2, 128, F16, 16, seed=4)
    q = c.q(300)
    starts = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    whole = ops.paged_prompt_attention(q, starts, 300, c.kc, c.vc, c.table, c.device_lens())
    for i in (0, 1, 17, 128, 299):
        one = ops.paged_attention(q[i:i + 1], c.kc, c.vc, c.table, torch.tensor([i + 1], dtype=torch.int32, device="cuda"))
        _, size = _reference(q[i:i + 1], [0, 1], c.kc, c.vc, c.table, [i + 1], 128 ** -0.5, 0)
        # both within the definition's bound
        tol = 2 * ((2 * UNIT[F16] + 2.0 ** -10) * size + UNIT[F16] * one.double().cpu().abs() + 2.0 ** -24)
        assert bool(((whole[i:i + 1].double().cpu() - one.double().cpu()).abs() <= tol).all())


def test_prompt_large_scores(cuda):
    """Running maxima that rise by hundreds from one block of keys to the next."""
    c = Case([400], 4, 2, 64, BF16, 16, seed=11)
    ramp = torch.arange(c.kc.shape[0], device="cuda", dtype=torch.float32)
    order = c.table[0].clamp_min(0).long()
    ramp[order[:25]] = torch.arange(25, device="cuda", dtype=torch.float32)
    c.kc[..., 0] = (ramp * 4)[:, None, None].to(BF16)
    c.kc[..., 1:] = 0
    from vllm_webgpu_b200 import ops
    q = torch.zeros(400, 4, 64, dtype=BF16, device="cuda")
    q[..., 0] = 32.0
    starts = torch.tensor([0, 400], dtype=torch.int32, device="cuda")
    for sign in (1.0, -1.0):
        got = ops.paged_prompt_attention(q * sign, starts, 400, c.kc, c.vc, c.table, c.device_lens())
        want, size = _reference(q * sign, [0, 400], c.kc, c.vc, c.table, [400], 0.125, 0)
        _check(got, want, size, BF16)


def test_prompt_strides_and_untouched_rows(cuda):
    from vllm_webgpu_b200 import ops
    c = Case([50, 20], 4, 2, 64, BF16, 16, seed=12, slots_first=True)
    wide = torch.randn(80, 12, 64, device="cuda").to(BF16)
    q = wide[:, 2:6]
    out = torch.full((80, 8, 64), 3.0, dtype=BF16, device="cuda")
    starts = torch.tensor([4, 54, 74], dtype=torch.int32, device="cuda")
    ops.paged_prompt_attention(q, starts, 50, c.kc, c.vc, c.table, c.device_lens(), out=out[:, 4:])
    want, size = _reference(q, [4, 54, 74], c.kc, c.vc, c.table, [50, 20], 0.125, 0)
    _check(out[4:74, 4:], want[4:74], size[4:74], BF16)
    rest = torch.full_like(out, 3.0)
    assert torch.equal(out[:, :4], rest[:, :4]) and torch.equal(out[:4], rest[:4]) and torch.equal(out[74:], rest[74:])


def test_empty_batches(cuda):
    from vllm_webgpu_b200 import ops
    c = Case([4], 4, 2, 64, BF16, 16)
    q = torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    none, table = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    assert ops.paged_attention(q, c.kc, c.vc, table, none).shape == (0, 4, 64)
    assert ops.paged_prompt_attention(q, torch.zeros(1, dtype=torch.int32, device="cuda"), 0, c.kc, c.vc, table,
                                      none).shape == (0, 4, 64)
    got = ops.paged_prompt_attention(q, torch.zeros(2, dtype=torch.int32, device="cuda"), 0, c.kc, c.vc, c.table,
                                     c.device_lens())
    assert got.shape == (0, 4, 64)
    no_pages = torch.zeros(1, 0, dtype=torch.int32, device="cuda")
    z = ops.paged_attention(c.q(1), c.kc, c.vc, no_pages, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert int(z.count_nonzero()) == 0


def test_refusals(cuda):
    from vllm_webgpu_b200 import ops
    c = Case([20, 20], 4, 2, 64, BF16, 16)
    good = dict(q=c.q(2), k_cache=c.kc, v_cache=c.vc, block_tables=c.table, lens=c.device_lens())

    def refused(fn=ops.paged_attention, **other):
        with pytest.raises(ValueError):
            fn(**{**good, **other})
    refused(q=c.q(3))                                                        # three tokens, two sequences
    refused(q=good["q"].float())
    refused(q=good["q"].half())                                              # not the cache's type
    refused(q=good["q"][:, :3].contiguous())                                 # 3 heads on 2
    refused(q=good["q"][..., :32].contiguous())
    refused(q=good["q"].cpu())
    refused(k_cache=c.kc.float(), v_cache=c.vc.float(), q=good["q"].float())
    refused(k_cache=c.kc[..., :60], v_cache=c.vc[..., :60], q=good["q"][..., :60])  # 60 is no multiple of 8
    refused(k_cache=c.kc[:, :, :12], v_cache=c.vc[:, :, :12])                # a page of 12 slots
    refused(lens=good["lens"][:1])
    refused(block_tables=c.table[0])
    refused(window=-1)
    refused(scale=float("inf"))
    refused(out=torch.empty(2, 4, 64, device="cuda"))
    refused(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda"))
    many = torch.zeros(2, 130, 64, dtype=BF16, device="cuda")
    refused(q=many)                                                          # 65 query heads to one
    flat = torch.zeros(2 * 4 * 64 + 1, dtype=BF16, device="cuda")[1:]
    refused(q=flat.view(2, 4, 64))                                           # not 16-byte aligned
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    refused(ops.paged_prompt_attention, q_starts=starts, max_q=3)            # longer than q
    refused(ops.paged_prompt_attention, q_starts=starts, max_q=-1)
    refused(ops.paged_prompt_attention, q_starts=starts[:2], max_q=1)
    assert bool(ops.paged_attention(**good).isfinite().all())
