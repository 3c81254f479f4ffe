"""ggufmm_rms_norm against the definition in 64 bits: dtypes, odd widths, strides, in place,
extremes and refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # relative error of one rounding
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}  # spacing of the subnormals


def _ref(x, w, eps, r, add):
    s = x.double() if r is None else x.double() + r.double()
    y = s / torch.sqrt((s * s).mean(dim=-1, keepdim=True) + eps)
    return s, y if w is None else y * (w.double() + add)


def _check(got, want, n, dtype):
    # 32-bit work: the sum of squares adds n values in at most n/32 + 16 steps, each of one
    # rounding, halved by the root; six more roundings along the way; then the store's own
    rel = UNIT[F32] * ((n / 32 + 16) / 2 + 6) + UNIT[dtype]
    err = (got.double() - want).abs()
    assert bool((err <= rel * want.abs() + TINY[dtype]).all()), float((err / want.abs().clamp_min(1e-30)).max())


def _make(m, n, dtype, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, n, generator=g) * gain).to(dtype).cuda()


@pytest.mark.parametrize("m,n", [(1, 4096), (3, 1), (5, 7), (1, 2815), (33, 128), (2, 8192), (9, 2048), (300, 320),
                                 (1, 65536), (2, 50001), (4, 16392)])
@pytest.mark.parametrize("xt,rt,yt,wt", [(F32, BF16, BF16, F32), (BF16, None, BF16, BF16), (F16, F16, F32, F16),
                                         (F32, None, F16, None), (BF16, F32, F16, F32), (F16, BF16, BF16, BF16)])
def test_norm_matches_the_definition(cuda, m, n, xt, rt, yt, wt):
    from vllm_webgpu_b200 import ops
    x = _make(m, n, xt, 1)
    r = _make(m, n, rt, 2, 3.0) if rt is not None else None
    w = (1 + _make(1, n, F32, 3, 0.1)[0]).to(wt) if wt is not None else None
    s, y = _ref(x, w, 1e-5, r, 0.25 if wt is not None else 0.0)
    got = ops.rms_norm(x, w, 1e-5, r, out_dtype=yt, weight_add=0.25 if wt is not None else 0.0)
    if r is not None:
        got, ro = got
        assert ro.dtype == rt
        assert torch.equal(ro, (x.float() + r.float()).to(rt))  # one 32-bit sum, rounded once
    assert got.dtype == yt
    _check(got, y, n, yt)


@pytest.mark.parametrize("n", [4096, 515])
def test_in_place_and_strided(cuda, n):
    """residual_out = residual, out = x, rows of wider tensors; what lies around stays."""
    from vllm_webgpu_b200 import ops
    m = 6
    xw, rw = _make(m, n + 37, BF16, 4), _make(m, n + 13, BF16, 5)
    x, r = xw[:, 5:5 + n], rw[:, 1:1 + n]
    x0, r0, xw0, rw0 = x.clone(), r.clone(), xw.clone(), rw.clone()
    w = torch.ones(n, device="cuda")
    s, y = _ref(x0, w, 1e-6, r0, 0.0)
    out, ro = ops.rms_norm(x, w, 1e-6, r, out=x, residual_out=r)
    assert out.data_ptr() == x.data_ptr() and ro.data_ptr() == r.data_ptr()
    _check(x, y, n, BF16)
    assert torch.equal(r, (x0.float() + r0.float()).to(BF16))
    assert torch.equal(xw[:, :5], xw0[:, :5]) and torch.equal(xw[:, 5 + n:], xw0[:, 5 + n:])
    assert torch.equal(rw[:, :1], rw0[:, :1]) and torch.equal(rw[:, 1 + n:], rw0[:, 1 + n:])


@pytest.mark.parametrize("n", [1, 2, 3, 5, 9, 15, 17, 250, 254, 1006, 1009, 1010, 1011, 1023, 4095, 16367, 16369, 16371])
@pytest.mark.parametrize("xt,rt,yt,wt", [(F32, BF16, BF16, F32), (F16, None, F16, F16), (BF16, F32, F32, BF16)])
def test_packed_rows_of_odd_width(cuda, n, xt, rt, yt, wt):
    """Rows without a gap that begin anywhere between 16-byte boundaries, in place; what lies
    behind the last row stays."""
    from vllm_webgpu_b200 import ops
    m = 11
    store = _make(1, m * n + 64, xt, 8)[0]
    x, behind = store[:m * n].view(m, n), store[m * n:].clone()
    r = _make(m, n, rt, 9, 2.0) if rt is not None else None
    w = (1 + _make(1, n, F32, 3, 0.1)[0]).to(wt)
    s, y = _ref(x, w, 1e-5, r, 0.0)
    want_ro = None if r is None else (x.float() + r.float()).to(rt)
    same = xt == yt
    got = ops.rms_norm(x, w, 1e-5, r, out=x if same else None, out_dtype=None if same else yt, residual_out=r)
    if r is not None:
        got, ro = got
        assert torch.equal(ro, want_ro)
    assert (got.data_ptr() == x.data_ptr()) == same
    _check(got, y, n, yt)
    assert torch.equal(store[m * n:], behind)


def test_same_bits_on_every_call_and_row(cuda):
    """A row's result depends on that row alone, and not on the number of rows beside it."""
    from vllm_webgpu_b200 import ops
    x = _make(1, 4096, F32, 6).expand(700, 4096).contiguous()
    many = ops.rms_norm(x, None, out_dtype=F32)
    assert torch.equal(many, many[:1].expand_as(many))
    assert torch.equal(many, ops.rms_norm(x, None, out_dtype=F32))


def test_extremes(cuda):
    from vllm_webgpu_b200 import ops
    n = 256
    x = torch.zeros(5, n, device="cuda")
    x[1] = 1e-25            # squares vanish in 32 bits: eps holds the norm
    x[2, 3] = float("inf")
    x[3, 4] = float("nan")
    x[4] = 2.0
    y = ops.rms_norm(x, None, 1e-6)
    assert torch.equal(y[0], torch.zeros(n, device="cuda"))
    assert torch.allclose(y[1], torch.full((n,), 1e-22, device="cuda"), rtol=1e-5)
    assert bool(y[2, 3].isnan()) and bool((y[2, 4:] == 0).all())  # inf / inf and 2 / inf
    assert bool(y[3].isnan().all())
    assert torch.allclose(y[4], torch.ones(n, device="cuda"), rtol=1e-6)
    z = ops.rms_norm(torch.zeros(1, n, device="cuda"), None, 0.0)  # 0 * inf, as the formula says
    assert bool(z.isnan().all())


def test_shapes_of_other_ranks_and_no_rows(cuda):
    from vllm_webgpu_b200 import ops
    x = _make(24, 64, BF16, 7)
    y = ops.rms_norm(x, None)
    assert torch.equal(ops.rms_norm(x.view(2, 3, 4, 64), None), y.view(2, 3, 4, 64))
    assert torch.equal(ops.rms_norm(x[0], None), y[0])
    assert torch.equal(ops.rms_norm(x.t().contiguous().t(), None), y)  # columns first: copied
    e = ops.rms_norm(torch.empty(0, 64, device="cuda"), None, residual=torch.empty(0, 64, device="cuda"))
    assert e[0].shape == (0, 64) and e[1].shape == (0, 64)


def test_on_another_stream_and_in_a_graph(cuda):
    from vllm_webgpu_b200 import ops
    x, w = _make(17, 1000, BF16, 8), torch.ones(1000, device="cuda")
    want = ops.rms_norm(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(x)
    with torch.cuda.stream(s):
        ops.rms_norm(x, w, out=out)
        g = torch.cuda.CUDAGraph()
        buf = torch.zeros_like(x)
        with torch.cuda.graph(g, stream=s):
            ops.rms_norm(x, w, out=buf)
        g.replay()
    s.synchronize()
    assert torch.equal(out, want) and torch.equal(buf, want)


def test_refusals(cuda):
    from vllm_webgpu_b200 import ops
    x = torch.zeros(2, 64, device="cuda")
    with pytest.raises(ValueError):
        ops.rms_norm(x, torch.ones(63, device="cuda"))
    with pytest.raises(ValueError):
        ops.rms_norm(x, None, residual=torch.zeros(2, 63, device="cuda"))
    with pytest.raises(ValueError):
        ops.rms_norm(x, None, residual_out=torch.zeros(2, 64, device="cuda"))
    with pytest.raises(ValueError):
        ops.rms_norm(x, None, out=torch.zeros(64, 2, device="cuda").t())
    with pytest.raises(ValueError):
        ops.rms_norm(x, None, residual=x, residual_out=torch.zeros(2, 64, device="cuda", dtype=BF16))
    with pytest.raises(ValueError):
        ops.rms_norm(x.double(), None)
    with pytest.raises(ValueError):
        ops.rms_norm(x, None, eps=-1.0)
    with pytest.raises(ValueError):
        ops.rms_norm(x, None, eps=float("nan"))
    with pytest.raises(ValueError):
        ops.rms_norm(torch.zeros(1, 65537, device="cuda"), None)
    with pytest.raises(ValueError):
        ops.rms_norm(x.cpu(), None)
    with pytest.raises(ValueError):
        ops.rms_norm(torch.zeros(2, 0, device="cuda"), None)
    assert np.isfinite(ops.rms_norm(x, None).cpu().numpy()).all()  # the context is as before
